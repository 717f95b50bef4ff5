"""Refusals of the 8-bit product: no GPU needed."""
import ctypes as C

import pytest
import torch

from titanet_amd import _lib
from titanet_amd.int8 import Int8Linear, Int8Rows, int8_matmul, quantize_rows
from titanet_amd.metrics import cosine_scores, verification_test


def test_operands_must_live_on_a_device():
    for call in (lambda: quantize_rows(torch.ones(2, 3)), lambda: Int8Rows(torch.ones(2, 3, dtype=torch.int8), torch.ones(2)),
                 lambda: Int8Linear(torch.ones(2, 3))):
        with pytest.raises(RuntimeError, match="no CPU execution path"):
            call()


def test_types_and_shapes_it_does_not_take():
    for bad in (torch.ones(2, 3, dtype=torch.float64), torch.ones(2, 3, dtype=torch.int8), [1.0]):
        with pytest.raises(TypeError):
            quantize_rows(bad)
    for bad in (torch.ones(3), torch.ones(2, 3, 4), torch.ones(2, 0), torch.empty(1, 131072)):
        with pytest.raises(ValueError):
            quantize_rows(bad)
    with pytest.raises(TypeError):
        Int8Rows(torch.ones(2, 3), torch.ones(2))
    with pytest.raises(TypeError):
        Int8Rows(torch.ones(2, 3, dtype=torch.int8), torch.ones(3))
    with pytest.raises(TypeError):
        Int8Rows(torch.ones(2, 3, dtype=torch.int8), torch.ones(2, dtype=torch.float64))
    with pytest.raises(TypeError):
        int8_matmul(torch.ones(2, 3), torch.ones(2, 3))


def test_c_entries_refuse_before_they_touch_the_device():
    lib = _lib.load()
    at, none = C.c_void_p(4096), C.c_void_p(0)
    bad, unsupported = -1, -2

    def quantize(x=at, dtype=0, rows=1, cols=3, ldx=3, ld=64, scales=at):
        return lib.tn_int8_quantize_rows(x, dtype, rows, cols, ldx, at, ld, scales, none)

    assert quantize(rows=0) == 0 and quantize(rows=-1) == bad and quantize(x=none) == bad and quantize(scales=none) == bad
    assert quantize(cols=0) == bad and quantize(ld=63) == bad and quantize(cols=65) == bad and quantize(ldx=-1) == bad
    assert quantize(dtype=3) == unsupported and quantize(cols=131072, ld=131072) == unsupported

    def matmul(a=at, b=at, y=at, dtype=0, lda=64, ldb=64, ldy=5, m=4, n=5, k=3):
        return lib.tn_int8_matmul(a, at, lda, b, at, ldb, none, y, dtype, ldy, m, n, k, none)

    assert matmul(m=0) == 0 and matmul(n=0) == 0 and matmul(m=-1) == bad and matmul(k=0) == bad
    assert matmul(a=none) == bad and matmul(y=none) == bad and matmul(b=C.c_void_p(4097)) == bad
    assert matmul(lda=32) == bad and matmul(k=65) == bad and matmul(ldy=4) == bad
    assert matmul(dtype=-1) == unsupported and matmul(lda=131072, ldb=131072, k=131072) == unsupported

    def linear(x=at, xd=0, yd=0, m=4, ws=none, size=0, ldx=3, ldb=64):
        return lib.tn_int8_linear(x, xd, ldx, at, at, ldb, none, at, yd, 5, m, 5, 3, ws, size, none)

    assert linear(m=0) == 0 and linear(x=none) == bad and linear(ldx=-1) == bad and linear(ldb=63) == bad
    assert linear(xd=5) == unsupported and linear(yd=5) == unsupported
    need = lib.tn_int8_linear_workspace(100, 3)
    assert need == 100 * 64 + 400 and lib.tn_int8_linear_workspace(4, 3) == 0 and lib.tn_int8_linear_workspace(4, 0) == bad
    assert linear(m=100) == bad and linear(m=100, ws=at, size=need - 1) == bad and linear(m=100, ws=C.c_void_p(4104), size=need) == bad


def test_tiles_refuse_rows_further_apart_than_they_can_address():
    """128 rows of a tile have to lie within 2^31 - 1 bytes: a pitch beyond that is refused before anything is launched"""
    lib = _lib.load()
    at, none, unsupported = C.c_void_p(4096), C.c_void_p(0), -2
    most = (2 ** 31 - 1) // 128 // 64 * 64
    for lda, ldb in ((most + 64, 64), (64, most + 64), (2 ** 25, 64), (64, 2 ** 33), (2 ** 40, 2 ** 40)):
        for m, k in ((33, 3), (100, 64), (4, 20000)):
            lda_, ldb_ = max(lda, 20032), max(ldb, 20032)
            assert lib.tn_int8_matmul(at, at, lda_, at, at, ldb_, none, at, 0, 5, m, 5, k, none) == unsupported
            if ldb_ > most:
                size = lib.tn_int8_linear_workspace(m, k)
                assert lib.tn_int8_linear(at, 0, k, at, at, ldb_, none, at, 0, 5, m, 5, k, at, size, none) == unsupported


def test_products_of_operands_that_left_the_device():
    """rows and layers whose buffers were moved to the host: refused before a kernel gets their addresses"""
    rows = Int8Rows._of(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4), 3)
    layer = Int8Linear.__new__(Int8Linear)
    torch.nn.Module.__init__(layer)
    layer.in_features, layer.out_features = 3, 4
    for name, t in (("codes", rows._padded), ("scales", rows.scales), ("bias", torch.zeros(4))):
        layer.register_buffer(name, t)
    for call in (lambda: int8_matmul(torch.ones(2, 3), rows), lambda: int8_matmul(torch.ones(64, 3), rows), lambda: int8_matmul(rows, rows),
                 lambda: layer(torch.ones(2, 3)), lambda: layer(torch.ones(64, 3, dtype=torch.bfloat16)), lambda: layer(torch.ones(0, 3))):
        with pytest.raises(RuntimeError, match="no CPU execution path"):
            call()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
def test_cosine_scores_are_float32_whatever_the_embeddings_are(dtype):
    """a row of zeros scores 0 against everything (in half precision the norm's lower bound of 1e-8 is no number of the type)"""
    g = torch.Generator().manual_seed(1)
    e, other = torch.randn(5, 24, generator=g).to(dtype), torch.randn(3, 24, generator=g).to(dtype)
    e[2] = 0
    for args in ((e,), (e, other)):
        y = cosine_scores(*args)
        a, b = (t.double() / t.double().norm(dim=1, keepdim=True).clamp(min=1e-8) for t in (args[0], args[-1]))
        # both unit rows and a sum of 24 products, each rounded in float32
        assert y.dtype == torch.float32 and float((y - a @ b.t()).abs().max()) <= 40 * 2.0 ** -24 and not y[2].any()


def test_scores_refuse_before_they_compute():
    rows = Int8Rows._of(torch.zeros(4, 64, dtype=torch.int8), torch.ones(4), 3)
    with pytest.raises(TypeError, match="bits=8"):
        cosine_scores(torch.ones(2, 3), rows)
    with pytest.raises(ValueError, match="score_bits"):
        verification_test(None, [], [], score_bits=16)
