"""The 8-bit product and its row quantiser against exact integer sums.

Codes and scales equal the definition's (the scale is one correctly rounded division, codes are decided by exact remainders).  The
product then differs from the exact one by u = 2^-24 for each of: the sum's conversion to float32, the two scales, the bias, and
half a step of a 16-bit output."""
import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from tests import int8_oracle as O
from titanet_amd import LOSSES
from titanet_amd.int8 import Int8Linear, Int8Rows, int8_matmul, quantize_rows

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {"fp32": 0.0, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def _np(t):
    return t.detach().double().cpu().numpy()


def _x(m, k, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g))).to(dtype).cuda()


def _compare(y, want, part, dtype):
    bound = U * (3 * np.abs(part) + np.abs(want) + np.abs(part))
    bound = bound + HALF_STEP[dtype] * (np.abs(want) + bound) + (2.0 ** -25 if dtype == "fp16" else 1e-38)
    off = np.abs(_np(y) - want)
    assert (off <= bound).all(), (off.max(), np.unravel_index(off.argmax(), off.shape))


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("m,k", [(1, 1), (3, 15), (5, 64), (130, 65), (7, 192), (4, 1000), (33, 1536), (2, 5001), (1, 131071)])
def test_quantised_rows(m, k, dtype):
    x = _x(m, k, 1, TYPES[dtype])
    if m > 2:
        x[1] = 0
    q = quantize_rows(x)
    codes, scales = O.quantize(_np(x))
    assert np.array_equal(q.codes.cpu().numpy(), codes) and np.array_equal(q.scales.cpu().numpy(), scales)
    assert not q._padded[:, k:].any() and q.shape == (m, k) and len(q) == m
    np.testing.assert_allclose(_np(q.dequantize()), codes * scales.astype(np.float64)[:, None], rtol=U, atol=1e-44)


def test_quantised_borders():
    """half way goes to the even code; rows around the smallest and largest floats; what is not finite"""
    row = torch.tensor([127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -126.5, 126.49999], device="cuda")
    assert quantize_rows(row[None]).codes.tolist() == [[127, 0, 2, 2, 0, -2, -126, 126]]
    g = torch.Generator().manual_seed(2)
    near = (torch.randint(-254, 255, (64, 512), generator=g) * 0.5).cuda()
    near = torch.cat([near, torch.nextafter(near, torch.full_like(near, 1e9)), torch.nextafter(near, torch.full_like(near, -1e9))], 1)
    near[:, 0] = 127.0
    for x in (near, near * 0.37, near * 1e30, near * 2.0 ** -120, near * 2.0 ** -133, near * 2.0 ** -140):
        q = quantize_rows(x)
        codes, scales = O.quantize(_np(x))
        assert np.array_equal(q.scales.cpu().numpy(), scales) and np.array_equal(q.codes.cpu().numpy(), codes)
    top = torch.full((2, 70), torch.finfo(torch.float32).max, device="cuda")
    assert bool((quantize_rows(top).codes == 127).all())
    x = _x(4, 100, 3)
    x[1, 5], x[2, 99], x[3, 0] = float("nan"), float("inf"), -float("inf")
    q = quantize_rows(x)
    assert torch.isnan(q.scales).tolist() == [False, True, True, True] and not q.codes[1:].any()
    y = int8_matmul(x, quantize_rows(_x(9, 100, 4)))
    assert torch.isnan(y).all(1).tolist() == [False, True, True, True] and not bool(torch.isnan(y[0]).any())


@pytest.mark.parametrize("m", [1, 2, 5, 16, 17, 33, 64, 129, 300])
@pytest.mark.parametrize("n,k", [(1, 1), (7, 15), (64, 64), (251, 192), (192, 1536), (513, 65), (130, 4100)])
def test_product(m, n, k):
    for x_type, out, bias in (("fp32", "fp32", True), ("bf16", "bf16", False), ("fp16", "fp32", True), ("codes", "fp16", False)):
        x, w = _x(m, k, 5, TYPES.get(x_type, torch.float32)), _x(n, k, 6) * (0.1 / k ** 0.5)
        b = torch.randn(n, device="cuda") if bias else None
        qb = quantize_rows(w)
        y = int8_matmul(quantize_rows(x) if x_type == "codes" else x, qb, bias=b, out_dtype=TYPES[out])
        want, part = O.product(*O.quantize(_np(x)), *O.quantize(_np(w)), None if b is None else _np(b))
        assert y.shape == (m, n) and y.dtype == TYPES[out]
        _compare(y, want, part, out)


@pytest.mark.parametrize("m,n,k", [(1000, 777, 300), (9631, 512, 512), (257, 7205, 192), (2049, 130, 2000), (1, 100003, 192), (16, 4099, 1024)])
def test_larger_products(m, n, k):
    x, w = _x(m, k, 7, torch.bfloat16), _x(n, k, 8)
    b = torch.randn(n, device="cuda")
    want, part = O.product(*[a.astype(np.float64) for a in O.quantize(_np(x))], *[a.astype(np.float64) for a in O.quantize(_np(w))], _np(b))
    _compare(int8_matmul(x, quantize_rows(w), bias=b, out_dtype=torch.float32), want, part, "fp32")


@pytest.mark.parametrize("m", [1, 40, 200])
def test_longest_sums(m):
    """codes of -128 and 127 over the longest rows the product takes: no sum leaves 32 bits"""
    k = 131071
    a, b = torch.full((m, k), -128, dtype=torch.int8, device="cuda"), torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    b[1] = 127
    b[2, ::2] = 127
    one = torch.ones(m, device="cuda")
    y = int8_matmul(Int8Rows(a, one), Int8Rows(b, torch.ones(3, device="cuda")))
    want = (a[:1].cpu().numpy().astype(np.int64) @ b.cpu().numpy().astype(np.int64).T).astype(np.float32)
    assert np.array_equal(y.cpu().numpy(), np.repeat(want, m, 0))
    with pytest.raises(ValueError):
        Int8Rows(torch.zeros(1, k + 1, dtype=torch.int8, device="cuda"), one[:1])


def test_strides_shapes_and_empty_operands():
    w = quantize_rows(_x(40, 96, 9))
    x = _x(24, 200, 10)
    plain = int8_matmul(x[:, 8:104].contiguous(), w)
    assert torch.equal(int8_matmul(x[:, 8:104], w), plain)                                        # rows of a larger matrix
    assert torch.equal(int8_matmul(x[:, 8:104].t().contiguous().t(), w), plain)                   # columns first
    assert torch.equal(int8_matmul(x[:, 8:104].contiguous().view(2, 3, 4, 96), w), plain.view(2, 3, 4, 40))
    assert torch.equal(int8_matmul(x[3, 8:104], w), plain[3])
    assert torch.equal(int8_matmul(x[3:4, 8:104].expand(5, 96), w), plain[3:4].expand(5, 40))
    assert torch.equal(int8_matmul(x[::3, 8:104], w), plain[::3])
    assert int8_matmul(x[:0, 8:104], w).shape == (0, 40) and int8_matmul(x[:, :5], quantize_rows(x[:0, :5])).shape == (24, 0)
    for t in (torch.bfloat16, torch.float16, torch.float32):                                      # rows that begin at any element
        odd = x.to(t).view(-1)[1:24 * 199 + 1].view(24, 199)
        for first in (1, 2, 5):
            for m in (3, 24):
                part = odd[:m, first:first + 96]
                assert torch.equal(int8_matmul(part, w), int8_matmul(part.contiguous(), w)) and torch.equal(quantize_rows(part).codes, quantize_rows(part.contiguous()).codes)
        tall = x.to(t).repeat(3, 1)[:, 3:99]
        assert torch.equal(int8_matmul(tall, w), int8_matmul(tall.contiguous(), w))
    inner = torch.zeros(40, 200, dtype=torch.int8, device="cuda")
    inner[:, 3:99] = w.codes
    inner[:, 99:] = 77                                                                            # what lies behind the codes is no part of them
    assert torch.equal(int8_matmul(x[:, 8:104], Int8Rows(inner[:, 3:99], w.scales)), plain)
    bias = torch.randn(80, device="cuda")[::2]
    torch.testing.assert_close(int8_matmul(x[:, 8:104], w, bias=bias), plain + bias, rtol=4 * U, atol=4 * U * float(plain.abs().max()))


def test_refusals_on_the_device():
    w, x = quantize_rows(_x(4, 8, 1)), _x(3, 8, 2)
    for bad in (x.double(), x.to(torch.int32)):
        with pytest.raises(TypeError):
            int8_matmul(bad, w)
    with pytest.raises(TypeError):
        int8_matmul(x, w, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        int8_matmul(x[:, :7], w)
    with pytest.raises(ValueError):
        int8_matmul(x.cpu(), w)
    for bias in (torch.zeros(3, device="cuda"), torch.zeros(4), torch.zeros(4, device="cuda", dtype=torch.float16)):
        with pytest.raises(ValueError):
            int8_matmul(x, w, bias=bias)
    with pytest.raises(RuntimeError, match="no backward pass"):
        int8_matmul(x.requires_grad_(True), w)
    with torch.no_grad():
        assert int8_matmul(x, w).shape == (3, 4)


def test_streams_and_graphs():
    w = quantize_rows(_x(700, 192, 11))
    xs = [_x(5, 192, 12 + k) for k in range(4)]
    want = [int8_matmul(x, w) for x in xs]
    big = [_x(300, 192, 22 + k) for k in range(4)]
    want_big = [int8_matmul(x, w, out_dtype=torch.bfloat16) for x in big]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for k in range(4):                                        # two calls at once
        with torch.cuda.stream(sides[k % 2]):
            got.append((int8_matmul(xs[k], w), int8_matmul(big[k], w, out_dtype=torch.bfloat16)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(c, d) for (a, c), b, d in zip(got, want, want_big))
    x, y = xs[0].clone(), big[0].clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        int8_matmul(x, w), int8_matmul(y, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        small, large = int8_matmul(x, w), int8_matmul(y, w, out_dtype=torch.bfloat16)
    for k in (1, 2, 3, 0):
        x.copy_(xs[k])
        y.copy_(big[k])
        graph.replay()
        other = int8_matmul(xs[(k + 1) % 4], w)               # eager work between the replays
        torch.cuda.synchronize()
        assert torch.equal(small, want[k]) and torch.equal(large, want_big[k]) and torch.equal(other, want[(k + 1) % 4])


def test_more_outputs_than_32_bits_count():
    n = 46350
    x, w = _x(n, 16, 13), _x(n, 16, 14)
    qx, qw = quantize_rows(x), quantize_rows(w)
    y = int8_matmul(qx, qw, out_dtype=torch.bfloat16)
    assert y.numel() > 2 ** 31
    for rows, cols in ((slice(0, 64), slice(0, 64)), (slice(n - 70, n), slice(n - 70, n)), (slice(n - 3, n), slice(0, 5))):
        want, part = O.product(*O.quantize(_np(x[rows])), *O.quantize(_np(w[cols])))
        _compare(y[rows, cols], want, part, "bf16")


def test_more_codes_than_32_bits_count():
    rows = 2 ** 31 // 64 + 77
    w = torch.zeros(rows, 3, dtype=torch.bfloat16, device="cuda")
    w[-100:] = _x(100, 3, 15, torch.bfloat16)
    w[:100] = _x(100, 3, 16, torch.bfloat16)
    q = quantize_rows(w)
    for x in (_x(1, 3, 17), _x(40, 3, 18)):
        for some in (slice(0, 100), slice(rows - 100, rows)):
            want, part = O.product(*O.quantize(_np(x)), *O.quantize(_np(w[some])))
            _compare(int8_matmul(x, q)[:, some], want, part, "fp32")
    back = int8_matmul(Int8Rows._of(q._padded, q.scales, 3), quantize_rows(_x(2, 3, 19)))
    want, part = O.product(*O.quantize(_np(w[-100:])), *O.quantize(_np(_x(2, 3, 19))))
    _compare(back[-100:], want, part, "fp32")


def test_a_head_served_in_8_bits():
    torch.manual_seed(1)
    loss = LOSSES["ce"](192, 251, device="cuda")
    layer = Int8Linear.from_linear(loss.fc)
    x = torch.randn(50, 192, device="cuda")
    with torch.no_grad():
        y = layer(x)
        full = x @ loss.fc.weight.t() + loss.fc.bias
    # rows of 192 values of unit size, each rounded by at most half a step of max / 127 in both operands
    assert float((y - full).norm() / (full - loss.fc.bias).norm()) < 0.02
    assert layer.in_features == 192 and layer.out_features == 251 and set(layer.state_dict()) == {"codes", "scales", "bias"}
    other = Int8Linear(torch.zeros(251, 192, device="cuda"), torch.zeros(251, device="cuda"))
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), y) and layer(x.bfloat16()).dtype == torch.bfloat16
    with pytest.raises(TypeError):
        layer.half()(x)


@pytest.mark.parametrize("m,n,k", [(20000, 1536, 1536), (30001, 300, 640), (700, 30000, 192), (5000, 512, 512)])
def test_every_output_of_large_products_time_after_time(m, n, k):
    """all outputs of launches of many workgroups, several times over: waves that run ahead of others may not overwrite what these read"""
    g = torch.Generator(device="cuda").manual_seed(20)
    a, b = (torch.randint(-127, 128, (r, k), generator=g, device="cuda", dtype=torch.int8) for r in (m, n))
    sa, sb = torch.rand(m, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda")
    want = a.float() @ b.float().t()                          # whole numbers below 2^24 on the way: exact
    assert float(want.abs().max()) < 2 ** 23
    want = want * sa[:, None] * sb[None, :]
    qa, qb = Int8Rows(a, sa), Int8Rows(b, sb)
    for _ in range(6):
        assert torch.equal(int8_matmul(qa, qb), want)


@pytest.mark.parametrize("m", [1, 5, 32, 33, 200])
@pytest.mark.parametrize("n,k", [(7, 64), (130, 192), (251, 700)])
def test_large_rows_against_small_weights(m, n, k):
    """rows whose sums times one scale leave float32 while the products do not, ordinary and tiny rows beside them"""
    x, w = _x(m, k, 30), _x(n, k, 31) * 1e-4
    x[::3] *= 3e37 / float(x.abs().max())
    x[1::3] *= 1e-30
    x[2::6] = 0
    for a, b, out in ((x, w, "fp32"), (x, w, "bf16"), (w, x, "fp32")):
        want, part = O.product(*O.quantize(_np(a)), *O.quantize(_np(b)))
        assert np.abs(want).max() < 3e38
        for left in (a, quantize_rows(a)):
            _compare(int8_matmul(left, quantize_rows(b), out_dtype={"fp32": torch.float32, "bf16": torch.bfloat16}[out]), want, part, out)


@pytest.mark.parametrize("m,k", [(31, 192), (32, 1), (32, 192), (32, 1984), (32, 1985), (31, 2048), (31, 2049)])
def test_products_at_the_ends_of_the_few_rows_kernel(m, k):
    """the most rows, and the longest for that many, that are quantised inside the product, and the next ones"""
    for n in (5, 130):
        x, w = _x(m, k, 32), _x(n, k, 33)
        want, part = O.product(*O.quantize(_np(x)), *O.quantize(_np(w)))
        for a in (x, quantize_rows(x)):
            _compare(int8_matmul(a, quantize_rows(w)), want, part, "fp32")


def test_gradients_are_not_dropped():
    x, w = _x(3, 8, 2).requires_grad_(True), quantize_rows(_x(4, 8, 1))
    with pytest.raises(RuntimeError, match="no backward pass"):
        quantize_rows(x)
    with pytest.raises(RuntimeError, match="no backward pass"):
        quantize_rows(x * 2)
    scales = torch.ones(4, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="no backward pass"):
        Int8Rows(w.codes, scales)
    with torch.no_grad():
        assert int8_matmul(quantize_rows(x), Int8Rows(w.codes, scales)).shape == (3, 4)
    assert quantize_rows(x.detach()).shape == (3, 8)
    layer = Int8Linear(torch.nn.Parameter(_x(4, 8, 1)), torch.nn.Parameter(torch.ones(4, device="cuda")))     # weights are laid out once, for serving
    assert layer(x.detach()).shape == (3, 4)
    with pytest.raises(RuntimeError, match="no backward pass"):
        layer(x)


def test_tangents_are_not_dropped():
    x, w, bias = _x(3, 8, 2), quantize_rows(_x(4, 8, 1)), torch.ones(4, device="cuda")
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="no backward pass"):
            int8_matmul(dual, w)
        with pytest.raises(RuntimeError, match="no backward pass"):
            quantize_rows(dual)
        with pytest.raises(RuntimeError, match="no backward pass"):
            int8_matmul(x, w, bias=forward_ad.make_dual(bias, bias))
        with pytest.raises(RuntimeError, match="no backward pass"):
            int8_matmul(quantize_rows(x), w, bias=forward_ad.make_dual(bias, bias))
        assert int8_matmul(x, w, bias=bias).shape == (3, 4)


def test_a_product_is_not_traced():
    x = _x(3, 8, 2)
    layer = Int8Linear(_x(4, 8, 1))
    for call in (layer, lambda a: int8_matmul(quantize_rows(a), quantize_rows(x)), lambda a: quantize_rows(a).codes):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, x, check_trace=False)
    assert layer(x).shape == (3, 4)


@pytest.mark.parametrize("m", [3, 40])
def test_scales_of_either_sign_and_any_size(m):
    """codes and scales in hand: the sum times one of them may leave float32, the product does not"""
    g = torch.Generator().manual_seed(34)
    a, b = (torch.randint(-127, 128, (r, 96), generator=g, dtype=torch.int8).cuda() for r in (m, 21))
    sa, sb = torch.full((m,), -2.0 ** 120, device="cuda"), torch.full((21,), 2.0 ** -30, device="cuda")
    sa[1::2], sb[::3] = 2.0 ** -140, -2.0 ** -20
    y = int8_matmul(Int8Rows(a, sa), Int8Rows(b, sb))
    want, part = O.product(a.cpu().numpy().astype(np.int64), _np(sa), b.cpu().numpy().astype(np.int64), _np(sb))
    _compare(y, want, part, "fp32")
    y = int8_matmul(Int8Rows(b, sb), Int8Rows(a, sa))
    _compare(y, want.T, part.T, "fp32")
