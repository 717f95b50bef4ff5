"""Matrix products in 8-bit integers with a scale for each token and each channel.

    gallery = quantize_rows(enrolled)                       # [speakers, E] float -> codes and scales, once
    scores = int8_matmul(embeddings, gallery)               # [utterances, speakers]: the embeddings are quantised in the call
    head = Int8Linear.from_linear(loss.fc)                  # a head or any other linear layer, for serving

The reference multiplies in float32 (the heads' ``nn.Linear``, reference src/losses.py:30; the cosine scores of its test, reference
src/learn.py:441-447).  Here both operands are int8 rows with one float32 scale each, the sums are exact 32-bit integers
(``tn_int8_matmul``, include/titanet_amd.h) and one multiplication by both scales follows.  For serving: there is no backward
pass and no CPU fallback.
"""
import torch
import torch.nn as nn

from . import _lib

MAX_K = 131071       # TN_INT8_MAX_K: 128 * 128 * MAX_K still fits 32 bits


def _need_device(t, what):
    if not t.is_cuda:
        raise RuntimeError(f"titanet_amd.int8: {what} must be a ROCm device tensor; there is no CPU execution path")


class Int8Rows:
    """Rows of int8 codes with a float32 scale each: row r stands for ``scales[r] * codes[r]``.  Held with every row padded by
    zeros to a multiple of 64 bytes, as the product reads them; ``codes`` is the unpadded view."""

    def __init__(self, codes, scales):
        if codes.dtype != torch.int8 or codes.dim() != 2 or codes.shape[1] < 1:
            raise TypeError(f"codes must be an int8 matrix, got {codes.dtype} {tuple(codes.shape)}")
        if scales.dtype != torch.float32 or tuple(scales.shape) != (codes.shape[0],):
            raise TypeError(f"scales must be float32, one for each of the {codes.shape[0]} rows, got {scales.dtype} {tuple(scales.shape)}")
        if codes.shape[1] > MAX_K:
            raise ValueError(f"rows of more than {MAX_K} codes could overflow the 32-bit sums")
        _need_device(codes, "codes")
        if scales.device != codes.device:
            raise ValueError(f"codes and scales are on different devices: {codes.device} and {scales.device}")
        if torch.is_grad_enabled() and scales.requires_grad:
            raise RuntimeError("Int8Rows has no backward pass: detach its scales or build it under torch.no_grad()")
        rows, cols = codes.shape
        padded = torch.zeros(rows, (cols + 63) // 64 * 64, dtype=torch.int8, device=codes.device)
        padded[:, :cols] = codes.detach()
        self._padded, self.scales, self.cols = padded, scales.detach().contiguous(), cols

    @classmethod
    def _of(cls, padded, scales, cols):
        r = cls.__new__(cls)
        r._padded, r.scales, r.cols = padded, scales, cols
        return r

    @property
    def codes(self):
        return self._padded[:, :self.cols]

    @property
    def shape(self):
        return torch.Size((self._padded.shape[0], self.cols))

    @property
    def device(self):
        return self._padded.device

    def __len__(self):
        return self._padded.shape[0]

    def dequantize(self):
        """the float32 values the rows stand for"""
        return self.codes.float() * self.scales[:, None]


def quantize_rows(x):
    """``Int8Rows`` of a float matrix (float32, bfloat16 or float16): scale max |row| / 127 (at least 2^-126; 0 for a row of
    zeros), codes the nearest integers to x / scale, even half way.  A row with a NaN or an infinity gets the scale NaN.  There is no backward
    pass: a matrix that needs a gradient is refused outside ``torch.no_grad()``."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"quantize_rows takes a float32, bfloat16 or float16 matrix, got {type(x).__name__}")
    padded, scales = _lib.load_host().quantize_rows(x)
    return Int8Rows._of(padded, scales, x.shape[1])


def int8_matmul(a, b, bias=None, out_dtype=None):
    """``a @ b.T (+ bias)`` in 8-bit integers: ``b`` an :class:`Int8Rows` [N, K], ``a`` one of [M, K] or a float tensor [..., K]
    whose rows are quantised in the call; ``bias`` float32 [N].  Returns [..., N] in ``out_dtype`` (float32, bfloat16, float16;
    default: that of a float ``a``, else float32)."""
    if not isinstance(b, Int8Rows):
        raise TypeError(f"the second operand must be Int8Rows (quantize_rows), got {type(b).__name__}")
    if isinstance(a, torch.Tensor):
        return _lib.load_host().matmul_float(a, b._padded, b.scales, b.cols, bias, out_dtype)
    if isinstance(a, Int8Rows):
        return _lib.load_host().matmul_rows(a._padded, a.scales, a.cols, b._padded, b.scales, b.cols, bias, out_dtype)
    raise TypeError(f"the first operand must be Int8Rows or a tensor, got {type(a).__name__}")


class Int8Linear(nn.Module):
    """A linear layer for serving: int8 weight rows with a scale per output channel, inputs quantised per token in the call."""

    def __init__(self, weight, bias=None):
        super().__init__()
        rows = quantize_rows(weight.detach())
        self.in_features, self.out_features = rows.cols, len(rows)
        self.register_buffer("codes", rows._padded)
        self.register_buffer("scales", rows.scales)
        self.register_buffer("bias", None if bias is None else bias.detach().float().clone())

    @classmethod
    def from_linear(cls, module):
        """from a module with ``weight`` [out, in] and optionally ``bias`` (an ``nn.Linear``, a loss head's ``fc``)"""
        return cls(module.weight, getattr(module, "bias", None))

    def forward(self, x, out_dtype=None):
        if self.scales.dtype != torch.float32:
            raise TypeError("Int8Linear keeps float32 scales: do not convert it to another type")
        return int8_matmul(x, Int8Rows._of(self.codes, self.scales, self.in_features), bias=self.bias, out_dtype=out_dtype)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
