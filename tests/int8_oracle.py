"""The 8-bit product in float64 / int64 (numpy), from the definition."""
import numpy as np


def quantize(x):
    """(int64 codes, float32 scales) of the rows of a float64 matrix of finite values"""
    top = np.abs(x).max(1)
    scale = np.where(top > 0, np.maximum(top / 127, 2.0 ** -126), 0).astype(np.float32)
    s = np.where(scale > 0, scale, 1).astype(np.float64)[:, None]
    return np.where(scale[:, None] > 0, np.rint(x / s), 0).astype(np.int64), scale


def product(qa, sa, qb, sb, bias=None):
    """(y, the product without its bias) in float64; the integer sums are exact"""
    y = (qa @ qb.T).astype(np.float64) * sa.astype(np.float64)[:, None] * sb.astype(np.float64)[None, :]
    return (y if bias is None else y + bias.astype(np.float64)), y
