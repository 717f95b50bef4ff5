"""AdamW and the 8-bit form of its moments in float64 (numpy), from the definitions."""
import numpy as np

BLOCK = 256
EDGES1 = ((np.arange(127) + 0.5) / 127) ** 2                             # between |codes| 0 .. 127 of exp_avg, relative to the block's scale
EDGES2 = np.concatenate([[0.0], ((np.arange(1, 255) + 0.5) / 255) ** 4])      # between codes 0 .. 255 of exp_avg_sq; above 0 is code 1 at least


def _blocks(x):
    n = x.size
    out = np.zeros(((n + BLOCK - 1) // BLOCK, BLOCK))
    out.reshape(-1)[:n] = x
    return out


def encode(x, second):
    """(codes, float32 scales) of one tensor's moment"""
    n, x = x.size, _blocks(np.asarray(x, np.float64).ravel())
    top = np.abs(x).max(1).astype(np.float32)
    ratio = np.abs(x) / np.where(top > 0, top, 1).astype(np.float64)[:, None]
    code = np.searchsorted(EDGES2 if second else EDGES1, ratio, side="left")
    code = np.where(top[:, None] > 0, code, 0)
    return (np.where(x < 0, -code, code)).reshape(-1)[:n], top


def decode(code, top, second):
    c = _blocks(np.asarray(code, np.float64))
    v = (c / 255) ** 4 if second else np.sign(c) * (c / 127) ** 2
    return (v * top.astype(np.float64)[:, None]).reshape(-1)[:code.size]


class Tensor:
    """one parameter with its moments; step() returns what the tolerances count with"""

    def __init__(self, p, bits):
        self.p, self.bits, self.t = np.asarray(p, np.float64).ravel().copy(), bits, 0
        self.m, self.v = np.zeros_like(self.p), np.zeros_like(self.p)
        self.c1 = self.c2 = None

    def step(self, g, lr, b1=0.9, b2=0.999, eps=1e-8, wd=0.01, factor=1.0):
        g = np.asarray(g, np.float64).ravel() * factor
        self.t += 1
        size = np.abs(b1 * self.m) + np.abs((1 - b1) * g)
        self.m = b1 * self.m + (1 - b1) * g
        self.v = b2 * self.v + (1 - b2) * g * g
        denom = np.sqrt(self.v) / np.sqrt(1 - b2 ** self.t) + eps
        rate = lr / (1 - b1 ** self.t)
        update = rate * self.m / denom
        self.p = self.p * (1 - lr * wd) - update
        if self.bits == 8:
            self.c1, self.s1 = encode(self.m, False)
            self.c2, self.s2 = encode(self.v, True)
            self.m, self.v = decode(self.c1, self.s1, False), decode(self.c2, self.s2, True)
        return size, np.abs(update), rate * size / denom


def clip_factor(norm, max_norm):
    return min(1.0, max_norm / (norm + 1e-6))
