"""Cases for the optimizer step over many tensors (titanet_amd.optim) and the 8-bit integer matrix product (titanet_amd.int8).

``run`` computes a case in its plain form with elementary torch operations; with ``own`` set it makes the calls a user makes
of the framework.  Every case is one of two kinds:

  op = "adamw"   one AdamW step over a list of tensors, its two moments held in 32 bits or as 8-bit codes with a scale for
                 each block of 256 elements, with or without clipping by the global gradient norm.  Returned: the parameters,
                 both moments as the values they stand for, the norm.
  op = "int8"    y[m, n] = sa[m] sb[n] sum_k qa[m, k] qb[n, k] (+ bias[n]): the weight's codes qb and channel scales sb are laid
                 out once; the activations' codes and token scales are computed in the call, or in hand (x = "codes").

The 8-bit forms, both rounding to the nearest value:
  moments   exp_avg = sign (c / 127)^2 M, c = 0..127, M = max |exp_avg| of the block;
            exp_avg_sq = (c / 255)^4 V, c = 0..255, V = max exp_avg_sq of the block, a value above 0 keeps c >= 1; c is the
            nearest in the root's domain, the lower one half way
  rows      q = x / s rounded to the nearest integer (even half way), s = max(max |row| / 127, 2^-126), 0 for a row of zeros
"""
import random

import torch

own = False

BLOCK = 256                       # elements that share a scale of the 8-bit moments; every tensor begins at such a boundary
LR, BETA1, BETA2, EPS, WD, STEPS_DONE = 1e-3, 0.9, 0.999, 1e-8, 0.01, 100
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the published small model, parameter by parameter, as its training loop steps it: 428 tensors from 16 x 256 to 1536 x 256
        {"name": "adamw32-small-model", "op": "adamw", "kind": "model", "hidden": 256, "blocks": 17, "taps": 3, "classes": 251, "bits": 32, "dtype": "fp32", "clip": 1.0},
        {"name": "adamw8-small-model", "op": "adamw", "kind": "model", "hidden": 256, "blocks": 17, "taps": 3, "classes": 251, "bits": 8, "dtype": "fp32", "clip": 1.0},
        # the large model with the speakers of a big corpus in its head, no clipping
        {"name": "adamw32-large-model", "op": "adamw", "kind": "model", "hidden": 1024, "blocks": 5, "taps": 11, "classes": 7205, "bits": 32, "dtype": "fp32", "clip": 0.0},
        # the table of a head over 333333 speakers: the one tensor that makes 8-bit moments worth having
        {"name": "adamw8-speaker-table", "op": "adamw", "kind": "table", "rows": 333333, "cols": 192, "bits": 8, "dtype": "fp32", "clip": 0.0},
        # a handful of biases and norms being fine-tuned: nothing but latency
        {"name": "adamw32-few-small", "op": "adamw", "kind": "ragged", "count": 7, "most": 1537, "bits": 32, "dtype": "bf16", "clip": 1.0},
        # adapters of every size, odd ones among them, in bf16
        {"name": "adamw8-ragged", "op": "adamw", "kind": "ragged", "count": 48, "most": 2000003, "bits": 8, "dtype": "bf16", "clip": 0.5},
        # one embedding against the speakers of a head: the answer to a single request
        {"name": "int8-one-row", "op": "int8", "m": 1, "n": 7205, "k": 192, "x": "bf16", "out": "fp32", "bias": True},
        # the decoder's last linear for a few utterances
        {"name": "int8-few-rows", "op": "int8", "m": 16, "n": 192, "k": 1536, "x": "fp32", "out": "fp32", "bias": True},
        # a training batch's worth of embeddings against a large head
        {"name": "int8-batch-head", "op": "int8", "m": 250, "n": 100003, "k": 192, "x": "fp16", "out": "fp16", "bias": False},
        # the frames of a ragged batch through a pointwise layer of the medium model
        {"name": "int8-ragged-frames", "op": "int8", "m": 9631, "n": 512, "k": 512, "x": "bf16", "out": "bf16", "bias": True},
        # every test utterance against an enrolled gallery, both quantised beforehand
        {"name": "int8-gallery", "op": "int8", "m": 4708, "n": 50021, "k": 192, "x": "codes", "out": "fp32", "bias": False},
        # the frames of a full batch (256 x 300) through a 1536-wide layer
        {"name": "int8-wide-frames", "op": "int8", "m": 76800, "n": 1536, "k": 1536, "x": "bf16", "out": "bf16", "bias": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    if rng.random() < 0.5:
        c = {"op": "adamw", "bits": rng.choice((8, 32)), "dtype": rng.choice(("fp32", "fp32", "bf16", "fp16")),
             "clip": rng.choice((0.0, 1.0, rng.choice((0.1, 20.0))))}
        kind = rng.choice(("model", "table", "ragged"))
        if kind == "model":
            hidden, taps = rng.choice(((256, 3), (512, 7), (1024, 11)))
            c.update(kind=kind, hidden=hidden, taps=taps, blocks=rng.randint(1, {256: 17, 512: 10, 1024: 5}[hidden]), classes=_log_int(rng, 2, 20000))
        elif kind == "table":
            c.update(kind=kind, rows=_log_int(rng, 1, 160000), cols=rng.choice((192, rng.randint(1, 256))))
        else:
            c.update(kind=kind, count=_log_int(rng, 1, 60), most=_log_int(rng, 3, 500000))
        return c
    k = rng.choice((192, 256, 512, 1024, 1536, _log_int(rng, 1, 1600)))
    m = _log_int(rng, 1, 60000)
    n = rng.choice((192, 256, 512, 1536, _log_int(rng, 1, 100000)))
    n = max(1, min(n, 150_000_000 // m, 90_000_000_000 // (m * k)))
    return {"op": "int8", "m": m, "n": n, "k": k, "x": rng.choice(("bf16", "fp32", "fp16", "codes")),
            "out": rng.choice(("bf16", "fp32", "fp16")), "bias": rng.random() < 0.5}


def _shapes(case):
    """the tensors of an optimizer case"""
    if case["kind"] == "table":
        return [(case["rows"], case["cols"])]
    if case["kind"] == "ragged":
        r = random.Random(case["count"] * 1000003 + case["most"])
        return [(case["most"],)] + [(_log_int(r, 1, case["most"]),) for _ in range(case["count"] - 1)]
    h, wide, att, emb, classes = case["hidden"], 1536, 128, 192, case["classes"]
    norm = lambda c: [(c,), (c,)]  # noqa: E731
    sub = [(h, 1, case["taps"]), (h,), (h, h, 1), (h,)] + norm(h)
    block = 3 * sub + [(h // 16, h), (h, h // 16), (h, h, 1), (h,)] + norm(h)
    return ([(h, 80, 3), (h,)] + norm(h) + case["blocks"] * block + [(wide, h, 1), (wide,)] + norm(wide) + [(att, wide), (att,), (wide, att), (wide,)]
            + norm(2 * wide) + [(emb, 2 * wide), (emb,)] + norm(emb) + [(classes, emb), (classes,)])


def _numel(shape):
    n = 1
    for s in shape:
        n *= s
    return n


# ----------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    if case["op"] == "int8":
        return _prepare_int8(case, g)
    shapes = _shapes(case)
    sizes = [_numel(s) for s in shapes]
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    dtype = DTYPES[case["dtype"]]
    # what lies between the tensors is 0 and stays 0
    live = torch.zeros(at // BLOCK, BLOCK, dtype=torch.bool, device="cuda")
    for s, n in zip(starts, sizes):
        live.view(-1)[s:s + n] = True
    def normal():
        return torch.randn(at // BLOCK, BLOCK, generator=g, device="cuda") * live
    # gradients whose size differs from block to block by orders of magnitude, as those of layers and speakers do
    size = torch.exp(1.5 * torch.randn(at // BLOCK, 1, generator=g, device="cuda") - 7.0)
    params, grads = (0.05 * normal()).to(dtype), (size * normal()).to(dtype)
    exp_avg = 0.3 * size * normal()
    exp_avg_sq = torch.exp(1.2 * torch.randn(at // BLOCK, BLOCK, generator=g, device="cuda")) * size * size * live
    state = {"case": case, "params": params.view(-1), "grads": grads.view(-1), "step": STEPS_DONE}
    if own:
        from titanet_amd.optim import AdamW
        tensors = []
        for s, n, shape in zip(starts, sizes, shapes):
            p = state["params"][s:s + n].view(shape).requires_grad_(True)
            p.grad = state["grads"][s:s + n].view(shape)
            tensors.append(p)
        state["optimizer"] = AdamW(tensors, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=WD, state_bits=case["bits"],
                                   max_grad_norm=case["clip"] or None)
        state["optimizer"].load_moments(exp_avg.view(-1), exp_avg_sq.view(-1), step=STEPS_DONE)
    elif case["bits"] == 8:
        state["exp_avg"], state["exp_avg_sq"] = _first_codes(exp_avg.double()), _second_codes(exp_avg_sq.double())
    else:
        state["exp_avg"], state["exp_avg_sq"] = exp_avg, exp_avg_sq
    return state


def _prepare_int8(case, g):
    m, n, k = case["m"], case["n"], case["k"]
    weight = torch.randn(n, k, generator=g, device="cuda") * torch.exp(0.5 * torch.randn(n, 1, generator=g, device="cuda")) * k ** -0.5
    x = torch.randn(m, k, generator=g, device="cuda") * torch.exp(torch.randn(m, 1, generator=g, device="cuda"))
    state = {"case": case, "b": _row_codes(weight), "bias": torch.randn(n, generator=g, device="cuda") if case["bias"] else None}
    if case["x"] == "codes":
        state["a"] = _row_codes(x)
    else:
        state["x"] = x.to(DTYPES[case["x"]])
    if own:
        from titanet_amd.int8 import Int8Rows
        state["b"] = Int8Rows(*state["b"])
        if case["x"] == "codes":
            state["x"] = Int8Rows(*state["a"])
    return state


# ------------------------------------------------------------------------------------------------------- the plain forms
def _first_codes(x):
    """codes and block scales of exp_avg, float64 [blocks, 256]: in 64 bits, since the codes turn at borders"""
    top = x.abs().amax(1, keepdim=True).float()
    ratio = x.abs() / torch.where(top > 0, top, torch.ones_like(top)).double()
    return torch.sign(x) * torch.clamp(torch.ceil(127 * torch.sqrt(ratio) - 0.5), 0, 127), top


def _second_codes(x):
    top = x.amax(1, keepdim=True).float()
    ratio = x / torch.where(top > 0, top, torch.ones_like(top)).double()
    return torch.where(x > 0, torch.clamp(torch.ceil(255 * torch.sqrt(torch.sqrt(ratio)) - 0.5), 1, 255), 0.0), top


def _first_values(codes, top):
    return torch.sign(codes) * (codes / 127) ** 2 * top.double()


def _second_values(codes, top):
    return (codes / 255) ** 4 * top.double()


def _row_codes(x):
    """int8 codes and float32 scales of the rows of x: in 64 bits, since the codes turn at borders"""
    x = x.double()
    top = x.abs().amax(1)
    scale = torch.where(top > 0, torch.clamp(top / 127, min=2.0 ** -126), 0.0).float()
    safe = torch.where(scale > 0, scale, torch.ones_like(scale)).double()
    return torch.round(x / safe[:, None]).to(torch.int8), scale


def run(state):
    case = state["case"]
    if case["op"] == "int8":
        return _run_int8(state, case)
    if own:
        opt = state["optimizer"]
        opt.step()
        exp_avg, exp_avg_sq = opt.moments()
        out = {"params": state["params"], "exp_avg": exp_avg, "exp_avg_sq": exp_avg_sq}
        if case["clip"]:
            out["norm"] = opt.last_grad_norm
        return out
    state["step"] += 1
    eight, clip = case["bits"] == 8, case["clip"]
    out = {}
    wide = torch.float64 if eight else torch.float32
    g = state["grads"].to(wide).view(-1, BLOCK)
    if clip:
        norm = torch.sqrt(state["grads"].double().square().sum())
        g = g * torch.clamp(clip / (norm + 1e-6), max=1.0).to(wide)
        out["norm"] = norm.float()
    m = _first_values(*state["exp_avg"]) if eight else state["exp_avg"]
    v = _second_values(*state["exp_avg_sq"]) if eight else state["exp_avg_sq"]
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * (g * g)
    rate, root = LR / (1 - BETA1 ** state["step"]), (1 - BETA2 ** state["step"]) ** 0.5
    p = state["params"].float().view(-1, BLOCK) * (1 - LR * WD)
    p = p - rate * (m.float() / (torch.sqrt(v.float()) / root + EPS))
    state["params"].copy_(p.view(-1))
    if eight:
        state["exp_avg"], state["exp_avg_sq"] = _first_codes(m), _second_codes(v)
        m, v = _first_values(*state["exp_avg"]).float(), _second_values(*state["exp_avg_sq"]).float()
    else:
        state["exp_avg"], state["exp_avg_sq"] = m, v
    out.update(params=state["params"], exp_avg=m.view(-1), exp_avg_sq=v.view(-1))
    return out


def _run_int8(state, case):
    out = DTYPES[case["out"]]
    if own:
        from titanet_amd.int8 import int8_matmul
        return int8_matmul(state["x"], state["b"], bias=state["bias"], out_dtype=out)
    a, sa = state["a"] if case["x"] == "codes" else _row_codes(state["x"])
    b, sb = state["b"]
    y = (a.float() @ b.float().t()) * sa[:, None] * sb[None, :]        # the products and their sums are whole numbers below 2^24
    if state["bias"] is not None:
        y = y + state["bias"]
    return y.to(out)


# ------------------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "int8":
        m, n, k = case["m"], case["n"], case["k"]
        size = {"fp32": 4, "bf16": 2, "fp16": 2}
        a = m * (k + 4) if case["x"] == "codes" else m * k * size[case["x"]]
        return {"bytes": a + n * (k + 4) + (4 * n if case["bias"] else 0) + m * n * size[case["out"]], "flops": 2 * m * n * k}
    sizes = [_numel(s) for s in _shapes(case)]
    n, blocks = sum(sizes), sum((s + BLOCK - 1) // BLOCK for s in sizes)
    p = 4 if case["dtype"] == "fp32" else 2
    # parameter read and written, gradient read; two moments read and written, or their codes and scales, and then their values
    each = 3 * p + (16 if case["bits"] == 32 else 4 + 8)
    return {"bytes": n * each + (16 * blocks if case["bits"] == 8 else 0), "flops": n * (16 if case["clip"] else 14)}


# ------------------------------------------------------------------------------------------------ the definition, 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "int8":
        def rows(x):
            x = x.to(torch.float64)
            most = torch.maximum(x.max(1).values, -x.min(1).values)
            s = (most / 127).float().double()
            s[(most > 0) & (s < 2.0 ** -126)] = 2.0 ** -126
            codes = torch.zeros_like(x)
            some = s > 0
            codes[some] = (x[some] / s[some].unsqueeze(1)).round()
            return codes, s
        a, sa = (t.double() for t in state["a"]) if "a" in state else rows(state["x"])
        b, sb = (t.double() for t in state["b"])
        y = torch.empty(case["m"], case["n"], dtype=torch.float64, device="cuda")
        for lo in range(0, case["m"], 8192):
            hi = min(case["m"], lo + 8192)
            torch.mm(a[lo:hi] * sa[lo:hi].unsqueeze(1), (b * sb.unsqueeze(1)).t().contiguous(), out=y[lo:hi])
        return y if state["bias"] is None else y.add_(state["bias"].double())
    t = STEPS_DONE + 1
    grads, params = state["grads"].double(), state["params"].double()
    length = torch.linalg.vector_norm(grads)
    if case["clip"] and float(length) + 1e-6 > case["clip"]:
        grads = grads * (case["clip"] / (float(length) + 1e-6))
    # the values the codes can take, relative to the block's largest, and the borders between neighbours in the root's domain
    table1 = torch.tensor([(c / 127.0) ** 2 for c in range(128)], dtype=torch.float64, device="cuda")
    edges1 = torch.tensor([((c + 0.5) / 127.0) ** 2 for c in range(127)], dtype=torch.float64, device="cuda")
    table2 = torch.tensor([(c / 255.0) ** 4 for c in range(256)], dtype=torch.float64, device="cuda")
    edges2 = torch.tensor([0.0] + [((c + 0.5) / 255.0) ** 4 for c in range(1, 255)], dtype=torch.float64, device="cuda")
    if case["bits"] == 8:
        c1, top1 = state["exp_avg"]
        c2, top2 = state["exp_avg_sq"]
        m = (table1[c1.abs().long()] * top1.double()).view(-1)
        m = torch.where(c1.view(-1) < 0, -m, m)
        v = (table2[c2.long()] * top2.double()).view(-1)
    else:
        m, v = state["exp_avg"].double().view(-1), state["exp_avg_sq"].double().view(-1)
    m.mul_(BETA1).add_(grads, alpha=1 - BETA1)
    v.mul_(BETA2).addcmul_(grads, grads, value=1 - BETA2)
    hat1, hat2 = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
    out = {"params": params - LR * WD * params - LR * hat1 / (hat2.sqrt() + EPS)}
    if case["clip"]:
        out["norm"] = length
    if case["bits"] == 8:
        def stored(x, table, edges):
            x = x.view(-1, BLOCK)
            top = x.abs().max(1, keepdim=True).values.float().double()
            code = torch.searchsorted(edges, (x.abs() / torch.where(top > 0, top, 1.0)).contiguous())
            return (torch.sign(x) * table[code] * top).view(-1)
        m, v = stored(m, table1, edges1), stored(v, table2, edges2)
    out.update(exp_avg=m, exp_avg_sq=v)
    return out
