"""AdamW over many tensors (32- and 8-bit moments) and the global gradient norm against float64.

Tolerances count roundings of u = 2^-24 (float32, half a step) per operation of the step:
  exp_avg     b1, 1 - b1 and the gradient's factor are rounded, then two products and a sum:   5 u (|b1 m| + |(1 - b1) g|)
  exp_avg_sq  the factor twice over, its product twice over, the square, 1 - b2, a product, a sum:  8 u v
  parameter   u (3 (|p| + |update|) + 16 rate (|b1 m| + |(1 - b1) g|) / denominator), and half a step of a 16-bit type
8-bit moments are decided in 64 bits: their codes equal the oracle's, scales are within one float32 step."""
import copy

import numpy as np
import pytest
import torch

from tests import optim_oracle as O
from titanet_amd import LOSSES, TitaNet
from titanet_amd.optim import BLOCK, AdamW, grad_norm

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {"fp32": 0.0, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
MIXED = [1, 3, 255, 256, 257, 1000, 4095, 4096, 4097, 12289]
MANY = [1 + (37 * i) % 700 for i in range(230)]                         # more tensors than one launch names


def _np(t):
    return t.detach().double().cpu().numpy().ravel()


def _tensors(sizes, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(n, generator=g)).to(dtype).cuda() for n in sizes]


def _grads(sizes, dtype, seed, scale=1e-2):
    """sizes differing by orders of magnitude from tensor to tensor"""
    g = torch.Generator().manual_seed(seed)
    return [(scale * float(torch.exp(2 * torch.randn((), generator=g))) * torch.randn(n, generator=g)).to(dtype).cuda() for n in sizes]


def _check(opt, params, oracles, before, dtype, bits):
    m, v = (x.cpu().numpy().astype(np.float64) for x in opt.moments())
    for i, (p, o) in enumerate(zip(params, oracles)):
        lo, n = int(opt._first[i]) * BLOCK, p.numel()
        size, update, reach = before[i]
        p_old = o.p_old
        bound = U * (3 * (np.abs(p_old) + update) + 16 * reach)
        bound = bound + HALF_STEP[dtype] * (np.abs(o.p) + bound) + (2.0 ** -25 if dtype == "fp16" else 1e-40)
        off = np.abs(_np(p) - o.p)
        assert (off <= bound).all(), (i, n, off.max(), bound[off.argmax()])
        if bits == 32:
            assert (np.abs(m[lo:lo + n] - o.m) <= 5 * U * size + 1e-44).all() and (np.abs(v[lo:lo + n] - o.v) <= 8 * U * o.v + 1e-44).all(), (i, n)
        else:
            codes1, codes2 = (x[lo:lo + n].cpu().numpy().astype(np.int64) for x in (opt._exp_avg, opt._exp_avg_sq))
            assert np.array_equal(codes1, o.c1) and np.array_equal(codes2, o.c2), (i, n)
            b, k = int(opt._first[i]), (n + BLOCK - 1) // BLOCK
            np.testing.assert_allclose(opt._scale1[b:b + k].cpu().numpy(), o.s1, rtol=2 * U, atol=1.5e-45)
            np.testing.assert_allclose(opt._scale2[b:b + k].cpu().numpy(), o.s2, rtol=2 * U, atol=1.5e-45)
            np.testing.assert_allclose(m[lo:lo + n], o.m, rtol=4 * U, atol=1.5e-45)
            np.testing.assert_allclose(v[lo:lo + n], o.v, rtol=4 * U, atol=1.5e-45)
        assert not m[lo + n:lo + (n + 255) // 256 * 256].any() and not v[lo + n:lo + (n + 255) // 256 * 256].any()


def _follow(opt, params, oracles, dtype, bits, grads, **hyper):
    """one step of both; the oracle goes on from the kernel's parameters and moments, so that every step is checked by itself"""
    m0, v0 = (x.cpu().numpy().astype(np.float64) for x in opt.moments())
    for i, (p, o, g) in enumerate(zip(params, oracles, grads)):
        p.grad = g
        o.p = o.p_old = _np(p)
        if bits == 32:
            lo = int(opt._first[i]) * BLOCK
            o.m, o.v = m0[lo:lo + p.numel()].copy(), v0[lo:lo + p.numel()].copy()
    opt.step()
    factor = hyper.pop("factor", 1.0)
    before = [o.step(_np(g), factor=factor, **hyper) for o, g in zip(oracles, grads)]
    _check(opt, params, oracles, before, dtype, bits)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("sizes,clip", [([1], None), (MIXED, None), (MIXED, 0.5), (MANY, 1e-3), ([70001], 1e9)])
def test_steps_against_float64(sizes, clip, dtype, bits):
    params = _tensors(sizes, TYPES[dtype], 1)
    opt = AdamW(params, lr=2e-3, betas=(0.9, 0.99), weight_decay=0.1, state_bits=bits, max_grad_norm=clip)
    oracles = [O.Tensor(_np(p), bits) for p in params]
    for k in range(4):
        grads = _grads(sizes, TYPES[dtype], 10 + k)
        norm = float(np.sqrt(sum((_np(g) ** 2).sum() for g in grads)))
        _follow(opt, params, oracles, dtype, bits, grads, lr=2e-3, b2=0.99, wd=0.1, factor=O.clip_factor(norm, clip) if clip else 1.0)
        if clip:
            assert abs(float(opt.last_grad_norm) - norm) <= 2 * U * norm


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_tensors_at_any_offset_and_their_neighbours(dtype, bits):
    """views that begin at odd elements of larger buffers: what lies around them keeps its values"""
    sizes, t = [1, 5, 255, 1023, 5000], TYPES[dtype]
    base, gbase = torch.full((9000,), 7.0, dtype=t, device="cuda"), torch.full((9000,), 3.0, dtype=t, device="cuda")
    inside = torch.zeros(9000, dtype=torch.bool, device="cuda")
    params, grads, at = [], [], 1
    for i, n in enumerate(sizes):
        params.append(base[at:at + n])
        grads.append(gbase[at + 2:at + 2 + n])
        params[-1].copy_(_tensors([n], t, 40 + i)[0])
        grads[-1].copy_(_tensors([n], t, 50 + i, 0.1)[0])
        inside[at:at + n] = True
        at += n + 3 + i
    opt = AdamW(params, lr=1e-2, state_bits=bits, max_grad_norm=1.0)
    oracles = [O.Tensor(_np(p), bits) for p in params]
    norm = float(np.sqrt(sum((_np(g) ** 2).sum() for g in grads)))
    for _ in range(2):
        _follow(opt, params, oracles, dtype, bits, grads, lr=1e-2, factor=O.clip_factor(norm, 1.0))
    assert bool((base[~inside] == 7.0).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_neighbouring_tensors_are_stepped_as_if_apart(bits):
    """parameters that follow one another in memory (a flat buffer's views) and ones that do not give the same numbers"""
    sizes = [256, 512, 192, 64, 768, 4096, 300, 256]
    values, grads = torch.cat(_tensors(sizes, torch.float32, 5)), torch.cat(_grads(sizes, torch.float32, 6))
    together, apart, at = [], [], 0
    for n in sizes:
        p = values[at:at + n]
        p.grad = grads[at:at + n]
        together.append(p)
        q = p.clone()
        q.grad = p.grad.clone()
        apart.append(q)
        at += n
    opts = [AdamW(x, state_bits=bits, max_grad_norm=0.1) for x in (together, apart)]
    for _ in range(3):
        for opt in opts:
            opt.step()
    for p, q in zip(together, apart):
        assert torch.equal(p, q)
    for a, b in zip(opts[0].moments(), opts[1].moments()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("scale", [0.0, 1e-30, 1e-12, 1e15, 1e30])
def test_small_and_large_gradients(scale, bits):
    """second moments from denormal to beyond float32 (8 bits: the block turns NaN there, 32 bits: infinity, as the formula's)"""
    params = _tensors([700], torch.float32, 3)
    opt = AdamW(params, state_bits=bits)
    o = O.Tensor(_np(params[0]), bits)
    g = scale * _tensors([700], torch.float32, 4)[0]
    if scale == 1e30:
        params[0].grad = g
        opt.step()
        m, v = opt.moments()
        if bits == 8:
            assert bool(torch.isnan(m[:700]).all()) and bool(torch.isnan(v[:700]).all())
        else:
            assert bool((v[:700] == float("inf")).any()) and bool(torch.isfinite(m).all())
        assert bool(torch.isfinite(params[0]).all())
        return
    if scale == 1e-30:                       # squares below float32's range vanish from the update's root, not from the double-precision codes
        params[0].grad = g
        opt.step()
        assert bool(torch.isfinite(params[0]).all()) and all(bool(torch.isfinite(x).all()) for x in opt.moments())
        return
    for _ in range(2):
        _follow(opt, params, [o], "fp32", bits, [g], lr=1e-3)


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_finite(bits):
    params = _tensors([600, 300], torch.float32, 8)
    kept = [p.clone() for p in params]
    opt = AdamW(params, state_bits=bits, max_grad_norm=1.0)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for p, g in zip(params, _grads([600, 300], torch.float32, 9)):
            p.grad = g
        params[0].grad[17] = bad
        opt.step()
        assert all(torch.equal(p, k) for p, k in zip(params, kept)) and not float(opt.last_grad_norm) < float("inf")
        assert not any(bool(x.any()) for x in opt.moments()) and opt.state_dict()["state"] == {}
    params[0].grad[17] = 0.25                     # the step after a skipped one is the first
    norm = float(np.sqrt(sum((_np(p.grad) ** 2).sum() for p in params)))
    _follow(opt, params, [O.Tensor(_np(p), bits) for p in params], "fp32", bits, [p.grad for p in params], lr=1e-3, factor=O.clip_factor(norm, 1.0))
    # without a norm to go by the value reaches its element, or its block of 256
    opt = AdamW(params, state_bits=bits)
    params[0].grad[300] = float("nan")
    opt.step()
    m = opt.moments()[0]
    nan = torch.isnan(m).nonzero().view(-1).tolist()
    assert nan == ([300] if bits == 32 else list(range(256, 512)))
    assert torch.isnan(params[0]).nonzero().view(-1).tolist() == [300] and bool(torch.isfinite(params[1]).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_without_gradients_keep_their_own_count(bits):
    sizes = [300, 10, 513]
    params = _tensors(sizes, torch.float32, 11)
    opt = AdamW(params, state_bits=bits, lr=1e-2)
    oracles = [O.Tensor(_np(p), bits) for p in params]
    for k, active in enumerate([(0, 1, 2), (0, 2), (2,), (0, 1, 2), (1,), (0, 1, 2)]):
        grads = _grads(sizes, torch.float32, 60 + k)
        kept = [p.clone() for p in params]
        m0, v0 = (x.cpu().numpy().astype(np.float64) for x in opt.moments())
        for i, p in enumerate(params):
            p.grad = grads[i] if i in active else None
            oracles[i].p = oracles[i].p_old = _np(p)
            if bits == 32:
                lo = int(opt._first[i]) * BLOCK
                oracles[i].m, oracles[i].v = m0[lo:lo + p.numel()].copy(), v0[lo:lo + p.numel()].copy()
        opt.step()
        before = {i: oracles[i].step(_np(grads[i]), lr=1e-2) for i in active}
        for i in active:
            size, update, reach = before[i]
            bound = U * (3 * (np.abs(oracles[i].p_old) + update) + 16 * reach)
            assert (np.abs(_np(params[i]) - oracles[i].p) <= bound).all(), (k, i)
        assert all(torch.equal(params[i], kept[i]) for i in range(3) if i not in active)
    steps = {i: int(e["step"]) for i, e in opt.state_dict()["state"].items()}
    assert steps == {0: 4, 1: 4, 2: 5}
    other = AdamW([p.clone() for p in params], state_bits=bits)
    other.load_state_dict(opt.state_dict())
    assert {i: int(e["step"]) for i, e in other.state_dict()["state"].items()} == steps
    with pytest.raises(RuntimeError):
        params[0].data = params[0].data[:10].clone()
        params[0].grad = torch.ones(10, device="cuda")
        opt.step()


def test_groups_types_and_a_scheduler():
    """two groups of their own hyper-parameters, types mixed within one, one norm over all of them; a torch scheduler sets lr"""
    a, b = _tensors([400, 33], torch.float32, 12), _tensors([777], torch.bfloat16, 13)
    c = _tensors([1000], torch.float32, 14)
    opt = AdamW([{"params": a + b, "lr": 1e-2, "weight_decay": 0.0}, {"params": c, "betas": (0.5, 0.75), "eps": 1e-3}], lr=3e-3, max_grad_norm=0.2)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, gamma=0.5)
    every = a + b + c
    oracles = [O.Tensor(_np(p), 32) for p in every]
    for k in range(3):
        grads = [g.to(p.dtype) for g, p in zip(_grads([400, 33, 777, 1000], torch.float32, 70 + k), every)]
        m0, v0 = (x.cpu().numpy().astype(np.float64) for x in opt.moments())
        for i, (p, g, o) in enumerate(zip(every, grads, oracles)):
            p.grad = g
            lo = int(opt._first[i]) * BLOCK
            o.p, o.m, o.v = _np(p), m0[lo:lo + p.numel()].copy(), v0[lo:lo + p.numel()].copy()
            o.p_old = o.p
        opt.step()
        norm = float(np.sqrt(sum((_np(g) ** 2).sum() for g in grads)))
        factor = O.clip_factor(norm, 0.2)
        assert abs(float(opt.last_grad_norm) - norm) <= 2 * U * norm
        for i, o in enumerate(oracles):
            kw = dict(lr=1e-2 * 0.5 ** k, wd=0.0) if i < 3 else dict(lr=3e-3 * 0.5 ** k, b1=0.5, b2=0.75, eps=1e-3)
            size, update, reach = o.step(_np(grads[i]), factor=factor, **kw)
            bound = U * (3 * (np.abs(o.p_old) + update) + 16 * reach)
            bound = bound + HALF_STEP["bf16" if i == 2 else "fp32"] * (np.abs(o.p) + bound)
            assert (np.abs(_np(every[i]) - o.p) <= bound).all(), (k, i)
        sched.step()
    opt.add_param_group({"params": _tensors([5], torch.float32, 15), "lr": 1.0})
    assert len(opt.state_dict()["param_groups"]) == 3 and opt.moments()[0].numel() == opt.blocks * BLOCK


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_replays(bits):
    sizes = [1000, 64, 2, 4097]
    params, twin = _tensors(sizes, torch.float32, 20), _tensors(sizes, torch.float32, 20)
    lr, lr2 = (torch.full((), 1e-2, device="cuda") for _ in range(2))
    opt, eager = AdamW(params, lr=lr, state_bits=bits, max_grad_norm=0.3), AdamW(twin, lr=lr2, state_bits=bits, max_grad_norm=0.3)
    for p, q in zip(params, twin):
        p.grad, q.grad = torch.zeros_like(p), torch.zeros_like(q)

    def give(k):
        for p, q, g in zip(params, twin, _grads(sizes, torch.float32, 80 + k)):
            if k == 3:
                g[0] = float("nan")              # one replay that is skipped
            p.grad.copy_(g)
            q.grad.copy_(g)
        lr.fill_(1e-2 / (k + 1))
        lr2.fill_(1e-2 / (k + 1))

    side = torch.cuda.Stream()
    give(0)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(1, 6):
        give(k)
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(params, twin)), k
        assert all(torch.equal(a, b) for a, b in zip(opt.moments(), eager.moments())), k
        assert torch.equal(opt.last_grad_norm, eager.last_grad_norm) or k == 3
    assert {int(e["step"]) for e in opt.state_dict()["state"].values()} == {5}
    frozen = AdamW([torch.ones(3, device="cuda")], lr=1e-3)
    frozen.param_groups[0]["params"][0].grad = torch.ones(3, device="cuda")
    with pytest.raises(RuntimeError, match="device tensor to capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            frozen.step()


def test_a_partial_step_is_not_captured_and_two_graphs_share_an_optimizer():
    """a graph for each of two gradient buffers, replayed in turn with eager steps between them"""
    p, q = _tensors([5000], torch.float32, 25)[0], _tensors([5000], torch.float32, 25)[0]
    lr, lr2 = (torch.full((), 1e-2, device="cuda") for _ in range(2))
    opt, eager = AdamW([p], lr=lr, max_grad_norm=1.0, state_bits=8), AdamW([q], lr=lr2, max_grad_norm=1.0, state_bits=8)
    grads, graphs = _grads([5000, 5000], torch.float32, 26), []
    p.grad = grads[0]
    opt.step()
    q.grad = grads[0]
    eager.step()
    for g in grads:
        p.grad = g
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            opt.step()
    for k in (0, 1, 1, 0, 2, 0, 1):
        if k < 2:
            graphs[k].replay()
            q.grad = grads[k]
        else:
            p.grad = q.grad = grads[0] * 0.5
            opt.step()
        eager.step()
        torch.cuda.synchronize()
        assert torch.equal(p, q) and all(torch.equal(a, b) for a, b in zip(opt.moments(), eager.moments())), k
    a, b = (torch.ones(300, device="cuda") for _ in range(2))
    some = AdamW([a, b], lr=lr)
    a.grad = torch.ones(300, device="cuda")
    with pytest.raises(RuntimeError, match="run such a step once"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            some.step()


def test_on_another_stream():
    params, twin = _tensors([100000], torch.float32, 21), _tensors([100000], torch.float32, 21)
    opt, plain = AdamW(params, max_grad_norm=0.1), AdamW(twin, max_grad_norm=0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for k in range(5):
        with torch.cuda.stream(side):
            params[0].grad = torch.sin(params[0] * (k + 1))
            opt.step()
        twin[0].grad = torch.sin(twin[0] * (k + 1))
        plain.step()
    side.synchronize()
    assert torch.equal(params[0], twin[0])


def test_checkpoints_of_either_width_and_torchs():
    sizes = [1000, 7, 256]
    params = _tensors(sizes, torch.float32, 22)
    ref = [torch.nn.Parameter(p.clone()) for p in params]
    torchs = torch.optim.AdamW(ref, lr=1e-2, weight_decay=0.1)
    for k in range(3):
        for p, g in zip(ref, _grads(sizes, torch.float32, 90 + k)):
            p.grad = g
        torchs.step()
    for p, q in zip(params, ref):
        p.copy_(q.detach())
    wide, narrow = AdamW(params, state_bits=32), AdamW([p.clone() for p in params], state_bits=8)
    wide.load_state_dict(torchs.state_dict())
    narrow.load_state_dict(torchs.state_dict())
    assert wide.param_groups[0]["lr"] == 1e-2 and wide.param_groups[0]["weight_decay"] == 0.1
    assert all(int(e["step"]) == 3 for e in wide.state_dict()["state"].values())
    grads = _grads(sizes, torch.float32, 99)
    for p, q, g in zip(params, ref, grads):
        p.grad, q.grad = g, g.clone()
    wide.step()
    torchs.step()
    for p, q in zip(params, ref):
        torch.testing.assert_close(p, q.detach(), rtol=1e-6, atol=1e-6)      # two float32 computations of updates up to lr = 1e-2
    # back to torch
    again = torch.optim.AdamW([torch.nn.Parameter(p.clone()) for p in params], lr=1e-2)
    again.load_state_dict(copy.deepcopy(wide.state_dict()))
    # 8 bits: codes survive their values, and a width change in between
    codes = copy.deepcopy(narrow.state_dict())
    assert codes["state"][0]["exp_avg"].dtype == torch.int8 and codes["state"][0]["exp_avg_sq"].dtype == torch.uint8
    wide.load_state_dict(codes)
    other = AdamW([p.clone() for p in params], state_bits=8)
    other.load_state_dict(wide.state_dict())
    for i, e in other.state_dict()["state"].items():
        for key, value in e.items():
            assert torch.equal(value, codes["state"][i][key]), (i, key)
    m, v = narrow.moments()
    other.load_moments(m, v, step=3)
    for a, b in zip((other._exp_avg, other._exp_avg_sq, other._scale1, other._scale2), (narrow._exp_avg, narrow._exp_avg_sq, narrow._scale1, narrow._scale2)):
        assert torch.equal(a, b)
    # a tensor lr stays the tensor it is (a captured step reads it) and takes the loaded value
    lr = torch.full((), 5.0, device="cuda")
    held = AdamW([p.clone() for p in params], lr=lr, state_bits=8)
    held.load_state_dict(codes)
    assert held.param_groups[0]["lr"] is lr and abs(float(lr) - 1e-2) < 1e-9
    with pytest.raises(TypeError, match="state_dict"):
        copy.deepcopy(other)
    with pytest.raises(ValueError):
        other.load_moments(m[1:], v[1:], step=1)
    with pytest.raises(ValueError):
        AdamW([p.clone() for p in params[:2]]).load_state_dict(codes)


def test_refusals_on_the_device():
    p = torch.ones(8, device="cuda")
    for bad in ([p, p], [p, p[2:5]]):
        with pytest.raises(ValueError):
            AdamW(bad)
    with pytest.raises(ValueError):
        AdamW([torch.ones(4, 6, device="cuda").t()])
    opt = AdamW([p])
    p.grad = torch.ones(8, device="cuda").to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()
    opt.param_groups[0]["lr"] = -1.0
    p.grad = torch.ones(8, device="cuda")
    with pytest.raises(ValueError):
        opt.step()
    assert bool((p == 1).all())


def test_gradients_with_strides_and_none_at_all():
    p, q = torch.ones(6, 4, device="cuda"), torch.ones(6, 4, device="cuda")
    opt, plain = AdamW([p]), AdamW([q])
    opt.step()                                          # nothing has a gradient: nothing happens
    assert bool((p == 1).all())
    for g in (torch.arange(24.0, device="cuda").view(4, 6).t(), torch.full((1, 1), 0.5, device="cuda").expand(6, 4)):
        p.grad, q.grad = g, g.contiguous()
        v = p._version
        opt.step()
        plain.step()
        assert p._version > v
    assert torch.equal(p, q)
    empty = torch.empty(0, device="cuda")
    empty.grad = torch.empty(0, device="cuda")
    AdamW([empty], max_grad_norm=1.0).step()
    loss = opt.step(lambda: torch.tensor(2.5))
    assert float(loss) == 2.5


@pytest.mark.parametrize("sizes", [[1], [3, 16384, 16385, 50000], MANY, [3_000_001]])
def test_grad_norm(sizes):
    ts = [t.to(d) for t, d in zip(_grads(sizes, torch.float32, 30, 1.0), [torch.float32, torch.bfloat16, torch.float16] * len(sizes))]
    want = float(np.sqrt(sum((_np(t) ** 2).sum() for t in ts)))
    got = grad_norm(ts)
    assert got.shape == () and got.dtype == torch.float32 and abs(float(got) - want) <= 2 * U * want
    assert torch.equal(got, grad_norm([t.clone() for t in ts]))              # a fixed order of summation, whatever the addresses
    assert float(grad_norm([torch.zeros(9, device="cuda")])) == 0.0
    huge = torch.full((1000,), 1e30, device="cuda")
    assert abs(float(grad_norm(huge)) / (1e30 * 1000 ** 0.5) - 1) < 1e-6
    assert np.isnan(float(grad_norm([ts[0], torch.full((3,), float("nan"), device="cuda")])))
    assert abs(float(grad_norm(torch.ones(4, 6, device="cuda").t()[::2])) - 12 ** 0.5) < 1e-6


def test_more_elements_than_32_bits_count():
    """a bfloat16 table of 2^31 + 1001 elements with 8-bit moments: its first and last elements are stepped like small tensors"""
    n = 2 ** 31 + 1001
    p = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    p.grad = torch.full((n,), 1e-3, dtype=torch.bfloat16, device="cuda")
    ends = [slice(0, 2048), slice(n - n % 256 - 2048, n)]
    for k, s in enumerate(ends):
        p[s] = _tensors([s.stop - s.start], torch.bfloat16, 31 + k)[0]
        p.grad[s] = _tensors([s.stop - s.start], torch.bfloat16, 33 + k, 1e-2)[0]
    small = [p[s].clone() for s in ends]
    for q, s in zip(small, ends):
        q.grad = p.grad[s].clone()
    opt, ref = AdamW([p], lr=1e-2, state_bits=8), AdamW(small, lr=1e-2, state_bits=8)
    for _ in range(2):
        opt.step()
        ref.step()
    assert all(torch.equal(p[s], q) for s, q in zip(ends, small))
    lo = ends[1].start
    assert torch.equal(opt._exp_avg[lo:n], ref._exp_avg[2048:2048 + n - lo]) and torch.equal(opt._exp_avg_sq[:2048], ref._exp_avg_sq[:2048])
    middle = p[2 ** 30:2 ** 30 + 5]
    assert bool((middle == middle[0]).all()) and float(middle[0]) != 0.5


@pytest.mark.parametrize("bits", [32, 8])
def test_titanet_parameters(bits):
    """the network's own parameters through autograd, against the same steps on its flat buffer"""
    torch.manual_seed(5)
    kw = dict(n_mels=80, n_mega_blocks=1, n_sub_blocks=3, encoder_hidden_size=256, encoder_output_size=1536, embedding_size=192,
              mega_block_kernel_size=3, dropout=0.0)
    model = TitaNet(loss_function=LOSSES["ce"](192, 11, device="cuda"), device="cuda", **kw).train()
    x, y = torch.randn(6, 80, 64, device="cuda"), torch.randint(0, 11, (6,), device="cuda")
    flat = model.flat_parameters().clone()
    opt, whole = AdamW(model.parameters(), lr=1e-3, state_bits=bits, max_grad_norm=1.0), AdamW([flat], lr=1e-3, state_bits=32, max_grad_norm=1.0)
    for k in range(4):
        opt.zero_grad()
        loss = model(x, speakers=y)[2]
        loss.backward()
        if k == 0:
            flat.grad = model.flat_gradients().clone()
            whole.step()
        opt.step()
        if k == 0:
            # the first step does not depend on how moments are held, but for the roundings of 32 bits
            torch.testing.assert_close(flat, model.flat_parameters(), rtol=6 * U, atol=1e-3 * 32 * U)
    assert bool(torch.isfinite(model.flat_parameters()).all())


@pytest.mark.parametrize("top", [3e38, 2.0 ** 127, 1.7e38, 2.0 ** 126, 2.0 ** 125, 1e30, 2.0 ** -99, 2.0 ** -100, 2.0 ** -101, 1e-31, 1e-37, 1e-40, 2.0 ** -149])
def test_codes_of_the_largest_and_smallest_scales(top):
    """blocks whose largest moment lies near either end of float32: codes and scales are the definition's"""
    top = float(np.float32(top))
    x = torch.randn(700, generator=torch.Generator().manual_seed(35), dtype=torch.float64)
    x = (x / x.abs().max() * top).float()
    x[[0, 256]], x[699] = top, -top
    m, v = (torch.zeros(768, device="cuda") for _ in range(2))
    m[:700], v[:700] = x.cuda(), x.abs().cuda()
    opt = AdamW([torch.zeros(700, device="cuda")], state_bits=8)
    opt.load_moments(m, v, step=5)
    for codes, scales, back, y, second in zip((opt._exp_avg, opt._exp_avg_sq), (opt._scale1, opt._scale2), opt.moments(), (x, x.abs()), (False, True)):
        want, tops = O.encode(y.double().numpy(), second)
        assert np.array_equal(scales.cpu().numpy(), tops) and np.array_equal(codes[:700].cpu().numpy().astype(np.int64), want)
        np.testing.assert_allclose(back[:700].cpu().numpy(), O.decode(want, tops, second), rtol=4 * U, atol=1.5e-45)


def test_8_bit_steps_whose_squares_come_near_the_largest_float():
    params = _tensors([700], torch.float32, 3)
    opt, o = AdamW(params, state_bits=8), O.Tensor(_np(params[0]), 8)
    for scale in (1.2e20, 1e19, 0.0):
        _follow(opt, params, [o], "fp32", 8, [scale * _tensors([700], torch.float32, 4)[0]], lr=1e-3)
        assert scale < 1e20 or 2.0 ** 126 < float(opt._scale2.max()) < float("inf")


@pytest.mark.parametrize("bits", [32, 8])
def test_a_graph_and_steps_of_some_tensors_count_together(bits):
    """replays, eager steps of all or of some tensors and loaded states, in any order: every tensor has its own count"""
    sizes = [256, 512, 300, 64]                  # the first ones follow one another in memory, whole blocks
    values, grads = torch.cat(_tensors(sizes, torch.float32, 36)), torch.cat(_grads(sizes, torch.float32, 37))

    def build():
        params, at = list(values.clone().split(sizes)), list(grads.clone().split(sizes))
        return params, at, AdamW(params, lr=torch.full((), 1e-2, device="cuda"), state_bits=bits, max_grad_norm=0.3)
    (p, g, opt), (q, h, eager) = build(), build()

    def give(active):
        for k in range(4):
            p[k].grad, q[k].grad = (g[k], h[k]) if k in active else (None, None)

    def same(what):
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(p, q)), what
        assert all(torch.equal(a, b) for a, b in zip(opt.moments(), eager.moments())), what
        a, b = ({i: int(e["step"]) for i, e in o.state_dict()["state"].items()} for o in (opt, eager))
        assert a == b, (what, a, b)

    def some(*active):
        give(active)
        opt.step()
        eager.step()
        same(("eager", active))

    def replay(graph):
        graph.replay()
        give(range(4))
        eager.step()
        same("replay")

    def capture():
        give(range(4))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
        return graph

    some(0, 1, 2, 3)
    first = capture()
    replay(first)
    for _ in range(3):
        some(0)
    replay(first)
    some(1, 3)
    second = capture()
    for graph in (second, first, second):
        replay(graph)
        some(0, 1, 2, 3)
    state = copy.deepcopy(eager.state_dict())
    unequal = copy.deepcopy(state)
    for e in state["state"].values():
        e["step"] = torch.tensor(7.0)
    for loaded in (state, unequal, state):
        opt.load_state_dict(copy.deepcopy(loaded))
        eager.load_state_dict(copy.deepcopy(loaded))
        for graph in (first, second):
            replay(graph)
            some(2)
            some(0, 1, 2, 3)
    m, v = (x.clone() for x in eager.moments())
    for o in (opt, eager):
        o.load_moments(m, v, step=2)
    replay(second)
    some(1)
    replay(first)
    some(0, 1, 2, 3)


@pytest.mark.parametrize("bits", [32, 8])
def test_no_group_is_added_once_a_step_is_captured(bits):
    """a graph writes the buffers that the optimizer had when it was captured: these stay where they are"""
    p, q = _tensors([300], torch.float32, 41)[0], _tensors([300], torch.float32, 41)[0]
    opt, eager = (AdamW([x], lr=torch.full((), 1e-2, device="cuda"), state_bits=bits) for x in (p, q))
    p.grad = q.grad = _grads([300], torch.float32, 42)[0]
    opt.step()
    eager.step()
    late = _tensors([70], torch.float32, 43)[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    held = [x.data_ptr() for x in (opt._exp_avg, opt._exp_avg_sq, opt._steps, opt._corr, opt._owner)]
    with pytest.raises(RuntimeError, match="add all groups before"):
        opt.add_param_group({"params": [late]})
    assert held == [x.data_ptr() for x in (opt._exp_avg, opt._exp_avg_sq, opt._steps, opt._corr, opt._owner)] and len(opt.param_groups) == 1
    opt.load_state_dict(opt.state_dict())
    assert held == [x.data_ptr() for x in (opt._exp_avg, opt._exp_avg_sq, opt._steps, opt._corr, opt._owner)]
    for _ in range(3):
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        assert torch.equal(p, q) and all(torch.equal(a, b) for a, b in zip(opt.moments(), eager.moments()))
    wide = []
    for x, o in ((p, opt), (q, eager)):                                                   # the way there is
        wide.append(AdamW([{"params": [x]}, {"params": [late.clone()]}], lr=1e-2, state_bits=bits))
        state = o.state_dict()
        wide[-1].load_state_dict({"state": state["state"], "param_groups": [state["param_groups"][0], {"params": [1]}]})
        wide[-1].param_groups[1]["params"][0].grad = torch.ones_like(late)
        wide[-1].step()
        assert {i: int(e["step"]) for i, e in wide[-1].state_dict()["state"].items()} == {0: 5, 1: 1}
    assert torch.equal(p, q)


def test_the_last_norm_is_the_last_steps_whoever_ran_it():
    p, q = _tensors([5000], torch.float32, 25)[0], _tensors([5000], torch.float32, 25)[0]
    opt, eager = (AdamW([x], lr=torch.full((), 1e-2, device="cuda"), max_grad_norm=1.0) for x in (p, q))
    grads, graphs = [2.0 ** k * x for k, x in enumerate(_grads([5000] * 3, torch.float32, 26))], []
    norms = []
    for g in grads:                                              # norms of eager steps can be collected
        p.grad = q.grad = g
        opt.step()
        eager.step()
        norms.append(opt.last_grad_norm)
    assert len({float(n) for n in norms}) == 3
    for g in grads:
        p.grad = g
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            opt.step()
    for k in (0, 1, 2, 3, 1, 0, 3, 2):
        if k < 3:
            graphs[k].replay()
            q.grad = grads[k]
        else:
            p.grad = q.grad = grads[0] * 0.5
            opt.step()
        eager.step()
        torch.cuda.synchronize()
        assert torch.equal(p, q) and torch.equal(opt.last_grad_norm, eager.last_grad_norm), k
    grads[1][3] = float("nan")                                  # a skipped replay says so
    graphs[0].replay()
    graphs[1].replay()
    assert not float(opt.last_grad_norm) < float("inf")


def test_state_dict_hooks_are_called():
    p = torch.ones(300, device="cuda")
    opt, calls = AdamW([p]), []
    p.grad = torch.ones(300, device="cuda")
    opt.step()
    opt.register_state_dict_pre_hook(lambda o: calls.append("pre"))
    opt.register_state_dict_post_hook(lambda o, sd: calls.append("post"))
    handle = opt.register_state_dict_post_hook(lambda o, sd: {**sd, "epoch": 4})
    sd = opt.state_dict()
    assert calls == ["pre", "post"] and sd["epoch"] == 4 and set(sd["state"]) == {0}
    handle.remove()
    assert "epoch" not in opt.state_dict()

    def twice(o, given):
        calls.append("before loading")
        return {"state": {0: {**given["state"][0], "step": torch.tensor(9.0)}}, "param_groups": given["param_groups"]}
    opt.register_load_state_dict_pre_hook(twice)
    opt.register_load_state_dict_post_hook(lambda o: calls.append("loaded"))
    opt.load_state_dict(sd)
    assert calls[-2:] == ["before loading", "loaded"] and int(sd["state"][0]["step"]) == 1
    assert int(opt.state_dict()["state"][0]["step"]) == 9


@pytest.mark.parametrize("bits", [32, 8])
def test_what_lies_between_loaded_moments_is_left_out(bits):
    sizes = [300, 7, 256]
    params = _tensors(sizes, torch.float32, 38)
    opts = [AdamW(params, state_bits=bits) for _ in range(2)]
    live = torch.zeros(opts[0].blocks * BLOCK, dtype=torch.bool, device="cuda")
    for first, n in zip(opts[0]._first, sizes):
        live[first * BLOCK:first * BLOCK + n] = True
    for fill in (float("nan"), float("inf"), -3.0):
        for opt, between in zip(opts, (0.0, fill)):
            m, v = (torch.full((len(live),), between, device="cuda") for _ in range(2))
            m[live], v[live] = _tensors([563], torch.float32, 39)[0], _tensors([563], torch.float32, 40)[0].abs()
            opt.load_moments(m, v, step=1)
        for a, b in zip(opts[0].moments(), opts[1].moments()):
            assert torch.equal(a, b) and not b[~live].any()


def test_parameters_taken_out_of_the_groups():
    """moments belong to positions: what is left is stepped with its own, or the step is refused"""
    ps = _tensors([300, 300, 300], torch.float32, 44)
    for p, g in zip(ps, _grads([300, 300, 300], torch.float32, 45)):
        p.grad = g
    opt = AdamW([{"params": [p]} for p in ps])
    opt.step()
    kept = [p.clone() for p in ps]
    last = opt.param_groups.pop()
    opt.step()
    assert not torch.equal(ps[0], kept[0]) and torch.equal(ps[2], kept[2]) and [int(e["step"]) for e in opt.state_dict()["state"].values()] == [2, 2]
    kept = [p.clone() for p in ps]
    first = opt.param_groups.pop(0)
    with pytest.raises(RuntimeError, match="parameter list changed"):
        opt.step()
    assert all(torch.equal(p, k) for p, k in zip(ps, kept))
    opt.param_groups[:] = [first] + opt.param_groups + [last]
    opt.step()
    assert [int(e["step"]) for e in opt.state_dict()["state"].values()] == [3, 3, 2]


@pytest.mark.parametrize("bits", [32, 8])
def test_two_groups_are_two_optimizers(bits):
    """no decay on the short tensors: a list of two groups gives the numbers of an optimizer for each"""
    sizes, short = [70000, 256, 30001], [300, 17, 20000]
    ps, qs = ([_tensors(s, torch.float32, 46 + k) for k, s in enumerate((sizes, short))] for _ in range(2))
    opt = AdamW([{"params": ps[0], "weight_decay": 0.1}, {"params": ps[1], "weight_decay": 0.0, "betas": (0.8, 0.95)}], lr=1e-2, state_bits=bits)
    apart = [AdamW(qs[0], lr=1e-2, weight_decay=0.1, state_bits=bits), AdamW(qs[1], lr=1e-2, weight_decay=0.0, betas=(0.8, 0.95), state_bits=bits)]
    for k in range(3):
        for group, twins, s in zip(ps, qs, (sizes, short)):
            for p, q, g in zip(group, twins, _grads(s, torch.float32, 50 + k)):
                p.grad = q.grad = g
        opt.step()
        for o in apart:
            o.step()
        assert all(torch.equal(p, q) for p, q in zip(ps[0] + ps[1], qs[0] + qs[1])), k
    for a, b, c in zip(opt.moments(), *(o.moments() for o in apart)):
        assert torch.equal(a, torch.cat([b, c]))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [None, 0.05, 1e9])
def test_gradients_summed_over_ranks(clip, bits):
    """two ranks' gradients added up and grad_mult = 1/2: the step of their mean, norm and clipping included"""
    sizes = [5000, 33]
    params = _tensors(sizes, torch.float32, 53)
    opt = AdamW(params, lr=2e-3, weight_decay=0.1, state_bits=bits, max_grad_norm=clip, grad_mult=0.5)
    oracles = [O.Tensor(_np(p), bits) for p in params]
    for k in range(3):
        a, b = _grads(sizes, torch.float32, 54 + k), _grads(sizes, torch.float32, 64 + k)
        summed = [x + y for x, y in zip(a, b)]
        norm = 0.5 * float(np.sqrt(sum((_np(g) ** 2).sum() for g in summed)))
        _follow(opt, params, oracles, "fp32", bits, summed, lr=2e-3, wd=0.1, factor=0.5 * (O.clip_factor(norm, clip) if clip else 1.0))
        if clip:
            assert abs(float(opt.last_grad_norm) - norm) <= 2 * U * norm


@pytest.mark.parametrize("sizes", [[700], [70001]])
@pytest.mark.parametrize("bits", [32, 8])
def test_clipping_by_factors_below_the_smallest_normal_float(bits, sizes):
    params = _tensors(sizes, torch.float32, 3)
    opt, oracles = AdamW(params, state_bits=bits, max_grad_norm=1e-9), [O.Tensor(_np(p), bits) for p in params]
    for scale in (1e30, 1e32):
        grads = [scale * g for g in _tensors(sizes, torch.float32, 4)]
        norm = float(np.sqrt(sum((_np(g) ** 2).sum() for g in grads)))
        assert O.clip_factor(norm, 1e-9) < 2.0 ** -130
        _follow(opt, params, oracles, "fp32", bits, grads, lr=1e-3, factor=O.clip_factor(norm, 1e-9))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("clip", [None, 1e9])
def test_more_tensors_than_one_launch_counts(clip, bits):
    """1300 tensors, empty ones among them, against optimizers of a quarter each; then a step of some and a captured one"""
    sizes = [(37 * i) % 300 for i in range(1300)]
    ps, qs = _tensors(sizes, torch.float32, 70), _tensors(sizes, torch.float32, 70)
    kw = dict(weight_decay=0.1, state_bits=bits, max_grad_norm=clip)
    opt = AdamW(ps, lr=torch.full((), 1e-2, device="cuda"), **kw)
    apart = [AdamW(qs[lo:lo + 325], lr=torch.full((), 1e-2, device="cuda"), **kw) for lo in range(0, 1300, 325)]
    graph = torch.cuda.CUDAGraph()
    held = _grads(sizes, torch.float32, 71)
    for k in range(6):
        captured = k >= 4
        for i, (p, q, g) in enumerate(zip(ps, qs, held if captured else _grads(sizes, torch.float32, 72 + k))):
            p.grad = q.grad = None if k == 2 and i % 3 == 0 else g
        if k == 4:
            with torch.cuda.graph(graph):
                opt.step()
        graph.replay() if captured else opt.step()
        for o in apart:
            o.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)), k
    steps = [int(e["step"]) for e in opt.state_dict()["state"].values()]
    assert steps == [int(e["step"]) for o in apart for e in o.state_dict()["state"].values()] and set(steps) == {5, 6}
