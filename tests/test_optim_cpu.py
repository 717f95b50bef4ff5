"""Refusals of the optimizer step and the gradient norm, and the oracle's 8-bit moments: no GPU needed."""
import ctypes as C

import numpy as np
import pytest
import torch

from tests import optim_oracle as O
from titanet_amd import _lib
from titanet_amd.optim import AdamW, grad_norm


def test_parameters_must_live_on_a_device():
    with pytest.raises(RuntimeError, match="no CPU execution path"):
        AdamW([torch.zeros(4)])
    with pytest.raises(RuntimeError, match="no CPU execution path"):
        grad_norm([torch.zeros(4)])


@pytest.mark.parametrize("kw", [dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(weight_decay=-0.1),
                                dict(state_bits=16), dict(max_grad_norm=0.0), dict(max_grad_norm=float("nan")), dict(lr=torch.zeros(2)),
                                dict(lr=torch.zeros((), dtype=torch.float64))])
def test_hyper_parameters_out_of_range(kw):
    with pytest.raises(ValueError):
        AdamW([torch.zeros(4)], **kw)


@pytest.mark.parametrize("p", [torch.zeros(4, dtype=torch.float64), torch.zeros(4, dtype=torch.int64), torch.zeros(4).to_sparse()])
def test_types_it_does_not_take(p):
    with pytest.raises(TypeError):
        AdamW([p])
    with pytest.raises(TypeError):
        grad_norm([p])
    with pytest.raises(TypeError):
        AdamW([1.0])


def test_grad_norm_of_nothing():
    with pytest.raises(ValueError):
        grad_norm([])


def test_c_entries_refuse_before_they_touch_the_device():
    lib = _lib.load()
    one, none = (C.c_void_p * 1)(4096), C.c_void_p(0)
    n, first, slot = (C.c_int64 * 1)(256), (C.c_int64 * 1)(0), (C.c_int32 * 1)(0)
    at, written = C.c_void_p(4096), C.c_int64()

    def call(entry, count=1, params=one, numel=n, first_block=first, slots=slot, dtype=0, bits=32, m=at, scale=at, blocks=1, b1=0.9, eps=1e-8, lr=1e-3,
             steps=at, corr=at, wd=0.0):
        p = lambda a: C.cast(a, C.c_void_p)  # noqa: E731
        lists = _lib.TnAdamwLists(count, dtype, p(params), p(one), p(numel), p(first_block), p(slots))
        state = _lib.TnAdamwState(bits, blocks, m, m, scale, scale, steps, corr)
        hyper = _lib.TnAdamwHyper(lr, b1, 0.999, eps, wd, none)
        if entry == "apply":
            return lib.tn_adamw_apply(lists, state, hyper, 1.0, none, none)
        if entry == "small":
            return lib.tn_adamw_step_small(lists, state, hyper, 1, p(slots), 1.0, 0.0, none, none)
        return lib.tn_adamw_tick(count, p(slots), state, hyper, none, 0, 1.0, 0.0, none, none, none)

    bad, unsupported = -1, -2
    assert call("apply", count=0) == 0 and call("tick", count=0) == 0
    for entry in ("apply", "small"):
        assert call(entry, count=-1) == bad and call(entry, m=none) == bad and call(entry, corr=none) == bad
        assert call(entry, params=(C.c_void_p * 1)(0)) == bad
        assert call(entry, numel=(C.c_int64 * 1)(-1)) == bad and call(entry, slots=(C.c_int32 * 1)(-1)) == bad
        assert call(entry, numel=(C.c_int64 * 1)(257)) == bad                      # more than the moment buffers hold
        assert call(entry, numel=(C.c_int64 * 1)(2 ** 62)) == bad
        assert call(entry, first_block=(C.c_int64 * 1)(1)) == bad and call(entry, first_block=(C.c_int64 * 1)(-1)) == bad
        assert call(entry, dtype=3) == unsupported and call(entry, bits=16) == unsupported and call(entry, bits=8, scale=none) == bad
        assert call(entry, blocks=1 << 33) == unsupported
    for entry in ("apply", "small", "tick"):
        assert call(entry, b1=1.0) == bad and call(entry, b1=float("nan")) == bad and call(entry, eps=-1.0) == bad and call(entry, lr=-1.0) == bad
        assert call(entry, wd=float("nan")) == bad
    assert call("small", steps=none) == bad and call("small", blocks=100, numel=(C.c_int64 * 1)(65 * 256)) == unsupported
    assert call("tick", steps=none) == bad and call("tick", corr=none) == bad and call("tick", slots=(C.c_int32 * 1)(-1)) == bad
    state, hyper = _lib.TnAdamwState(32, 1, at, at, none, none, at, at), _lib.TnAdamwHyper(1e-3, 0.9, 0.999, 1e-8, 0.0, none)
    assert lib.tn_adamw_tick(1, slot, state, hyper, at, 1, 1.0, 1.0, none, none, none) == bad          # partial sums, nowhere for the factor
    assert lib.tn_adamw_tick(1, slot, state, hyper, at, 1, 1.0, 0.0, none, at, none) == bad
    assert lib.tn_grad_sumsq_partials(-1, none) == bad and lib.tn_grad_sumsq_partials(0, none) == 0
    assert lib.tn_grad_sumsq_partials(1, n) == 1 and lib.tn_grad_sumsq_partials(1, (C.c_int64 * 1)(10 ** 6)) > 1
    assert lib.tn_grad_sumsq(1, one, n, 7, at, C.byref(written), none) == unsupported
    assert lib.tn_grad_sumsq(1, (C.c_void_p * 1)(0), n, 0, at, C.byref(written), none) == bad
    assert lib.tn_grad_norm_finish(at, -1, 1.0, 1.0, at, none, none) == bad and lib.tn_grad_norm_finish(at, 1, 1.0, 0.0, at, at, none) == bad
    assert lib.tn_moments_decode(none, at, at, at, at, at, 1, none) == bad and lib.tn_moments_encode(at, at, at, at, at, none, 1, none) == bad


def test_oracle_codes_are_the_nearest_and_survive_a_round_trip():
    rng = np.random.default_rng(3)
    x = rng.standard_normal(700) * np.exp(rng.standard_normal(700))
    for second in (False, True):
        y = x * x if second else x
        code, top = O.encode(y, second)
        back = O.decode(code, top, second)
        again, top2 = O.encode(back, second)
        assert np.array_equal(code, again) and np.array_equal(top, top2)
        # in the root's domain the codes are even steps: no value is further than half a step away (code 1 takes all below it)
        root = (lambda a: np.abs(a) ** 0.25) if second else (lambda a: np.abs(a) ** 0.5)
        scale = np.repeat(root(top.astype(np.float64)), O.BLOCK)[:700]
        off = np.abs(root(y) - root(back)) / scale
        step = 1 / 255 if second else 1 / 127
        assert off[code != 1].max() <= step / 2 * (1 + 1e-6) and off.max() <= step
        assert not second or (code[y > 0] >= 1).all()


def test_hooks_of_a_state_dict_run_in_torchs_order():
    """the same calls on torch's own optimizer and on this one, where there is no parameter that would need a device"""
    seen = []
    for opt in (torch.optim.AdamW([{"params": []}]), AdamW([{"params": []}])):
        calls = []
        seen.append(calls)
        opt.register_state_dict_pre_hook(lambda o: calls.append("pre"))
        opt.register_state_dict_post_hook(lambda o, sd: calls.append(("post", sorted(sd))))
        opt.register_state_dict_post_hook(lambda o, sd: {**sd, "epoch": 4}, prepend=True)
        opt.register_load_state_dict_pre_hook(lambda o, sd: calls.append(("before", sorted(sd))))
        opt.register_load_state_dict_pre_hook(lambda o, sd: {k: v for k, v in sd.items() if k != "epoch"}, prepend=True)
        opt.register_load_state_dict_post_hook(lambda o: calls.append("loaded"))
        sd = opt.state_dict()
        opt.load_state_dict(sd)
        assert sd["epoch"] == 4
    assert seen[0] == seen[1] and len(seen[0]) == 4


@pytest.mark.parametrize("bad", [dict(amsgrad=True), dict(maximize=True), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0)])
def test_a_refused_state_changes_nothing(bad):
    opt = AdamW([{"params": [], "lr": 0.5}, {"params": []}])
    state = opt.state_dict()
    state["param_groups"][0]["lr"] = 0.25
    state["param_groups"][1].update(bad)
    with pytest.raises(ValueError):
        opt.load_state_dict(state)
    assert [g["lr"] for g in opt.param_groups] == [0.5, 1e-3]


@pytest.mark.parametrize("bad", [0.0, -1.0, float("nan")])
def test_a_norm_assigned_later_is_checked(bad):
    opt = AdamW([{"params": []}], max_grad_norm=1.0)
    opt.step()
    opt.max_grad_norm = bad
    with pytest.raises(ValueError, match="max_grad_norm"):
        opt.step()
    opt.max_grad_norm = None
    opt.step()
    for mult in (float("nan"), float("inf")):
        with pytest.raises(ValueError, match="grad_mult"):
            AdamW([{"params": []}], grad_mult=mult)
