"""AdamW over many tensors at once, with moments in 32 or in 8 bits, and the global gradient norm.

    opt = AdamW(model.parameters(), lr=1e-3, weight_decay=0.01, state_bits=8, max_grad_norm=1.0)
    loss.backward()
    opt.step()

The reference steps one ``torch.optim.Adam`` (reference src/train.py:130-135, src/learn.py:116-118); :class:`AdamW` is its
decoupled-decay sibling for a whole list of tensors in a few launches (``tn_adamw_apply``, include/titanet_amd.h).  Step counts,
the clipping factor and a learning rate given as a device tensor are read on the device: a step can be captured into a graph and
replayed, and a step whose gradient norm is not finite leaves everything as it was.  There is no CPU fallback.
"""
import ctypes as C
import math

import numpy as np
import torch

from . import _lib
from ._lib import check

BLOCK = 256          # TN_OPT_BLOCK: elements that share a scale of the 8-bit moments
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _dev(tensor):
    return C.c_void_p(tensor.data_ptr() if tensor is not None else 0)


def grad_norm(tensors):
    """The 2-norm of all elements of ``tensors`` together, as a 0-dim float32 tensor on their device.  Summed in 64 bits in an
    order that goes by the tensors and by which of them lie next to each other in memory: two calls on the same tensors give the same
    number.  float32, bfloat16 and float16 may be mixed.  The number is for reading: it takes no part in autograd."""
    return _lib.load_host().grad_norm([tensors] if isinstance(tensors, torch.Tensor) else list(tensors))


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay; the update of ``torch.optim.AdamW``) over lists of dense float32, bfloat16 or float16
    tensors of one device.

    ``state_bits=32`` keeps both moments in float32, ``state_bits=8`` one byte per element and moment and a float32 scale per
    block of 256 elements of a tensor: 2.05 bytes of state per element instead of 8.  The step itself is computed from the
    moments before they are rounded; what is rounded is what the next step starts from (forms: include/titanet_amd.h).
    Parameters of 16 bits are rounded to the nearest value after every step: updates below half a step of their type are lost.

    ``max_grad_norm``: the gradients of all groups together are scaled to at most this 2-norm, as
    ``torch.nn.utils.clip_grad_norm_`` does (the ``.grad`` tensors themselves keep their values); ``last_grad_norm`` is the norm
    before that, on the device (once a step has been captured: one tensor that every step and replay writes).  A norm that is not finite skips the step — parameters, moments and step counts stay as they
    are; without ``max_grad_norm`` a gradient that is NaN or infinite reaches its element (8 bits: its block of 256).
    ``float("inf")`` measures the norm and skips, without scaling.

    ``grad_mult`` multiplies the gradients before everything else (1 / world size behind a summing all-reduce).

    ``lr`` may be a 0-dim float32 tensor on the device; a step can be captured into a graph only then (a number would be frozen
    into the graph, as the other hyper-parameters are).  The graph then reads and writes the optimizer's buffers: keep the optimizer as
    long as the graph.  No parameter group can be added any more; loading a state and eager steps of all or some parameters go on.

    Parameters whose ``.grad`` is None are left alone and keep a step count of their own."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, max_grad_norm=None, grad_mult=1.0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits!r}")
        self._check_norm(max_grad_norm)
        if not math.isfinite(grad_mult):
            raise ValueError(f"grad_mult must be a finite number, got {grad_mult!r}")
        self.state_bits, self.max_grad_norm, self.grad_mult = state_bits, max_grad_norm, float(grad_mult)
        self.last_grad_norm = None
        self._native = _lib.load()
        self._stepper = _lib.load_host().Stepper(state_bits)      # checks, collects and launches a step
        self._list, self._device = [], None          # all parameters, group after group
        self._exp_avg = self._exp_avg_sq = self._scale1 = self._scale2 = self._steps = self._corr = self._owner = None
        self._numel = self._first = np.zeros(0, dtype=np.int64)
        self.blocks = 0
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def __getstate__(self):
        raise TypeError("AdamW holds device buffers laid out for its parameters: save state_dict() instead of pickling or copying it")

    # ------------------------------------------------------------------ layout
    def add_param_group(self, param_group):
        if self._stepper.captured:
            raise RuntimeError("AdamW: a captured step holds this optimizer's moments, which a new group would move: add all groups before "
                               "capturing a step, or load state_dict() into a new optimizer")
        params = param_group["params"]
        params = [params] if isinstance(params, torch.Tensor) else list(params)
        new = [p[1] if isinstance(p, tuple) else p for p in params]
        hyper = {**self.defaults, **{k: v for k, v in param_group.items() if k != "params"}}
        self._check_hyper(hyper)
        seen = {id(p) for p in self._list}
        device = self._device
        for p in new:
            if not isinstance(p, torch.Tensor):
                raise TypeError(f"AdamW optimizes tensors, got {type(p).__name__}")
            if p.dtype not in _TYPES or p.layout != torch.strided:
                raise TypeError(f"AdamW takes dense float32, bfloat16 or float16 parameters, got {p.dtype} ({p.layout})")
            if not p.is_cuda:
                raise RuntimeError("titanet_amd.optim needs parameters on a ROCm device; there is no CPU execution path")
            if device is not None and p.device != device:
                raise ValueError(f"AdamW takes parameters of one device, got {device} and {p.device}")
            device = p.device
            if not p.is_contiguous():
                raise ValueError("AdamW takes contiguous parameters")
            if id(p) in seen:
                raise ValueError("a parameter appears more than once")
            seen.add(id(p))
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in self._list + new if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("two parameters share memory")
        lr = hyper["lr"]
        if isinstance(lr, torch.Tensor) and new and lr.device != device:
            raise ValueError(f"a tensor lr must be on the parameters' device {device}, got {lr.device}")
        param_group["params"] = params
        super().add_param_group(param_group)
        self._device = device
        self._extend(new)

    @staticmethod
    def _check_norm(max_grad_norm):
        if max_grad_norm is not None and not float(max_grad_norm) > 0.0:
            raise ValueError(f"max_grad_norm must be above 0 or None, got {max_grad_norm!r}")

    @staticmethod
    def _check_hyper(g):
        lr = g["lr"]
        if isinstance(lr, torch.Tensor):
            if lr.dtype != torch.float32 or lr.dim() != 0:
                raise ValueError("a tensor lr must be a 0-dim float32 tensor")
        elif not float(lr) >= 0.0:
            raise ValueError(f"Invalid learning rate: {lr}")
        if len(g["betas"]) != 2 or not all(0.0 <= float(b) < 1.0 for b in g["betas"]):
            raise ValueError(f"betas must be two numbers in [0, 1), got {g['betas']}")
        if not float(g["eps"]) >= 0.0:
            raise ValueError(f"Invalid epsilon value: {g['eps']}")
        if not float(g["weight_decay"]) >= 0.0:
            raise ValueError(f"Invalid weight_decay value: {g['weight_decay']}")

    def _extend(self, new):
        """moments and counts of the parameters of a new group, behind those there are"""
        if not new:
            return
        n0, b0 = len(self._list), self.blocks
        numel = np.array([p.numel() for p in new], dtype=np.int64)
        blocks = (numel + BLOCK - 1) // BLOCK
        first = b0 + np.concatenate([[0], np.cumsum(blocks)[:-1]]).astype(np.int64)
        self._list += new
        self._numel, self._first = np.concatenate([self._numel, numel]), np.concatenate([self._first, first])
        # the whole group is at one step count until some of its tensors go without a gradient
        sets = self._stepper.sets + [n0] * len(new)
        self.blocks = b0 + int(blocks.sum())

        def grown(old, size, dtype):
            t = torch.zeros(size, dtype=dtype, device=self._device)
            if old is not None:
                t[:old.shape[0]] = old
            return t
        eight = self.state_bits == 8
        self._exp_avg = grown(self._exp_avg, self.blocks * BLOCK, torch.int8 if eight else torch.float32)
        self._exp_avg_sq = grown(self._exp_avg_sq, self.blocks * BLOCK, torch.uint8 if eight else torch.float32)
        if eight:
            self._scale1, self._scale2 = grown(self._scale1, self.blocks, torch.float32), grown(self._scale2, self.blocks, torch.float32)
        self._steps = grown(self._steps, len(self._list), torch.int32)
        self._corr = torch.zeros(len(self._list), 4, dtype=torch.float32, device=self._device)
        every = (self._numel + BLOCK - 1) // BLOCK
        self._owner = torch.from_numpy(np.repeat(np.arange(len(every), dtype=np.int32), every)).to(self._device)      # each block's parameter
        self._stepper.layout(self._numel.tolist(), self._first.tolist(), sets, self.blocks, self._exp_avg, self._exp_avg_sq, self._scale1,
                             self._scale2, self._steps, self._corr, self._owner, self._list)

    def _groups(self):
        """(group, index of its first parameter) in order"""
        at = 0
        for group in self.param_groups:
            yield group, at
            at += len(group["params"])

    # ------------------------------------------------------------------ the step
    def step(self, closure=None):
        loss = None
        self._check_norm(self.max_grad_norm)          # (it may have been assigned)
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self._device is not None:
            norm = self._stepper.step(self.param_groups, 0.0 if self.max_grad_norm is None else float(self.max_grad_norm), self.grad_mult)
            self.last_grad_norm = self.last_grad_norm if norm is None else norm
        return loss

    # ------------------------------------------------------------------ moments as values
    def moments(self):
        """(exp_avg, exp_avg_sq) of all parameters as flat float32 tensors: parameter i's from ``BLOCK * first`` on, every
        parameter at a multiple of 256, zeros between them (8 bits: NaN in the rest of a block that is NaN).  32 bits: the buffers
        themselves; 8 bits: the values of the codes."""
        return self._stepper.moments() if self._device is not None else (self._exp_avg, self._exp_avg_sq)

    @torch.no_grad()
    def load_moments(self, exp_avg, exp_avg_sq, step):
        """Sets the moments from two flat tensors laid out as :meth:`moments` gives them, and every step count to ``step``.  What lies
        between the parameters is not read."""
        size = self.blocks * BLOCK
        if tuple(exp_avg.shape) != (size,) or tuple(exp_avg_sq.shape) != (size,):
            raise ValueError(f"moments of this optimizer are two tensors of {size} values, got {tuple(exp_avg.shape)} and {tuple(exp_avg_sq.shape)}")
        if not 0 <= int(step) < 2 ** 31:
            raise ValueError(f"step must be a count, got {step}")
        m, v = (t.detach().to(device=self._device, dtype=torch.float32, copy=True) for t in (exp_avg, exp_avg_sq))
        between = torch.ones(size, dtype=torch.bool, device=self._device)
        for first, n in zip(self._first, self._numel):
            between[first * BLOCK:first * BLOCK + n] = False
        for t in (m, v):
            t.masked_fill_(between, 0.0)          # (whatever lies between the parameters: NaN would not become 0 by a product)
        self._put_values(m, v)
        self._put_steps([int(step)] * len(self._list))

    def _put_values(self, m, v):
        if self.state_bits == 32:
            self._exp_avg.copy_(m)
            self._exp_avg_sq.copy_(v)
            return
        with torch.cuda.device(self._device):
            check(self._native.tn_moments_encode(_dev(m), _dev(v), _dev(self._exp_avg), _dev(self._exp_avg_sq), _dev(self._scale1),
                                                 _dev(self._scale2), self.blocks, C.c_void_p(torch.cuda.current_stream(self._device).cuda_stream)),
                  "tn_moments_encode")

    def _put_steps(self, steps):
        """Sets every parameter's count.  Those of a group that are at one count are stepped together; once a step has been captured, only
        those that were so before: replays advance what they hold, and only these are known to stay at one count."""
        old, first, sets = self._stepper.sets, {}, list(range(len(self._list)))
        for k, (group, at) in enumerate(self._groups()):
            for i in range(at, at + len(group["params"])):
                sets[i] = first.setdefault((k, steps[i], old[i] if self._stepper.captured else None), i)
        self._stepper.sets = sets
        counts = torch.zeros(len(self._list), dtype=torch.int32)
        counts[:len(steps)] = torch.tensor(steps, dtype=torch.int32)
        self._steps.copy_(counts)

    # ------------------------------------------------------------------ checkpoints
    def _views(self, i):
        """parameter i's part of the moment buffers (8 bits: codes and scales)"""
        lo, n, shape = int(self._first[i]) * BLOCK, int(self._numel[i]), self._list[i].shape
        out = {"exp_avg": self._exp_avg[lo:lo + n].view(shape), "exp_avg_sq": self._exp_avg_sq[lo:lo + n].view(shape)}
        if self.state_bits == 8:
            b, k = int(self._first[i]), (n + BLOCK - 1) // BLOCK
            out.update(exp_avg_scale=self._scale1[b:b + k], exp_avg_sq_scale=self._scale2[b:b + k])
        return out

    def state_dict(self):
        """``torch.optim.AdamW``'s layout, the moments as they are held: float32, or int8 / uint8 codes with ``exp_avg_scale`` /
        ``exp_avg_sq_scale`` per block of 256 elements.  Parameters that were never stepped have no entry.  (``self.state`` stays empty:
        the moments of all parameters lie in buffers of the whole list.)  Hooks registered on the optimizer are called as torch does."""
        for hook in self._optimizer_state_dict_pre_hooks.values():
            hook(self)
        state, groups = {}, []
        counts = self._steps.cpu().tolist() if self._device is not None else []
        for group, at in self._groups():
            index = list(range(at, at + len(group["params"])))
            groups.append({**{k: v for k, v in group.items() if k != "params"}, "params": index})
            for i in index:
                t = counts[i]
                if t:
                    state[i] = {"step": torch.tensor(float(t)), **self._views(i)}
        state_dict = {"state": state, "param_groups": groups}
        for hook in self._optimizer_state_dict_post_hooks.values():
            given = hook(self, state_dict)
            state_dict = state_dict if given is None else given
        return state_dict

    def load_state_dict(self, state_dict):
        """Takes the dict of :meth:`state_dict` of either width, or of ``torch.optim.AdamW`` / ``torch.optim.Adam``: moments held in
        another width are converted.  Hooks registered on the optimizer are called as torch does."""
        state_dict = dict(state_dict)
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            given = hook(self, state_dict)
            state_dict = state_dict if given is None else given
        self._load_state_dict(state_dict)
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    @torch.no_grad()
    def _load_state_dict(self, state_dict):
        groups, state = state_dict["param_groups"], state_dict["state"]
        if len(groups) != len(self.param_groups) or any(len(g["params"]) != len(o["params"]) for g, o in zip(groups, self.param_groups)):
            raise ValueError("loaded state dict has other parameter groups than this optimizer")
        order = [i for g in groups for i in g["params"]]
        entries = [state.get(i) for i in order]
        coded = {not e["exp_avg"].is_floating_point() for e in entries if e}
        if len(coded) > 1:
            raise ValueError("loaded state dict holds moments of both widths")
        coded = coded == {True}
        for e, n in zip(entries, self._numel):
            if e and (e["exp_avg"].numel() != n or e["exp_avg_sq"].numel() != n or (coded and (
                    e["exp_avg_scale"].numel() != (n + BLOCK - 1) // BLOCK or e["exp_avg_sq_scale"].numel() != (n + BLOCK - 1) // BLOCK))):
                raise ValueError("loaded state dict has moments of another size")
        hypers = []
        for g, o in zip(groups, self.param_groups):         # (everything is looked at before anything changes)
            if g.get("amsgrad") or g.get("maximize"):
                raise ValueError("loaded state dict is of a variant (amsgrad, maximize) that AdamW does not have")
            hypers.append({k: v for k, v in g.items() if k in ("lr", "betas", "eps", "weight_decay")})
            self._check_hyper({**o, **hypers[-1]})
        steps = [int(float(e["step"])) if e else 0 for e in entries]
        for g, o, hyper in zip(groups, self.param_groups, hypers):
            if "lr" in hyper and isinstance(o["lr"], torch.Tensor):
                o["lr"].fill_(hyper.pop("lr"))               # (a captured step reads this tensor)
            elif isinstance(hyper.get("lr"), torch.Tensor):
                hyper["lr"] = hyper["lr"].to(self._device or hyper["lr"].device).clone()
            o.update({**{k: v for k, v in g.items() if k not in ("params", "lr", "betas", "eps", "weight_decay")}, **hyper})
        if self._device is None:
            return
        size, dev = self.blocks * BLOCK, self._device
        m = torch.zeros(size, dtype=torch.int8 if coded else torch.float32, device=dev)
        v = torch.zeros(size, dtype=torch.uint8 if coded else torch.float32, device=dev)
        s1, s2 = torch.zeros(self.blocks, dtype=torch.float32, device=dev), torch.zeros(self.blocks, dtype=torch.float32, device=dev)
        for e, first, n in zip(entries, self._first, self._numel):
            if not e:
                continue
            lo, k = int(first) * BLOCK, int((n + BLOCK - 1) // BLOCK)
            m[lo:lo + int(n)] = e["exp_avg"].reshape(-1).to(dev)
            v[lo:lo + int(n)] = e["exp_avg_sq"].reshape(-1).to(dev)
            if coded:
                s1[int(first):int(first) + k] = e["exp_avg_scale"].to(dev)
                s2[int(first):int(first) + k] = e["exp_avg_sq_scale"].to(dev)
        if coded and self.state_bits == 8:
            for new, old in ((m, self._exp_avg), (v, self._exp_avg_sq), (s1, self._scale1), (s2, self._scale2)):
                old.copy_(new)
        elif coded:
            with torch.cuda.device(dev):
                check(self._native.tn_moments_decode(_dev(m), _dev(v), _dev(s1), _dev(s2), _dev(self._exp_avg), _dev(self._exp_avg_sq), self.blocks,
                                                     C.c_void_p(torch.cuda.current_stream(dev).cuda_stream)), "tn_moments_decode")
        else:
            self._put_values(m, v)
        self._put_steps(steps)
