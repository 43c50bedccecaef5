"""The optimiser half of a training step on this package's kernels (``hoic_amd/csrc/hoic_mlp.hip``): the norm of a list of gradients,
clipping by it, and AdamW over many tensors with its states in 32 or in 8 bits.

``AdamW`` takes the place of the reference's ``torch.optim.Adam`` (the policy / value optimisers of uhc/agents/agent_handmimic.py)
where a config asks for it: ``policy_optimizer`` / ``value_optimizer`` = "AdamW" or "AdamW8bit" (hoic_amd.agent.PPOLearner).
Everything runs on the current stream of the tensors' device and nothing synchronises; there is no CPU path in here.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import lib

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}         # enum hoic_type
BLOCK = 256                                                             # elements per block of an 8-bit state
_EMPTY_SCALE = 2.0 ** -126                                              # the scale of a block whose values are all zero


def _ptr(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream(dev):
    return C.c_void_p(torch.cuda.current_stream(dev).cuda_stream)


def _strides(t):
    return [st for n, st in zip(t.shape, t.stride()) if n > 1]


def _dense(t):
    """whether the elements fill one stretch of memory, in whatever order of the dimensions"""
    if t.is_contiguous():
        return True
    want = 1
    for st, n in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n > 1):
        if st != want:
            return False
        want *= n
    return True


def _check(t, what):
    if not isinstance(t, torch.Tensor) or t.layout != torch.strided:
        raise ValueError(f"{what}: a dense tensor is needed")
    if not t.is_cuda:
        raise lib.HoicError(f"{what}: the kernels run on the GPU only, this tensor is on {t.device}")
    if t.dtype not in TYPES:
        raise ValueError(f"{what}: float32, float16 or bfloat16, not {t.dtype}")


def _norm(grads, bound):
    """(norm: float32 scalar, float64 [2] = {norm, min(1, bound / (norm + 1e-6))}) of dense CUDA tensors of one device"""
    dev = grads[0].device
    by_type = {}
    for g in grads:
        if g.device != dev:
            raise ValueError(f"one norm over gradients on several devices ({dev}, {g.device})")
        if g.numel():
            by_type.setdefault(g.dtype, []).append(g if _dense(g) else g.contiguous())
    L = lib.load()
    lists, parts = [], 0
    for dt, gs in by_type.items():
        sizes = (C.c_int64 * len(gs))(*[g.numel() for g in gs])
        lists.append((dt, gs, (C.c_void_p * len(gs))(*[g.data_ptr() for g in gs]), sizes, parts))
        parts += L.hoic_grad_norm_parts(sizes, len(gs))
    buf = torch.empty(parts + 2, dtype=torch.float64, device=dev)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    base = buf.data_ptr() + 16
    with torch.cuda.device(dev):
        st = _stream(dev)
        for dt, gs, ptrs, sizes, at in lists:
            lib._chk(L.hoic_grad_norm_partial(ptrs, sizes, len(gs), TYPES[dt], C.c_void_p(base + 8 * at), st), "hoic_grad_norm_partial")
        lib._chk(L.hoic_grad_norm_finish(C.c_void_p(base), parts, float(bound), _ptr(buf), _ptr(norm), st), "hoic_grad_norm_finish")
    return norm, buf, lists


def _bound(max_norm):
    b = float(max_norm)
    if not b >= 0.0:
        raise ValueError(f"max_norm must be >= 0, not {max_norm}")
    return b


def grad_norm(tensors):
    """sqrt(sum of squares) over a list of tensors (float32 / float16 / bfloat16, any mix, one device) as a float32 scalar on the
    device; 64-bit sums in a fixed order: the same bits in every run."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    for t in tensors:
        _check(t, "grad_norm")
    if not tensors:
        return torch.zeros(())
    with torch.no_grad():
        return _norm(tensors, float("inf"))[0]


def clip_grad_norm_(parameters, max_norm):
    """``torch.nn.utils.clip_grad_norm_`` (norm 2) on this package's kernels: the gradients times min(1, max_norm / (norm + 1e-6)) in
    place, the norm before clipping returned as a float32 scalar on the device.  A factor of 1 reads and writes nothing; a norm
    that is not finite gives the factor that the formula gives (0 or NaN)."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    b = _bound(max_norm)
    for g in grads:
        _check(g, "clip_grad_norm_")
        if not _dense(g):
            raise ValueError("clip_grad_norm_: a gradient whose elements do not fill their memory cannot be scaled in place")
    if not grads:
        return torch.zeros(())
    with torch.no_grad():
        norm, clip, lists = _norm(grads, b)
        L, dev = lib.load(), grads[0].device
        with torch.cuda.device(dev):
            for dt, gs, ptrs, sizes, _ in lists:
                lib._chk(L.hoic_scale_list(ptrs, sizes, len(gs), TYPES[dt], _ptr(clip), _stream(dev)), "hoic_scale_list")
        for g in grads:
            torch.autograd.graph.increment_version(g)
    return norm


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over all tensors of a parameter list at once.

    ``state_bits``: 32 = float32 moments; 8 = one byte each, in blocks of 256 elements with a power-of-two scale per block, rounded
    stochastically by a hash of (``seed``, step, tensor, element) -- 2 bytes of state per parameter instead of 8, the same result in
    every run and on every rank.  Parameters: float32, float16 or bfloat16 on the GPU, dense; their new values are rounded to
    nearest (a bfloat16 parameter stays where it is once its step is under 2^-9 of it: keep float32 parameters for small
    learning rates).

    ``step(max_norm=b)`` clips by the norm of all gradients inside the step (the gradients themselves are left alone); the norm is in
    ``self.grad_norm`` afterwards, and a norm that is not finite leaves parameters and moments as they are.

    ``capturable``: the step count lives on the device, so that ``step()`` can be captured into a graph (after one eager step, which
    makes the states) and replayed; ``lr`` may then be a float32 CUDA tensor of one element, read at every replay."""

    grad_norm = None

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, *, state_bits=32, capturable=False, seed=0):
        if isinstance(lr, torch.Tensor):
            if not capturable or not lr.is_cuda or lr.dtype != torch.float32 or lr.numel() != 1:
                raise ValueError("lr: a float, or with capturable=True a float32 CUDA tensor of one element")
        elif not float(lr) >= 0.0:
            raise ValueError(f"lr must be >= 0, not {lr}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"betas must lie in [0, 1), not {betas}")
        if not float(eps) >= 0.0 or not float(weight_decay) >= 0.0:
            raise ValueError(f"eps and weight_decay must be >= 0, not {eps}, {weight_decay}")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, not {state_bits}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=int(state_bits),
                                      capturable=bool(capturable), seed=int(seed) & 0xFFFFFFFF))

    def add_param_group(self, group):
        group = dict(group)
        ps = group["params"]
        group["params"] = ps = [ps] if isinstance(ps, torch.Tensor) else list(ps)
        for key in ("state_bits", "capturable"):
            if group.get(key, self.defaults[key]) != self.defaults[key]:
                raise ValueError(f"{key} is one for all groups")
        for p in ps:
            _check(p, "AdamW")
            if not _dense(p):
                raise ValueError("AdamW: a parameter whose elements do not fill their memory (an expanded or cut view)")
        super().add_param_group(group)

    def _make_state(self, p, step=0):
        bits, s = self.defaults["state_bits"], {}
        s["step"] = torch.full((), step, dtype=torch.int32, device=p.device) if self.defaults["capturable"] else step
        for key in ("exp_avg", "exp_avg_sq"):
            if bits == 32:
                s[key] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
            else:
                s[key] = torch.zeros(p.numel(), dtype=torch.uint8, device=p.device)
                s[key + "_scale"] = torch.full(((p.numel() + BLOCK - 1) // BLOCK,), _EMPTY_SCALE, dtype=torch.float32, device=p.device)
        return s

    def load_state_dict(self, state_dict):
        """Also takes the state of a ``torch.optim.Adam`` / ``AdamW`` over the same parameters (``state_bits=32``).  The moments are
        copied, and keep their own types whatever the parameters' are."""
        old = [p for g in state_dict["param_groups"] for p in g["params"]]
        new = [p for g in self.param_groups for p in g["params"]]
        want = {"exp_avg", "exp_avg_sq"} if self.defaults["state_bits"] == 32 else {"exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale"}
        if len(old) != len(new):
            raise ValueError(f"a state of {len(old)} parameters for {len(new)}")
        states = {}
        for k, p in zip(old, new):
            s = state_dict["state"].get(k)
            if s is None:
                continue
            if set(s) - {"step"} != want:
                raise ValueError(f"a state of {sorted(s)}: this optimiser holds {sorted(want)} (state_bits={self.defaults['state_bits']})")
            mine = self._make_state(p, int(s["step"]))
            for key in want:
                if s[key].numel() != mine[key].numel() or (mine[key].dtype == torch.uint8) != (s[key].dtype == torch.uint8):
                    raise ValueError(f"{key}: {tuple(s[key].shape)} {s[key].dtype} for a parameter of {p.numel()} elements")
                mine[key].copy_(s[key] if s[key].shape == mine[key].shape else s[key].reshape(mine[key].shape))
            states[p] = mine
        fixed = {k: self.defaults[k] for k in ("state_bits", "capturable")}
        super().load_state_dict({**state_dict, "state": {}})
        for g in self.param_groups:
            for key, value in self.defaults.items():
                g.setdefault(key, value)
            g.update(fixed)
        self.state.update(states)

    @torch.no_grad()
    def step(self, closure=None, *, max_norm=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        capturable = self.defaults["capturable"]
        bound = None if max_norm is None else _bound(max_norm)
        ordinal, work, capturing = -1, {}, None
        for gi, group in enumerate(self.param_groups):
            for p in group["params"]:
                ordinal += 1
                g = p.grad
                if g is None:
                    continue
                if g.dtype != p.dtype or g.layout != torch.strided:
                    raise ValueError(f"AdamW: a {g.dtype} gradient (dense ones only) of a {p.dtype} parameter")
                if not ((p.is_contiguous() and g.is_contiguous()) or _strides(g) == _strides(p)):
                    g = torch.empty_like(p).copy_(g)                   # the parameter's order of elements
                work.setdefault((p.device, gi, p.dtype), []).append((ordinal, p, g))
        self.grad_norm = None
        clip = None
        if work:
            for dev in {k[0] for k in work}:
                with torch.cuda.device(dev):
                    capturing = torch.cuda.is_current_stream_capturing()
                if capturing and not capturable:
                    raise lib.HoicError("AdamW: a captured step needs capturable=True (its step count would stand still)")
                if capturing and any(not self.state[p] for k in work if k[0] == dev for _, p, _ in work[k]):
                    raise lib.HoicError("AdamW: take one eager step before a capture (the states would be made anew at every replay)")
        if bound is not None:
            if work:
                self.grad_norm, clip, _ = _norm([g for todo in work.values() for _, _, g in todo], bound)
            else:
                self.grad_norm = torch.zeros(())
        L = lib.load()
        bits = self.defaults["state_bits"]
        for (dev, gi, dtype), todo in work.items():
            group = self.param_groups[gi]
            flat = []
            for o, p, g in todo:
                s = self.state[p]
                if not s:
                    s.update(self._make_state(p))
                if capturable:
                    t, d_step = 0, s["step"].data_ptr()
                else:
                    s["step"] = t = s["step"] + 1
                    d_step = 0
                ms, vs = (s["exp_avg_scale"].data_ptr(), s["exp_avg_sq_scale"].data_ptr()) if bits == 8 else (0, 0)
                flat += (p.data_ptr(), g.data_ptr(), s["exp_avg"].data_ptr(), s["exp_avg_sq"].data_ptr(), ms, vs, p.numel(), t, d_step, o)
            a = lib.AdamWArgs()
            lr = group["lr"]
            a.type, a.state_bits = TYPES[dtype], bits
            if isinstance(lr, torch.Tensor):
                if not capturable or lr.device != dev or lr.dtype != torch.float32:
                    raise ValueError("lr: a float, or with capturable=True a float32 tensor on the parameters' device")
                a.lr, a.d_lr = 0.0, lr.data_ptr()
            else:
                a.lr = float(lr)
            (a.b1, a.b2), a.eps, a.weight_decay, a.seed = group["betas"], group["eps"], group["weight_decay"], group["seed"]
            consts = torch.empty(4 * len(todo), dtype=torch.float32, device=dev) if capturable else None
            a.d_clip = None if clip is None else clip.data_ptr()
            a.d_consts = None if consts is None else consts.data_ptr()
            with torch.cuda.device(dev):
                lib._chk(L.hoic_adamw((C.c_int64 * len(flat))(*flat), len(todo), C.byref(a), _stream(dev)), "hoic_adamw")
            for _, p, _ in todo:
                torch.autograd.graph.increment_version(p)
        return loss

    @torch.no_grad()
    def state_values(self):
        """([m, ...], [v, ...]): both moments of every parameter in float32 (8-bit states: the values that their codes stand for, made
        anew by one launch per 48 tensors; 32-bit ones: the states themselves); zeros where a parameter has no state yet."""
        params = [p for g in self.param_groups for p in g["params"]]
        if self.defaults["state_bits"] == 32:
            get = lambda key: [self.state[p][key] if p in self.state and self.state[p] else torch.zeros_like(p, dtype=torch.float32) for p in params]
            return get("exp_avg"), get("exp_avg_sq")
        L, out, work = lib.load(), ({}, {}), {}
        for p in params:
            work.setdefault(p.device, []).append(p)
        for dev, ps in work.items():
            with torch.cuda.device(dev):
                # one buffer for all values: each tensor's stretch starts at a multiple of 4 elements
                at, ends = [], 0
                for p in ps:
                    at.append(ends)
                    ends += (p.numel() + 3) // 4 * 4
                bufs = (torch.empty(ends, dtype=torch.float32, device=dev), torch.empty(ends, dtype=torch.float32, device=dev))
                flat, n = [], 0
                for p, i in zip(ps, at):
                    for o, b in zip(out, bufs):
                        o[p] = b.as_strided(p.shape, p.stride(), i)
                    s = self.state.get(p)
                    if not s:
                        out[0][p].zero_(), out[1][p].zero_()
                        continue
                    flat += (bufs[0].data_ptr() + 4 * i, bufs[1].data_ptr() + 4 * i, s["exp_avg"].data_ptr(), s["exp_avg_sq"].data_ptr(),
                             s["exp_avg_scale"].data_ptr(), s["exp_avg_sq_scale"].data_ptr(), p.numel(), 1, 0, 0)
                    n += 1
                lib._chk(L.hoic_adamw_values((C.c_int64 * len(flat))(*flat), n, _stream(dev)), "hoic_adamw_values")
        return [out[0][p] for p in params], [out[1][p] for p in params]

