"""The optimiser half of a training step on this package's kernels (``hoic_amd/csrc/hoic_mlp.hip``): the norm of a list of gradients,
clipping by it, and AdamW over many tensors with its states in 32 or in 8 bits.

``AdamW`` takes the place of the reference's ``torch.optim.Adam`` (the policy / value optimisers of uhc/agents/agent_handmimic.py)
where a config asks for it: ``policy_optimizer`` / ``value_optimizer`` = "AdamW" or "AdamW8bit" (hoic_amd.agent.PPOLearner).
Everything runs on the current stream of the tensors' device and nothing synchronises; there is no CPU path in here.
"""
from __future__ import annotations

import struct

import torch
import torch.optim.optimizer as _opt

from . import lib

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}         # enum hoic_type
BLOCK = 256                                                             # elements per block of an 8-bit state
_EMPTY_SCALE = 2.0 ** -126                                              # the scale of a block whose values are all zero


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
    if not isinstance(t, torch.Tensor) or t.layout is not torch.strided:
        raise ValueError(f"{what}: a dense tensor is needed")
    if not t.is_cuda:
        raise lib.HoicError(f"{what}: the kernels run on the GPU only, this tensor is on {t.device}")
    if t.dtype not in TYPES:
        raise ValueError(f"{what}: float32, float16 or bfloat16, not {t.dtype}")


def _pack(x):
    """64-bit integers as a host array (a third of the time of a ctypes array)"""
    return struct.pack(f"{len(x)}q", *x)


def _list_args(ptrs, sizes, types):
    """(pointers, sizes, types, count) of the hoic_grad_norm family, and the number of partial sums"""
    n = len(ptrs)
    sizes = _pack(sizes)
    return (_pack(ptrs), sizes, bytes(types), n), lib.load().hoic_grad_norm_parts(sizes, n)


def _tensor_list(tensors, what):
    """_list_args of dense CUDA tensors of one device"""
    ptrs, sizes, types, at = [], [], [], None
    for t in tensors:
        if not (isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in TYPES and t.layout is torch.strided):
            _check(t, what)
        if t.get_device() != at:
            if at is not None:
                raise ValueError(f"{what}: one norm over tensors on several devices (cuda:{at}, {t.device})")
            at = t.get_device()
        if not t.is_contiguous() and not _dense(t):
            raise ValueError(f"{what}: a tensor whose elements do not fill their memory (an expanded or cut view)")
        ptrs.append(t.data_ptr())
        sizes.append(t.numel())
        types.append(TYPES[t.dtype])
    return _list_args(ptrs, sizes, types)


def _bound(max_norm):
    b = float(max_norm)
    if not b >= 0.0:
        raise ValueError(f"max_norm must be >= 0, not {max_norm}")
    return b


def _check_options(group):
    """options of torch.optim.Adam's / AdamW's groups that the step does not have"""
    for key in ("maximize", "amsgrad"):
        if group.get(key):
            raise ValueError(f"AdamW: {key}=True is not supported")
    if group.get("weight_decay") and group.get("decoupled_weight_decay") is False:
        raise ValueError("AdamW: its weight decay is decoupled, these options ask for a coupled one (torch.optim.Adam with weight_decay)")


def grad_norm(tensors):
    """sqrt(sum of squares) over a list of tensors (float32 / float16 / bfloat16, any mix, one device) as a float32 scalar on the
    device; 64-bit sums in a fixed order: the same bits in every run."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        return torch.zeros(())
    for i, t in enumerate(tensors):
        _check(t, "grad_norm")
        if not _dense(t):
            tensors[i] = t.detach().contiguous()
    args, parts = _tensor_list(tensors, "grad_norm")
    dev = tensors[0].device
    norm = torch.empty((), dtype=torch.float32, device=dev)
    if parts == 0:
        return norm.zero_()
    buf = torch.empty(parts + 2, dtype=torch.float64, device=dev)
    with lib.Launch(dev) as st:
        lib._chk(lib.load().hoic_grad_norm(*args, buf.data_ptr(), norm.data_ptr(), st), "hoic_grad_norm")
    return norm


def clip_grad_norm_(parameters, max_norm):
    """``torch.nn.utils.clip_grad_norm_`` (norm 2) on this package's kernels: the gradients times min(1, max_norm / (norm + 1e-6)) in
    place, the norm before clipping returned as a float32 scalar on the device.  A factor of 1 reads and writes nothing; a norm
    that is not finite in float32 gives the factor that the formula gives (0 or NaN)."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [g for g in [p.grad for p in parameters] if g is not None]
    bound = _bound(max_norm)
    if not grads:
        return torch.zeros(())
    args, parts = _tensor_list(grads, "clip_grad_norm_")
    dev = grads[0].device
    norm = torch.empty((), dtype=torch.float32, device=dev)
    if parts == 0:
        return norm.zero_()
    buf = torch.empty(parts + 2, dtype=torch.float64, device=dev)
    with lib.Launch(dev) as st:
        rc = lib.load().hoic_clip_grads(*args, bound, buf.data_ptr(), norm.data_ptr(), st)
    if rc != 0:
        error = lib.load().hoic_last_error().decode()
        raise (ValueError if "same memory" in error else lib.HoicError)(f"clip_grad_norm_: {error}")
    torch.autograd.graph.increment_version(grads)
    return norm


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over all tensors of a parameter list at once.

    ``state_bits``: 32 = float32 moments; 8 = one byte each, in blocks of 256 elements with a power-of-two scale per block, rounded
    stochastically by a hash of (``seed``, step, tensor, element) -- 2 bytes of state per parameter instead of 8, the same result in
    every run and on every rank.  Parameters: float32, float16 or bfloat16 on the GPU, dense; their new values are rounded to
    nearest (a bfloat16 parameter stays where it is once its step is under 2^-9 of it: keep float32 parameters for small
    learning rates).

    ``step(max_norm=b)`` clips by the norm of all gradients inside the step (the gradients themselves are left alone); the norm is in
    ``self.grad_norm`` afterwards, and a norm that is not finite leaves parameters and moments as they are (the step counts all the same:
    the host does not wait for the norm).

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
        _check_options({**self.defaults, **group})
        for p in ps:
            _check(p, "AdamW")
            if not _dense(p):
                raise ValueError("AdamW: a parameter whose elements do not fill their memory (an expanded or cut view)")
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in [p for g in self.param_groups for p in g["params"]] + ps if p.numel())
        if any(b[0] < a[1] for a, b in zip(spans, spans[1:])):
            raise ValueError("AdamW: two parameters in the same memory")
        super().add_param_group(group)

    def _make_state(self, p, step=0, filled=True):
        bits, s = self.defaults["state_bits"], {}
        s["step"] = torch.full((), step, dtype=torch.int32, device=p.device) if self.defaults["capturable"] else step
        if not p.is_contiguous():
            s["order"] = _strides(p)
        for key in ("exp_avg", "exp_avg_sq"):
            if bits == 32:
                s[key] = torch.empty_like(p, dtype=torch.float32, memory_format=torch.preserve_format, requires_grad=False)
            else:
                s[key] = torch.empty(p.numel(), dtype=torch.uint8, device=p.device)
                s[key + "_scale"] = torch.empty((p.numel() + BLOCK - 1) // BLOCK, dtype=torch.float32, device=p.device)
            if filled:
                s[key].zero_()
                if bits == 8:
                    s[key + "_scale"].fill_(_EMPTY_SCALE)
        return s

    def _new_order(self, p, s, capturing):
        """moments of a parameter that lies in another order in memory than when they were made"""
        if self.defaults["state_bits"] == 8:
            raise ValueError("AdamW: 8-bit moments lie in blocks in the parameter's order in memory, which has changed since they were made")
        if capturing:
            raise lib.HoicError("AdamW: a parameter's order in memory has changed: take one eager step before a capture")
        for key in ("exp_avg", "exp_avg_sq"):
            s[key] = torch.empty_like(p, dtype=torch.float32, requires_grad=False).copy_(s[key].reshape(p.shape))
        s.pop("order", None)
        if not p.is_contiguous():
            s["order"] = _strides(p)

    def load_state_dict(self, state_dict):
        """Also takes the state of a ``torch.optim.Adam`` / ``AdamW`` over the same parameters (``state_bits=32``; refused with options that
        this step does not have: ``maximize``, ``amsgrad``, ``Adam``'s coupled weight decay).  The moments are copied, and keep their own
        types whatever the parameters' are.  (8-bit ones need parameters in the order in memory that they were made for.)"""
        state_dict = dict(state_dict)
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        for g in state_dict["param_groups"]:
            _check_options(g)
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
            if set(s) - {"step", "order"} != want:
                raise ValueError(f"a state of {sorted(s)}: this optimiser holds {sorted(want)} (state_bits={self.defaults['state_bits']})")
            mine = self._make_state(p, int(s["step"]), filled=False)
            if self.defaults["state_bits"] == 8 and list(s.get("order", ())) != list(mine.get("order", ())):
                raise ValueError("8-bit moments of a parameter that lay in another order in memory")
            for key in want:
                if s[key].numel() != mine[key].numel() or (mine[key].dtype == torch.uint8) != (s[key].dtype == torch.uint8):
                    raise ValueError(f"{key}: {tuple(s[key].shape)} {s[key].dtype} for a parameter of {p.numel()} elements")
                mine[key].copy_(s[key] if s[key].shape == mine[key].shape else s[key].reshape(mine[key].shape))
            states[p] = mine
        fixed = {k: self.defaults[k] for k in ("state_bits", "capturable")}
        hooks = self._optimizer_load_state_dict_pre_hooks, self._optimizer_load_state_dict_post_hooks
        self._optimizer_load_state_dict_pre_hooks, self._optimizer_load_state_dict_post_hooks = {}, {}
        try:                        # (the base class would bring the moments to the parameters' types; its hooks run here, around the whole call)
            super().load_state_dict({**state_dict, "state": {}})
        finally:
            self._optimizer_load_state_dict_pre_hooks, self._optimizer_load_state_dict_post_hooks = hooks
        for g in self.param_groups:
            for key, value in self.defaults.items():
                g.setdefault(key, value)
            g.update(fixed)
        self.state.update(states)
        for hook in hooks[1].values():
            hook(self)

    def step(self, closure=None, *, max_norm=None):
        if (self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _opt._global_optimizer_pre_hooks
                or _opt._global_optimizer_post_hooks or torch.autograd.profiler._is_profiler_enabled):
            return self._step_hooked(closure, max_norm=max_norm)
        return self._step(closure, max_norm=max_norm)

    step.hooked = True          # (hooks and profiler ranges are taken care of above; the base class would add 6 us to every step)

    def _step(self, closure=None, *, max_norm=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        bound = None if max_norm is None else _bound(max_norm)
        bits, capturable = self.defaults["state_bits"], self.defaults["capturable"]
        capturing, state = torch.cuda.is_current_stream_capturing(), self.state
        # rows of the list (hoic_adamw_tensor) per device, group and type
        ordinal, work, rows, params, held, touched = -1, {}, None, [], [], []
        t = d_step = m_scale = v_scale = 0
        for gi, group in enumerate(self.param_groups):
            rows_at = rows_dtype = None
            for p in group["params"]:
                ordinal += 1
                g = p.grad
                if g is None:
                    continue
                dtype, at, n, contiguous = p.dtype, p.get_device(), p.numel(), p.is_contiguous()
                if g.dtype is not dtype or g.layout is not torch.strided or g.numel() != n or g.get_device() != at:
                    raise ValueError(f"AdamW: a gradient {tuple(g.shape)} {g.dtype} on {g.device} (dense ones only) of a parameter {tuple(p.shape)} {dtype} on {p.device}")
                if not (contiguous and g.is_contiguous()):
                    if not _dense(p) or g.shape != p.shape:          # (dense when it was added, but ``p.data`` may have been replaced since)
                        raise ValueError(f"AdamW: a parameter {tuple(p.shape)} whose elements do not fill their memory, or a gradient of another shape, {tuple(g.shape)}")
                    if _strides(g) != _strides(p):
                        g = torch.empty_like(p, requires_grad=False).copy_(g.detach())      # the parameter's order of elements
                        held.append(g)
                s = state[p]
                if not s or capturing:
                    if capturing and not capturable:
                        raise lib.HoicError("AdamW: a captured step needs capturable=True (its step count would stand still)")
                    if capturing and not s:
                        raise lib.HoicError("AdamW: take one eager step before a capture (the states would be made anew at every replay)")
                    if not s:
                        s.update(self._make_state(p))
                m = s["exp_avg"]
                if m.numel() != n or m.get_device() != at:
                    raise ValueError(f"AdamW: moments of {m.numel()} elements on {m.device} for a parameter of {n} on {p.device}")
                if not contiguous or "order" in s:
                    if s.get("order") != (None if contiguous else _strides(p)):
                        self._new_order(p, s, capturing)
                        m = s["exp_avg"]
                if at != rows_at or dtype is not rows_dtype:
                    _check(p, "AdamW")
                    rows_at, rows_dtype = at, dtype
                    rows = work.setdefault((at, gi, dtype), [])
                if capturable:
                    d_step = s["step"].data_ptr()
                else:
                    t = s["step"] + 1
                if bits == 8:
                    m_scale, v_scale = s["exp_avg_scale"].data_ptr(), s["exp_avg_sq_scale"].data_ptr()
                rows += (p.data_ptr(), g.data_ptr(), m.data_ptr(), s["exp_avg_sq"].data_ptr(), m_scale, v_scale, n, t, d_step, ordinal)
                params.append(p)
                touched.append(s)
        self.grad_norm = None
        if not work:
            if bound is not None:
                self.grad_norm = torch.zeros(())
            return loss
        for at, gi, _ in work:               # before any launch: a step is taken by all groups or by none
            lr = self.param_groups[gi]["lr"]
            if isinstance(lr, torch.Tensor) and (not capturable or lr.get_device() != at or lr.dtype != torch.float32 or lr.numel() != 1):
                raise ValueError("lr: a float, or with capturable=True a float32 tensor of one element on the parameters' device")
        L = lib.load()
        buf_ptr = norm_ptr = parts = 0
        if bound is not None:
            if len({k[0] for k in work}) > 1:
                raise ValueError("AdamW: one norm over gradients on several devices")
            dev = params[0].device
            self.grad_norm = norm = torch.empty((), dtype=torch.float32, device=dev)
            ptrs, sizes, types = [], [], []
            for (_, _, dtype), rows in work.items():
                ptrs += rows[1::10]
                sizes += rows[6::10]
                types += [TYPES[dtype]] * (len(rows) // 10)
            args, parts = _list_args(ptrs, sizes, types)
            if parts:
                buf = torch.empty(parts + 2, dtype=torch.float64, device=dev)
                buf_ptr, norm_ptr = buf.data_ptr(), norm.data_ptr()
                with lib.Launch(dev) as st:
                    lib._chk(L.hoic_grad_norm_partial(*args, buf_ptr, st), "hoic_grad_norm_partial")
            else:
                norm.zero_()
        for (at, gi, dtype), rows in work.items():
            group, dev, n = self.param_groups[gi], torch.device("cuda", at), len(rows) // 10
            lr, (b1, b2) = group["lr"], group["betas"]
            lr_ptr = 0
            if isinstance(lr, torch.Tensor):
                lr, lr_ptr = 0.0, lr.data_ptr()
            consts = torch.empty(4 * n, dtype=torch.float32, device=dev) if capturable else None
            a = lib.ADAMW_ARGS.pack(TYPES[dtype], bits, lr, b1, b2, group["eps"], group["weight_decay"], lr_ptr,
                                    0 if consts is None else consts.data_ptr(), buf_ptr, norm_ptr, bound or 0.0, parts, group["seed"], 0)
            with lib.Launch(dev) as st:
                lib._chk(L.hoic_adamw(_pack(rows), n, a, st), "hoic_adamw")
        if not capturable:
            for s in touched:
                s["step"] += 1
        torch.autograd.graph.increment_version(params)
        return loss

    def state_values(self):
        """([m, ...], [v, ...]): both moments of every parameter in float32 (8-bit states: the values that their codes stand for, made
        anew by one launch per 48 tensors; 32-bit ones: the states themselves); zeros where a parameter has no state yet."""
        bits, groups = self.defaults["state_bits"], self.param_groups
        states = [(p, self.state.get(p)) for group in groups for p in group["params"]]
        if not states:
            return [], []
        if bits == 32 and all(s for _, s in states):
            return [s["exp_avg"] for _, s in states], [s["exp_avg_sq"] for _, s in states]
        changed = "AdamW: 8-bit moments of a parameter whose size, device or order in memory has changed since"
        at, work = states[0][0].get_device(), {}
        if bits == 8 and all([s and p.is_contiguous() and p.get_device() == at for p, s in states]):
            # one buffer, cut into the parameters' shapes (an allocation a parameter costs more than the launch)
            sizes = [p.numel() for p, _ in states]
            n, k = sum(sizes), len(sizes)
            buf = torch.empty(2 * n, dtype=torch.float32, device=states[0][0].device)
            mp, rows = buf.data_ptr(), []
            for (_, s), size in zip(states, sizes):
                m = s["exp_avg"]
                if m.numel() != size or m.get_device() != at or "order" in s:
                    raise ValueError(changed)
                rows += (mp, mp + 4 * n, m.data_ptr(), s["exp_avg_sq"].data_ptr(), s["exp_avg_scale"].data_ptr(), s["exp_avg_sq_scale"].data_ptr(), size, 1, 0, 0)
                mp += 4 * size
            work[buf.device] = rows
            out = [x if p.dim() == 1 else x.view(p.shape) for (p, _), x in zip(states + states, torch.split_with_sizes(buf, sizes + sizes))]
            ms, vs = out[:k], out[k:]
        else:
            new = lambda p: torch.empty_like(p, dtype=torch.float32, requires_grad=False)
            ms = [s["exp_avg"] if s and bits == 32 else new(p) if s else new(p).zero_() for p, s in states]
            vs = [s["exp_avg_sq"] if s and bits == 32 else new(p) if s else new(p).zero_() for p, s in states]
            for (p, s), m, v in zip(states, ms, vs):
                if s and bits == 8:
                    if s["exp_avg"].numel() != p.numel() or s["exp_avg"].device != p.device or s.get("order") != (None if p.is_contiguous() else _strides(p)):
                        raise ValueError(changed)
                    work.setdefault(p.device, []).extend((m.data_ptr(), v.data_ptr(), s["exp_avg"].data_ptr(), s["exp_avg_sq"].data_ptr(), s["exp_avg_scale"].data_ptr(),
                                                          s["exp_avg_sq_scale"].data_ptr(), p.numel(), 1, 0, 0))
        for dev, rows in work.items():
            with lib.Launch(dev) as st:
                lib._chk(lib.load().hoic_adamw_values(_pack(rows), len(rows) // 10, st), "hoic_adamw_values")
        return ms, vs


AdamW._step_hooked = torch.optim.Optimizer.profile_hook_step(AdamW._step)
