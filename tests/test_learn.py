"""The clipped policy loss with a KL term (hoic_amd.rl), gradient norm / clipping and AdamW with 32- or 8-bit states (hoic_amd.optim)
against plain implementations in 64 bits.

Tolerances: a rounding to type t is off by at most finfo(t).eps / 2 of the value (``half``).  The loss's kernel works in 64 bits per row
and rounds once (twice to 16-bit types, through float32): half(t) + 2^-24 of the value, plus 1e-12 of the largest term for the 64-bit
arithmetic (log-probabilities around 100 in magnitude: 100 x 2^-53 in the exponent).  AdamW's bounds count the float32 roundings
of each formula where they are used.
"""
import copy
import math

import numpy as np
import pytest
import torch

from hoic_amd import lib, optim, rl

gpu = pytest.mark.gpu
U32 = 2.0 ** -24


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float64: 0.0}[t]


# ================================================================================================ policy loss
def loss_case(M, N, mean="f32", act="f32", per_row=False, ref=True, ref_row=None, mask=0.0, first=False, seed=0, device="cpu", spread=0.3):
    T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g)
    old = rn(M, N)
    s0 = 0.2 * rn(M if (per_row if ref_row is None else ref_row) else 1, N) - 0.4
    act_ = old + torch.exp(s0) * rn(M, N)
    mu = old + spread / math.sqrt(N) * rn(M, N)
    s = (s0 if s0.shape[0] == (M if per_row else 1) else 0.2 * rn(M if per_row else 1, N) - 0.4) + 0.1 / math.sqrt(N) * rn(M if per_row else 1, N)
    d = act_ - old
    fixed = (-(d * d) / (2 * torch.exp(2 * s0)) - s0 - 0.5 * math.log(2 * math.pi)).sum(1)
    x = dict(mean=mu.to(T[mean]), log_std=s, actions=act_.to(T[act]), advantages=rn(M), fixed_log_probs=None if first else fixed,
             ref_mean=old.to(T[mean]) if ref else None, ref_log_std=s0 if ref else None, valid=None)
    if mask:
        x["valid"] = torch.rand(M, generator=g) >= mask
        bad = ~x["valid"]
        x["mean"][bad] = float("nan"); x["actions"][bad] = float("inf")
        x["advantages"][bad] = float("-inf")
        if x["fixed_log_probs"] is not None:
            x["fixed_log_probs"][bad] = float("nan")
        if ref:
            x["ref_mean"][bad] = torch.finfo(x["ref_mean"].dtype).min
    return {k: None if v is None else v.to(device) for k, v in x.items()}


def loss_reference(x, clip=(0.2, 0.2), kl_coef=0.0, weight=1.0):
    """float64 on the CPU, gradients by the formulas (not by differentiation)."""
    c = {k: None if v is None else v.detach().cpu() for k, v in x.items()}
    M, N = c["mean"].shape
    ok = torch.ones(M, dtype=torch.bool) if c["valid"] is None else c["valid"].bool()
    n = max(int(ok.sum()), 1)
    f = lambda t: t.double().expand(M, N)[ok] if t.dim() == 2 or t.shape[0] == N else t.double()
    mu, a, s = c["mean"].double()[ok], c["actions"].double()[ok], f(c["log_std"].reshape(-1, N))
    A = c["advantages"].reshape(-1).double()[ok]
    sig2 = torch.exp(2 * s)
    d = a - mu
    lp = (-(d ** 2) / (2 * sig2) - s - 0.5 * math.log(2 * math.pi)).sum(1)
    r = torch.ones_like(lp) if c["fixed_log_probs"] is None else torch.exp(lp - c["fixed_log_probs"].reshape(-1).double()[ok])
    lo, hi = 1 - clip[0], 1 + clip[1]
    s1, s2 = r * A, torch.clamp(r, lo, hi) * A
    moving = (s1 < s2) | ((r >= lo) & (r <= hi))
    surr = -torch.minimum(s1, s2).sum() / n
    dlp = torch.where(moving, -s1, torch.zeros_like(s1)) / n
    g_mu, g_s = dlp[:, None] * d / sig2, dlp[:, None] * (d ** 2 / sig2 - 1)
    kl = torch.zeros((), dtype=torch.float64)
    if c["ref_mean"] is not None:
        s0 = f(c["ref_log_std"].reshape(-1, N))
        dk = mu - c["ref_mean"].double()[ok]
        kl = (s - s0 + (torch.exp(2 * s0) + dk ** 2) / (2 * sig2) - 0.5).sum() / n
        g_mu = g_mu + kl_coef / n * dk / sig2
        g_s = g_s + kl_coef / n * (1 - (torch.exp(2 * s0) + dk ** 2) / sig2)
    full = lambda t: torch.zeros(M, N, dtype=torch.float64).index_copy_(0, ok.nonzero()[:, 0], weight * t)
    g_s_rows = full(g_s)
    shared = c["log_std"].reshape(-1, N).shape[0] == 1
    d_s = g_s_rows.sum(0, keepdim=True) if shared else g_s_rows
    lps = torch.zeros(M, 1, dtype=torch.float64).index_copy_(0, ok.nonzero()[:, 0], lp[:, None])
    clipped = (~moving).sum().double() / n
    return dict(loss=surr + kl_coef * kl, info=torch.stack([surr, kl, clipped, ok.sum().double()]), d_mean=full(g_mu),
                d_log_std=d_s.reshape(c["log_std"].shape), log_probs=lps, terms=g_s_rows.abs().sum(0).max() if M else torch.zeros(()))


def close(got, want, what, floor=0.0):
    """one rounding to got's type (through float32), and 64-bit arithmetic on terms as large as the largest value"""
    t = got.dtype
    got, want = got.detach().cpu().double().reshape(-1), want.reshape(-1)
    if not want.numel():
        return
    tol = (half(t) + U32) * want.abs() + 1e-12 * float(want.abs().max()) + tiny(t) + floor
    bad = ((got - want).abs() > tol) | torch.isnan(got)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() - tol).max())} over its bound"


def check_loss(x, clip=(0.2, 0.2), kl_coef=0.3, weight=1.0):
    kl_coef = kl_coef if x["ref_mean"] is not None else 0.0
    ref = loss_reference(x, clip, kl_coef, weight)
    args = {k: v for k, v in x.items()}
    o = rl.clipped_policy_loss_grad(**args, clip_epsilon=clip, kl_coef=kl_coef, weight=weight)
    f = 1e-12 * max(1.0, float(ref["info"][:2].abs().max()))
    close(o.loss, ref["loss"], "loss", f); close(o.info, ref["info"], "info", f)
    close(o.d_mean, ref["d_mean"], "d_mean"); close(o.d_log_std, ref["d_log_std"], "d_log_std", 1e-12 * float(ref["terms"]))
    assert o.d_mean.dtype == x["mean"].dtype and o.d_log_std.dtype == x["log_std"].dtype and o.d_log_std.shape == x["log_std"].shape
    if x["fixed_log_probs"] is None:
        close(o.log_probs, ref["log_probs"], "log_probs")
        assert o.log_probs.shape == (x["mean"].shape[0], 1)
    else:
        assert o.log_probs is None
    # the differentiable form: the same value, gradients scaled by what comes in
    mu, s = x["mean"].detach().requires_grad_(), x["log_std"].detach().requires_grad_()
    p = rl.clipped_policy_loss(**{**args, "mean": mu, "log_std": s}, clip_epsilon=clip, kl_coef=kl_coef)
    close(p.loss, ref["loss"], "loss", f); close(p.info, ref["info"], "info", f)
    (p.loss * weight).backward()
    close(mu.grad, ref["d_mean"], "autograd d_mean"); close(s.grad, ref["d_log_std"], "autograd d_log_std", 1e-12 * float(ref["terms"]))
    return o


SHAPES = [(1, 1), (1, 32), (2, 3), (33, 4), (64, 5), (257, 32), (100, 26), (31, 33), (19, 100), (5, 256), (4099, 32)]


@gpu
@pytest.mark.parametrize("M,N", SHAPES)
@pytest.mark.parametrize("kind", ["plain", "kl", "mask", "per_row", "first"])
def test_policy_loss_matches_float64(M, N, kind):
    x = loss_case(M, N, ref=kind != "plain", mask=0.4 if kind in ("mask", "per_row") else 0.0, per_row=kind == "per_row", first=kind == "first",
                  seed=M + N, device="cuda")
    check_loss(x, kl_coef=0.0 if kind == "plain" else 0.3)


@gpu
@pytest.mark.parametrize("mean,act", [("bf16", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("M,N", [(300, 32), (77, 7), (40, 130)])
def test_policy_loss_in_16_bits(mean, act, M, N):
    check_loss(loss_case(M, N, mean, act, mask=0.3, seed=3, device="cuda"), weight=float(M))
    check_loss(loss_case(M, N, mean, act, per_row=True, seed=4, device="cuda"), weight=float(M))
    x = loss_case(M, N, mean, act, per_row=True, seed=5, device="cuda")          # log_std from the same 16-bit network
    x["log_std"], x["ref_log_std"] = x["log_std"].to(x["mean"].dtype), x["ref_log_std"].to(x["mean"].dtype)
    check_loss(x, weight=float(M))


@gpu
def test_policy_loss_clips_and_references_of_other_shapes():
    for clip in ((0.0, 0.0), (0.1, 0.4), (0.0, 3.0)):
        check_loss(loss_case(500, 12, spread=1.0, seed=7, device="cuda"), clip=clip)
    check_loss(loss_case(500, 12, per_row=True, ref_row=False, seed=8, device="cuda"))
    check_loss(loss_case(500, 12, per_row=False, ref_row=True, seed=9, device="cuda"))
    x = loss_case(64, 6, seed=10, device="cuda")
    for k in ("log_std", "ref_log_std"):
        x[k] = x[k].reshape(-1)                                                # [N]
    x["advantages"], x["fixed_log_probs"] = x["advantages"][:, None], x["fixed_log_probs"][:, None]
    check_loss(x)


@gpu
@pytest.mark.parametrize("mean", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["both", "log_std", "ref_log_std"])
def test_policy_loss_deviations_of_masked_rows_are_not_used(kind, mean):
    """rows outside the batch (the first and the last among them) hold log-deviations that are no numbers, the policy's, the reference's or
    both (a shared one of the policy's with the reference's per row, too): their gradients are 0 and nobody else's see them"""
    for M, N in ((2, 3), (33, 4), (70, 32), (19, 100)):
        x = loss_case(M, N, mean=mean, per_row=kind != "ref_log_std", ref_row=kind != "log_std", mask=0.4, seed=M)
        bad = ~x["valid"]
        bad[0] = bad[-1] = True                                                           # (of two rows none is left)
        x["valid"] = ~bad
        for value in (float("nan"), float("inf"), float("-inf")):
            for name in ("log_std", "ref_log_std"):
                if kind in ("both", name):
                    x[name][bad] = value
            o = check_loss({k: None if v is None else v.cuda() for k, v in x.items()})
            assert not bool(o.d_mean.cpu()[bad].any())
        # a shared deviation that is no number reaches the rows of the batch only, and none if there are none
        y = dict(x, log_std=torch.full((1, N), float("nan")), ref_log_std=torch.full((1, N), float("inf")))
        y = {k: v.cuda() for k, v in y.items()}
        o = rl.clipped_policy_loss_grad(**y, kl_coef=0.3)
        assert not bool(o.d_mean.cpu()[bad].any()) and (bool(bad.all()) or bool(torch.isnan(o.d_log_std).all()))
        o = rl.clipped_policy_loss_grad(**dict(y, valid=torch.zeros(M, dtype=torch.bool, device="cuda")), kl_coef=0.3)
        assert float(o.loss) == 0.0 and not bool(o.d_mean.any()) and not bool(o.d_log_std.any())


@gpu
@pytest.mark.parametrize("M", [15, 16, 17, 4095, 4097, 12304, 16383, 16384, 16401, 65535, 65536, 65537, 70001, (1 << 20) + 5])
def test_policy_loss_counts_the_valid_rows(M):
    """flags as bool and as bytes of any value, at every alignment, in batches that every workgroup counts by itself and in larger ones: the
    number is in ``info`` and divides the gradient (advantage 1, ratio 1: each valid row's d_mean is -(a - mean) / sigma^2 / n)"""
    g = torch.Generator().manual_seed(M)
    for shift, kind in ((0, "bool"), (1, "bytes"), (7, "bytes"), (3, "one"), (2, "none")):
        flags = torch.zeros(M + 8, dtype=torch.uint8)
        if kind == "one":
            flags[shift + int(torch.randint(M, (), generator=g))] = 128
        elif kind != "none":
            keep = torch.rand(M, generator=g) < 0.6
            flags[shift:shift + M][keep] = torch.randint(1, 256, (int(keep.sum()),), generator=g).to(torch.uint8) if kind == "bytes" else 1
        n = int((flags[shift:shift + M] != 0).sum())
        ok = (flags[shift:shift + M] != 0).cuda()
        valid = flags.cuda()[shift:shift + M]
        valid = valid.bool() if kind == "bool" else valid
        mean = torch.zeros(M, 1, device="cuda")
        o = rl.clipped_policy_loss_grad(mean, torch.zeros(1, device="cuda"), torch.ones(M, 1, device="cuda"), torch.ones(M, device="cuda"), valid=valid)
        assert float(o.info[3]) == n
        want = torch.where(ok, torch.full((M,), -1.0 / max(n, 1), device="cuda"), torch.zeros(M, device="cuda"))
        assert torch.equal(o.d_mean[:, 0], want)


@gpu
def test_policy_loss_strides_and_expanded_rows():
    """row strides that are no multiple of the dimensions, columns that are not adjacent, one row expanded over the batch"""
    base = loss_case(200, 9, per_row=True, seed=11, device="cuda")
    want = check_loss(base)
    wide = lambda t: torch.nn.functional.pad(t, (1, 4), value=float("nan"))[:, 1:10]
    x = {**base, **{k: wide(base[k]) for k in ("mean", "actions", "log_std", "ref_mean", "ref_log_std")}}
    assert x["mean"].stride() == (14, 1)
    o = check_loss(x)
    for a, b in zip(o[:4], want[:4]):
        assert torch.equal(a, b)
    x = {**base, **{k: base[k].t().contiguous().t() for k in ("mean", "actions", "log_std", "ref_mean", "ref_log_std")}}
    for a, b in zip(check_loss(x)[:4], want[:4]):
        assert torch.equal(a, b)
    # four dimensions a load at every alignment of a type, a mask that starts anywhere
    for dt, at in ((torch.float32, 1), (torch.bfloat16, 1), (torch.float16, 3)):
        b = loss_case(150, 8, mask=0.3, per_row=True, seed=21, device="cuda")
        for k in ("mean", "actions", "ref_mean"):
            b[k] = b[k].to(dt)
        cut = lambda t: torch.nn.functional.pad(t, (at, 2))[:, at:at + t.shape[1]]
        shift = lambda t: torch.cat([t[:at], t])[at:]
        y = {**b, **{k: cut(b[k]) for k in ("mean", "actions", "log_std", "ref_mean", "ref_log_std")}, "valid": shift(b["valid"]), "advantages": shift(b["advantages"])}
        assert y["mean"].data_ptr() % 16 and y["valid"].data_ptr() % 4
        for a, c in zip(rl.clipped_policy_loss_grad(**y, kl_coef=0.3)[:4], rl.clipped_policy_loss_grad(**b, kl_coef=0.3)[:4]):
            assert torch.equal(a, c)
    one = {**base, "mean": base["mean"][:1].expand(200, 9), "log_std": base["log_std"][:1].expand(200, 9)}
    check_loss(one)


@gpu
def test_policy_loss_without_rows():
    """no valid row and no row at all: value 0, gradients 0, nothing from what the rows hold"""
    x = loss_case(70, 8, mask=0.5, seed=12, device="cuda")
    x["valid"].fill_(False)
    for t in ("mean", "actions"):
        x[t].fill_(float("nan"))
    o = rl.clipped_policy_loss_grad(**x, kl_coef=0.5)
    assert float(o.loss) == 0 and o.info.tolist() == [0, 0, 0, 0] and not o.d_mean.any() and not o.d_log_std.any()
    mu, s = x["mean"].requires_grad_(), x["log_std"].requires_grad_()
    p = rl.clipped_policy_loss(**{**x, "mean": mu, "log_std": s}, kl_coef=0.5)
    p.loss.backward()
    assert float(p.loss.detach()) == 0 and not mu.grad.any() and not s.grad.any()
    x = loss_case(0, 8, seed=13, device="cuda")
    o = rl.clipped_policy_loss_grad(**x, kl_coef=0.5)
    assert float(o.loss) == 0 and o.d_mean.shape == (0, 8) and not o.d_log_std.any()


@gpu
def test_policy_loss_extremes():
    """non-finite values in valid rows reach that row's gradient only; a ratio past float32's range keeps its sign; rows exactly on a
    clip border pass their gradient"""
    x = loss_case(50, 4, ref=False, seed=14, device="cuda")
    x["mean"][7, 2] = float("nan")
    o = rl.clipped_policy_loss_grad(**x)
    assert math.isnan(float(o.loss)) and bool(torch.isnan(o.d_mean[7]).all())
    rest = torch.arange(50, device="cuda") != 7
    assert bool(torch.isfinite(o.d_mean[rest]).all())
    y = {k: v[rest] if v is not None and v.shape[0] == 50 else v for k, v in x.items()}
    ref = loss_reference(y, weight=49 / 50)
    close(o.d_mean[rest], ref["d_mean"], "the other rows")
    # e^200: beyond float32; A < 0 passes the gradient of the unclipped branch, A > 0 none
    x = loss_case(2, 4, ref=False, seed=15, device="cuda")
    lp = rl.clipped_policy_loss_grad(**{**x, "fixed_log_probs": None}).log_probs[:, 0]
    x["fixed_log_probs"] = lp - 80.0
    x["advantages"] = torch.tensor([1e-20, -1e-20], device="cuda")
    check_loss(x)
    # ratio exactly 1 with an interval of width 0
    x = loss_case(9, 4, ref=False, first=True, seed=16, device="cuda")
    o = check_loss(x, clip=(0.0, 0.0), kl_coef=0.0)
    assert float(o.info[2]) == 0 and bool(o.d_mean.any(1).all())


@gpu
def test_policy_loss_gradient_against_differences():
    """central differences of the value in 64 bits (the tensor form) at a point away from the clip borders"""
    x = loss_case(6, 3, seed=17, spread=0.05)
    o = rl.clipped_policy_loss_grad(**{k: None if v is None else v.cuda() for k, v in x.items()}, kl_coef=0.4)
    x64 = {k: v.double() if v is not None and v.dtype != torch.bool else v for k, v in x.items()}
    # truncation h^2 / 6 of a third derivative (a handful of units here: 1e3 allowed), cancellation 2^-53 / h
    h = 1e-5
    for name, grad in (("mean", o.d_mean), ("log_std", o.d_log_std)):
        for i in range(x64[name].numel()):
            v = []
            for sgn in (1, -1):
                y = {**x64, name: x64[name].clone()}
                y[name].view(-1)[i] += sgn * h
                v.append(float(rl.clipped_policy_loss(**y, kl_coef=0.4).loss))
            want = (v[0] - v[1]) / (2 * h)
            assert abs(float(grad.view(-1)[i]) - want) <= U32 * 2 * abs(want) + 1e3 * h * h / 6 + 2 ** -50 / h


@gpu
@pytest.mark.parametrize("mean", ["f32", "bf16"])
def test_policy_loss_backward_twice_and_in_part(mean):
    """a graph kept for a second backward call, gradients taken over by the leaves and changed there, one input without gradient"""
    x = loss_case(300, 8, mean, mask=0.3, seed=30, device="cuda")
    ref = loss_reference(x, kl_coef=0.3)
    mu, s = x["mean"].detach().requires_grad_(), x["log_std"].detach().requires_grad_()
    p = rl.clipped_policy_loss(**{**x, "mean": mu, "log_std": s}, kl_coef=0.3)
    p.loss.backward(retain_graph=True)
    close(mu.grad, ref["d_mean"], "first"); close(s.grad, ref["d_log_std"], "first", 1e-12 * float(ref["terms"]))
    mu.grad.zero_(); s.grad.fill_(7.0)
    g = torch.autograd.grad(p.loss, (mu, s), grad_outputs=torch.tensor(4.0, device="cuda"), retain_graph=True)
    for a, k in zip(g, ("d_mean", "d_log_std")):
        close(a, 4 * ref[k], "second", 1e-11 * float(ref["terms"]))
    (2.0 * p.loss + 1.0).backward()
    close(mu.grad, 2 * ref["d_mean"], "third")
    for only in ("mean", "log_std"):
        leaf = x[only].detach().requires_grad_()
        rl.clipped_policy_loss(**{**x, only: leaf}, kl_coef=0.3).loss.backward()
        close(leaf.grad, ref["d_" + only], only, 1e-12 * float(ref["terms"]))
    with torch.no_grad():
        assert not rl.clipped_policy_loss(**{**x, "mean": mu}, kl_coef=0.3).loss.requires_grad
    q = rl.clipped_policy_loss(**{**x, "mean": mu}, kl_coef=0.3)
    with torch.no_grad():
        mu.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        q.loss.backward()


@gpu
def test_policy_loss_matches_the_existing_losses():
    """kl_coef 0: rl.ppo_loss on the CPU in float64, and the fused head step's loss kernel's gradient, on the learner's own shapes"""
    x = loss_case(1000, 32, ref=False, seed=18, device="cuda")
    class P:
        def get_log_prob(self, states, action, hidden):
            mean, s = states
            return (-((action - mean) ** 2) / (2 * torch.exp(2 * s)) - s - 0.5 * math.log(2 * math.pi)).sum(1, keepdim=True)
    c = {k: None if v is None else v.cpu().double() for k, v in x.items()}
    want = rl.ppo_loss(P(), (c["mean"], c["log_std"]), c["actions"], c["advantages"][:, None], c["fixed_log_probs"][:, None], 0.2)
    close(rl.clipped_policy_loss(**x).loss, want, "loss", 1e-12)


@gpu
def test_policy_loss_on_a_side_stream_and_in_a_graph():
    x = loss_case(3000, 32, mask=0.2, seed=19, device="cuda")
    want = rl.clipped_policy_loss_grad(**x, kl_coef=0.3)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        got = rl.clipped_policy_loss_grad(**x, kl_coef=0.3)
    torch.cuda.current_stream().wait_stream(st)
    for a, b in zip(got[:4], want[:4]):
        assert torch.equal(a, b)
    # captured, with a fresh leaf of its own; replayed on changing inputs, eager work between the replays
    mu, s = x["mean"].clone().requires_grad_(), x["log_std"].clone().requires_grad_()
    args = {**x, "mean": mu, "log_std": s}
    with torch.cuda.stream(st):
        for _ in range(2):
            torch.autograd.grad(rl.clipped_policy_loss(**args, kl_coef=0.3).loss, (mu, s))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p = rl.clipped_policy_loss(**args, kl_coef=0.3)
        gm, gs = torch.autograd.grad(p.loss * 2.0, (mu, s))
    for rep in range(4):
        with torch.no_grad():
            mu.add_(0.01)
        graph.replay()
        torch.cuda.synchronize()
        e = rl.clipped_policy_loss_grad(**{**x, "mean": mu.detach()}, kl_coef=0.3, weight=2.0)
        assert torch.equal(p.loss, e.loss) and torch.equal(gm, e.d_mean) and torch.equal(gs, e.d_log_std) and torch.equal(p.info, e.info), rep
    # the one-pass form with its count of the valid rows, beside the norm and the clipping of what it made
    grads = [torch.nn.Parameter(torch.zeros_like(x["mean"])), torch.nn.Parameter(torch.zeros_like(x["log_std"]))]
    for p_ in grads:
        p_.grad = torch.zeros_like(p_)
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        o = rl.clipped_policy_loss_grad(**{**x, "mean": mu.detach()}, kl_coef=0.3, weight=100.0)
        grads[0].grad.copy_(o.d_mean); grads[1].grad.copy_(o.d_log_std)
        norm = optim.clip_grad_norm_(grads, 0.5)
        after = optim.grad_norm([p_.grad for p_ in grads])
    for rep in range(4):
        x["valid"].copy_(torch.rand(3000, device="cuda") < 0.2 * (rep + 1))
        x["mean"].nan_to_num_(0.0); x["actions"].nan_to_num_(0.0, 0.0, 0.0); x["advantages"].nan_to_num_(0.0, 0.0, 0.0); x["fixed_log_probs"].nan_to_num_(-10.0)
        with torch.no_grad():
            mu.copy_(x["mean"]).add_(0.01 * rep)
        second.replay(); graph.replay()                   # (two graphs of the same operators, one after the other)
        torch.cuda.synchronize()
        e = rl.clipped_policy_loss_grad(**{**x, "mean": mu.detach()}, kl_coef=0.3, weight=100.0)
        assert torch.equal(o.loss, e.loss) and torch.equal(o.info, e.info) and torch.equal(o.d_mean, e.d_mean) and torch.equal(o.d_log_std, e.d_log_std), rep
        total = float(optim.grad_norm([e.d_mean, e.d_log_std]))
        # (rows that were padding are valid now, their reference means at float32's lowest value: where the norm is not finite, what was
        #  scaled by 0 is NaN in the infinite places)
        assert float(norm) == total and total > 0.5, rep
        assert abs(float(after) - 0.5) <= 0.5 * (1e-6 / 0.5 + 8 * U32) if math.isfinite(total) else math.isnan(float(after)), rep


@gpu
def test_policy_loss_offsets_past_32_bits():
    """2^31 elements and more a tensor: the last rows against a call on them alone"""
    M, N = (1 << 26) + 5, 32
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("needs 60 GB")
    mean = torch.zeros(M, N, device="cuda"); act = torch.full((M, N), 0.5, device="cuda")
    x = loss_case(7, N, ref=False, seed=20, device="cuda")
    mean[-7:], act[-7:] = x["mean"], x["actions"]
    adv = torch.zeros(M, device="cuda"); fixed = torch.zeros(M, device="cuda")
    adv[-7:], fixed[-7:] = x["advantages"], x["fixed_log_probs"]
    o = rl.clipped_policy_loss_grad(mean, x["log_std"], act, adv, fixed, weight=float(M))
    ref = loss_reference(x, weight=7.0)
    close(o.d_mean[-7:], ref["d_mean"], "last rows")
    assert not o.d_mean[:-7].any() and float(o.info[3]) == float(torch.tensor(M, dtype=torch.float32))
    close(o.d_log_std, ref["d_log_std"], "d_log_std", 1e-12 * float(ref["terms"]))


def test_policy_loss_tensor_form_and_refusals():
    """the tensor form (CPU, float64) against the formulas, and every call that is refused"""
    for kind in range(4):
        x = loss_case(40, 5, per_row=kind == 1, mask=0.4 if kind == 2 else 0.0, first=kind == 3, seed=kind)
        x = {k: v.double() if v is not None and v.dtype != torch.bool else v for k, v in x.items()}
        ref = loss_reference(x, kl_coef=0.3, weight=2.0)
        o = rl.clipped_policy_loss_grad(**x, kl_coef=0.3, weight=2.0)
        for k in ("loss", "info", "d_mean", "d_log_std"):
            torch.testing.assert_close(getattr(o, k), ref[k], rtol=1e-12, atol=1e-13)
        if kind == 3:
            torch.testing.assert_close(o.log_probs, ref["log_probs"], rtol=1e-12, atol=1e-13)
    x = loss_case(6, 3)
    bad = [dict(mean=x["mean"][0]), dict(mean=x["mean"].int()), dict(actions=x["actions"][:, :2]), dict(actions=x["actions"].half()), dict(log_std=x["log_std"][:, :2]),
           dict(log_std=x["log_std"].expand(5, 3)), dict(advantages=x["advantages"][:5]), dict(advantages=x["advantages"].double()),
           dict(fixed_log_probs=x["fixed_log_probs"].half()), dict(valid=torch.ones(5, dtype=torch.bool)), dict(valid=torch.ones(6)), dict(ref_mean=None),
           dict(ref_log_std=None), dict(ref_mean=x["ref_mean"].half()), dict(ref_log_std=x["ref_log_std"].double()), dict(clip_epsilon=-0.1),
           dict(clip_epsilon=(0.1, math.nan)), dict(kl_coef=math.inf), dict(ref_mean=None, ref_log_std=None, kl_coef=0.1), dict(mean=torch.zeros(6, 0))]
    for b in bad:
        with pytest.raises(ValueError):
            rl.clipped_policy_loss_grad(**{**x, "kl_coef": 0.0, **b})


def test_policy_loss_entry_point_refuses_on_the_host():
    """hoic_policy_loss checks its arguments before any launch (no GPU is needed to see it)"""
    L = lib.load()
    assert L.hoic_policy_loss(None, None) == -1
    names = ("rows dims t_mean t_act t_std mean act log_std ref_mean ref_log_std ld_mean ld_act ld_std ld_ref_mean ld_ref_std ld_dmean adv fixed valid upstream count "
             "clip_lo clip_hi kl_coef weight d_mean d_log_std log_probs loss info n_out scratch").split()
    at = 64
    good = dict.fromkeys(names, 0) | dict(rows=4, dims=4, mean=at, act=at, log_std=at, adv=at, loss=at, info=at, scratch=at)
    for change in (dict(dims=0), dict(dims=257), dict(rows=-1), dict(t_mean=3), dict(t_mean=2, t_act=1), dict(t_std=1), dict(mean=0), dict(scratch=0), dict(loss=0), dict(info=0),
                   dict(ref_mean=at), dict(ref_log_std=at), dict(d_log_std=at), dict(count=at)):
        assert L.hoic_policy_loss(lib.POLICY_LOSS_ARGS.pack(*(good | change).values()), None) == -1, change
    assert L.hoic_policy_loss_scratch_bytes(0) == 0


def test_policy_loss_entry_point_refuses_rows_beyond_its_counts():
    L = lib.load()
    at = 64
    for rows in ((1 << 32) + 1, 1 << 40):
        args = lib.POLICY_LOSS_ARGS.pack(rows, 4, 0, 0, 0, at, at, at, 0, 0, 4, 4, 0, 0, 0, 4, at, 0, 0, 0, 0, 0.2, 0.2, 0.0, 1.0, 0, 0, 0, at, at, 0, at)
        assert L.hoic_policy_loss(args, None) == -1 and b"2^32" in L.hoic_last_error()


# ================================================================================================ norm and clipping
def tensor_list(sizes, dtype=torch.float32, seed=0, scale=1.0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(s, generator=g) * math.exp(2 * math.sin(i))).to(dtype).to(device) for i, s in enumerate(sizes)]


SIZES = [[1], [3, 0, 5], [8191, 8192, 8193], [1000003], [(64, 617), (64,), (32, 64), (32,)], [17] * 300, [5, 1 << 22, 7]]


@gpu
@pytest.mark.parametrize("sizes", SIZES, ids=[f"{len(s)}x{s[0]}" for s in SIZES])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_grad_norm_and_clipping(sizes, dtype):
    """norm: 64-bit sums, one rounding to float32; clipped gradients: factor rounded to float32, product, result type"""
    gs = tensor_list(sizes, dtype, seed=len(sizes))
    want = math.sqrt(sum(float((g.cpu().double() ** 2).sum()) for g in gs))
    got = optim.grad_norm(gs)
    assert got.dtype == torch.float32 and got.dim() == 0 and abs(float(got) - want) <= (U32 + 1e-12) * want
    assert torch.equal(got, optim.grad_norm(gs))
    for bound in (0.5 * want, 2.0 * want):
        ps = [torch.nn.Parameter(torch.zeros_like(g)) for g in gs]
        for p, g in zip(ps, gs):
            p.grad = g.clone()
        n = optim.clip_grad_norm_(ps, bound)
        assert torch.equal(n, got)
        c = min(1.0, bound / (want + 1e-6))
        for p, g in zip(ps, gs):
            if c == 1.0:
                assert torch.equal(p.grad, g)
            else:
                w = g.cpu().double() * c
                assert bool(((p.grad.cpu().double() - w).abs() <= (half(dtype) + 2.1 * U32) * w.abs() + tiny(dtype)).all())


@gpu
def test_grad_norm_of_mixed_types_strides_and_values():
    gs = tensor_list([100, 200], torch.float32) + tensor_list([300], torch.bfloat16, 1) + tensor_list([(40, 50)], torch.float16, 2)
    gs[3] = gs[3].t()
    gs.append(torch.randn(64, 10, device="cuda")[:, 2:7])
    want = math.sqrt(sum(float((g.cpu().double() ** 2).sum()) for g in gs))
    assert abs(float(optim.grad_norm(gs)) - want) <= (U32 + 1e-12) * want
    big = [torch.full((1000,), 3e38, device="cuda"), torch.full((10,), 1e-30, device="cuda")]       # squares past float32's range
    assert abs(float(optim.grad_norm([big[0][:1]])) / 3e38 - 1) < 1e-6 and math.isinf(float(optim.grad_norm([big[0]])) ) is (3e38 * math.sqrt(1000) > 3.4e38)
    assert abs(float(optim.grad_norm([big[1]])) / (1e-30 * math.sqrt(10)) - 1) < 1e-6
    p = torch.nn.Parameter(torch.zeros(4, device="cuda"))
    p.grad = torch.tensor([1.0, float("inf"), 2.0, 0.0], device="cuda")
    q = torch.nn.Parameter(torch.zeros(4, device="cuda")); q.grad = p.grad.clone()
    n = optim.clip_grad_norm_([p], 1.0); m = torch.nn.utils.clip_grad_norm_([q], 1.0)
    assert math.isinf(float(n)) and math.isinf(float(m)) and torch.equal(torch.isnan(p.grad), torch.isnan(q.grad)) and float(p.grad[0]) == float(q.grad[0]) == 0
    assert float(optim.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3, device="cuda"))], 1.0)) == 0      # no gradient anywhere
    assert float(optim.grad_norm([torch.zeros(0, device="cuda")])) == 0
    flat = torch.randn(1000, device="cuda")
    twice = [torch.nn.Parameter(torch.zeros(500, device="cuda")) for _ in range(2)]
    for p in twice:
        p.grad = flat[3:503]
    with pytest.raises(ValueError, match="same memory"):
        optim.clip_grad_norm_(twice, 1.0)
    with pytest.raises(ValueError, match="fill their memory"):
        twice[0].grad = flat[::2]
        optim.clip_grad_norm_(twice[:1], 1.0)
    # views of one buffer at odd offsets, as a network's gradients in a bucket
    want = float(flat[1:].double().norm())
    for p, (i, j) in zip(twice, ((1, 501), (501, 1000))):
        p.data = torch.zeros(j - i, device="cuda"); p.grad = flat[i:j]
    first = flat.clone()
    assert abs(float(optim.clip_grad_norm_(twice, 0.5 * want)) - want) <= (U32 + 1e-12) * want
    assert float(flat[0]) == float(first[0]) and bool(((flat[1:] - 0.5 * first[1:]).abs() <= (4 * U32 + 1e-6 / want) * first[1:].abs()).all())


def test_norm_refusals():
    for t in (torch.zeros(3), [torch.zeros(3)]):
        with pytest.raises(lib.HoicError):
            optim.grad_norm(t)
    p = torch.nn.Parameter(torch.zeros(3)); p.grad = torch.ones(3)
    for b in (-1.0, math.nan):
        with pytest.raises(ValueError):
            optim.clip_grad_norm_([p], b)
    with pytest.raises(lib.HoicError):
        optim.clip_grad_norm_([p], 1.0)
    import ctypes as C
    L = lib.load()
    one, none = (C.c_int64 * 1)(4), (C.c_int64 * 1)(0)
    null, some = (C.c_void_p * 1)(None), (C.c_void_p * 1)(8)
    assert L.hoic_grad_norm_parts(None, 1) == -1 and L.hoic_grad_norm_parts(one, 1) == 1
    for g, n, t, nt, buf, norm in ((null, one, b"\0", 1, 8, 8), (some, one, b"\5", 1, 8, 8), (some, (C.c_int64 * 1)(-1), b"\0", 1, 8, 8), (some, one, None, 1, 8, 8),
                                   (some, one, b"\0", -1, 8, 8), (some, one, b"\0", 1, None, 8)):
        assert L.hoic_grad_norm(g, n, t, nt, buf, norm, None) == -1 and L.hoic_clip_grads(g, n, t, nt, 1.0, buf, norm, None) == -1
        assert L.hoic_grad_norm_partial(g, n, t, nt, buf, None) == -1
    for n, norm, bound in ((one, None, 1.0), (none, 8, 1.0), (one, 8, -1.0), (one, 8, math.nan)):
        assert L.hoic_clip_grads(some, n, b"\0", 1, bound, 8, norm, None) == -1
    assert L.hoic_grad_norm(some, none, b"\0", 1, 8, 8, None) == -1
    assert L.hoic_scale_list(some, one, b"\0", 1, None, None) == -1 and L.hoic_scale_list(null, one, b"\0", 1, 8, None) == -1


# ================================================================================================ AdamW
def test_lists_that_overlap_are_refused_on_the_host():
    """any two tensors that are written, in whatever order they are listed; neighbours may touch"""
    import ctypes as C
    L = lib.load()
    base = 1 << 20

    def lists(spans, types):
        return (C.c_void_p * len(spans))(*[base + at for at, _ in spans]), (C.c_int64 * len(spans))(*[n for _, n in spans]), bytes(types), len(spans)

    cases = [([(0, 4), (0, 4)], (0, 0)), ([(0, 4), (12, 4)], (0, 0)), ([(12, 4), (0, 4)], (0, 0)), ([(0, 5), (8, 1)], (1, 0)), ([(64, 4), (0, 4), (32, 2), (34, 1)], (0, 0, 2, 1)),
             ([(0, 100), (40, 1), (200, 1)], (2, 0, 1))]
    for spans, types in cases:
        assert L.hoic_clip_grads(*lists(spans, types), 1.0, 8, 8, None) == -1 and b"same memory" in L.hoic_last_error()
        assert L.hoic_scale_list(*lists(spans, types), 8, None) == -1 and b"same memory" in L.hoic_last_error()
    fields = dict(type=0, state_bits=32, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, weight_decay=0.0, d_lr=0, d_consts=0, d_norm_buf=0, d_norm=0, bound=0.0, norm_parts=0, seed=0,
                  reserved=0)
    for type_, spans in ((0, [(0, 4), (12, 4)]), (2, [(12, 2), (6, 4)]), (1, [(0, 1), (0, 1)])):
        rows = [v for at, n in spans for v in (base + at, 8, 8, 8, 0, 0, n, 1, 0, 0)]
        assert L.hoic_adamw((C.c_int64 * len(rows))(*rows), len(spans), lib.ADAMW_ARGS.pack(*(fields | dict(type=type_)).values()), None) == -1
        assert b"same memory" in L.hoic_last_error()


@gpu
def test_clipping_and_adamw_of_views_of_one_buffer():
    """neighbours in one buffer, listed in any order, are taken; views that share an element are refused and left as they are"""
    flat, g = torch.randn(64, device="cuda"), torch.randn(64, device="cuda")
    cuts = [(32, 64), (0, 7), (7, 32)]
    ps = [torch.nn.Parameter(flat[a:b]) for a, b in cuts]
    for p, (a, b) in zip(ps, cuts):
        p.grad = g[a:b]
    want = g.double() * min(1.0, 0.5 / (float(g.double().norm()) + 1e-6))
    optim.clip_grad_norm_(ps, 0.5)
    assert bool(((g.double() - want).abs() <= 2 * 1.001 * U32 * want.abs() + 2.0 ** -149).all())
    opt, before = optim.AdamW(ps, lr=0.1), flat.clone()
    opt.step()
    assert bool((flat != before).all())
    ps[0].grad = g[31:63]
    keep = g.clone()
    with pytest.raises(ValueError, match="same memory"):
        optim.clip_grad_norm_(ps, 0.1)
    ps[0].data = flat[31:63]
    before = flat.clone()
    with pytest.raises(lib.HoicError, match="same memory"):
        opt.step()
    assert torch.equal(g, keep) and torch.equal(flat, before) and all(opt.state[p]["step"] == 1 for p in ps)


def random_bits(n, seed, step, ordinal, first=0):
    """the stochastic rounding's 32 bits per element, in NumPy"""
    def mix(x):
        x = np.asarray(x, dtype=np.uint64) & np.uint64(0xFFFFFFFF)
        x = x ^ (x >> np.uint64(17)); x = (x * np.uint64(0x743B8C43)) & np.uint64(0xFFFFFFFF)
        x = x ^ (x >> np.uint64(12)); x = (x * np.uint64(0xAB2209AB)) & np.uint64(0xFFFFFFFF)
        return x ^ (x >> np.uint64(15))
    i = np.arange(first, first + n, dtype=np.uint64)
    key = mix(mix(mix(mix(np.uint64(seed)) + np.uint64(step)) + np.uint64(ordinal)) + (i >> np.uint64(32)))
    return mix((i & np.uint64(0xFFFFFFFF)) + key)


def ladder(signed):
    """the values of the codes 0 .. (126 | 254) without sign, in units of the block's scale"""
    low = -6 if signed else -14
    c = np.arange(127 if signed else 255)
    e, man = c >> 3, c & 7
    return np.where(e == 0, man * 2.0 ** (low - 3), (1 + man / 8) * 2.0 ** (e - 1 + low))


def store8(x, signed, r16):
    """float64 values -> (codes, scales): the place on the ladder by search, up with the probability of the part cut off"""
    vals, top = ladder(signed), 7 if signed else 15
    codes, scales = np.zeros(x.size, np.uint8), []
    for b in range(0, x.size, 256):
        v = x[b:b + 256]
        a = np.abs(v)
        fin = np.isfinite(a)
        amax = a[fin].max() if fin.any() else 0.0
        e = max(math.frexp(amax)[1] - 1 - top, -126) if amax > 0 else -126
        k = 2.0 ** e
        scales.append(k)
        y = np.where(fin, a, 0.0) / k
        i = np.searchsorted(vals, y, side="right") - 1
        step = vals[np.minimum(i + 1, len(vals) - 1)] - vals[i]
        part = np.divide(y - vals[i], step, out=np.zeros_like(y), where=step > 0)
        i = i + (part + (r16[b:b + 256] + 0.5) / 65536.0 >= 1.0)
        if not signed:
            i = np.where((a > 0) & (i == 0), 1, i)
        c = i.astype(np.uint8)
        if signed:
            c = np.where(v < 0, c + 128, c).astype(np.uint8)
        codes[b:b + 256] = np.where(fin, c, 0x7F if signed else 0xFF)
    return codes, np.array(scales, np.float32)


def load8(codes, scales, signed):
    vals = np.append(ladder(signed), np.nan)
    c = codes.astype(np.int64)
    v = vals[c & 127] * np.where(c >= 128, -1.0, 1.0) if signed else vals[c]
    return v * np.repeat(scales.astype(np.float64), 256)[:codes.size]


HYP = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def reference_step(p, g, m, v, t, lr, betas, eps, weight_decay, coef=1.0):
    """float64 arrays -> (p', m', v', step size * m' / denominator, the error bounds of a float32 m' and of p' in float32)"""
    b1, b2 = betas
    x = g * coef
    m1, v1 = b1 * m + (1 - b1) * x, b2 * v + (1 - b2) * x * x
    den = np.sqrt(v1) / math.sqrt(1 - b2 ** t) + eps
    size = lr / (1 - b1 ** t)
    u = size * m1 / den
    p1 = p - (lr * weight_decay * p + u)
    # float32 roundings: b1, c1, the clipped gradient (factor and product), c1 x, the FMA
    em = 1.001 * U32 * (np.abs(b1 * m) + 4 * np.abs((1 - b1) * x) + np.abs(m1)) + 2.0 ** -149
    # b2, c2, twice the clipped gradient, two products, the FMA
    ev = 1.001 * U32 * (b2 * v + 7 * (1 - b2) * x * x + v1) + 3 * 2.0 ** -149
    # of the step: size, product, quotient, square root (each at most 2 half-units), its factor, eps, the FMA: under 16; v' to half its relative error
    ep = 1.01 * (U32 * (np.abs(p1) + 3 * lr * weight_decay * np.abs(p) + 16 * np.abs(u)) + size * em / den
                 + np.abs(u) * ev / (2 * np.maximum(v1, 1e-300))) + 2.0 ** -149
    return p1, m1, v1, em, ev, ep


def np64(t):
    return t.detach().cpu().double().numpy().reshape(-1)


def make_params(sizes, dtype, seed=0, gscale=1.0):
    ps = [torch.nn.Parameter(p) for p in tensor_list(sizes, dtype, seed)]
    for p, g in zip(ps, tensor_list(sizes, dtype, seed + 1, gscale)):
        p.grad = g
    return ps


LISTS = [[1], [4, 0, 255, 256, 257], [(617, 33), (33,), (5, 33)], [4095, 4096, 4097, 12289], [9] * 100]


@gpu
@pytest.mark.parametrize("sizes", LISTS, ids=[f"{len(s)}x{s[0]}" for s in LISTS])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("clip", [None, 1.5])
def test_adamw32_matches_float64(sizes, dtype, clip):
    ps = make_params(sizes, dtype)
    opt = optim.AdamW(ps, **HYP)
    state = [(np64(p), np.zeros(p.numel()), np.zeros(p.numel())) for p in ps]
    for t in (1, 2, 3):
        gs = [np64(p.grad) for p in ps]
        norm = math.sqrt(sum(float((g ** 2).sum()) for g in gs))
        opt.step(max_norm=clip)
        coef = 1.0 if clip is None else min(1.0, clip / (norm + 1e-6))
        ms, vs = opt.state_values()
        for i, p in enumerate(ps):
            p1, m1, v1, em, ev, ep = reference_step(*state[i][:1], gs[i], *state[i][1:], t, coef=coef, **HYP)
            got = np64(p)
            assert (np.abs(np64(ms[i]) - m1) <= em).all() and (np.abs(np64(vs[i]) - v1) <= ev).all(), (i, t)
            assert (np.abs(got - p1) <= ep + (half(dtype) * np.abs(p1) * 1.01 + tiny(dtype) if dtype != torch.float32 else 0)).all(), (i, t)
            state[i] = (got, np64(ms[i]), np64(vs[i]))               # the next step from what is held
            p.grad = (p.grad.float() * 0.7 + 0.1).to(dtype)
        if clip is not None:
            assert abs(float(opt.grad_norm) - norm) <= (U32 + 1e-12) * norm
    if dtype == torch.float32 and clip is None:                       # and torch's own AdamW from the same start
        qs = [torch.nn.Parameter(torch.as_tensor(np64(p), dtype=torch.float32).view(p.shape)) for p in make_params(sizes, dtype)]
        ref = torch.optim.AdamW(qs, lr=HYP["lr"], betas=HYP["betas"], eps=HYP["eps"], weight_decay=HYP["weight_decay"])
        hs = make_params(sizes, dtype)
        for _ in range(3):
            for q, h in zip(qs, hs):
                q.grad = h.grad.cpu()
                h.grad = h.grad * 0.7 + 0.1
            ref.step()
        for q, p in zip(qs, ps):           # three steps of at most 2 lr; relative errors of a few float32 roundings each
            assert float((q.detach() - p.detach().cpu()).abs().max() if p.numel() else 0.0) <= 3 * (64 * U32 * 2 * HYP["lr"] + 4 * U32 * float(q.detach().abs().max() if q.numel() else 0.0))


@gpu
@pytest.mark.parametrize("sizes", LISTS, ids=[f"{len(s)}x{s[0]}" for s in LISTS])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("clip", [None, 1.5])
def test_adamw8_matches_float64(sizes, dtype, clip):
    """codes and scales exactly (the kernel places values between codes in 64 bits), parameters to float32 roundings"""
    ps = make_params(sizes, dtype, gscale=1e-2)
    opt = optim.AdamW(ps, **HYP, state_bits=8, seed=77)
    before = [np64(p) for p in ps]
    state = [(np.zeros(p.numel()), np.zeros(p.numel())) for p in ps]
    for t in (1, 2, 3):
        gs = [np64(p.grad) for p in ps]
        norm = math.sqrt(sum(float((g ** 2).sum()) for g in gs))
        coef = 1.0 if clip is None else min(1.0, clip / (norm + 1e-6))
        opt.step(max_norm=clip)
        ms, vs = opt.state_values()
        for i, p in enumerate(ps):
            p1, m1, v1, em, ev, ep = reference_step(before[i], gs[i], *state[i], t, coef=coef, **HYP)
            h = random_bits(p.numel(), 77, t, i).astype(np.int64)
            s = opt.state[p]
            for key, x, signed, r, values in (("exp_avg", m1, True, h & 0xFFFF, ms[i]), ("exp_avg_sq", v1, False, h >> 16, vs[i])):
                codes, scales = store8(x, signed, r)
                np.testing.assert_array_equal(s[key + "_scale"].cpu().numpy(), scales)
                np.testing.assert_array_equal(s[key].cpu().numpy(), codes)
                np.testing.assert_array_equal(np64(values), load8(codes, scales, signed).astype(np.float32))
            got = np64(p)
            assert (np.abs(got - p1) <= ep + (half(dtype) * np.abs(p1) * 1.01 + tiny(dtype) if dtype != torch.float32 else 0)).all(), (i, t)
            before[i], state[i] = got, (np64(ms[i]), np64(vs[i]))
            p.grad = (p.grad.float() * 0.7 + 1e-3).to(dtype)


def tensor_form8(x, signed, bits):
    """store8 and its values as float64 tensor operations on the GPU (blocks of 256 throughout)"""
    top, low = (7, -6) if signed else (15, -14)
    b = x.abs().view(-1, 256)
    e = torch.clamp(torch.frexp(b.max(1).values)[1] - 1 - top, min=-126)
    k = torch.ldexp(torch.ones((), dtype=torch.float64, device=x.device), e)
    y = (b / k[:, None]).view(-1)
    ey = torch.clamp(torch.where(y > 0, torch.frexp(y)[1] - 1, low), min=low)
    code = torch.floor(torch.ldexp(y, 3 - ey) + (bits.double() + 0.5) / 65536.0).long() + (ey.long() - low) * 8
    code = code + 128 * (x < 0).long() if signed else torch.where(x > 0, torch.clamp(code, min=1), code)
    return code.to(torch.uint8), k.float()


def tensor_form8_values(code, k, signed):
    low = -6 if signed else -14
    c = torch.arange(256, device=code.device)
    e, man = (c & 127 if signed else c) >> 3, c & 7
    v = torch.where(e == 0, torch.ldexp(man.double(), torch.full_like(e, low - 3)), torch.ldexp(man.double() + 8.0, e - 1 + low - 3))
    v = torch.where(c >= 128, -v, v) if signed else v
    return v[code.long()] * k.double().repeat_interleave(256)


@gpu
@pytest.mark.parametrize("seed", [0, 1])
def test_adamw8_borders_fall_as_in_tensor_operations(seed):
    """Decimal fractions that lie exactly between up and down come up once in 10^7 values at b1 = 0.9: 2^26 elements, gradients with few
    bits so that they come up often, a first step and one on states of every code: the same codes as the float64 tensor form"""
    n = 1 << 26
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g = torch.randint(1, 4096, (n,), device="cuda", generator=gen).float() * (2.0 ** torch.randint(-20, -10, (n,), device="cuda", generator=gen))
    p = torch.nn.Parameter(torch.zeros(n, device="cuda")); p.grad = g
    opt = optim.AdamW([p], lr=0.0, state_bits=8, seed=seed)
    i = torch.arange(n, device="cuda")
    def mix(x):
        x = x ^ (x >> 17); x = (x * 0x743B8C43) & 0xFFFFFFFF
        x = x ^ (x >> 12); x = (x * 0xAB2209AB) & 0xFFFFFFFF
        return x ^ (x >> 15)
    m = v = torch.zeros(n, dtype=torch.float64, device="cuda")
    for t in (1, 2):
        opt.step()
        m = 0.9 * m + (1.0 - 0.9) * g.double(); v = 0.999 * v + (1.0 - 0.999) * g.double() * g.double()
        h = mix((i + mix(mix(mix(mix(seed) + t & 0xFFFFFFFF) + 0) + 0 & 0xFFFFFFFF)) & 0xFFFFFFFF)
        s = opt.state[p]
        for key, x, signed, r in (("exp_avg", m, True, h & 0xFFFF), ("exp_avg_sq", v, False, h >> 16)):
            code, k = tensor_form8(x, signed, r)
            assert int((code != s[key]).sum()) == 0 and torch.equal(k, s[key + "_scale"]), (key, t)
        m, v = tensor_form8_values(s["exp_avg"], s["exp_avg_scale"], True), tensor_form8_values(s["exp_avg_sq"], s["exp_avg_sq_scale"], False)
        p.grad = g = -g.flip(0)


@gpu
def test_adamw8_extreme_values():
    """zero blocks, single large and tiny values, non-finite gradients (their own element only), squares past float32's range"""
    g = torch.zeros(256 * 6)
    g[256:512] = torch.logspace(-30, 0, 256)                    # 30 decades in one block
    g[512] = 1e30; g[513:520] = 1.0                             # v beyond float32's range: held at its largest value
    g[768] = float("nan"); g[769] = float("inf"); g[770] = float("-inf"); g[771:1024] = 0.01
    g[1024:1280] = -1e-25                                       # scales below float32's normal range
    g[1280:1536] = 3.0
    p = torch.nn.Parameter(torch.ones(g.numel(), device="cuda")); p.grad = g.cuda()
    opt = optim.AdamW([p], **HYP, state_bits=8, seed=5)
    opt.step()
    x = g.double().numpy()
    with np.errstate(over="ignore", invalid="ignore"):
        m1, v1 = (1 - 0.9) * x, (1 - 0.999) * x * x
        v1 = np.where(np.isfinite(v1) & (v1 > np.finfo(np.float32).max), np.finfo(np.float32).max, v1)
    h = random_bits(g.numel(), 5, 1, 0).astype(np.int64)
    s = opt.state[p]
    for key, want, signed, r in (("exp_avg", m1, True, h & 0xFFFF), ("exp_avg_sq", v1, False, h >> 16)):
        codes, scales = store8(want, signed, r)
        np.testing.assert_array_equal(s[key + "_scale"].cpu().numpy(), scales)
        np.testing.assert_array_equal(s[key].cpu().numpy(), codes)
    out = p.detach().cpu()
    bad = torch.zeros(g.numel(), dtype=torch.bool); bad[768:771] = True
    assert torch.equal(torch.isnan(out), bad)
    m, v = opt.state_values()
    assert torch.equal(torch.isnan(m[0]).cpu(), bad) and torch.equal(torch.isnan(v[0]).cpu(), bad)
    assert abs(float(out[0]) - (1 - HYP["lr"] * HYP["weight_decay"])) <= U32           # no gradient: the decay alone
    # v > 0 is never lost, so that nothing jumps where the gradient stops (but at 1e30, whose v is held too small): after bias correction
    # m / sqrt(v) is at most 0.24 lr x (a quantum of m over the least r: 2 x 0.1 x 2^-16 / (0.7 x 0.032 x 2^-16) = 9), 10 lr allowed
    bad[512] = True
    p.grad = torch.zeros_like(p)
    for _ in range(5):
        q = p.detach().clone()
        opt.step()
        assert float((p.detach() - q)[~bad.cuda()].abs().max()) <= 10 * HYP["lr"]


@gpu
def test_adamw8_rounding_keeps_the_mean():
    """v decays by 0.1 % a step without gradients, far less than the distance of two codes (6 to 12 %): the mean over many elements
    follows 0.999^t.  Per element and step the variance is at most 0.001 x 2^-3 of v^2 (a move of 2^-3 v at most with probability
    0.001 v over its size): relative std over 500 steps < sqrt(500 / 8000) = 0.25, of the mean over 2^16 elements < 0.001."""
    n = 1 << 16
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    p.grad = (1.0 + torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)))
    opt = optim.AdamW([p], lr=0.0, state_bits=8, seed=3)
    opt.step()
    v0 = opt.state_values()[1][0].double()
    p.grad = torch.zeros_like(p)
    for _ in range(500):
        opt.step()
    v = opt.state_values()[1][0].double()
    assert abs(float(v.mean() / v0.mean()) / 0.999 ** 500 - 1) < 6 * 0.001
    assert bool((v > 0).all())


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_layouts_groups_and_missing_gradients(bits):
    """transposed parameters (states in their order), gradients of another order, several groups and types, a parameter that joins later"""
    a = torch.nn.Parameter(torch.randn(30, 20, device="cuda").t()); b = torch.nn.Parameter(torch.randn(40, device="cuda"))
    c = torch.nn.Parameter(torch.randn(50, device="cuda").bfloat16()); d = torch.nn.Parameter(torch.randn(8, device="cuda"))
    start = [t.detach().clone() for t in (a, b, c, d)]
    opt = optim.AdamW([{"params": [a, c], "lr": 1e-3}, {"params": [b, d], "weight_decay": 0.5, "betas": (0.8, 0.99)}], lr=1e-2, state_bits=bits, seed=1)
    a.grad = torch.randn(20, 30, device="cuda")                  # contiguous, the parameter is not
    a_grad = a.grad.clone()
    b.grad = torch.randn(40, device="cuda"); c.grad = torch.randn(50, device="cuda").bfloat16()
    va, vb = a._version, b._version
    opt.step()
    assert a._version > va and b._version > vb and torch.equal(d.detach(), start[3]) and not opt.state[d]
    assert torch.equal(a.grad, a_grad)
    for p, s, kw in ((a, start[0], dict(lr=1e-3, weight_decay=0.0, betas=(0.9, 0.999))), (b, start[1], dict(lr=1e-2, weight_decay=0.5, betas=(0.8, 0.99)))):
        p1, *_, ep = reference_step(np64(s), np64(p.grad), np.zeros(s.numel()), np.zeros(s.numel()), 1, eps=1e-8, **kw)
        assert (np.abs(np64(p) - p1) <= ep).all()
    m, _ = opt.state_values()
    assert m[0].stride() == a.stride()
    tol = U32 * 4 if bits == 32 else 2.0 ** -3
    assert bool(((m[0].double() - 0.1 * a.grad.double()).abs() <= tol * 0.1 * a.grad.double().abs() + 2.0 ** -16).all())
    d.grad = torch.ones(8, device="cuda")
    opt.step()                                                   # d's first step: its own bias correction
    p1, *_, ep = reference_step(np64(start[3]), np.ones(8), np.zeros(8), np.zeros(8), 1, lr=1e-2, weight_decay=0.5, betas=(0.8, 0.99), eps=1e-8)
    assert (np.abs(np64(d) - p1) <= ep).all() and opt.state[d]["step"] == 1 and opt.state[b]["step"] == 2


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_after_a_parameter_was_changed_underneath(bits):
    """``p.data`` of another order in memory (32 bits: the moments follow; 8: refused, their blocks do not), size, device or type, gradients left
    behind: nothing is launched, parameters, moments and counts stay"""
    w = torch.randn(6, 5, 4, device="cuda")
    a, b = torch.nn.Parameter(w.clone()), torch.nn.Parameter(w.clone())
    g = torch.randn(6, 5, 4, device="cuda")
    opts = [optim.AdamW([p], **HYP, state_bits=bits, seed=4) for p in (a, b)]
    for p, o in zip((a, b), opts):
        p.grad = g.clone()
        o.step()
    for order in ((2, 0, 1), (0, 1, 2)):                         # to an order of its own, and back
        inverse = [order.index(i) for i in range(3)]
        b.data = b.data.permute(order).contiguous().permute(inverse)
        assert b.is_contiguous() == (order == (0, 1, 2))
        if bits == 8 and order != (0, 1, 2):
            for call in (opts[1].step, opts[1].state_values, lambda: optim.AdamW([b], state_bits=8).load_state_dict(opts[1].state_dict())):
                with pytest.raises(ValueError):
                    call()
            continue
        for p, o in zip((a, b), opts):
            o.step(max_norm=1.0)
        assert torch.equal(a, b) and opts[0].state[a]["step"] == opts[1].state[b]["step"]
        for x, y in zip(opts[0].state_values(), opts[1].state_values()):
            assert torch.equal(x[0], y[0]) and y[0].stride() == b.stride()
    keep = b.detach().clone()
    before = {k: v.clone() if torch.is_tensor(v) else v for k, v in opts[1].state[b].items()}
    inner = torch.randn(6, 5, 8, device="cuda")
    for data in (torch.randn(7, 5, 4, device="cuda"), torch.randn(6, 5, 3, device="cuda"), inner[:, :, :4], inner[:1, :, :4].expand(6, 5, 4), b.data.cpu(), b.data.double(),
                 b.data.half()):
        c = torch.nn.Parameter(b.detach().clone())
        o = optim.AdamW([c], **HYP, state_bits=bits, seed=4)
        o.load_state_dict(opts[1].state_dict())
        c.grad = g.clone()
        saved = data.clone()
        c.data = data
        for kw in ({}, {"max_norm": 1.0}):
            with pytest.raises((ValueError, lib.HoicError)):
                o.step(**kw)
        assert torch.equal(data, saved) and o.state[c]["step"] == before["step"] and torch.equal(o.state[c]["exp_avg"], before["exp_avg"])
        if data.numel() != b.numel() and data.is_cuda:           # a gradient that fits, moments that do not
            c.grad = torch.ones_like(data)
            with pytest.raises(ValueError):
                o.step()
            if bits == 8:
                with pytest.raises(ValueError):
                    o.state_values()
    assert torch.equal(b.detach(), keep) and torch.equal(opts[1].state[b]["exp_avg"], before["exp_avg"])
    c = torch.nn.Parameter(torch.randn(5, 6, device="cuda").t())                # an order of its own through a saved state
    c.grad = torch.randn(6, 5, device="cuda")
    o = optim.AdamW([c], **HYP, state_bits=bits, seed=4)
    o.step()
    d = torch.nn.Parameter(c.detach().clone(memory_format=torch.preserve_format))
    d.grad = c.grad.clone()
    q = optim.AdamW([d], **HYP, state_bits=bits, seed=4)
    q.load_state_dict(copy.deepcopy(o.state_dict()))
    o.step(); q.step()
    assert d.stride() == c.stride() and torch.equal(c, d)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_resumes_from_its_state(bits):
    """state_dict / load_state_dict (also through torch.save) and deepcopy continue bit for bit; the moments keep their types"""
    import io
    ps = make_params([300, (7, 9), 1], torch.bfloat16)
    opt = optim.AdamW(ps, **HYP, state_bits=bits, seed=9)
    opt.step(); opt.step()
    buf = io.BytesIO()
    torch.save(opt.state_dict(), buf); buf.seek(0)
    sd = torch.load(buf, weights_only=True)
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p, q in zip(ps, qs):
        q.grad = p.grad.clone()
    other = optim.AdamW(qs, lr=1.0, state_bits=bits)
    other.load_state_dict(sd)
    assert other.param_groups[0]["lr"] == HYP["lr"] and other.param_groups[0]["seed"] == 9
    both = copy.deepcopy((ps, opt))
    for p, q in zip(ps, both[0]):
        q.grad = p.grad.clone()
    for o in (opt, other, both[1]):
        o.step(max_norm=1.0); o.step()
    for p, q, r in zip(ps, qs, both[0]):
        assert torch.equal(p, q) and torch.equal(p, r)
        for k, t in opt.state[p].items():
            assert (torch.equal(t, other.state[q][k]) and t.dtype == other.state[q][k].dtype) if isinstance(t, torch.Tensor) else t == other.state[q][k]
    if bits == 32:                                               # torch's own optimiser's state
        xs = make_params([300, (7, 9), 1], torch.float32)
        ref = torch.optim.AdamW(xs, **HYP); ref.step()
        ys = [torch.nn.Parameter(x.detach().clone()) for x in xs]
        mine = optim.AdamW(ys); mine.load_state_dict(ref.state_dict())
        for x, y in zip(xs, ys):
            y.grad = x.grad.clone()
            assert mine.state[y]["step"] == 1 and torch.equal(mine.state[y]["exp_avg"], ref.state[x]["exp_avg"])
        ref.step(); mine.step()
        for x, y in zip(xs, ys):
            assert float((x - y).abs().max()) <= 64 * U32 * 2 * HYP["lr"] + 4 * U32 * float(x.abs().max())
    with pytest.raises(ValueError):
        optim.AdamW(qs, state_bits=40 - bits).load_state_dict(sd)
    with pytest.raises(ValueError):
        optim.AdamW(qs[:2], state_bits=bits).load_state_dict(sd)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_skips_a_step_whose_norm_is_not_finite(bits):
    ps = make_params([500, 60], torch.float32)
    opt = optim.AdamW(ps, **HYP, state_bits=bits)
    opt.step(max_norm=1.0)
    held = copy.deepcopy([(p.detach(), {k: v for k, v in opt.state[p].items() if k != "step"}) for p in ps])
    for value in (float("inf"), float("nan")):
        ps[1].grad[3] = value
        opt.step(max_norm=1.0)
        assert not math.isfinite(float(opt.grad_norm))
        for p, (q, s) in zip(ps, held):
            assert torch.equal(p.detach(), q) and all(torch.equal(opt.state[p][k], v) for k, v in s.items())
    ps[1].grad[3] = 0.0
    opt.step(max_norm=1.0)
    assert all(bool(torch.isfinite(p).all()) for p in ps) and not torch.equal(ps[0].detach(), held[0][0])


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [60, 5 << 20])
def test_adamw_skips_a_step_whose_norm_is_past_float32(bits, n):
    """gradients of float32's largest values: the norm is finite in 64 bits and infinite in the float32 that the caller sees -- the step is
    skipped like any whose ``grad_norm`` is not finite (joined in the step's launch, and before it in a large list)"""
    p = torch.nn.Parameter(torch.ones(n, device="cuda"))
    p.grad = torch.full((n,), 3.0e38, device="cuda")
    opt = optim.AdamW([p], **HYP, state_bits=bits)
    opt.step(max_norm=1.0)
    assert math.isinf(float(opt.grad_norm)) and bool((p == 1).all()) and not bool(opt.state[p]["exp_avg"].any()) and not bool(opt.state[p]["exp_avg_sq"].any())
    p.grad[1:] = 0.0
    opt.step(max_norm=1.0)
    assert abs(float(opt.grad_norm) / 3.0e38 - 1) <= 2 * U32 and float(p.detach()[0]) < 1.0


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_captured_and_replayed(bits):
    """capturable: a captured step, replayed with other gradients and another lr and eager work between, is the eager optimiser's;
    two optimisers captured into two graphs and replayed in turn do not disturb one another"""
    sizes = [1000, (33, 7)] + [5] * 60
    lr = torch.full((1,), 3e-3, device="cuda")
    pairs = []
    for seed in (0, 10):
        ps, qs = make_params(sizes, torch.float32, seed), make_params(sizes, torch.float32, seed)
        cap = optim.AdamW(ps, **{**HYP, "lr": lr}, state_bits=bits, capturable=True, seed=seed)
        eager = optim.AdamW(qs, **HYP, state_bits=bits, seed=seed)
        cap.step(max_norm=2.0); eager.step(max_norm=2.0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cap.step(max_norm=2.0)
        pairs.append((ps, qs, cap, eager, graph))
    for rep in range(4):
        lr.fill_(3e-3 * (1 + rep))
        for k, (ps, qs, cap, eager, graph) in enumerate(pairs):
            for p, q in zip(ps, qs):
                p.grad.mul_(0.5).add_(0.01 * (k + 1)); q.grad.copy_(p.grad)
            graph.replay()
            eager.param_groups[0]["lr"] = float(lr)
            eager.step(max_norm=2.0)
        torch.cuda.synchronize()
        for ps, qs, cap, eager, graph in pairs:
            for p, q in zip(ps, qs):
                for key in set(eager.state[q]) - {"step"}:
                    assert torch.equal(cap.state[p][key], eager.state[q][key]), (rep, key)
                # the step size's float32 lr is 2^-24 off the double's, on top of the device's pow: a rounding or two of the step
                assert float((p - q).abs().max()) <= (rep + 2) * (8 * U32 * 2 * 1.2e-2 + 2 * U32 * float(q.abs().max()))
                assert int(cap.state[p]["step"]) == eager.state[q]["step"] == rep + 2
    bad = optim.AdamW(make_params([10], torch.float32), state_bits=bits)
    bad.step()
    fresh = optim.AdamW(make_params([10], torch.float32), state_bits=bits, capturable=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(lib.HoicError, match="capturable"):
            bad.step()
        with pytest.raises(lib.HoicError, match="eager step"):
            fresh.step()


@gpu
def test_adamw_offsets_past_32_bits():
    """a tensor of more than 2^32 elements: its last block against the reference (the random numbers' upper half counts)"""
    n = (1 << 32) + 300
    if torch.cuda.get_device_properties(0).total_memory < 120 << 30:
        pytest.skip("needs 120 GB")
    p = torch.nn.Parameter(torch.ones(n, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    tail = tensor_list([300], torch.bfloat16, 4)[0]
    p.grad[-300:] = tail
    opt = optim.AdamW([p], **HYP, state_bits=8, seed=2)
    opt.step(max_norm=1e9)
    g = np64(tail)
    h = random_bits(300, 2, 1, 0, first=1 << 32).astype(np.int64)
    codes, scales = store8((1 - 0.9) * g, True, h & 0xFFFF)
    s = opt.state[p]
    np.testing.assert_array_equal(s["exp_avg"][-300:].cpu().numpy(), codes)
    np.testing.assert_array_equal(s["exp_avg_scale"][-2:].cpu().numpy(), scales)
    assert not s["exp_avg"][:-300].any() and not s["exp_avg_sq"][:-300].any()
    norm = math.sqrt(float((g ** 2).sum()))
    assert abs(float(opt.grad_norm) - norm) <= (U32 + 1e-12) * norm


def test_adamw_refusals():
    with pytest.raises(lib.HoicError):
        optim.AdamW([torch.nn.Parameter(torch.zeros(3))])
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(weight_decay=-1.0), dict(state_bits=16), dict(lr=torch.zeros(1)),
               dict(lr=math.nan)):
        with pytest.raises(ValueError):
            optim.AdamW([torch.nn.Parameter(torch.zeros(3))], **kw)
    import ctypes as C
    L = lib.load()
    fields = dict(type=0, state_bits=32, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, weight_decay=0.0, d_lr=0, d_consts=0, d_norm_buf=0, d_norm=0, bound=0.0, norm_parts=0, seed=0,
                  reserved=0)
    args = lambda **kw: lib.ADAMW_ARGS.pack(*(fields | kw).values())
    row = lambda **kw: (C.c_int64 * 10)(*[kw.get(k, d) for k, d in zip(("p", "g", "m", "v", "ms", "vs", "n", "step", "d_step", "ordinal"), (8, 8, 8, 8, 0, 0, 4, 1, 0, 0))])
    for a, t in ((args(type=3), row()), (args(state_bits=16), row()), (args(b1=1.0), row()), (args(eps=-1.0), row()), (args(), row(p=0)), (args(), row(g=0)), (args(), row(m=0)),
                 (args(), row(v=0)), (args(), row(n=-1)), (args(), row(step=0)), (args(state_bits=8), row()), (args(d_consts=8), row()), (args(), row(n=1 << 60)),
                 (args(d_norm_buf=8, d_norm=8), row()), (args(d_norm_buf=8, norm_parts=1), row()), (args(d_norm_buf=8, d_norm=8, norm_parts=1, bound=-1.0), row())):
        assert L.hoic_adamw(t, 1, a, None) == -1
    assert L.hoic_adamw(None, 1, args(), None) == -1 and L.hoic_adamw(row(), 1, None, None) == -1 and L.hoic_adamw(row(), -1, args(), None) == -1
    assert L.hoic_adamw_values(row(), 1, None) == -1 and L.hoic_adamw_values(None, 1, None) == -1


@gpu
def test_adamw_refuses_what_it_cannot_hold():
    for t in (torch.zeros(3, dtype=torch.float64, device="cuda"), torch.zeros(8, device="cuda")[::2], torch.zeros(1, device="cuda").expand(4)):
        with pytest.raises(ValueError):
            optim.AdamW([torch.nn.Parameter(t)])
    p = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    opt = optim.AdamW([p])
    with pytest.raises(ValueError):
        opt.step(max_norm=-1.0)
    assert not opt.state[p]
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(3, device="cuda"))], state_bits=8))
    with pytest.raises(ValueError, match="same memory"):
        optim.AdamW([torch.nn.Parameter(p.data), torch.nn.Parameter(p.data)])
    with pytest.raises(ValueError, match="same memory"):
        opt.add_param_group(dict(params=[torch.nn.Parameter(p.data)]))


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_hooks_closure_scheduler_and_profiler(bits):
    """what a torch optimiser offers around its step keeps working"""
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    opt = optim.AdamW([p], lr=1e-2, state_bits=bits)
    sched = torch.optim.lr_scheduler.StepLR(opt, 1, 0.5)
    seen = []
    opt.register_step_pre_hook(lambda o, a, k: seen.append("pre")); opt.register_step_post_hook(lambda o, a, k: seen.append("post"))
    def closure():
        opt.zero_grad()
        loss = (p ** 2).sum()
        loss.backward()
        return loss
    assert float(opt.step(closure, max_norm=1.0).detach()) == 300.0 and seen == ["pre", "post"] and float(opt.grad_norm) > 0
    sched.step()
    assert opt.param_groups[0]["lr"] == 5e-3
    with torch.autograd.profiler.profile():
        opt.step(closure)
    assert seen == ["pre", "post"] * 2 and opt.grad_norm is None and opt.state[p]["step"] == 2
    opt.zero_grad(set_to_none=True)
    before = p.detach().clone()
    opt.step(max_norm=1.0)                                       # nothing to do
    assert torch.equal(before, p.detach()) and float(opt.grad_norm) == 0 and opt.state[p]["step"] == 2


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_unaligned_views_and_a_side_stream(bits):
    """parameters and gradients that are views at odd offsets of one buffer, stepped on another stream: the same bits as aligned copies"""
    for dt in (torch.float32, torch.bfloat16):
        flat, grad = tensor_list([20000], dt, 1)[0], tensor_list([20000], dt, 2)[0]
        cuts = [(1, 4098), (4099, 9000), (9001, 9002), (9003, 19999)]
        ps = [torch.nn.Parameter(flat[i:j]) for i, j in cuts]; qs = [torch.nn.Parameter(flat[i:j].clone()) for i, j in cuts]
        for p, q, (i, j) in zip(ps, qs, cuts):
            p.grad, q.grad = grad[i:j], grad[i:j].clone()
        edges = flat[[0, 4098, 9000, 9002, 19999]].clone()
        a, b = optim.AdamW(ps, **HYP, state_bits=bits), optim.AdamW(qs, **HYP, state_bits=bits)
        st = torch.cuda.Stream(); st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            a.step(max_norm=1.0); a.step()
        torch.cuda.current_stream().wait_stream(st)
        b.step(max_norm=1.0); b.step()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and torch.equal(flat[[0, 4098, 9000, 9002, 19999]], edges)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_two_learners_on_two_streams(bits):
    """loss -> gradients -> clipping -> step -> values of two learners, interleaved launch by launch on two streams, and one after the other on
    one: the same bits (nothing is shared between calls)"""
    def learner(seed):
        x = loss_case(20000 if seed else 900, 32, mask=0.3, seed=seed, device="cuda")
        mu, s = torch.nn.Parameter(x["mean"].nan_to_num(0.0)), torch.nn.Parameter(x["log_std"].clone())
        return x, mu, s, optim.AdamW([mu, s], lr=1e-3, weight_decay=0.01, state_bits=bits, seed=seed)

    def update(x, mu, s, opt):
        o = rl.clipped_policy_loss_grad(**{**x, "mean": mu.detach(), "log_std": s.detach()}, kl_coef=0.2, weight=100.0)
        mu.grad, s.grad = o.d_mean, o.d_log_std
        norm = optim.clip_grad_norm_([mu, s], 0.7)
        opt.step(max_norm=0.5)
        return [o.loss, o.info, norm, opt.grad_norm, *sum(opt.state_values(), [])]

    want = []
    for seed in (0, 1):
        w = learner(seed)
        want.append([[t.clone() for t in update(*w)] for _ in range(6)] + [[w[1].detach(), w[2].detach()]])
    streams, both = [torch.cuda.Stream(), torch.cuda.Stream()], [learner(0), learner(1)]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(6):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append([t.clone() for t in update(*both[k])])
    torch.cuda.synchronize()
    for k in (0, 1):
        got[k].append([both[k][1].detach(), both[k][2].detach()])
        for a, b in zip(got[k], want[k]):
            for x, y in zip(a, b):
                assert torch.equal(x, y)
        assert bool(torch.isfinite(got[k][-1][0]).all())


def test_rounding_bits_are_uniform():
    """chi-square of the hash's two halves in 256 cells (255 degrees of freedom: mean 255, std 22.6; 6 std allowed), and the
    correlation of neighbours, halves, steps and tensors (2^18 samples: std 2^-9; 6 std allowed)"""
    n = 1 << 18
    u = lambda step, o: random_bits(n, 123, step, o).astype(np.int64)
    h, k, l = u(10, 0), u(11, 0), u(10, 1)
    for x in (h & 0xFFFF, h >> 16):
        c = np.bincount(x >> 8, minlength=256)
        assert ((c - n / 256) ** 2 / (n / 256)).sum() < 255 + 6 * 22.6
    f = lambda x: (x & 0xFFFF) / 65536.0 - 0.5
    s = lambda x: (x >> 16) / 65536.0 - 0.5
    for a, b in ((f(h)[1:], f(h)[:-1]), (f(h), s(h)), (f(h), f(k)), (s(h), s(k)), (f(h), f(l)), (s(h), f(l)), (f(h)[256:], f(h)[:-256])):
        assert abs(float((a * b).mean()) * 12) < 6 * 2.0 ** -9


# ================================================================================================ together: the learner's update
def learner_config(hsize, **kw):
    from hoic_amd.config import Config, release_cfg_dict
    return Config("box_future5_light_add_geom", cfg_dict={**release_cfg_dict("box"), "policy_hsize": hsize, "value_hsize": hsize, "fix_std": False, **kw})


def learner_batch(T, N, D, A, dtype, dev, seed=5):
    from types import SimpleNamespace
    g = torch.Generator().manual_seed(seed)
    mk = lambda *sh: torch.randn(*sh, generator=g)
    b = dict(states=torch.clamp(mk(T, N, D), -5, 5), actions=mk(T, N, A) * 0.1, rewards=torch.rand(T, N, generator=g), masks=(torch.rand(T, N, generator=g) > 0.05).float(),
             next_values=torch.zeros(N))
    return SimpleNamespace(valid=None, **{k: v.to(dev, dtype) for k, v in b.items()})


def test_learner_kl_update_is_the_formula():
    """PPOLearner on the CPU in float64 with kl_coef: five epochs against a loop written out here, to rounding"""
    from hoic_amd.agent import PPOLearner
    cfg = learner_config([24, 16], kl_coef=0.7, policy_lr=1e-2)
    torch.manual_seed(3)
    L = PPOLearner(cfg, 20, 5, "cpu", torch.float64)
    assert L.kl_coef == 0.7 and type(L.optimizer_policy) is torch.optim.Adam
    net = copy.deepcopy(L.policy_net)
    b = learner_batch(4, 50, 20, 5, torch.float64, "cpu")
    adv = torch.randn(200, 1, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
    states, actions = b.states.reshape(200, 20), b.actions.reshape(200, 5)
    L.optimize(states, actions, adv, torch.zeros(200, 1, dtype=torch.float64))
    opt = torch.optim.Adam(net.parameters(), lr=1e-2)
    logp = lambda mu, s: (-(actions - mu) ** 2 / (2 * torch.exp(2 * s)) - s - 0.5 * math.log(2 * math.pi)).sum(1, keepdim=True)
    mu0, s0 = (t.detach().clone() for t in net(states))
    for ep in range(5):
        mu, s = net(states)
        r = torch.exp(logp(mu, s) - logp(mu0, s0))
        kl = (s - s0 + (torch.exp(2 * s0) + (mu - mu0) ** 2) / (2 * torch.exp(2 * s)) - 0.5).sum(1, keepdim=True)
        loss = (-torch.min(r * adv, torch.clamp(r, 0.8, 1.2) * adv) + 0.7 * kl).mean()
        opt.zero_grad(); loss.backward()
        if ep == 0:
            torch.nn.utils.clip_grad_norm_(net.parameters(), 40)
        opt.step()
    for p, q in zip(L.policy_net.parameters(), net.parameters()):
        assert float((p - q).abs().max()) < 1e-10             # five Adam steps of lr 1e-2: rounding of 1e-16 grows by 1 / (eps-like small gradients), 1e6 allowed
    assert abs(L.last_losses[1] - float(loss)) < 1e-12


def test_learner_optimizers_follow_the_config():
    from hoic_amd.agent import PPOLearner
    L = PPOLearner(learner_config([8], policy_optimizer="AdamW", value_optimizer="Adam", policy_weightdecay=0.1), 6, 2, "cpu")
    assert type(L.optimizer_policy) is torch.optim.AdamW and type(L.optimizer_value) is torch.optim.Adam and L.optimizer_policy.param_groups[0]["weight_decay"] == 0.1
    with pytest.raises(lib.HoicError):
        PPOLearner(learner_config([8], policy_optimizer="AdamW8bit"), 6, 2, "cpu")


@gpu
@pytest.mark.parametrize("update_dtype,streams", [("f16x3", 3), ("f16x3", 1), ("f32", 3), ("bf16", 3)])
def test_learner_update_with_kl_adamw_and_clipping(update_dtype, streams):
    """loss with KL -> gradients -> norm and clipping -> AdamW in a learner's update (five epochs, both networks), against the same update
    in float64 with torch's AdamW: as close as the float32 library path is (Adam divides rounding noise by its own size: any two
    float32 computations differ there); with 8-bit moments within a quarter of the way moved (a code is 1/8 of its value
    at most: 20 % of a step); the same bits in two runs."""
    from hoic_amd.agent import PPOLearner
    dev = torch.device("cuda")

    def run(ud, optimizer, dtype=torch.float32):
        torch.manual_seed(0)
        cfg = learner_config([512, 256, 256], kl_coef=0.5, policy_optimizer=optimizer, value_optimizer=optimizer, policy_weightdecay=0.01, value_weightdecay=0.01)
        # (float64 networks need the optimiser of float64 parameters: made before the first step)
        L = PPOLearner(cfg, 617, 32, dev, update_dtype=ud, strict_reference=False, update_streams=streams)
        if dtype == torch.float64 or optimizer == "torch":
            for n, lr in (("policy", cfg.policy_lr), ("value", cfg.value_lr)):
                getattr(L, n + "_net").to(dtype)
                setattr(L, "optimizer_" + n, torch.optim.AdamW(getattr(L, n + "_net").parameters(), lr=lr, weight_decay=0.01))
        start = {n: [p.detach().double().clone() for p in getattr(L, n + "_net").parameters()] for n in ("policy", "value")}
        L.update_params(learner_batch(16, 256, 617, 32, dtype, dev))
        return {n: [p.detach().double() for p in getattr(L, n + "_net").parameters()] for n in ("policy", "value")}, start, L

    dist = lambda a, b: math.sqrt(sum(float(((x - y) ** 2).sum()) for x, y in zip(a, b)))
    ref, start, L64 = run("f32", "torch", torch.float64)
    lib32 = run("f32", "torch")[0]
    got, _, L = run(update_dtype, "AdamW")
    again = run(update_dtype, "AdamW")[0]
    low, _, L8 = run(update_dtype, "AdamW8bit")
    assert type(L.optimizer_policy) is optim.AdamW and L8.optimizer_policy.defaults["state_bits"] == 8
    assert float(L.optimizer_policy.grad_norm) > 0 and all(L.optimizer_policy.state[p]["step"] == 5 for p in L.policy_net.parameters())
    for n in ("policy", "value"):
        moved = dist(ref[n], start[n])
        assert moved > 0
        if update_dtype != "bf16":
            assert dist(got[n], ref[n]) <= 1.5 * dist(lib32[n], ref[n]) + 1e-3 * moved, n
            assert dist(low[n], ref[n]) <= 0.25 * moved, n
            assert all(torch.equal(x, y) for x, y in zip(got[n], again[n]))
        else:                    # bfloat16 products: 2^-8 of a gradient and sign changes of small ones; the update's direction stays
            assert dist(got[n], ref[n]) <= 0.5 * moved, n
    if update_dtype != "bf16":
        assert abs(L.last_losses[1] - L64.last_losses[1]) < 1e-4 * abs(L64.last_losses[1]) + 1e-6


@gpu
def test_learner_kl_holds_the_policy_back():
    """the KL term's gradient reaches the networks: a large kl_coef leaves the policy nearer to where it was"""
    from hoic_amd.agent import PPOLearner
    moved = []
    for kl in (0.0, 100.0):
        torch.manual_seed(0)
        L = PPOLearner(learner_config([512, 256, 256], kl_coef=kl, policy_lr=1e-3), 617, 32, torch.device("cuda"), update_dtype="f16x3")
        b = learner_batch(16, 256, 617, 32, torch.float32, "cuda")
        with torch.no_grad():
            before = L.policy_net(b.states.reshape(-1, 617))[0]
        L.update_params(b)
        with torch.no_grad():
            moved.append(float((L.policy_net(b.states.reshape(-1, 617))[0] - before).pow(2).mean()))
    assert moved[1] < moved[0]


@gpu
def test_train_script_with_the_new_options(tmp_path):
    """scripts/train_hand_mimic.py --optimizer / --kl_coef: two iterations each way, checkpoint"""
    import importlib.util
    import os
    from conftest import ROOT
    spec = importlib.util.spec_from_file_location("train_hand_mimic", os.path.join(ROOT, "scripts", "train_hand_mimic.py"))
    mod = importlib.util.module_from_spec(spec); spec.loader.exec_module(mod)
    base = ["--cfg", "box_future5_light_add_geom", "--num_threads", "16", "--no_log", "--num_epoch", "2", "--base_dir", str(tmp_path)]
    for more, bits in ((["--n_envs", "128", "--optimizer", "AdamW8bit", "--kl_coef", "0.2"], 8), (["--sample_mode", "episodes", "--optimizer", "AdamW"], 32)):
        agent = mod.main(base + more)
        assert type(agent.optimizer_policy) is optim.AdamW and agent.optimizer_value.defaults["state_bits"] == bits
        assert agent.learner.kl_coef == (0.2 if bits == 8 else 0.0) and agent.epoch == 1
        assert all(bool(torch.isfinite(p).all()) for p in agent.policy_net.parameters())
        assert agent.optimizer_policy.param_groups[0]["lr"] == float(agent.cfg.adp_policy_lr)
        agent.save_checkpoint(1)
        agent.env.close()
