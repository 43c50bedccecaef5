"""Calls of the learning operators (hoic_amd.rl, hoic_amd.optim) that their documentation allows or has to refuse, beside tests/test_learn.py: what
must reach no kernel is tested on the CPU, with the entry points replaced by recorders."""
import copy
import math

import numpy as np
import pytest
import torch

import test_learn as T
from hoic_amd import lib, optim, rl

gpu = pytest.mark.gpu
U32 = T.U32


class Recorder:
    """the library with every entry point a recorder of its calls; the gradient lists' sizes are the real ones"""

    def __init__(self):
        self.calls, self.real = [], lib.load()

    def hoic_grad_norm_parts(self, sizes, n):
        return self.real.hoic_grad_norm_parts(sizes, n)

    def __getattr__(self, name):
        return lambda *args: self.calls.append((name, args)) or 0


class NoLaunch:
    def __init__(self, dev):
        pass

    def __enter__(self):
        return 0

    def __exit__(self, *exc):
        pass


@pytest.fixture
def recorder(monkeypatch):
    """optim on CPU tensors that pass for tensors of cuda:0"""
    r = Recorder()
    monkeypatch.setattr(lib, "load", lambda: r)
    monkeypatch.setattr(lib, "Launch", NoLaunch)
    monkeypatch.setattr(optim, "_check", lambda t, what: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    return r


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("stepped", [False, True])
def test_adamw_cut_or_expanded_parameters_reach_no_kernel(recorder, bits, stepped):
    """``p.data`` replaced by a view whose elements do not fill their memory, the gradient a view of the same strides: a kernel that takes the
    elements in a row would write its neighbours (a cut view) or past the allocation (an expanded one)"""
    cut = lambda: torch.randn(6, 8)[:, :4]
    views = [(cut(), cut()), (torch.randn(1, 4).expand(6, 4), torch.randn(1, 4).expand(6, 4)), (torch.randn(6, 1).expand(6, 4), torch.randn(6, 1).expand(6, 4)),
             (torch.randn(48)[::2].view(6, 4), torch.randn(48)[::2].view(6, 4)), (torch.randn(8, 6).t()[:, ::2], torch.randn(8, 6).t()[:, ::2])]
    for data, grad in views:
        p = torch.nn.Parameter(torch.zeros(6, 4)); p.grad = torch.ones(6, 4)
        opt = optim.AdamW([p], state_bits=bits)
        if stepped:
            opt.step()
            assert [name for name, _ in recorder.calls] == ["hoic_adamw"]
            recorder.calls.clear()
        before = {k: v.clone() if torch.is_tensor(v) else v for k, v in opt.state[p].items()} if stepped else {}
        keep = data.clone()
        p.grad = None
        p.data = data
        p.grad = grad
        for kw in ({}, {"max_norm": 1.0}):
            with pytest.raises(ValueError, match="fill their memory"):
                opt.step(**kw)
            assert not recorder.calls and torch.equal(data, keep)
        state = opt.state[p]
        assert state.keys() == before.keys() and all(torch.equal(state[k], v) if torch.is_tensor(v) else state[k] == v for k, v in before.items())
    # a gradient of the parameter's strides and number of elements, but of another shape
    p = torch.nn.Parameter(torch.randn(3, 2))
    p.grad = torch.zeros(16).as_strided((3, 2), (1, 2))
    opt = optim.AdamW([p], state_bits=bits)
    p.data = torch.randn(3, 2).t()
    with pytest.raises(ValueError, match="another shape"):
        opt.step()
    assert not recorder.calls


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_dense_parameters_of_any_order_reach_the_kernel(recorder, bits):
    """views that fill one stretch of memory are taken as they are, a gradient of another order in a copy of the parameter's"""
    base, gbase = torch.randn(40), torch.randn(40)
    p = torch.nn.Parameter(base[7:31].view(4, 6).t()); p.grad = gbase[5:29].view(4, 6).t()
    optim.AdamW([p], state_bits=bits).step()
    (name, (rows, n, _, _)), = recorder.calls
    row = np.frombuffer(rows, np.int64)
    assert name == "hoic_adamw" and n == 1 and row[0] == p.data_ptr() and row[1] == p.grad.data_ptr() and row[6] == 24
    recorder.calls.clear()
    p.grad = torch.randn(6, 4)
    optim.AdamW([p], state_bits=bits).step()
    (name, (rows, n, _, _)), = recorder.calls
    assert np.frombuffer(rows, np.int64)[1] != p.grad.data_ptr()


@pytest.mark.parametrize("stepped", [False, True])
def test_adamw_refuses_options_that_it_does_not_have(recorder, stepped):
    """a group of torch's optimisers that maximises, keeps maxima or couples its weight decay is not taken over in silence, with a state or
    before the first step; one without them is, with its moments"""
    def foreign(cls, **kw):
        q = torch.nn.Parameter(torch.randn(5, 3))
        o = cls([q], lr=0.25, **kw)
        if stepped:
            q.grad = torch.randn(5, 3)
            o.step()
        return o.state_dict()

    p = torch.nn.Parameter(torch.randn(5, 3))
    opt = optim.AdamW([p], lr=0.5)
    for cls, kw, word in ((torch.optim.AdamW, dict(maximize=True), "maximize"), (torch.optim.Adam, dict(maximize=True), "maximize"),
                          (torch.optim.AdamW, dict(amsgrad=True), "amsgrad"), (torch.optim.Adam, dict(weight_decay=0.1), "decoupled")):
        with pytest.raises(ValueError, match=word):
            opt.load_state_dict(foreign(cls, **kw))
        assert opt.param_groups[0]["lr"] == 0.5 and not opt.state.get(p)
        group = {k: v for k, v in kw.items()} | ({"decoupled_weight_decay": False} if word == "decoupled" else {})
        with pytest.raises(ValueError, match=word):
            opt.add_param_group(dict(params=[torch.nn.Parameter(torch.randn(2))], **group))
    for cls, kw in ((torch.optim.AdamW, dict(weight_decay=0.1)), (torch.optim.Adam, {})):
        sd = foreign(cls, **kw)
        opt.load_state_dict(sd)
        assert opt.param_groups[0]["lr"] == 0.25 and opt.param_groups[0]["weight_decay"] == kw.get("weight_decay", 0.0)
        if stepped:
            assert opt.state[p]["step"] == 1 and torch.equal(opt.state[p]["exp_avg"], sd["state"][0]["exp_avg"])
    opt.load_state_dict(copy.deepcopy(opt.state_dict()))


@pytest.mark.parametrize("mean", [torch.float32, torch.bfloat16])
def test_policy_loss_makes_gradients_only_for_a_backward_call(monkeypatch, mean):
    """a value under no_grad, or of tensors that require no gradient, is a pass without gradients, whether or not leaves stand behind it"""
    asked = []

    def launch(x, kl_coef, weight, grad, upstream=None, count=None, want_count=False):
        asked.append((grad, want_count))
        made = lambda t: torch.zeros_like(t) if grad else None
        return torch.zeros(()), torch.zeros(4), torch.ones(1, dtype=torch.float64) if want_count else None, made(x[0]), made(x[1]), None

    monkeypatch.setattr(rl, "_on_kernel", lambda t: True)
    monkeypatch.setattr(rl, "_policy_loss_launch", launch)
    x = T.loss_case(7, 3, mean={torch.float32: "f32", torch.bfloat16: "bf16"}[mean])
    direct = mean == torch.float32                    # (gradients of 16-bit means are made in the backward call, which needs the count)
    for leaves in ((), ("mean",), ("log_std",), ("mean", "log_std")):
        y = {**x, **{k: x[k].detach().requires_grad_() for k in leaves}}
        with torch.no_grad():
            assert not rl.clipped_policy_loss(**y, kl_coef=0.3).loss.requires_grad
        assert asked.pop() == (False, False) and not asked
        p = rl.clipped_policy_loss(**y, kl_coef=0.3)
        assert p.loss.requires_grad == bool(leaves)
        assert asked.pop() == ((direct, not direct) if leaves else (False, False)) and not asked


def test_policy_loss_tensor_form_is_differentiable_in_the_policy_alone():
    """actions, advantages (a value network's, say), old log-probabilities and the reference get no gradient on the CPU either"""
    others = ("actions", "advantages", "fixed_log_probs", "ref_mean", "ref_log_std")
    x = {k: v.double() if v is not None and v.dtype != torch.bool else v for k, v in T.loss_case(9, 4, seed=3).items()}
    want = T.loss_reference(x, kl_coef=0.3)
    y = {k: v.detach().requires_grad_() if k != "valid" else v for k, v in x.items()}
    rl.clipped_policy_loss(**y, kl_coef=0.3).loss.backward()
    assert all(y[k].grad is None for k in others)
    for k in ("mean", "log_std"):
        torch.testing.assert_close(y[k].grad, want["d_" + k], rtol=1e-12, atol=1e-13)
    z = {k: v.detach().requires_grad_(k in others) if k != "valid" else v for k, v in x.items()}
    assert not rl.clipped_policy_loss(**z, kl_coef=0.3).loss.requires_grad


def test_adamw_checks_every_group_before_the_first_launch(recorder):
    """a learning rate that the second group cannot use: nothing is launched, no step counted, so that the corrected call takes one step"""
    ps = [torch.nn.Parameter(torch.randn(4)) for _ in range(2)]
    for p in ps:
        p.grad = torch.randn(4)
    opt = optim.AdamW([dict(params=[p]) for p in ps])
    for lr in (torch.tensor(0.1), torch.zeros(2), torch.tensor(0.1, dtype=torch.float64)):
        opt.param_groups[1]["lr"] = lr
        for kw in ({}, {"max_norm": 1.0}):
            with pytest.raises(ValueError, match="lr"):
                opt.step(**kw)
            assert not recorder.calls
    opt.param_groups[1]["lr"] = 0.1
    opt.step()
    assert [name for name, _ in recorder.calls] == ["hoic_adamw"] * 2 and all(opt.state[p]["step"] == 1 for p in ps)


def test_adamw_refuses_parameters_that_overlap_in_any_group(recorder):
    """views that share some elements, in one group or in two, of one type or of two: an element would be stepped twice; neighbours are taken"""
    flat = torch.randn(64)
    make = lambda a, b, dtype=torch.float32: torch.nn.Parameter(flat[a:b].view(dtype))
    for first, second in (((0, 8), (7, 12)), ((7, 12), (0, 8)), ((0, 8), (0, 8)), ((0, 32), (4, 5)), ((4, 5), (0, 32))):
        for dtype in (torch.float32, torch.bfloat16):
            with pytest.raises(ValueError, match="same memory"):
                optim.AdamW([make(*first), make(*second, dtype)])
            opt = optim.AdamW([make(*first)])
            with pytest.raises(ValueError, match="same memory"):
                opt.add_param_group(dict(params=make(*second, dtype)))
            assert len(opt.param_groups) == 1
    opt = optim.AdamW([make(8, 16), make(0, 8), make(8, 8)])
    opt.add_param_group(dict(params=[make(16, 20, torch.bfloat16), make(16, 16)]))


@gpu
@pytest.mark.parametrize("n", [60, 5 << 20])
def test_clipping_by_a_norm_past_float32(n):
    """gradients whose norm float32 cannot hold: the norm that is shown is infinite, and the factor is that norm's, 0, as torch's own clipping
    gives; a norm just inside the range still gives its quotient (lists joined by the scaling launch and in front of it)"""
    for parts in (1, min(n, 300)):
        g = torch.full((n // parts * parts,), 3e38, device="cuda")
        ps = [torch.nn.Parameter(torch.empty_like(x)) for x in g.split(n // parts)]
        for p, x in zip(ps, g.split(n // parts)):
            p.grad = x
        assert math.isinf(float(optim.clip_grad_norm_(ps, 40.0))) and not bool(g.any())
        g.zero_()
        g[::g.numel() // 4][:4] = -1.5e38               # norm 3e38
        norm = float(optim.clip_grad_norm_(ps, 3e37))
        assert abs(norm / 3e38 - 1) <= 4 * U32 and bool(torch.isfinite(g).all())
        # the value 1.5e38 (half a unit off), the factor 0.1 and the product: three roundings
        assert bool(((g[::g.numel() // 4][:4].double() / -1.5e37 - 1).abs() <= 3.01 * U32).all()) and int((g != 0).sum()) == 4


def exact_pow2(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def exact_place8(x, signed, r16):
    """float64 values in whole blocks -> (place on the ladder with the random part, in codes: its whole part is the code without sign; scales), every
    power of two from its bits"""
    top, low = (7, -6) if signed else (15, -14)
    b = x.abs().view(-1, 256)
    e = torch.clamp(torch.frexp(b.max(1).values)[1] - 1 - top, min=-126)
    e = torch.where(b.max(1).values > 0, e, torch.full_like(e, -126))
    y = (b * exact_pow2(-e)[:, None]).view(-1)
    ey = torch.clamp(torch.where(y > 0, torch.frexp(y)[1] - 1, torch.full_like(e, low).repeat_interleave(256)), min=low)
    return y * exact_pow2(3 - ey) + (r16.double() + 0.5) / 65536.0 + ((ey - low) * 8).double(), exact_pow2(e)


def exact_values8(code, k, signed):
    low = -6 if signed else -14
    c = torch.arange(256, device=code.device)
    e, man = (c & 127 if signed else c) >> 3, c & 7
    v = torch.where(e == 0, man.double(), man.double() + 8.0) * exact_pow2(torch.clamp(e, min=1) - 4 + low)
    return torch.where(c >= 128, -v, v)[code.long()] * k.repeat_interleave(256) if signed else v[code.long()] * k.repeat_interleave(256)


@pytest.mark.parametrize("signed", [True, False])
def test_exact_forms_of_8_bit_values_agree(signed):
    """the tensor form with exact powers of two, which the next test uses, against the search on the ladder"""
    gen = np.random.default_rng(1)
    x = gen.standard_normal(256 * 40) * 10.0 ** gen.uniform(-12, 0, 256 * 40)
    x = x if signed else np.abs(x)
    x[:300] = 0
    r = gen.integers(0, 65536, x.size)
    codes, scales = T.store8(x, signed, r)
    place, k = exact_place8(torch.tensor(x), signed, torch.tensor(r))
    code = torch.floor(place) if signed else torch.where(torch.tensor(x) > 0, torch.clamp(torch.floor(place), min=1), torch.floor(place))
    assert np.array_equal(code.numpy(), codes & 127 if signed else codes) and np.array_equal(k.float().numpy(), scales)
    assert np.array_equal(exact_values8(torch.tensor(codes), k, signed).numpy(), T.load8(codes, scales, signed))


@gpu
@pytest.mark.parametrize("bits_of_gradient", [12, 24])
def test_adamw8_codes_are_those_of_exact_powers_but_on_a_border(bits_of_gradient):
    """the documented format -- code times a power of two, up with the probability of the part cut off -- with exact powers of two, over a first step
    and three on states of every code: the same scales and the same codes, but where the exact place lies on a border (within 2^-30 of a step: a
    last bit of a power of two moves a value of 2^8 of its scale by 2^-44 of it, 2^-35 of the smallest step, a scale that falls by 2^5
    in a step makes 2^-30 of that).  Such places come up once in 10^7 values, and a code then is one of the two beside it."""
    n = 1 << 24
    gen = torch.Generator(device="cuda").manual_seed(bits_of_gradient)
    g = torch.randint(1, 1 << bits_of_gradient, (n,), device="cuda", generator=gen).float() * (2.0 ** torch.randint(-20, -10, (n,), device="cuda", generator=gen))
    p = torch.nn.Parameter(torch.zeros(n, device="cuda")); p.grad = g
    opt = optim.AdamW([p], lr=0.0, state_bits=8, seed=7)
    i = torch.arange(n, device="cuda")
    def mix(x):
        x = x ^ (x >> 17); x = (x * 0x743B8C43) & 0xFFFFFFFF
        x = x ^ (x >> 12); x = (x * 0xAB2209AB) & 0xFFFFFFFF
        return x ^ (x >> 15)
    m = v = torch.zeros(n, dtype=torch.float64, device="cuda")
    for t in (1, 2, 3, 4):
        opt.step()
        m = 0.9 * m + (1.0 - 0.9) * g.double(); v = 0.999 * v + (1.0 - 0.999) * g.double() * g.double()
        h = mix((i + mix(mix(mix(mix(7) + t & 0xFFFFFFFF) + 0) + 0 & 0xFFFFFFFF)) & 0xFFFFFFFF)
        s = opt.state[p]
        for key, x, signed, r in (("exp_avg", m, True, h & 0xFFFF), ("exp_avg_sq", v, False, h >> 16)):
            place, k = exact_place8(x, signed, r)
            assert torch.equal(k.float(), s[key + "_scale"])
            code, got = torch.floor(place), (s[key] & 127 if signed else s[key]).double()
            code = code if signed else torch.where(x > 0, torch.clamp(code, min=1), code)
            far = (place - torch.round(place)).abs() >= 2.0 ** -30
            assert torch.equal(got[far], code[far]), (key, t)
            assert int((~far).sum()) < 2 ** -12 * n and bool(((got - torch.round(place))[~far] <= 0).all() & ((got - torch.round(place))[~far] >= -1).all())
            if signed:
                held = got != 0                                # (a sum that cancels to its last bits has either sign: codes 0 and 128 both stand for 0)
                assert torch.equal((s[key] >= 128)[held], (x < 0)[held])
        m, v = exact_values8(s["exp_avg"], s["exp_avg_scale"].double(), True), exact_values8(s["exp_avg_sq"], s["exp_avg_sq_scale"].double(), False)
        assert torch.equal(opt.state_values()[0][0], m.float()) and torch.equal(opt.state_values()[1][0], v.float())
        p.grad = g = -g.flip(0)


# ================================================================================================ the learner's head step with a KL term
def head_case(rows, seed=5, trainable=True):
    from hoic_amd.config import Config
    from hoic_amd.rl import PolicyGaussian
    torch.manual_seed(seed)                        # (the network's initial weights)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    pol = PolicyGaussian(Config("box_future5_light_add_geom"), 32, 617).cuda()
    with torch.no_grad():
        pol.action_log_std.add_(rn(1, 32) * 0.2)
        pol.action_mean.weight.mul_(3.0)
    pol.action_log_std.requires_grad_(trainable)
    h = rn(rows, 512)
    actions = pol.action_mean(h).detach() + torch.exp(pol.action_log_std.detach()) * rn(rows, 32)
    before = copy.deepcopy(pol)
    with torch.no_grad():
        before.action_mean.weight.add_(rn(32, 512) * 2e-4)
        before.action_log_std.add_(rn(1, 32) * 0.01)
        fixed, old = before.get_log_prob(None, actions, hidden=h), dict(mean=before.action_mean(h), log_std=before.action_log_std.clone())
    return pol, h, actions, rn(rows, 1), fixed, old


def head_reference(pol, h, actions, adv, fixed, old, kl_coef, weight, mean, clip=0.2):
    """float64 autograd at the float32 means that the head's kernel gives (so that a row is on the side of the clip border that the kernel sees):
    (loss, weight * its gradients of hidden, weight, bias, log_std; log-probabilities, ratio; the surrogate's part of each row in the gradients
    of the means and of log_std)"""
    pol64, h64 = copy.deepcopy(pol).double(), h.double().requires_grad_()
    pol64.action_log_std.requires_grad_(True)
    mu, s, a = pol64.action_mean(h64), pol64.action_log_std, actions.double()
    mu = mu + (mean.double() - mu).detach()
    logp = (-((a - mu) ** 2) / (2 * torch.exp(2 * s)) - s - 0.5 * math.log(2 * math.pi)).sum(1, keepdim=True)
    ratio = torch.exp(logp - (logp.detach() if fixed is None else fixed.double()))
    mu0, s0 = (mu.detach(), s.detach()) if fixed is None else (old["mean"].double(), old["log_std"].double())
    kl = (s - s0 + (torch.exp(2 * s0) + (mu - mu0) ** 2) / (2 * torch.exp(2 * s)) - 0.5).sum(1, keepdim=True)
    loss = (-torch.min(ratio * adv.double(), torch.clamp(ratio, 1 - clip, 1 + clip) * adv.double()) + kl_coef * kl).mean()
    g = torch.autograd.grad(weight * loss, (h64, pol64.action_mean.weight, pol64.action_mean.bias, s))
    with torch.no_grad():
        part = weight / h.shape[0] * ratio * adv.double()
        parts = part * (a - mu) / torch.exp(2 * s), part * ((a - mu) ** 2 / torch.exp(2 * s) - 1)
    return loss.item(), g, logp.detach(), ratio.detach().reshape(-1), parts


@gpu
@pytest.mark.parametrize("rows", [53248, 1003])
@pytest.mark.parametrize("weight", [1.0, 0.75])
@pytest.mark.parametrize("trainable", [True, False])
def test_kl_head_step_matches_float64(rows, weight, trainable):
    """mlp.ppo_kl_head_step against float64 autograd, epoch 0 and a later one: value, gradients of the hidden activation and of every
    parameter of the head, log-probabilities, means.  Its head kernels are ppo_head_step's, and so are the tolerances (tests/test_mlp.py: float32
    head forward and backward); the loss between them is in 64 bits on the head's float32 means, as the reference's is."""
    from hoic_amd import mlp as M
    pol, h, actions, adv, fixed, given = head_case(rows, trainable=trainable)
    def close(a, b, rel, what):
        err, mag = float((a.double() - b).abs().max()), float(b.abs().max())
        assert err <= rel * mag + 1e-12, f"{what}: {err:.3e} against magnitude {mag:.3e}"
    for first in (True, False):
        old = {} if first else dict(given)
        pol.action_mean.weight.grad = pol.action_mean.bias.grad = pol.action_log_std.grad = None
        loss, dh, lp = M.ppo_kl_head_step(h, pol, actions, adv, None if first else fixed, 0.2, 0.7, old, weight)
        with torch.no_grad():
            mean = M.action_head(h, pol.action_mean.weight, pol.action_mean.bias)
        want, (g_h, g_w, g_b, g_s), logp, ratio, _ = head_reference(pol, h, actions, adv, None if first else fixed, given, 0.7, weight, mean)
        assert abs(float(loss) - want) <= 2e-5 * max(1.0, abs(want))
        close(mean, torch.nn.functional.linear(h.double(), pol.action_mean.weight.double(), pol.action_mean.bias.double()).detach(), 1e-5, "means")
        if first:
            close(lp, logp, 2e-6, "log-probabilities")
            assert lp.shape == (rows, 1) and torch.equal(old["log_std"], pol.action_log_std) and old["log_std"].data_ptr() != pol.action_log_std.data_ptr()
            assert torch.equal(old["mean"], mean)
        else:
            assert lp is fixed and set(old) == {"mean", "log_std"}
            assert 0.05 < float(((ratio < 0.8) | (ratio > 1.2)).double().mean()) < 0.95
        close(dh, g_h, 5e-5, "d loss / d hidden")
        close(pol.action_mean.weight.grad, g_w, 5e-5, "action_mean.weight.grad")
        close(pol.action_mean.bias.grad, g_b, 5e-5, "action_mean.bias.grad")
        if trainable:
            close(pol.action_log_std.grad, g_s, 5e-5, "action_log_std.grad")
            assert pol.action_log_std.grad.shape == pol.action_log_std.shape
        else:
            assert pol.action_log_std.grad is None


@gpu
def test_kl_head_step_without_kl_is_the_head_step():
    """kl_coef 0: value, gradients and log-probabilities of ppo_head_step, whose loss kernel is in float32 (twice the tolerances against float64).
    That kernel's log-probabilities, around 50 in size, are some ten roundings off: 50 x 10 x 2^-24 = 3e-5, so that a row whose ratio is within
    1e-4 of a clip border may pass its gradient there and not here: such a row adds at most its whole part to a difference."""
    from hoic_amd import mlp as M
    pol, h, actions, adv, fixed, old = head_case(4099, seed=9)
    with torch.no_grad():
        mean = M.action_head(h, pol.action_mean.weight, pol.action_mean.bias)
    _, _, _, ratio, parts = head_reference(pol, h, actions, adv, fixed, old, 0.0, 0.75, mean)
    near = ((ratio - 0.8).abs() < 1e-4) | ((ratio - 1.2).abs() < 1e-4)
    part_mean, part_std = (x[near].abs() for x in parts)
    slack = [0.0, 0.0, 0.0, part_mean.t() @ h[near].double().abs(), part_mean.sum(0), part_std.sum(0, keepdim=True)]
    out = []
    for step in (lambda f: M.ppo_kl_head_step(h, pol, actions, adv, f, 0.2, 0.0, {} if f is None else old, 0.75), lambda f: M.ppo_head_step(h, pol, actions, adv, f, 0.2, 0.75)):
        for f in (None, fixed):
            loss, dh, lp = step(f)
            out.append([loss, dh[~near] if f is not None else dh, lp] + [p.grad.clone() for p in (pol.action_mean.weight, pol.action_mean.bias, pol.action_log_std)])
    for k in range(2):
        for a, b, rel, more in zip(out[k], out[2 + k], (4e-5, 1e-4, 4e-6, 1e-4, 1e-4, 1e-4), slack if k else [0.0] * 6):
            assert bool(((a.double() - b.double()).abs() <= rel * max(float(b.abs().max()), 1.0 if rel == 4e-5 else 0.0) + 1e-12 + more).all())


def learner_run(streams=1, overlap=False, optimizer="AdamW", kl_coef=0.5, fix_std=False):
    from hoic_amd.agent import PPOLearner
    torch.manual_seed(0)
    cfg = T.learner_config([512, 256, 256], kl_coef=kl_coef, policy_optimizer=optimizer, value_optimizer=optimizer, policy_weightdecay=0.01, value_weightdecay=0.01, fix_std=fix_std)
    L = PPOLearner(cfg, 617, 32, torch.device("cuda"), update_dtype="f16x3", strict_reference=False, update_streams=streams)
    L.overlap_value_update = overlap
    start = [p.detach().clone() for n in ("policy", "value") for p in getattr(L, n + "_net").parameters()]
    for seed in (5, 6):
        L.update_params(T.learner_batch(16, 256, 617, 32, torch.float32, "cuda", seed=seed))
    L.finish_update()
    torch.cuda.synchronize()
    return start, [p.detach().clone() for n in ("policy", "value") for p in getattr(L, n + "_net").parameters()], L


@gpu
@pytest.mark.parametrize("optimizer", ["AdamW", "AdamW8bit"])
def test_learner_update_with_kl_is_the_same_on_any_streams(optimizer):
    """one stream, the value chain on a side stream, each chain's small kernels on a stream of its own, the value phase behind the policy's: the same
    kernels on the same operands in the same order within a chain, so the same bits after two updates, losses included"""
    _, want, L = learner_run(1, optimizer=optimizer)
    for streams, overlap in ((2, False), (3, False), (3, True)):
        _, got, K = learner_run(streams, overlap, optimizer=optimizer)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), (streams, overlap)
        assert K.last_losses == L.last_losses


@gpu
@pytest.mark.parametrize("fix_std", [False, True])
def test_learner_update_with_kl_through_autograd_heads(monkeypatch, fix_std):
    """heads and losses through autograd (what runs where the heads do not fit the fused kernels): the same update as the fused form to float32
    rounding -- Adam's quotients carry a gradient's relative error, 5e-5 by the head step's tests, into the step, and small gradients' signs: a
    hundredth of the way moved allowed"""
    from hoic_amd import mlp as M
    start, fused, L = learner_run(fix_std=fix_std)
    monkeypatch.setattr(M, "FORCE_AUTOGRAD_HEADS", True)
    _, plain, K = learner_run(fix_std=fix_std)
    dist = lambda x, y: math.sqrt(sum(float(((a.double() - b.double()) ** 2).sum()) for a, b in zip(x, y)))
    assert 0.0 < dist(fused, start) and dist(fused, plain) <= 1e-2 * dist(fused, start)
    assert abs(L.last_losses[1] - K.last_losses[1]) <= 1e-4 * max(1.0, abs(L.last_losses[1]))


@gpu
@pytest.mark.parametrize("update_dtype", ["f16x3", "f32"])
@pytest.mark.parametrize("scale,strict", [(1.0, True), (1e5, True), (1e5, False)])
def test_learner_clips_with_its_own_kernels(monkeypatch, update_dtype, scale, strict):
    """Adam on the GPU: the policy's gradient through optim.clip_grad_norm_ (once a run as the reference does, or every step), as torch clips it:
    the same gradient where the norm is under the bound, a factor of float32 roundings beside torch's above it (its norm: some 10 roundings
    of partial norms, the factor and the product two more: under 16 U32)"""
    from hoic_amd import agent as A
    torch.manual_seed(0)
    L = A.PPOLearner(T.learner_config([512, 256, 256], policy_lr=1e-3), 617, 32, torch.device("cuda"), update_dtype=update_dtype, strict_reference=strict)
    norms, own, theirs = [], optim.clip_grad_norm_, torch.nn.utils.clip_grad_norm_

    def both(params, bound):
        twins = [torch.nn.Parameter(torch.empty_like(p)) for p in params]
        for q, p in zip(twins, params):
            q.grad = None if p.grad is None else p.grad.clone()
        norms.append(float(own(params, bound)))
        want = float(theirs(twins, bound))
        assert bound == 40 and abs(norms[-1] - want) <= 16 * U32 * want
        for q, p in zip(twins, params):
            if p.grad is not None:
                assert torch.equal(p.grad, q.grad) if want < 39.9 else bool(((p.grad - q.grad).abs() <= 16 * U32 * q.grad.abs() + 2.0 ** -149).all())
        return norms[-1]

    monkeypatch.setattr(optim, "clip_grad_norm_", both)
    monkeypatch.setattr(torch.nn.utils, "clip_grad_norm_", None)
    b = T.learner_batch(16, 256, 617, 32, torch.float32, "cuda")
    monkeypatch.setattr(A, "estimate_advantages", lambda *a, **k: tuple(x * s for x, s in zip(rl.estimate_advantages(*a, **k), (scale, 1.0))))
    for _ in range(2):
        L.update_params(b)
    L.finish_update()
    assert len(norms) == (1 if strict else 10) and (norms[0] > 40) == (scale > 1)


def test_kernels_claim_no_alignment_that_views_lack(tmp_path):
    """the compiler's own check of the unit's vector accesses: a view of a tensor is aligned to one element, so that a load or store that goes by
    a wider type's alignment is an error (here a piece of code that does, to see that the check is on)"""
    import os
    import re
    import shutil
    import subprocess
    from conftest import ROOT
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    csrc = os.path.join(ROOT, "hoic_amd", "csrc")
    assert re.search(r"^GEMMFLAGS .*-Werror=align-mismatch", open(os.path.join(csrc, "Makefile")).read(), re.M)
    check = lambda path: subprocess.run([hipcc, "-std=c++17", "--offload-arch=gfx950", "--cuda-device-only", "-fsyntax-only", "-Werror=align-mismatch", path],
                                        capture_output=True, text=True)
    bad = tmp_path / "bad.hip"
    bad.write_text("""#include <hip/hip_runtime.h>
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
template <class V> __device__ V get(const V* x) { return *x; }
__global__ void k(const float* x, float* y) { y[0] = get((const f4u*)x).x; }
""")
    r = check(str(bad))
    assert r.returncode != 0 and "align-mismatch" in r.stderr
    r = check(os.path.join(csrc, "hoic_mlp.hip"))
    assert r.returncode == 0, r.stderr[-2000:]


def test_adamw_load_hooks_see_and_change_the_whole_state(recorder):
    """a hook before loading may hand over another state, one behind it finds the moments in place, each runs once"""
    ps = [torch.nn.Parameter(torch.randn(6)) for _ in range(2)]
    for p in ps:
        p.grad = torch.randn(6)
    opt = optim.AdamW(ps[:1], lr=0.25)
    opt.step()
    opt.state[ps[0]]["exp_avg"].fill_(3.0)
    other, seen = optim.AdamW(ps[1:], lr=0.5), []

    def before(o, sd):
        seen.append("before")
        moments = {k: {**s, "exp_avg": s["exp_avg"] * 2} for k, s in sd["state"].items()}
        return {"state": moments, "param_groups": [{**g, "lr": 0.125} for g in sd["param_groups"]]}

    def after(o):
        seen.append(float(o.state[ps[1]]["exp_avg"][0]))

    handles = other.register_load_state_dict_pre_hook(before), other.register_load_state_dict_post_hook(after)
    other.load_state_dict(opt.state_dict())
    assert seen == ["before", 6.0] and other.param_groups[0]["lr"] == 0.125 and other.state[ps[1]]["step"] == 1
    for h in handles:
        h.remove()
    other.load_state_dict(opt.state_dict())
    assert seen == ["before", 6.0] and other.param_groups[0]["lr"] == 0.25 and float(other.state[ps[1]]["exp_avg"][0]) == 3.0


def test_policy_loss_entry_point_refuses_strides_that_it_cannot_take():
    """negative row strides, and a gradient whose rows would be written over one another: refused before any launch"""
    L = lib.load()
    names = ("rows dims t_mean t_act t_std mean act log_std ref_mean ref_log_std ld_mean ld_act ld_std ld_ref_mean ld_ref_std ld_dmean adv fixed valid upstream count "
             "clip_lo clip_hi kl_coef weight d_mean d_log_std log_probs loss info n_out scratch").split()
    at = 64
    good = dict.fromkeys(names, 0) | dict(rows=4, dims=4, mean=at, act=at, log_std=at, adv=at, loss=at, info=at, scratch=at, ld_mean=4, ld_act=4, ld_dmean=4)
    changes = [{k: -1} for k in ("ld_mean", "ld_act", "ld_std", "ld_ref_mean", "ld_ref_std")] + [dict(d_mean=at, ld_dmean=k) for k in (3, 0, -4)]
    for change in changes:
        assert L.hoic_policy_loss(lib.POLICY_LOSS_ARGS.pack(*(good | change).values()), None) == -1 and b"strides" in L.hoic_last_error(), change
