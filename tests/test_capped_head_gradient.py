"""Gradients of the capped head where a difference of rounded numbers would lose them: targets that have nearly all of the probability, and logits far beyond the cap. Bounds are
relative to what is left.

Tolerances count roundings. A target's p - 1 is minus what the others have, so an error of relative size e in each of the others' p is one of e in it, however small it is.
The others' p come from t = tanh(x w / cap) in 16 bits, H = 2^-11: t itself up to tanh(1), and the root of 1 - |t| from there on, so t is off by H of itself or by 2 H of 1 - |t|, and the derivative
1 - t^2 by 2 t^2 H / (1 - t^2) or 2 H, relative. The product (2^-17 of sum |x w|) is off by as much over the cap times 1 - t^2, and the tanh's polynomial by 6.8e-7; the normaliser is formed from
unrounded logits. The gradient of a logit is p or p - 1 times the derivative, rounded to bf16 (U = 2^-8); dx and dw are sums of it in fp32, rounded once."""
import pytest
import torch

from mini_trainer_b200.ops.torch_ref import TorchOps

U = torch.finfo(torch.bfloat16).eps / 2
H = torch.finfo(torch.float16).eps / 2
TANH = 6.8e-7


def rows(levels, width, V, seed=0, gain=0.5, device="cpu"):
    """``(x, w, targets)``: row r's product with its target's weight is ``levels[r]``, up to x's rounding; the others' are normal, of about ``gain``."""
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, width, generator=g).bfloat16()
    t = torch.randperm(V, generator=g)[:len(levels)]
    noise = torch.randn(len(levels), width, generator=g) * gain / width ** 0.5
    wt = w[t].float()
    along = (torch.tensor(levels) - (noise * wt).sum(1)) / wt.square().sum(1)
    return (noise + along[:, None] * wt).bfloat16().to(device), w.to(device), t.to(device)


def exact(x, w, t, cap, grad_scale):
    """``(loss, dx, dw)`` in 64 bits, their bounds, and what the others have of the probability."""
    x, w, t = x.double().cpu(), w.double().cpu(), t.cpu()[:, None]
    z = x @ w.t()
    th = torch.tanh(z / cap)
    l, c = cap * th, torch.cosh(z / cap).reciprocal().square()
    others = torch.logsumexp(l.scatter(1, t, float("-inf")), 1, keepdim=True)
    lt = l.gather(1, t)
    loss = torch.nn.functional.softplus(others - lt)[:, 0]
    whole = torch.logaddexp(others, lt)
    p, left = torch.exp(l - whole), torch.exp(others - whole)
    p1 = p.scatter(1, t, -left)
    dz = p1 * c * grad_scale
    ez = 2.0 ** -17 * (x.abs() @ w.abs().t())
    at = (z / cap).abs()
    below, above = th.abs().clamp_min(2.0 ** -14) * H * (at <= 1.01), (1 - th.abs()) * 2 * H * (at > 1)   # of t; around the bend by either
    el = c * ez + (TANH + 2.0 ** -21) * l.abs() + 2.0 ** -21 * cap * (z.abs() > cap)
    mine = el.gather(1, t)
    among = ((p.scatter(1, t, 0.0) / left) * el).sum(1, keepdim=True)   # of the others' sum, relative
    norm = left * (among + mine)                                        # of the normaliser
    rel = (el + cap * (below + above) + norm + 2.0 ** -18).scatter(1, t, among + norm + 2.0 ** -18)
    slope = 2 * th.abs() * (below / c + ez / cap) + 2 * H * (at > 1) + 2 * TANH * th.square() / c * (at <= 1.01) + 2.0 ** -18
    edz = (U + 1.02 * rel + 1.02 * slope) * dz.abs() + 2.0 ** -124   # what is no normal number of fp32 may be zero
    bl = left[:, 0] * (among + mine + 2.0 ** -18)[:, 0] * 1.02 + 2.0 ** -21 * loss
    dx, dw = dz @ w, dz.t() @ x
    bx, bw = (1.01 * edz + 2.0 ** -17 * dz.abs()) @ w.abs() + U * dx.abs(), (1.01 * edz + 2.0 ** -17 * dz.abs()).t() @ x.abs() + U * dw.abs()
    return (loss, dx, dw), (bl, bx, bw), left[:, 0]


def run(ops, x, w, t, cap, grad_scale=1.0):
    dw = torch.empty_like(w)
    loss, dx = ops.linear_ce(x, w, t, grad_scale, dw, softcap=cap)
    return loss, dx, dw


def check(ops, x, w, t, cap, grad_scale=1.0):
    got, (want, bound, left) = run(ops, x, w, t, cap, grad_scale), exact(x, w, t, cap, grad_scale)
    for name, g, v, b in zip(("loss", "dx", "dw"), got, want, bound):
        d = (g.double().cpu() - v).abs()
        assert torch.isfinite(g).all() and (d <= b).all(), (name, int((d > b).sum()), float((d / b).max()))
        if name != "loss":   # the bound says something: a gradient of zero is far outside
            assert b.norm() <= 0.5 * v.norm(), (name, float(b.norm() / v.norm()))
    return got, left


LEVELS = [9.0, 11.0, 13.0, 16.0, 18.0, 20.0, 22.0, 24.0, 12.0, 17.0, 19.0, 21.0]


def test_plain_backend_keeps_confident_targets():
    """In fp32, to 2^-22 of a target's own p: down to a p - 1 of 1e-3 that is within the bound."""
    for cap in (30.0, 60.0):
        x, w, t = rows(LEVELS[:3], 64, 520)
        _, left = check(TorchOps(), x, w, t, cap)
        assert 1e-3 < left.min() and left.max() < 0.2


@pytest.fixture(scope="module")
def ops():
    from mini_trainer_b200.ops.native import NativeOps
    return NativeOps("cuda:0")


@pytest.mark.gpu
@pytest.mark.parametrize("pair", [0, 1])
@pytest.mark.parametrize("cap", [30.0, 60.0, 500.0])
@pytest.mark.parametrize("T,width,V", [(1, 64, 8), (12, 64, 520), (12, 256, 4096), (150, 128, 8200), (3, 1032, 40008)])
def test_confident_targets_keep_their_gradient(ops, T, width, V, cap, pair, monkeypatch):
    """Targets with all but 0.2 to 1e-9 of the probability, in whole rows and divided ones: loss and gradients are off by a part of what is left, not of one."""
    from mini_trainer_b200.ops import gemm_plan
    monkeypatch.setattr(gemm_plan, "capped_form", lambda *a: pair)
    levels = [LEVELS[(5 * k + 5) % len(LEVELS)] for k in range(T)]
    x, w, t = rows(levels, width, V, seed=T, device="cuda")
    (_, dx, _), left = check(ops, x, w, t, cap, 1.0 / T)
    assert left.min() < 5e-3
    assert ((dx.double() * w[t].double()).sum(1) < 0).all()   # every step goes up along the target's weight
    ops.check_status()


@pytest.mark.gpu
def test_a_confident_target_between_ignored_and_missing_ones(ops):
    """Rows without a target keep the softmax of all columns; their neighbours are what they are alone."""
    x, w, t = rows(LEVELS, 128, 4096, device="cuda")
    alone = run(ops, x, w, t, 30.0)
    t2 = t.clone()
    t2[1::3], t2[2::3] = -100, 4096
    loss, dx, _ = run(ops, x, w, t2, 30.0)
    assert torch.equal(loss[::3], alone[0][::3]) and torch.equal(dx[::3], alone[1][::3])
    assert not loss[1::3].any() and not dx[1::3].any() and torch.isnan(loss[2::3]).all()
    z = x.double() @ w.double().t()
    th = torch.tanh(z / 30.0)
    want = (torch.softmax(30.0 * th, 1) * (1 - th * th) @ w.double())[2::3]
    assert ((dx[2::3].double() - want).norm(dim=1) <= 0.05 * want.norm(dim=1)).all()
    ops.check_status()


def saturated(V, caps, sign, cap, seed=0, device="cpu"):
    """One row whose logits are ``caps`` caps and more away from zero, on either side; the target's on that of ``sign``. Only the first entry of x is not zero, so dw holds every logit's gradient."""
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, 32, generator=g)
    w[:, 0] = torch.where(torch.rand(V, generator=g) < 0.5, -1.0, 1.0) * cap * (caps + torch.rand(V, generator=g))
    w[V // 3, 0] = sign * cap * (caps + 0.5)
    x = torch.zeros(1, 32)
    x[0, 0] = 1.0
    return x.bfloat16().to(device), w.bfloat16().to(device), torch.tensor([V // 3], device=device)


def test_plain_backend_keeps_the_slope_of_saturated_logits():
    """1 - t^2 of a t in fp32: off by 2^-23 / (1 - t^2), 1e-5 at three caps."""
    check(TorchOps(), *saturated(72, 3.0, -1.0, 2.0), 2.0)


@pytest.mark.gpu
@pytest.mark.parametrize("sign", [-1.0, 1.0])
@pytest.mark.parametrize("cap", [2.0, 30.0])
@pytest.mark.parametrize("caps", [0.2, 0.9, 2.0, 3.0, 4.5, 6.0, 9.0, 11.3])
def test_saturated_logits_keep_their_slope(ops, caps, cap, sign):
    """A target that is certain of the wrong side (sign -1, a p - 1 of one) has the gradient that 1 - tanh^2 leaves it, 2e-10 of it at twelve caps, and so have the others."""
    for V in (72, 4104):
        check(ops, *saturated(V, caps, sign, cap, device="cuda"), cap)
    ops.check_status()


@pytest.mark.gpu
def test_logits_beyond_all_caps_have_hardly_any_gradient(ops):
    """From 12.4 caps on the derivative stays at what it is there; p and p - 1 are what they are."""
    least = (4 / (torch.exp(torch.tensor(12.4257)) + torch.exp(torch.tensor(-12.4257))) ** 2).item()
    for caps, x, w, t in ((k, *saturated(72, k, -1.0, 30.0, device="cuda")) for k in (12.5, 30.0, 1000.0)):
        loss, dx, dw = run(ops, x, w, t, 30.0)
        assert abs(float(loss) - float(torch.logsumexp(30.0 * torch.tanh(w.double()[:, 0] / 30.0), 0) + 30.0)) < 1e-4
        assert torch.isfinite(dx).all() and 0 < -dw[24, 0] <= 1.02 * least and dw.abs().max() <= 1.02 * least
    ops.check_status()
