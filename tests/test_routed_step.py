"""A routed layer's whole training step on the operators together: router with its balance losses, experts, likelihoods weighted by what they are, and the matrices' update, against autograd in
64 bits, reproducible, and captured."""
import math

import pytest
import torch

from mini_trainer_b200.ops.newton_schulz import NS
from mini_trainer_b200.ops.torch_ref import TorchOps

T, H, E, K, V = 90, 64, 6, 2, 200
LENS = [30, 0, 41, 15]   # and four tokens behind the last sample
BAL, Z, HEADZ, LR, MU, WD = 0.02, 1e-3, 1e-3, 0.02, 0.9, 0.1


def model(device, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = {"router": torch.randn(E, H, generator=g) * 0.3, "experts": torch.randn(E, H, H, generator=g) / math.sqrt(H), "head": torch.randn(V, H, generator=g) * 2 / math.sqrt(H)}
    x, t = torch.randn(T, H, generator=g), torch.randint(0, V, (T,), generator=g)
    t[torch.rand(T, generator=g) < 0.2] = -100
    t[sum(LENS):] = -100
    cu = torch.tensor([0] + LENS).cumsum(0).to(torch.int32)
    put = lambda a: a.to(dtype).to(device)
    return {k: put(v) for k, v in w.items()}, put(x), t.to(device), cu.to(device), (t != -100).to(device)


def weigh(loss, ok):
    """Tokens that are harder than the mean count more: weights that depend on the losses themselves, and are constants of the gradient."""
    mean = loss[ok].mean()
    return torch.where(ok, torch.clamp(loss / mean, 0.2, 3.0), torch.zeros_like(loss)) / ok.sum()


def forward_backward(ops, w, x, t, cu, ok):
    """``(outputs, gradients)`` of one step; experts as plain products, whose gradients are written out."""
    S = len(LENS)
    logits = x.float() @ w["router"].float().t()   # in fp32, as routers are kept: a choice is not to turn on a rounding
    probs, topi, p, bal = ops.route_balanced(logits, K, True, cu, ok)
    h_all = torch.einsum("th,eoh->teo", x.float(), w["experts"].float())                    # [T, E, H]
    picked = h_all.gather(1, topi[:, :, None].expand(-1, -1, H))                            # [T, K, H]
    y = (x.float() + (p[:, :, None] * picked).sum(1)).to(x.dtype)
    loss, lse = ops.linear_nll(y, w["head"], t)
    weight = weigh(loss, ok)
    dhead = torch.empty_like(w["head"])
    dy = ops.linear_nll_bwd(weight, y, w["head"], t, loss, lse, dhead, dlse=2 * HEADZ * lse / T).float()
    dp = (dy[:, None] * picked).sum(-1)
    dl = ops.route_balanced_bwd(probs, topi, p, dp, True, bal, torch.full((S,), BAL / S, device=x.device), torch.full((S,), Z / S, device=x.device), torch.float32)
    dexp = torch.zeros(E, H, H, dtype=torch.float32, device=x.device)
    for e in range(E):
        c = torch.where(topi == e, p, 0.0).sum(1)
        dexp[e] = (dy * c[:, None]).t() @ x.float()
    return (loss, lse, bal.loss, bal.z_loss, bal.counts), {"router": dl.t() @ x.float(), "experts": dexp, "head": dhead.float()}


def exact(w, x, t, cu, ok, weight):
    w = {k: v.double().cpu().requires_grad_() for k, v in w.items()}
    x, t, ok, weight = x.double().cpu(), t.cpu(), ok.cpu(), weight.double().cpu()
    logits = x @ w["router"].t()
    p = torch.softmax(logits, 1)
    topi = torch.argsort(logits.detach(), dim=1, descending=True, stable=True)[:, :K]
    top = p.gather(1, topi)
    top = top / top.sum(1, keepdim=True)
    picked = torch.einsum("th,eoh->teo", x, w["experts"]).gather(1, topi[:, :, None].expand(-1, -1, H))
    y = x + (top[:, :, None] * picked).sum(1)
    z = y @ w["head"].t()
    lse = torch.logsumexp(z, 1)
    loss = torch.where(ok, lse - z.gather(1, t.clamp_min(0)[:, None])[:, 0], 0.0)
    total = (loss * weight).sum() + (HEADZ / T * lse[ok] ** 2).sum()
    b = cu.tolist()
    for s in range(len(LENS)):
        rows = torch.arange(b[s], b[s + 1])[ok[b[s]:b[s + 1]]]
        n = len(rows)
        if n:
            c = torch.bincount(topi[rows].reshape(-1), minlength=E).double()
            total = total + BAL / len(LENS) * E * (c * p[rows].sum(0)).sum() / n ** 2 + Z / len(LENS) * torch.logsumexp(logits[rows], 1).square().mean()
    total.backward()
    return loss.detach(), {k: v.grad for k, v in w.items()}


def orthogonal(u):
    a, b, c = NS
    u = u.double()
    x = u / (torch.linalg.matrix_norm(u, keepdim=True) + 1e-7)
    for _ in range(5):
        g = x @ x.mT
        x = a * x + (b * g + c * g @ g) @ x
    return x


def step(ops, device, dtype):
    w, x, t, cu, ok = model(device, dtype)
    out, grads = forward_backward(ops, w, x, t, cu, ok)
    loss, want = exact(w, x, t, cu, ok, weigh(out[0], ok))
    # three roundings to 16 bits are on the way to a gradient (y, the logits' gradients as operands, dy or the head's gradient), each of at most half a step of an entry; a loss is off by y's, through logits that
    # are sums of 64 products of numbers of about 1 and 0.25: 2^-8 * 64 * 0.8 * 0.2 = 0.04 were all of one sign
    tol = 1e-5 if dtype is torch.float32 else 3 * torch.finfo(dtype).eps / 2
    assert float((out[0].double().cpu() - loss).abs().max()) <= (1e-5 if dtype is torch.float32 else 0.04)
    for k, g in grads.items():
        assert float((g.double().cpu() - want[k]).norm() / want[k].norm()) <= tol, k
    # the update
    moment = {k: torch.zeros_like(g) for k, g in grads.items()}
    master = {k: w[k].float().clone() for k in grads}
    coef = torch.full((1,), 0.5, device=device)
    for k in grads:
        param = w[k].clone()
        ops.muon_step(master[k], moment[k], grads[k], param if dtype is torch.bfloat16 else None, LR, MU, WD, coef)
        u = 0.5 * grads[k].double()
        scale = 0.2 * math.sqrt(max(grads[k].shape[-2:]))
        upd = LR * scale * orthogonal(u * (1 + MU)).to(device)
        exp = (1 - LR * WD) * w[k].double() - upd
        assert float((master[k].double() - exp).norm()) <= 0.006 * float(upd.norm()) + 2.0 ** -22 * float(exp.norm()), k
        if dtype is torch.bfloat16:
            assert torch.equal(param, master[k].bfloat16())
    return out, grads, master


def test_step_on_the_cpu():
    step(TorchOps(), "cpu", torch.float32)


@pytest.mark.gpu
def test_step_on_the_kernels():
    from mini_trainer_b200.ops import get_ops
    ops = get_ops(torch.device("cuda:0"))
    first, again = (step(ops, "cuda", torch.bfloat16) for _ in range(2))
    for a, b in zip(first[0], again[0]):
        assert torch.equal(a, b)
    for part in (1, 2):
        for k in first[part]:
            assert torch.equal(first[part][k], again[part][k])
    ops.check_status()


@pytest.mark.gpu
def test_steps_captured_into_a_graph():
    """Three steps replayed are three steps run: losses, gradients and updated weights."""
    from mini_trainer_b200.ops import get_ops
    ops = get_ops(torch.device("cuda:0"))

    def make():
        w, x, t, cu, ok = model("cuda", torch.bfloat16, 3)
        moment = {k: torch.zeros(v.shape, device="cuda") for k, v in w.items()}
        master = {k: v.float().clone() for k, v in w.items()}
        coef = torch.ones(1, device="cuda")
        weight = ok.float() / ok.sum()

        def run():
            logits = x.float() @ w["router"].float().t()
            probs, topi, p, bal = ops.route_balanced(logits, K, True, cu, ok)
            h_all = torch.einsum("th,eoh->teo", x.float(), w["experts"].float())
            y = (x.float() + (p[:, :, None] * h_all.gather(1, topi[:, :, None].expand(-1, -1, H))).sum(1)).bfloat16()
            loss, lse = ops.linear_nll(y, w["head"], t)
            dhead = torch.empty_like(w["head"])
            dy = ops.linear_nll_bwd(weight, y, w["head"], t, loss, lse, dhead).float()
            dl = ops.route_balanced_bwd(probs, topi, p, (dy[:, None] * h_all.gather(1, topi[:, :, None].expand(-1, -1, H))).sum(-1), True, bal,
                                        torch.full((len(LENS),), BAL, device="cuda"), None, torch.float32)
            for k, g in (("head", dhead), ("router", dl.t() @ x.float())):
                ops.muon_step(master[k], moment[k], g.contiguous(), w[k], LR, MU, WD, coef)
            return loss, bal.loss
        return run, w, master
    run, w, master = make()
    want = [tuple(t.clone() for t in run()) for _ in range(3)]
    run2, w2, master2 = make()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run2()
    for a in want:   # (products that split their reduction do not under capture: sums in another order, which a step's rounding may turn)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(a, held):
            assert torch.allclose(x, y, rtol=2e-2, atol=2e-2)
    for k in ("head", "router"):
        assert float((master[k] - master2[k]).norm() / master[k].norm()) < 1e-2 and not torch.equal(master2[k], make()[2][k])
    ops.check_status()
