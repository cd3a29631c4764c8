"""A decoder block and its head as the operators for shaped scores are used together: attention under a rule, norms on both sides of the branches, a capped head.
Forward and every gradient against autograd in 64 bits, on the CPU in fp32 and by the kernels in bf16."""
import pytest
import torch

from mini_trainer_b200.ops.attention_rule import AttentionRule
from mini_trainer_b200.ops.torch_ref import TorchOps

HQ, HKV, D, H, F, V = 4, 2, 64, 128, 192, 264
LENS = [70, 1, 0, 133]
CU = [0, 70, 71, 71, 204]
EPS, CAP, LOGIT_CAP, SCALE = 1e-5, 30.0, 20.0, 0.5


def weights(seed=0):
    g = torch.Generator().manual_seed(seed)

    def t(*shape, gain=None, mean=0.0):
        return (torch.randn(*shape, generator=g) * (shape[-1] ** -0.5 if gain is None else gain) + mean).bfloat16()

    T = CU[-1]
    p = {"x": t(T, H, gain=1.0), "ln": t(H, gain=0.1, mean=1.0), "wqkv": t((HQ + 2 * HKV) * D, H, gain=2 * H ** -0.5), "wo": t(H, HQ * D), "post": t(H, gain=0.1, mean=0.8),
         "pre": t(H, gain=0.1, mean=1.0), "wgu": t(2 * F, H), "wd": t(H, F), "post2": t(H, gain=0.1, mean=0.8), "norm": t(H, gain=0.1, mean=1.0), "lm": t(V, H, gain=3 * H ** -0.5)}
    targets = torch.randint(0, V, (T,), generator=g)
    targets[::5] = -100
    return p, targets, torch.rand(T, generator=g) + 0.5


def rule(device="cpu"):
    return AttentionRule(cap=CAP, window=60, prefix=[20, 0, 0, 90], slopes=torch.tensor([0.5, 0.1, 0.02, 0.0], device=device))


def block(ops, p, targets, gate, r):
    """``(loss, gradients)`` by the backend's calls."""
    T, dw = p["x"].shape[0], {k: torch.empty_like(v) for k, v in p.items()}
    n, rstd = ops.rmsnorm(p["x"], p["ln"], EPS)
    qkv = ops.linear(n, p["wqkv"])
    attn, lse = ops.attention(qkv, None, CU, max(LENS), HQ, HKV, D, rule=r)
    ao = ops.linear(attn, p["wo"])
    h, z, st = ops.residual_norm(p["x"], ao, p["post"], p["pre"], EPS, scale=SCALE, gate=gate)
    gu = ops.linear(z, p["wgu"])
    act = ops.swiglu(gu)
    mo = ops.linear(act, p["wd"])
    h2, y, st2 = ops.residual_norm(h, mo, p["post2"], p["norm"], EPS)
    loss, dy = ops.linear_ce(y, p["lm"], targets, 1.0 / T, dw["lm"], softcap=LOGIT_CAP)
    dh, dmo, _ = ops.residual_norm_bwd(None, dy, mo, h2, st2, p["post2"], p["norm"], dw["post2"], dw["norm"])
    dact = ops.linear_dgrad(dmo, p["wd"])
    ops.linear_wgrad(dmo, act, dw["wd"])
    dgu = ops.swiglu_bwd(dact, gu)
    dz = ops.linear_dgrad(dgu, p["wgu"])
    ops.linear_wgrad(dgu, z, dw["wgu"])
    dx, dao, dgate = ops.residual_norm_bwd(dh, dz, ao, h, st, p["post"], p["pre"], dw["post"], dw["pre"], scale=SCALE, gate=gate)
    dattn = ops.linear_dgrad(dao, p["wo"])
    ops.linear_wgrad(dao, attn, dw["wo"])
    dqkv = ops.attention_bwd(dattn, qkv, attn, lse, None, CU, max(LENS), HQ, HKV, D, rule=r)
    dn = ops.linear_dgrad(dqkv, p["wqkv"])
    ops.linear_wgrad(dqkv, n, dw["wqkv"])
    dw["x"] = ops.rmsnorm_bwd(dn, p["x"], rstd, p["ln"], dw["ln"], add_to=dx)
    return loss, {**dw, "gate": dgate}


def oracle(p, targets, gate):
    """The same in 64 bits, written on its own, gradients by autograd."""
    p = {k: v.double().requires_grad_() for k, v in p.items()}
    gate = gate.double().requires_grad_()
    T = p["x"].shape[0]
    r = rule()

    def rms(t, w):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * w

    qkv = (rms(p["x"], p["ln"]) @ p["wqkv"].t()).view(T, HQ + 2 * HKV, D)
    outs = []
    for (a, b), prefix in zip(zip(CU[:-1], CU[1:]), r.prefix):
        i = torch.arange(b - a)
        dist = i[:, None] - i[None]
        see = ((dist >= 0) & (dist < r.window)) | (i[None] < prefix)
        heads = []
        for hd in range(HQ):
            s = CAP * torch.tanh(qkv[a:b, hd] @ qkv[a:b, HQ + hd // 2].t() / D ** 0.5 / CAP) - r.slopes[hd].double() * dist.abs()
            heads.append(torch.softmax(s.masked_fill(~see, float("-inf")), 1) @ qkv[a:b, HQ + HKV + hd // 2])
        outs.append(torch.cat(heads, 1))
    h = p["x"] + SCALE * gate[:, None] * rms(torch.cat(outs) @ p["wo"].t(), p["post"])
    gate_up = rms(h, p["pre"]) @ p["wgu"].t()
    act = torch.nn.functional.silu(gate_up[:, :F]) * gate_up[:, F:]
    h = h + rms(act @ p["wd"].t(), p["post2"])
    logits = LOGIT_CAP * torch.tanh(rms(h, p["norm"]) @ p["lm"].t() / LOGIT_CAP)
    loss = torch.nn.functional.cross_entropy(logits, targets, ignore_index=-100, reduction="none")
    grads = torch.autograd.grad(loss.sum() / T, [*p.values(), gate])
    return loss.detach(), dict(zip([*p, "gate"], grads))


def compare(got, want, far):
    for k in want[1]:
        d = (got[1][k].double().cpu() - want[1][k]).norm() / want[1][k].norm()
        assert d <= far, (k, float(d))
    assert (got[0].double().cpu() - want[0]).norm() <= far * want[0].norm()


def test_block_in_fp32():
    """Sums of up to 264 terms and a dozen operations behind one another in fp32: 2^-24 each, with room for their conditioning."""
    p, targets, gate = weights()
    compare(block(TorchOps(), {k: v.float() for k, v in p.items()}, targets, gate, rule()), oracle(p, targets, gate), 2e-5)


@pytest.mark.gpu
def test_block_by_the_kernels():
    """A gradient has at most sixteen tensors that are rounded to bf16 between it and the loss, forward and backward, each off by up to 2^-8 and by 2^-8 / sqrt(3) in its
    norm: sqrt(16) of those add up to 0.9e-2; tensors behind a norm or a softmax enter twice."""
    from mini_trainer_b200.ops.native import NativeOps
    ops = NativeOps("cuda:0")
    p, targets, gate = weights()
    got = block(ops, {k: v.cuda() for k, v in p.items()}, targets.cuda(), gate.cuda(), rule("cuda"))
    compare(got, oracle(p, targets, gate), 1.8e-2)
    ops.check_status()
