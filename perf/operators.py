"""Operators around a decoder block whose scores are shaped, as cases that can be timed and checked against plain torch.

Three operators, each through the entry points of the kernel backend (``ops.get_ops``):

* ``attention``  packed (varlen) GQA attention under an ``AttentionRule``: scores capped by a tanh, a bias that falls with distance, a sliding
                 window, a prefix that every token of its sample sees; forward alone, or forward and backward
                 (``attention(..., rule=)`` / ``attention_bwd(..., rule=)``)
* ``norm``       the norm behind a branch, its gate and residual scale, the residual sum and the norm in front of the next branch
                 (``residual_norm``), and its gradient (``residual_norm_bwd``)
* ``head``       LM head and cross-entropy on logits capped by a tanh, with their gradients (``linear_ce(..., softcap=)``)

``listed()`` holds one case per use, ``draw(rng)`` another one of the same ranges. ``run`` computes a case in its plain form, elementary torch
operations in fp32, or, with ``own`` set, by the calls that a program makes. ``exact`` is the definition in 64 bits, its gradients by autograd.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-5
SCORES = 2_150_000_000   # most entries that the scores of a padded batch have in the plain form (8.6 GB in fp32)

_OPS = None


def _ops():
    """The kernel backend: a program makes one and uses it for everything."""
    global _OPS
    if _OPS is None:
        from mini_trainer_b200.ops import get_ops
        _OPS = get_ops(torch.device(DEV, torch.cuda.current_device()))
    return _OPS


# ------------------------------------------------------------------------------------------ cases
def listed() -> list:
    return [
        # the smallest call: one short sample of the smoke run's heads, looked at without gradients
        {"name": "attention_tiny", "kind": "attention", "hq": 4, "hkv": 1, "d": 128, "tokens": 127, "samples": 1, "cap": 50.0, "window": 0,
         "bias": False, "prefix": False, "train": False},
        # one long document of the 8B model's heads through a sliding window: the case a long context is windowed for
        {"name": "attention_window", "kind": "attention", "hq": 32, "hkv": 8, "d": 128, "tokens": 8192, "samples": 1, "cap": 0.0, "window": 1024,
         "bias": False, "prefix": False, "train": True},
        # a minibatch of chat samples, the 8B model's heads with capped scores: the layers without a window of a model that caps
        {"name": "attention_capped", "kind": "attention", "hq": 32, "hkv": 8, "d": 128, "tokens": 8192, "samples": 3, "cap": 50.0, "window": 0,
         "bias": False, "prefix": False, "train": True},
        # many short samples, head_dim 64, a bias by distance in place of a rotation
        {"name": "attention_bias", "kind": "attention", "hq": 16, "hkv": 4, "d": 64, "tokens": 12345, "samples": 41, "cap": 0.0, "window": 0,
         "bias": True, "prefix": False, "train": True},
        # prompts that are read in both directions in front of answers that are not; heads of the q/k-norm block
        {"name": "attention_prefix", "kind": "attention", "hq": 16, "hkv": 8, "d": 128, "tokens": 4099, "samples": 7, "cap": 0.0, "window": 0,
         "bias": False, "prefix": True, "train": True},
        # everything at once on a minibatch the packer could not fill, forward only: the recompute of a block, or an evaluation
        {"name": "attention_forward", "kind": "attention", "hq": 12, "hkv": 2, "d": 128, "tokens": 5987, "samples": 4, "cap": 30.0, "window": 1000,
         "bias": True, "prefix": True, "train": False},
        # the norms of the smoke run's hidden size on a handful of tokens: launch latency
        {"name": "norm_tiny", "kind": "norm", "tokens": 5, "hidden": 512, "post": True, "pre": True, "gate": False, "scale": 1.0, "train": False},
        # both norms of the 8B block on a quarter of its token budget, forward and backward
        {"name": "norm_8b", "kind": "norm", "tokens": 16384, "hidden": 4096, "post": True, "pre": True, "gate": False, "scale": 1.0, "train": False},
        {"name": "norm_8b_backward", "kind": "norm", "tokens": 16384, "hidden": 4096, "post": True, "pre": True, "gate": False, "scale": 1.0,
         "train": True},
        # a gated, scaled branch of the 1.5B model on a ragged minibatch, backward
        {"name": "norm_gated_backward", "kind": "norm", "tokens": 5987, "hidden": 1536, "post": True, "pre": True, "gate": True, "scale": 0.22,
         "train": True},
        # a capped head of the tiny benchmark model's vocabulary on a short, odd batch
        {"name": "head_tiny", "kind": "head", "tokens": 129, "hidden": 256, "vocab": 32000, "cap": 30.0, "ignored": 0.2},
        # the 151 936-token vocabulary on a minibatch with its prompts taken out
        {"name": "head_1b5", "kind": "head", "tokens": 3720, "hidden": 1536, "vocab": 151936, "cap": 30.0, "ignored": 0.02},
    ]


def _log(rng, lo: float, hi: float, step: int = 1) -> int:
    return max(step, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["attention", "attention", "attention", "norm", "norm", "head"])
    if kind == "attention":
        hkv = rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 3, 4])
        samples = _log(rng, 1, 50)
        c = {"kind": kind, "hq": hq, "hkv": hkv, "d": rng.choice([64, 128]), "tokens": _log(rng, max(100, 30 * samples), 12500), "samples": samples,
             "cap": round(rng.uniform(20.0, 60.0), 1) if rng.random() < 0.5 else 0.0, "window": _log(rng, 16, 4096) if rng.random() < 0.5 else 0,
             "bias": rng.random() < 0.35, "prefix": rng.random() < 0.35, "train": rng.random() < 0.7}
        if not (c["cap"] or c["window"] or c["bias"] or c["prefix"]):
            c["cap"] = 50.0
        while c["samples"] * max(_lengths(c)) ** 2 * hq > SCORES:
            c["tokens"] = int(c["tokens"] * 0.8)
        return c
    if kind == "norm":
        hidden = _log(rng, 256, 8192, 8)
        post, pre = rng.choice([(True, True), (True, True), (True, False), (False, True)])
        return {"kind": kind, "tokens": _log(rng, 1, min(16384, 67e6 / hidden)), "hidden": hidden, "post": post, "pre": pre,
                "gate": rng.random() < 0.4, "scale": rng.choice([1.0, 0.22, round(rng.uniform(0.1, 2.0), 3)]), "train": rng.random() < 0.5}
    hidden = _log(rng, 256, 4096, 8)
    vocab = _log(rng, 4096, 152064, 8)
    return {"kind": kind, "tokens": _log(rng, 16, min(9000, 0.86e12 / (hidden * vocab))), "hidden": hidden, "vocab": vocab,
            "cap": round(rng.uniform(15.0, 60.0), 1), "ignored": round(rng.uniform(0.0, 0.5), 2)}


# ------------------------------------------------------------------------------------------ inputs
def _lengths(case: dict) -> list:
    """Lengths of the packed samples: lognormal, as chat data is, and fixed by the case."""
    n, t = case["samples"], case["tokens"]
    r = random.Random(1000003 * t + n)
    w = [r.lognormvariate(0.0, 0.8) for _ in range(n)]
    lens = [max(1, int(x / sum(w) * (t - n))) for x in w]
    lens[0] += t - sum(lens)
    return lens


def _prefixes(case: dict) -> list:
    """How much of every sample is prompt: nothing of some, all of others."""
    r = random.Random(77 + case["tokens"])
    return [min(n, max(0, int(n * r.uniform(-0.2, 1.1)))) for n in _lengths(case)]


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(1_000_003 * (seed + 1))

    def normal(*shape, gain=1.0, mean=0.0):
        return (torch.randn(*shape, generator=gen, device=DEV) * gain + mean).bfloat16()

    s = dict(case)
    T = case["tokens"]
    if case["kind"] == "attention":
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        qkv = normal(T, (hq + 2 * hkv) * d)
        qkv[:, : hq * d] *= 3.0   # scores of a trained model: a standard deviation of three, single ones of fifteen and more
        lens = _lengths(case)
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        s.update(qkv=qkv, cu_host=cu, cu=torch.tensor(cu, dtype=torch.int32, device=DEV), longest=max(lens),
                 prefix_host=_prefixes(case) if case["prefix"] else None,
                 slopes=torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], device=DEV) if case["bias"] else None)
        s["prefix_dev"] = None if s["prefix_host"] is None else torch.tensor(s["prefix_host"], device=DEV)
        if case["train"]:
            s["dout"] = normal(T, hq * d)
    elif case["kind"] == "norm":
        H = case["hidden"]
        s.update(y=normal(T, H, gain=1.7), w_post=normal(H, gain=0.2, mean=0.7) if case["post"] else None,
                 w_pre=normal(H, gain=0.2, mean=1.0) if case["pre"] else None,
                 g=torch.rand(T, generator=gen, device=DEV) if case["gate"] else None)
        if case["train"]:   # what the forward has left: the residual stream behind the sum, and the row statistics
            s["h"] = normal(T, H, gain=2.5)
            s["rstd"] = tuple(torch.rsqrt(t.double().square().mean(-1) + EPS).float() if has else None
                              for t, has in ((s["y"], case["post"]), (s["h"], case["pre"])))
            s["dh"], s["dz"] = normal(T, H), normal(T, H) if case["pre"] else None
        else:
            s["x"] = normal(T, H, gain=2.5)
    else:
        H, V = case["hidden"], case["vocab"]
        t = torch.randint(0, V, (T,), generator=gen, device=DEV)
        t[torch.rand(T, generator=gen, device=DEV) < case["ignored"]] = -100
        s.update(x=normal(T, H), w=normal(V, H, gain=3.0 / math.sqrt(H)), targets=t, grad_scale=1.0 / T)
    return s


# ------------------------------------------------------------------------------------------ plain forms
def _visible(s: dict, lens, L: int):
    """``[B, L, L]``: whether a query (second axis) of a sample sees a key (last axis). Rows behind a sample's end see themselves."""
    i, j = torch.arange(L, device=DEV)[:, None], torch.arange(L, device=DEV)[None, :]
    see = j <= i
    if s["window"]:
        see = see & (i - j < s["window"])
    see = see[None].expand(len(lens), L, L)
    if s["prefix_host"] is not None:
        see = see | (j[None] < s["prefix_dev"][:, None, None])
    return see


def _plain_attention(s: dict):
    hq, hkv, d, L, cap = s["hq"], s["hkv"], s["d"], s["longest"], s["cap"]
    T, B, g, scale = s["tokens"], s["samples"], hq // hkv, d ** -0.5
    cu = s["cu"].long()
    lens = cu[1:] - cu[:-1]
    pos = torch.arange(L, device=DEV)
    inside = pos[None] < lens[:, None]                                  # [B, L]
    rows = torch.where(inside, cu[:-1, None] + pos[None], 0)
    x = torch.where(inside[..., None], s["qkv"].float()[rows], 0.0)     # [B, L, (hq + 2 hkv) d]: samples padded to the longest
    q = x[..., : hq * d].view(B, L, hkv, g, d).permute(0, 2, 3, 1, 4)
    k = x[..., hq * d: (hq + hkv) * d].view(B, L, hkv, 1, d).permute(0, 2, 3, 1, 4)
    v = x[..., (hq + hkv) * d:].view(B, L, hkv, 1, d).permute(0, 2, 3, 1, 4)
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)                # [B, hkv, g, L, L]
    t = None
    if cap:
        t = p.mul_(1.0 / cap).tanh_()
        p = t * cap
    if s["slopes"] is not None:
        p -= s["slopes"].view(1, hkv, g, 1, 1) * (pos[:, None] - pos[None, :]).abs()
    p.masked_fill_(~_visible(s, lens, L)[:, None, None], float("-inf"))
    m = p.amax(-1, keepdim=True)
    l = p.sub_(m).exp_().sum(-1, keepdim=True)
    p /= l
    o = torch.matmul(p, v)

    def packed(a, heads):   # [B, hkv, *, L, d] -> [T, heads * d]
        return a.permute(0, 3, 1, 2, 4).reshape(B, L, heads * d)[inside]

    out = packed(o, hq).to(s["qkv"].dtype)
    if not s["train"]:
        return {"out": out, "lse": (m + l.log()).permute(0, 3, 1, 2, 4).reshape(B, L, hq)[inside].t().contiguous()}
    do = torch.where(inside[..., None], s["dout"].float()[rows], 0.0).view(B, L, hkv, g, d).permute(0, 2, 3, 1, 4)
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2, keepdim=True)
    ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    if cap:
        ds *= t.square_().neg_().add_(1.0)
    dq = torch.matmul(ds, k).mul_(scale)
    dk = torch.matmul(ds.transpose(-1, -2), q).sum(2, keepdim=True).mul_(scale)
    return {"out": out, "dqkv": torch.cat([packed(dq, hq), packed(dk, hkv), packed(dv, hkv)], 1).to(s["qkv"].dtype)}


def _plain_norm(s: dict):
    dt, f = s["y"].dtype, s["scale"] if s["g"] is None else (s["scale"] * s["g"])[:, None]
    y = s["y"].float()
    if not s["train"]:
        n = y if s["w_post"] is None else y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * s["w_post"].float()
        h = s["x"].float() + f * n
        z = None if s["w_pre"] is None else (h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["w_pre"].float()).to(dt)
        return {"h": h.to(dt), "z": z}
    ry, rh = s["rstd"]
    dx, h, dwq, dwp = s["dh"].float(), s["h"].float(), None, None
    if s["w_pre"] is not None:
        dz, hh = s["dz"].float(), h * rh[:, None]
        gz = dz * s["w_pre"].float()
        dx = dx + rh[:, None] * (gz - hh * (gz * hh).mean(-1, keepdim=True))
        dwq = (dz * hh).sum(0).to(dt)
    if s["w_post"] is None:
        dy, n = f * dx, y
    else:
        yh = y * ry[:, None]
        n, gn = yh * s["w_post"].float(), f * dx * s["w_post"].float()
        dy = ry[:, None] * (gn - yh * (gn * yh).mean(-1, keepdim=True))
        dwp = (f * dx * yh).sum(0).to(dt)
    dgate = None if s["g"] is None else s["scale"] * (dx * n).sum(-1)
    return {"dx": dx.to(dt), "dy": dy.to(dt), "dgate": dgate, "dw_post": dwp, "dw_pre": dwq}


def _plain_head(s: dict):
    x, w, cap = s["x"].float(), s["w"].float(), s["cap"]
    valid = s["targets"] != -100
    safe = s["targets"].clamp_min(0)[:, None]
    t = torch.matmul(x, w.t()).mul_(1.0 / cap).tanh_()
    p = t * cap
    m = p.amax(-1, keepdim=True)
    picked = p.gather(1, safe) - m
    l = p.sub_(m).exp_().sum(-1, keepdim=True)
    loss = torch.where(valid, (l.log() - picked)[:, 0], 0.0)
    p.div_(l).scatter_add_(1, safe, torch.full_like(picked, -1.0))
    p.mul_(t.square_().neg_().add_(1.0)).mul_((valid * s["grad_scale"])[:, None])
    return {"loss": loss, "dx": torch.matmul(p, w).to(s["x"].dtype), "dw": torch.matmul(p.t(), x).to(s["x"].dtype)}


# ------------------------------------------------------------------------------------------ the calls of a program
def _own_attention(s: dict):
    from mini_trainer_b200.ops.attention_rule import AttentionRule
    ops, hq, hkv, d = _ops(), s["hq"], s["hkv"], s["d"]
    rule = AttentionRule(cap=s["cap"] or None, window=s["window"] or None, prefix=s["prefix_host"], slopes=s["slopes"])
    out, lse = ops.attention(s["qkv"], s["cu"], s["cu_host"], s["longest"], hq, hkv, d, rule=rule)
    if not s["train"]:
        return {"out": out, "lse": lse}
    return {"out": out, "dqkv": ops.attention_bwd(s["dout"], s["qkv"], out, lse, s["cu"], s["cu_host"], s["longest"], hq, hkv, d, rule=rule)}


def _own_norm(s: dict):
    ops = _ops()
    if not s["train"]:
        h, z, _ = ops.residual_norm(s["x"], s["y"], s["w_post"], s["w_pre"], EPS, scale=s["scale"], gate=s["g"])
        return {"h": h, "z": z}
    dwp, dwq = (None if w is None else torch.empty_like(w) for w in (s["w_post"], s["w_pre"]))
    dx, dy, dgate = ops.residual_norm_bwd(s["dh"], s["dz"], s["y"], s["h"], s["rstd"], s["w_post"], s["w_pre"], dwp, dwq, scale=s["scale"], gate=s["g"])
    return {"dx": dx, "dy": dy, "dgate": dgate, "dw_post": dwp, "dw_pre": dwq}


def _own_head(s: dict):
    dw = torch.empty_like(s["w"])
    loss, dx = _ops().linear_ce(s["x"], s["w"], s["targets"], s["grad_scale"], dw, softcap=s["cap"])
    return {"loss": loss, "dx": dx, "dw": dw}


def run(state: dict):
    if own:
        return {"attention": _own_attention, "norm": _own_norm, "head": _own_head}[state["kind"]](state)
    return {"attention": _plain_attention, "norm": _plain_norm, "head": _plain_head}[state["kind"]](state)


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def _pairs(case: dict) -> int:
    """(query, key) pairs of one head that see each other."""
    total = 0
    for n, p in zip(_lengths(case), _prefixes(case) if case["prefix"] else [0] * case["samples"]):
        i = torch.arange(n)
        lo = (i - case["window"] + 1).clamp_min(0) if case["window"] else torch.zeros_like(i)
        total += int((p + (i + 1 - lo.clamp_min(p)).clamp_min(0)).sum())
    return total


def work(case: dict) -> dict:
    T = case["tokens"]
    if case["kind"] == "attention":
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        qkv, out = 2 * T * (hq + 2 * hkv) * d, 2 * T * hq * d
        products = 7 if case["train"] else 2   # S and P V; then S again, dV, dP, dQ and dK
        return {"bytes": 2 * qkv + 2 * out if case["train"] else qkv + out + 4 * hq * T, "flops": products * 2 * d * hq * _pairs(case)}
    if case["kind"] == "norm":
        e, pre, post, gate = 2 * T * case["hidden"], case["pre"], case["post"], case["gate"]
        if not case["train"]:
            return {"bytes": e * (3 + pre) + 4 * T * gate, "flops": 8 * T * case["hidden"]}
        return {"bytes": e * (3 + 2 * pre + (post or gate)) + 4 * T * (pre + post + 2 * gate), "flops": 24 * T * case["hidden"]}
    H, V = case["hidden"], case["vocab"]
    return {"bytes": 4 * T * H + 4 * V * H + 12 * T, "flops": 6 * T * H * V}


# ------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_attention(s: dict):
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    T, g = s["tokens"], hq // hkv
    out = torch.empty(T, hq, d, dtype=torch.float64, device=DEV)
    lse = torch.empty(hq, T, dtype=torch.float64, device=DEV)
    grads = torch.empty(T, hq + 2 * hkv, d, dtype=torch.float64, device=DEV)
    x = s["qkv"].view(T, hq + 2 * hkv, d)
    for b in range(s["samples"]):
        a, e = s["cu_host"][b], s["cu_host"][b + 1]
        n = e - a
        delta = torch.arange(n, device=DEV).unsqueeze(1) - torch.arange(n, device=DEV)   # query minus key
        hidden = delta < 0
        if s["window"]:
            hidden = hidden | (delta >= s["window"])
        if s["prefix_host"] is not None:
            hidden[:, : s["prefix_host"][b]] = False
        for head in range(hq):
            kv = head // g
            with torch.enable_grad():
                q, k, v = (x[a:e, c].double().requires_grad_(s["train"]) for c in (head, hq + kv, hq + hkv + kv))
                z = (q @ k.mT) / math.sqrt(d)
                if s["cap"]:
                    z = s["cap"] * torch.tanh(z / s["cap"])
                if s["slopes"] is not None:
                    z = z - s["slopes"][head].double() * delta.abs()
                z = z.masked_fill(hidden, -math.inf)
                r = torch.softmax(z, 1) @ v
                if s["train"]:
                    dq, dk, dv = torch.autograd.grad(r, (q, k, v), s["dout"].view(T, hq, d)[a:e, head].double())
            out[a:e, head] = r.detach()
            lse[head, a:e] = torch.logsumexp(z.detach(), 1)
            if s["train"]:
                grads[a:e, head] = dq
                if head % g == 0:
                    grads[a:e, hq + kv], grads[a:e, hq + hkv + kv] = dk, dv
                else:
                    grads[a:e, hq + kv] += dk
                    grads[a:e, hq + hkv + kv] += dv
    if s["train"]:
        return {"out": out.view(T, -1), "dqkv": grads.view(T, -1)}
    return {"out": out.view(T, -1), "lse": lse}


def _exact_norm(s: dict):
    def rms(t, w):
        return t / torch.sqrt((t * t).mean(1, True) + EPS) * w

    def leaf(t):
        return None if t is None else t.double().requires_grad_(s["train"])

    with torch.enable_grad():
        y, wp, wq, gate = leaf(s["y"]), leaf(s["w_post"]), leaf(s["w_pre"]), leaf(s["g"])
        branch = s["scale"] * (y if wp is None else rms(y, wp))
        if gate is not None:
            branch = branch * gate.unsqueeze(1)
        if not s["train"]:
            h = s["x"].double() + branch
            return {"h": h, "z": None if wq is None else rms(h, wq)}
        h = leaf(s["h"])   # the sum as the forward has stored it
        dx, dwq = s["dh"].double(), None
        if wq is not None:
            more, dwq = torch.autograd.grad(rms(h, wq), (h, wq), s["dz"].double())
            dx = dx + more
        there = [t for t in (y, gate, wp) if t is not None]
        grads = dict(zip(map(id, there), torch.autograd.grad(branch, there, dx)))
        dy, dgate, dwp = (grads.get(id(t)) for t in (y, gate, wp))
    return {"dx": dx, "dy": dy, "dgate": dgate, "dw_post": dwp, "dw_pre": dwq}


def _exact_head(s: dict):
    with torch.enable_grad():
        x, w = s["x"].double().requires_grad_(), s["w"].double().requires_grad_()
        logits = s["cap"] * torch.tanh(x @ w.mT / s["cap"])
        loss = torch.nn.functional.cross_entropy(logits, s["targets"], ignore_index=-100, reduction="none")
        dx, dw = torch.autograd.grad(loss.sum() * s["grad_scale"], (x, w))
    return {"loss": loss.detach(), "dx": dx, "dw": dw}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "norm": _exact_norm, "head": _exact_head}[case["kind"]](s)
