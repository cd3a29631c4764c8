"""What a training step of a routed model learns from beyond its blocks, and the update of its matrices, as cases that can be timed and checked against plain torch.

Three operators, each through the entry points of the kernel backend (``ops.get_ops``):

* ``route``  a router with its balance loss, its z-loss and the experts' counts, per packed sample (``route_balanced``), and the gradient of the
             router's logits through weights and losses together (``route_balanced_bwd``)
* ``nll``    per-token negative log-likelihoods of an LM head that keeps no logits (``linear_nll``), and their gradients for any upstream weights
             per token, the vocabulary in pieces (``linear_nll_bwd``)
* ``orth``   matrices orthogonalised by Newton-Schulz products (``orthogonalise``), one or a stack of them; ``muon``: the whole update of a
             parameter by its orthogonalised momentum (``muon_step``)

``listed()`` holds one case per use, ``draw(rng)`` another one of the same ranges. ``run`` computes a case in its plain form, elementary torch
operations in fp32, or, with ``own`` set, by the calls that a program makes. ``exact`` is the definition in 64 bits, the losses' gradients by autograd.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
NS = (3.4445, -4.7750, 2.0315)   # x -> a x + b x^3 + c x^5, of every singular value
STEPS = 5
MOMENTUM = 0.95
MOST = 5.6e12                    # most operations of a drawn stack of matrices, whole products

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
        # the smallest call: five tokens through a router of eight experts, looked at without gradients
        {"name": "route_tiny", "kind": "route", "tokens": 5, "experts": 8, "chosen": 2, "samples": 1, "counted": 1.0, "renorm": True, "fp32": False, "train": False},
        # the eight-expert layer on a quarter of the 8B model's token budget, the batch as one sample
        {"name": "route_8x", "kind": "route", "tokens": 16384, "experts": 8, "chosen": 2, "samples": 1, "counted": 1.0, "renorm": True, "fp32": False, "train": True},
        # many small experts on a full minibatch of chat samples, prompts not counted, each sample balanced for itself; logits kept in fp32
        {"name": "route_many", "kind": "route", "tokens": 64000, "experts": 128, "chosen": 8, "samples": 41, "counted": 0.7, "renorm": True, "fp32": True, "train": True},
        # log-likelihoods of one short answer under the tiny benchmark model's head
        {"name": "nll_tiny", "kind": "nll", "tokens": 129, "hidden": 256, "vocab": 32000, "ignored": 0.2, "z": False, "train": False},
        # scoring a minibatch that the packer could not fill with the 151 936-token vocabulary: an evaluation, no gradients
        {"name": "nll_scores", "kind": "nll", "tokens": 5987, "hidden": 1536, "vocab": 151936, "ignored": 0.4, "z": False, "train": False},
        # weights per token on an odd vocabulary, with the gradient of the log-partition too
        {"name": "nll_odd", "kind": "nll", "tokens": 1777, "hidden": 2048, "vocab": 50021, "ignored": 0.1, "z": True, "train": True},
        # the 8B model's head, losses first and gradients for weights that depend on them: the largest case
        {"name": "nll_8b", "kind": "nll", "tokens": 8192, "hidden": 4096, "vocab": 128256, "ignored": 0.05, "z": False, "train": True},
        # a matrix of the tiny benchmark model: launch latency
        {"name": "orth_tiny", "kind": "orth", "stack": 1, "rows": 688, "cols": 256, "fp32": True},
        # all experts' down projections of a layer with 64 experts, as one stack
        {"name": "orth_experts", "kind": "orth", "stack": 64, "rows": 2048, "cols": 1024, "fp32": False},
        # an odd matrix, as an adapter's or a router's: rows that start off 16 bytes
        {"name": "orth_odd", "kind": "orth", "stack": 1, "rows": 1001, "cols": 4097, "fp32": True},
        # the attention output's matrix of the 1.5B model, the whole update
        {"name": "muon_1b5", "kind": "muon", "stack": 1, "rows": 1536, "cols": 1536, "lr": 5e-5, "decay": 0.1, "nesterov": True},
        # a matrix of the 8B model's MLP, the whole update
        {"name": "muon_8b", "kind": "muon", "stack": 1, "rows": 14336, "cols": 4096, "lr": 2e-5, "decay": 0.0, "nesterov": True},
    ]


def _log(rng, lo: float, hi: float, step: int = 1) -> int:
    return max(step, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)


def _whole(c: dict) -> float:
    """Operations of a stack's products, each computed whole."""
    r, n = sorted((c["rows"], c["cols"]))
    return c["stack"] * STEPS * (4.0 * r * r * n + 2.0 * r ** 3)


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["route", "route", "nll", "nll", "orth", "orth", "muon"])
    if kind == "route":
        experts = _log(rng, 2, 512)
        samples = _log(rng, 1, 60)
        return {"kind": kind, "tokens": _log(rng, samples, min(65536, 8.4e6 / experts)), "experts": experts, "chosen": rng.randint(1, min(experts, 10)),
                "samples": samples, "counted": rng.choice([1.0, round(rng.uniform(0.0, 1.0), 2)]), "renorm": rng.random() < 0.6, "fp32": rng.random() < 0.5,
                "train": rng.random() < 0.7}
    if kind == "nll":
        hidden = _log(rng, 128, 4096, 8)
        vocab = _log(rng, 1000, 152064)
        return {"kind": kind, "tokens": _log(rng, 1, min(16384, 4.3e12 / (hidden * vocab), 1.05e9 / vocab)), "hidden": hidden, "vocab": vocab,
                "ignored": round(rng.uniform(0.0, 0.5), 2), "z": rng.random() < 0.3, "train": rng.random() < 0.6}
    step = rng.choice([1, 8, 64])
    c = {"kind": kind, "stack": rng.choice([1, 1, 1, _log(rng, 2, 64)]), "rows": _log(rng, 16, 8192, step), "cols": _log(rng, 16, 16384, step)}
    while _whole(c) > MOST or c["stack"] * c["rows"] * c["cols"] > 1.4e8:
        c["stack"], c["rows"], c["cols"] = max(1, c["stack"] // 2), max(step, c["rows"] * 3 // (4 * step) * step), max(step, c["cols"] * 3 // (4 * step) * step)
    if kind == "orth":
        return c | {"fp32": rng.random() < 0.5}
    return c | {"lr": round(10 ** rng.uniform(-5.5, -4.3), 8), "decay": rng.choice([0.0, 0.1]), "nesterov": rng.random() < 0.7}


# ------------------------------------------------------------------------------------------ inputs
def _lengths(case: dict) -> list:
    """Lengths of the packed samples: lognormal, as chat data is, and fixed by the case."""
    n, t = case["samples"], case["tokens"]
    r = random.Random(1000003 * t + n)
    w = [r.lognormvariate(0.0, 0.8) for _ in range(n)]
    lens = [max(1, int(x / sum(w) * (t - n))) for x in w]
    lens[0] += t - sum(lens)
    return lens


def _gradient(case: dict, gen, gain: float):
    """Stack of matrices as a step's products leave them: sums over half as many tokens as the shorter side of outer products whose features differ
    in size, so that singular values fall over decades and half of them are only what the storage type's rounding makes of zero."""
    e, m, n = case["stack"], case["rows"], case["cols"]
    t = max(1, min(m, n) // 2)
    y = torch.randn(e, t, m, generator=gen, device=DEV) * torch.randn(e, 1, m, generator=gen, device=DEV).exp()
    x = torch.randn(e, t, n, generator=gen, device=DEV) * torch.randn(e, 1, n, generator=gen, device=DEV).exp()
    g = torch.matmul(y.bfloat16().transpose(1, 2), x.bfloat16()).float().mul_(gain / math.sqrt(t))
    return g if e > 1 else g[0]


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(1_000_003 * (seed + 1))

    def normal(*shape, gain=1.0):
        return torch.randn(*shape, generator=gen, device=DEV) * gain

    s = dict(case)
    if case["kind"] == "route":
        T, E, k, S = case["tokens"], case["experts"], case["chosen"], case["samples"]
        logits = normal(T, E, gain=1.5) + normal(E, gain=0.7)   # some experts are liked more than others: what the loss is there for
        cu = [0]
        for n in _lengths(case):
            cu.append(cu[-1] + n)
        s.update(logits=logits if case["fp32"] else logits.bfloat16(), cu=torch.tensor(cu, dtype=torch.int32, device=DEV) if S > 1 else None,
                 mask=torch.rand(T, generator=gen, device=DEV) < case["counted"] if case["counted"] < 1.0 else None)
        if case["train"]:
            s.update(dw=normal(T, k, gain=1e-2), dbalance=(1.0 + normal(S, gain=0.1)) * 1e-2 / S, dz=(1.0 + normal(S, gain=0.1)) * 1e-3 / S)
    elif case["kind"] == "nll":
        T, H, V = case["tokens"], case["hidden"], case["vocab"]
        t = torch.randint(0, V, (T,), generator=gen, device=DEV)
        t[torch.rand(T, generator=gen, device=DEV) < case["ignored"]] = -100
        s.update(x=normal(T, H).bfloat16(), w=normal(V, H, gain=3.0 / math.sqrt(H)).bfloat16(), targets=t)
        if case["train"]:   # advantages: of either sign, another one for every token
            s.update(dloss=normal(T, gain=1.0 / T), dlse=normal(T, gain=0.1 / T) if case["z"] else None)
    elif case["kind"] == "orth":
        g = _gradient(case, gen, 1e-3)
        s.update(g=g if case["fp32"] else g.bfloat16())
    else:
        g, m = _gradient(case, gen, 1e-3), _gradient(case, gen, 1e-2)
        w = normal(*g.shape, gain=0.02)
        s.update(grad=g, moment=m, master=w, param=w.bfloat16(), coef=torch.rand(1, generator=gen, device=DEV) * 0.5 + 0.5)   # coef: clips the gradient's norm
    return s


# ------------------------------------------------------------------------------------------ plain forms
def _plain_route(s: dict):
    T, E, k, S = s["tokens"], s["experts"], s["chosen"], s["samples"]
    l = s["logits"].float()
    m = l.amax(-1, keepdim=True)
    p = (l - m).exp_()
    total = p.sum(-1, keepdim=True)
    p /= total
    lse = (m + total.log())[:, 0]
    topi = l.sort(dim=-1, descending=True, stable=True)[1][:, :k].contiguous()
    top = p.gather(1, topi)
    w = top / top.sum(-1, keepdim=True) if s["renorm"] else top
    counted = torch.ones(T, dtype=torch.bool, device=DEV) if s["mask"] is None else s["mask"]
    sample = torch.zeros(T, dtype=torch.long, device=DEV) if s["cu"] is None else torch.searchsorted(s["cu"][1:].contiguous(), torch.arange(T, device=DEV, dtype=torch.int32), right=True)
    of = ((sample[None] == torch.arange(S, device=DEV)[:, None]) & counted[None]).double()   # [S, T]: long sums, so in 64 bits
    n = of.sum(1).clamp_min(1.0)
    chose = torch.zeros(T, E, dtype=torch.float64, device=DEV).scatter_(1, topi, 1.0)
    counts = torch.matmul(of, chose)
    share = torch.matmul(of, p.double())
    out = {"probs": p, "topi": topi, "w": w, "balance": (E * (counts * share).sum(1) / n.square()).float(), "z": (torch.matmul(of, lse.double().square()) / n).float(),
           "counts": counts.to(torch.int32)}
    if not s["train"]:
        return out
    dtop = (s["dw"] - (s["dw"] * w).sum(-1, keepdim=True)) / top.sum(-1, keepdim=True) if s["renorm"] else s["dw"]
    gain = torch.where(counted, 1.0, 0.0)[:, None]
    db = (s["dbalance"].double() * E / n.square())[:, None] * counts
    g = torch.zeros_like(p).scatter_(1, topi, dtop) + db.float()[sample] * gain
    dz = gain[:, 0] * 2.0 * lse * (s["dz"].double() / n).float()[sample]
    out["dlogits"] = (p * (g - (g * p).sum(-1, keepdim=True) + dz[:, None])).to(s["logits"].dtype)
    return out


def _plain_nll(s: dict):
    x, w = s["x"].float(), s["w"].float()
    valid = s["targets"] != -100
    safe = s["targets"].clamp_min(0)[:, None]
    p = torch.matmul(x, w.t())
    m = p.amax(-1, keepdim=True)
    picked = p.gather(1, safe) - m
    total = p.sub_(m).exp_().sum(-1, keepdim=True)
    loss = torch.where(valid, (total.log() - picked)[:, 0], 0.0)
    out = {"loss": loss, "lse": (m + total.log())[:, 0]}
    if not s["train"]:
        return out
    d = torch.where(valid, s["dloss"], 0.0)
    both = d if s["dlse"] is None else d + torch.where(valid, s["dlse"], 0.0)
    p.mul_((both / total[:, 0])[:, None]).scatter_add_(1, safe, -d[:, None])
    out["dx"] = torch.matmul(p, w).to(s["x"].dtype)
    out["dw"] = torch.matmul(p.t(), x).to(s["w"].dtype)
    return out


def _newton_schulz(x):
    a, b, c = NS
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2) if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + 1e-7)
    for _ in range(STEPS):
        g = torch.matmul(x, x.transpose(-1, -2))
        x = a * x + torch.matmul(b * g + c * torch.matmul(g, g), x)
    return x.transpose(-1, -2) if tall else x


def _plain_orth(s: dict):
    return {"o": _newton_schulz(s["g"].float()).to(torch.bfloat16).contiguous()}


def _plain_muon(s: dict):
    g = s["grad"] * s["coef"]
    m = s["moment"].mul_(MOMENTUM).add_(g)
    o = _newton_schulz(g + MOMENTUM * m if s["nesterov"] else m)
    w = s["master"].mul_(1.0 - s["lr"] * s["decay"]).sub_(o, alpha=s["lr"] * 0.2 * math.sqrt(max(s["rows"], s["cols"])))
    return {"master": w, "moment": m, "param": s["param"].copy_(w)}


# ------------------------------------------------------------------------------------------ the calls of a program
def _own_route(s: dict):
    ops = _ops()
    probs, topi, w, bal = ops.route_balanced(s["logits"], s["chosen"], s["renorm"], cu_seqlens=s["cu"], counted=s["mask"])
    out = {"probs": probs, "topi": topi, "w": w, "balance": bal.loss, "z": bal.z_loss, "counts": bal.counts}
    if s["train"]:
        out["dlogits"] = ops.route_balanced_bwd(probs, topi, w, s["dw"], s["renorm"], bal, s["dbalance"], s["dz"], s["logits"].dtype)
    return out


def _own_nll(s: dict):
    ops = _ops()
    loss, lse = ops.linear_nll(s["x"], s["w"], s["targets"])
    if not s["train"]:
        return {"loss": loss, "lse": lse}
    dw = torch.empty_like(s["w"])
    dx = ops.linear_nll_bwd(s["dloss"], s["x"], s["w"], s["targets"], loss, lse, dw, dlse=s["dlse"])
    return {"loss": loss, "lse": lse, "dx": dx, "dw": dw}


def _own_orth(s: dict):
    return {"o": _ops().orthogonalise(s["g"])}


def _own_muon(s: dict):
    _ops().muon_step(s["master"], s["moment"], s["grad"], s["param"], s["lr"], MOMENTUM, s["decay"], s["coef"], nesterov=s["nesterov"])
    return {"master": s["master"], "moment": s["moment"], "param": s["param"]}


def run(state: dict):
    if own:
        return {"route": _own_route, "nll": _own_nll, "orth": _own_orth, "muon": _own_muon}[state["kind"]](state)
    return {"route": _plain_route, "nll": _plain_nll, "orth": _plain_orth, "muon": _plain_muon}[state["kind"]](state)


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case: dict) -> dict:
    if case["kind"] == "route":
        T, E, k, S = case["tokens"], case["experts"], case["chosen"], case["samples"]
        e = (4 if case["fp32"] else 2) * T * E
        once = T * (case["counted"] < 1.0) + 4 * S
        n = e + 4 * T * E + 12 * T * k + once + 4 * S * (E + 2)
        if case["train"]:   # dw and the losses' factors come in, the logits' gradient goes out; what the forward has left need not be read again
            n += e + 4 * T * k + 8 * S
        return {"bytes": n, "flops": (14 if case["train"] else 6) * T * E}
    if case["kind"] == "nll":
        T, H, V = case["tokens"], case["hidden"], case["vocab"]
        if not case["train"]:
            return {"bytes": 2 * T * H + 2 * V * H + 16 * T, "flops": 2 * T * H * V}
        return {"bytes": 4 * T * H + 4 * V * H + (20 + 4 * case["z"]) * T, "flops": 8 * T * H * V}   # logits twice: none are kept between loss and gradient
    r, c = sorted((case["rows"], case["cols"]))
    numel = case["stack"] * r * c
    flops = case["stack"] * STEPS * (3 * r * r * c + r ** 3)   # two of the three products are symmetric: half of each
    if case["kind"] == "orth":
        return {"bytes": numel * ((4 if case["fp32"] else 2) + 2), "flops": flops}
    return {"bytes": numel * (4 * 5 + 2), "flops": flops}


# ------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_route(s: dict):
    T, E, k, S = s["tokens"], s["experts"], s["chosen"], s["samples"]
    bounds = [0, T] if s["cu"] is None else s["cu"].tolist()
    with torch.enable_grad():
        l = s["logits"].double().requires_grad_(s["train"])
        p = torch.softmax(l, 1)
        topi = torch.argsort(s["logits"].double(), dim=1, descending=True, stable=True)[:, :k]
        w = torch.take_along_dim(p, topi, 1)
        if s["renorm"]:
            w = w / w.sum(1, True)
        balance, z, counts = [], [], []
        for a, b in zip(bounds[:-1], bounds[1:]):
            rows = torch.arange(a, b, device=DEV)
            if s["mask"] is not None:
                rows = rows[s["mask"][a:b]]
            n = max(1, len(rows))
            c = torch.bincount(topi[rows].reshape(-1), minlength=E)
            counts.append(c)
            balance.append(E * (c / n * (p[rows].sum(0) / n)).sum())
            z.append(torch.logsumexp(l[rows], 1).square().sum() / n)
        balance, z = torch.stack(balance), torch.stack(z)
        out = {"probs": p.detach(), "topi": topi, "w": w.detach(), "balance": balance.detach(), "z": z.detach(), "counts": torch.stack(counts).to(torch.int32)}
        if s["train"]:
            total = (w * s["dw"].double()).sum() + (balance * s["dbalance"].double()).sum() + (z * s["dz"].double()).sum()
            out["dlogits"] = torch.autograd.grad(total, l)[0]
    return out


def _exact_nll(s: dict):
    with torch.enable_grad():
        x, w = s["x"].double().requires_grad_(s["train"]), s["w"].double().requires_grad_(s["train"])
        logits = x @ w.mT
        lse = torch.logsumexp(logits, 1)
        valid = s["targets"] != -100
        loss = torch.nn.functional.cross_entropy(logits, s["targets"], ignore_index=-100, reduction="none")
        out = {"loss": loss.detach(), "lse": lse.detach()}
        if s["train"]:
            total = (loss * s["dloss"].double()).sum()
            if s["dlse"] is not None:
                total = total + (lse * s["dlse"].double())[valid].sum()
            out["dx"], out["dw"] = torch.autograd.grad(total, (x, w))
    return out


def _exact_orthogonal(g):
    """By the polynomial of the Gram matrix of the shorter side, from the right or the left."""
    a, b, c = NS
    x = g / (torch.linalg.matrix_norm(g, "fro", keepdim=True) + 1e-7)
    right = g.shape[-1] <= g.shape[-2]
    one = torch.eye(min(g.shape[-2:]), dtype=torch.float64, device=DEV)
    for _ in range(STEPS):
        k = x.mT @ x if right else x @ x.mT
        q = a * one + k @ (b * one + c * k)
        x = x @ q if right else q @ x
    return x


def _exact_orth(s: dict):
    return {"o": _exact_orthogonal(s["g"].double())}


def _exact_muon(s: dict):
    g = s["grad"].double() * s["coef"].double()
    m = MOMENTUM * s["moment"].double() + g
    o = _exact_orthogonal(g + MOMENTUM * m if s["nesterov"] else m)
    w = s["master"].double() * (1.0 - s["lr"] * s["decay"]) - s["lr"] * 0.2 * math.sqrt(max(s["rows"], s["cols"])) * o
    return {"master": w, "moment": m, "param": w}


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"route": _exact_route, "nll": _exact_nll, "orth": _exact_orth, "muon": _exact_muon}[case["kind"]](s)
