"""A router with its balance losses (``route_balanced`` and its gradient), on the CPU and by the kernels, against 64 bits.

Tolerances count roundings of 2^-24. A probability is an exponential of a rounded difference (|l - m| roundings of an argument below 30, two of the function) over a sum of up to
16 + 5 terms a chain: below 64 of itself, R = 2^-18, and so are weights (three probabilities' worth: 3 R). logsumexp is off by R / 4 of |m| + log E + 1. Balance losses are sums of positive terms: R of themselves, with the
rounding of sums over up to a few hundred tokens a chain in fp32 (2^-15 at most). The gradient is off by 4 R of the absolute values of its terms and half a step of its type."""
import pytest
import torch

from mini_trainer_b200.ops.torch_ref import TorchOps

R = 2.0 ** -18


def inputs(T, E, k, lens=None, counted=None, dtype=torch.float32, seed=0, device="cpu", gain=1.5):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(T, E, generator=g) * gain + 0.5 * torch.randn(E, generator=g)).to(dtype)
    cu = None if lens is None else torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32)
    S = 1 if lens is None else len(lens)
    v = {"logits": logits, "cu": cu, "counted": None if counted is None else torch.rand(T, generator=g) < counted, "dw": torch.randn(T, k, generator=g),
         "dloss": torch.randn(S, generator=g), "dz": torch.randn(S, generator=g) * 0.1}
    return {n: None if t is None else t.to(device) for n, t in v.items()}


def exact(v, k, renorm):
    l = v["logits"].double().cpu().requires_grad_()
    T, E = l.shape
    bounds = [0, T] if v["cu"] is None else v["cu"].tolist()
    counted = torch.ones(T, dtype=torch.bool) if v["counted"] is None else v["counted"].cpu()
    p = torch.softmax(l, 1)
    topi = torch.argsort(l.detach(), dim=1, descending=True, stable=True)[:, :k]
    top = p.gather(1, topi)
    w = top / top.sum(1, keepdim=True) if renorm else top
    loss, z, counts, tokens = [], [], [], []
    for a, b in zip(bounds[:-1], bounds[1:]):
        rows = torch.arange(a, b)[counted[a:b]]
        n = max(1, rows.numel())
        c = torch.bincount(topi[rows].reshape(-1), minlength=E)
        loss.append(E * (c.double() * p[rows].sum(0)).sum() / n ** 2)
        z.append(torch.logsumexp(l[rows], 1).square().sum() / n)
        counts.append(c)
        tokens.append(rows.numel())
    return l, p, topi, w, torch.stack(loss), torch.stack(z), torch.stack(counts), tokens


def check(ops, v, k, renorm, dw=True, dloss=True, dz=True):
    logits, dtype = v["logits"], v["logits"].dtype
    probs, topi, w, bal = ops.route_balanced(logits, k, renorm, cu_seqlens=v["cu"], counted=v["counted"])
    l, p, ti, wt, loss, z, counts, tokens = exact(v, k, renorm)
    d = lambda t: t.detach().double().cpu()
    assert (probs.dtype, topi.dtype, w.dtype, bal.counts.dtype) == (torch.float32, torch.int64, torch.float32, torch.int32)
    assert torch.equal(topi.cpu(), ti) and torch.equal(bal.counts.cpu().long(), counts) and bal.tokens.tolist() == tokens
    assert ((d(probs) - d(p)).abs() <= R * d(p) + 1e-37).all() and ((d(w) - d(wt)).abs() <= 3 * R * d(wt) + 1e-37).all()
    size = d(l).amax(1).abs() + torch.log(torch.tensor(float(l.shape[1]))) + 1
    lse = torch.logsumexp(d(l), 1)
    assert ((d(bal.lse) - lse).abs() <= R / 4 * size).all()
    assert ((d(bal.loss) - d(loss)).abs() <= 8 * R * d(loss)).all()
    top = size.max() if len(size) else 1.0
    assert ((d(bal.z_loss) - d(z)).abs() <= 8 * R * d(z) + R * top * d(z).sqrt() + R * R * top ** 2).all()
    cpu = lambda t: t.double().cpu()
    total = 0.0
    if dw:
        total = total + (wt * cpu(v["dw"])).sum()
    if dloss:
        total = total + (loss * cpu(v["dloss"])).sum()
    if dz:
        total = total + (z * cpu(v["dz"])).sum()
    want = torch.autograd.grad(total, l)[0]
    got = ops.route_balanced_bwd(probs, topi, w, v["dw"] if dw else None, renorm, bal, v["dloss"] if dloss else None, v["dz"] if dz else None, dtype)
    assert got.dtype == dtype and got.shape == logits.shape
    # absolute values of a gradient's terms
    T, E = l.shape
    terms = torch.zeros(T, E, dtype=torch.float64)
    bounds = [0, T] if v["cu"] is None else v["cu"].tolist()
    zt = torch.zeros(T, 1, dtype=torch.float64)
    for s, (a, b) in enumerate(zip(bounds[:-1], bounds[1:])):
        n = max(1, tokens[s])
        if dloss:
            terms[a:b] += cpu(v["dloss"])[s].abs() * E * counts[s] / n ** 2
        if dz:
            zt[a:b] += 2 * (lse[a:b, None].abs() + size[a:b, None] / 4) * cpu(v["dz"])[s].abs() / n
    if dw:
        adw = cpu(v["dw"]).abs()
        t = (adw + (adw * d(wt)).sum(1, keepdim=True)) / d(p).gather(1, ti).sum(1, keepdim=True) if renorm else adw
        terms.scatter_add_(1, ti, t)
    bound = d(p) * (terms + (d(p) * terms).sum(1, keepdim=True) + zt)
    assert ((d(got) - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 4 * R * bound + 1e-37).all()
    return probs, topi, w, bal, got


CASES = [(5, 8, 2, None, None, True), (1, 1, 1, None, None, True), (57, 9, 3, [10, 0, 1, 46], 0.5, False), (300, 64, 8, [100, 200], None, True),
         (77, 33, 5, [77], 0.0, True), (130, 128, 8, [1] * 130, 0.7, True), (513, 60, 4, [0, 0, 513, 0], None, False), (64, 100, 10, [7, 13, 20], 0.8, True),
         (40, 512, 32, [40], None, True), (33, 384, 8, [11, 22], 0.5, True), (100, 2, 2, None, None, True), (31, 257, 6, [30], None, False)]


@pytest.mark.parametrize("T,E,k,lens,counted,renorm", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_plain_form(T, E, k, lens, counted, renorm, dtype):
    check(TorchOps(), inputs(T, E, k, lens, counted, dtype), k, renorm)


def test_gradient_against_differences():
    """Balance and z-loss alone are smooth where the choice does not change."""
    ops, v = TorchOps(), inputs(12, 6, 2, [5, 7], 0.8, seed=3)
    _, topi, _, bal = ops.route_balanced(v["logits"], 2, True, v["cu"], v["counted"])
    probs, topi, w, bal = ops.route_balanced(v["logits"], 2, True, v["cu"], v["counted"])
    grad = ops.route_balanced_bwd(probs, topi, w, None, True, bal, v["dloss"], v["dz"], torch.float32)

    def f(x):
        l, p, ti, wt, loss, z, counts, tokens = exact({**v, "logits": x}, 2, True)
        return float(((loss * v["dloss"].double()).sum() + (z * v["dz"].double()).sum()).detach())
    x = v["logits"].double()
    for t in range(12):
        for e in range(6):
            hi, lo = x.clone(), x.clone()
            hi[t, e] += 1e-5
            lo[t, e] -= 1e-5
            assert abs((f(hi) - f(lo)) / 2e-5 - float(grad[t, e])) <= 1e-6


def test_balanced_use_has_the_least_loss():
    """``k`` for experts that are used alike, and else the experts' number times the sum of the products of two means: pairs per token and probabilities."""
    ops = TorchOps()
    assert abs(float(ops.route_balanced(torch.eye(8).repeat(5, 1) * 1e-3, 8, True)[3].loss) - 8.0) < 1e-4
    logits = torch.randn(64, 8, generator=torch.Generator().manual_seed(1))
    mask = ((torch.arange(64).view(2, 32) % 32) < torch.tensor([[20], [32]])).reshape(-1)
    for counted in (None, mask):
        p = logits.double().softmax(1)[slice(None) if counted is None else counted]
        pairs = torch.zeros_like(p).scatter_(1, p.topk(2, dim=1).indices, 1.0)
        want = 8 * float((pairs.mean(0) * p.mean(0)).sum())
        assert abs(float(ops.route_balanced(logits, 2, True, counted=counted)[3].loss) - want) < 1e-5


def special(ops, device):
    """Ties, masked experts, rows that are not numbers: the choice, and that uncounted rows stay out of the losses."""
    inf, low = float("inf"), torch.finfo(torch.float32).min
    l = torch.tensor([[1.0, 2.0, 2.0, 1.0], [0.0, -0.0, 0.0, -0.0], [-inf, 3.0, -inf, 1.0], [low, low, 0.0, low], [float("nan"), 1.0, 2.0, 3.0], [1.0, inf, 0.0, 2.0],
                      [-inf, -inf, -inf, -inf], [-inf, -inf, 5.0, -inf]], device=device)
    counted = torch.tensor([1, 1, 1, 1, 0, 0, 0, 1], dtype=torch.bool, device=device)
    probs, topi, w, bal = ops.route_balanced(l, 3, True, counted=counted)
    assert topi.tolist() == [[1, 2, 0], [0, 1, 2], [1, 3, 0], [2, 0, 1], [0, 3, 2], [1, 3, 0], [0, 1, 2], [2, 0, 1]]
    assert bal.tokens.tolist() == [5] and bal.counts.sum() == 15 and torch.isfinite(bal.loss).all() and torch.isfinite(bal.z_loss).all()
    assert torch.isnan(probs[4]).all() and torch.equal(probs[7].cpu(), torch.tensor([0.0, 0.0, 1.0, 0.0]))
    one = torch.ones(1, device=device)
    g = ops.route_balanced_bwd(probs, topi, w, None, True, bal, one, one, torch.float32)
    assert torch.isfinite(g[counted]).all() and not torch.isfinite(g[4]).any()


def test_special_rows():
    special(TorchOps(), "cpu")


def outside(ops, device):
    """Tokens in front of the first sample and behind the last one are routed, and have no part in a loss."""
    v = inputs(50, 12, 3, device=device)
    cu = torch.tensor([7, 20, 20, 44], dtype=torch.int32, device=device)
    probs, topi, w, bal = ops.route_balanced(v["logits"], 3, True, cu)
    inner = v["logits"][7:44].contiguous()
    p2, t2, w2, b2 = ops.route_balanced(inner, 3, True, (cu - 7).to(torch.int32))
    assert torch.equal(topi[7:44], t2) and torch.equal(probs[7:44], p2) and torch.equal(bal.counts, b2.counts) and torch.allclose(bal.loss, b2.loss, rtol=1e-6)
    assert bal.tokens.tolist() == [13, 0, 24] and bal.sample.tolist() == [-1] * 7 + [0] * 13 + [2] * 24 + [-1] * 6
    d, one = v["dw"], torch.ones(3, device=device)
    g = ops.route_balanced_bwd(probs, topi, w, d, True, bal, one, one, torch.float32)
    alone = ops.route_balanced_bwd(probs, topi, w, d, True, bal, dtype=torch.float32)
    assert torch.equal(g[:7], alone[:7]) and torch.equal(g[44:], alone[44:])
    g2 = ops.route_balanced_bwd(p2, t2, w2, d[7:44].contiguous(), True, b2, one, one, torch.float32)
    assert torch.allclose(g[7:44], g2, rtol=1e-5, atol=1e-7)


def test_tokens_outside_all_samples():
    outside(TorchOps(), "cpu")


def test_no_tokens():
    probs, topi, w, bal = TorchOps().route_balanced(torch.empty(0, 4), 2, True, torch.zeros(3, dtype=torch.int32))
    assert probs.shape == (0, 4) and bal.loss.tolist() == [0.0, 0.0] and bal.counts.tolist() == [[0] * 4] * 2


@pytest.mark.parametrize("backend", ["plain", "native"])
def test_refusals(backend):
    from .test_native_host import make_ops
    ops = TorchOps() if backend == "plain" else make_ops()
    l, cu = torch.zeros(6, 8), torch.tensor([0, 6], dtype=torch.int32)
    for bad in (dict(logits=l.half()), dict(logits=l.t()), dict(logits=l[:, :, None]), dict(logits=torch.zeros(6, 513)), dict(logits=torch.zeros(6, 0)), dict(k=0), dict(k=9), dict(k=2.0),
                dict(k=True), dict(logits=torch.zeros(6, 64), k=33), dict(cu_seqlens=cu.long()), dict(cu_seqlens=cu[:1]), dict(cu_seqlens=cu[None]), dict(counted=torch.ones(6)),
                dict(counted=torch.ones(5, dtype=torch.bool)), dict(logits=torch.empty(1 << 30, 2, device="meta"))):
        with pytest.raises(ValueError):
            ops.route_balanced(**{"logits": l, "k": 2, "renorm": True, **bad})
    probs, topi, w, bal = TorchOps().route_balanced(l, 2, True, cu)
    one = torch.ones(1)
    for bad in (dict(dloss=None), dict(dloss=torch.ones(2)), dict(dloss=one.double()), dict(dz=torch.ones(2)), dict(probs=probs[:5]), dict(topi=topi.int()), dict(w=w.double()),
                dict(dw=torch.ones(6, 3)), dict(dtype=torch.float16), dict(probs=probs.t())):
        with pytest.raises(ValueError):
            ops.route_balanced_bwd(**{"probs": probs, "topi": topi, "w": w, "dw": None, "renorm": True, "balance": bal, "dloss": one, **bad})
    if backend == "native":
        with pytest.raises(ValueError, match="made for"):   # tensors of another device
            ops.route_balanced(l, 2, True)
        assert not ops.calls


# ------------------------------------------------------------------------------------------ kernels
@pytest.fixture(scope="module")
def native():
    from mini_trainer_b200.ops import get_ops
    return get_ops(torch.device("cuda:0"))


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k,lens,counted,renorm", CASES + [(4099, 8, 2, None, None, True), (20011, 128, 8, [5000, 1, 14000, 1000], 0.6, True), (3001, 160, 6, [300] * 10, 0.9, False),
                                                               (9001, 24, 4, [29] * 300, 0.5, True), (5003, 37, 7, None, 0.5, True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_kernels(native, T, E, k, lens, counted, renorm, dtype):
    v = inputs(T, E, k, lens, counted, dtype, device="cuda", seed=T)
    first = check(native, v, k, renorm)
    again = check(native, v, k, renorm)
    for a, b in zip(first[:3] + (first[3].loss, first[3].z_loss, first[4]), again[:3] + (again[3].loss, again[3].z_loss, again[4])):
        assert torch.equal(a, b)
    for only in ("dw", "dloss", "dz"):
        check(native, v, k, renorm, **{n: n == only for n in ("dw", "dloss", "dz")})
    native.check_status()


@pytest.mark.gpu
def test_kernels_on_special_rows(native):
    special(native, "cuda")
    outside(native, "cuda")
    probs, topi, w, bal = native.route_balanced(torch.empty(0, 4, device="cuda"), 2, True, torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert bal.loss.tolist() == [0.0, 0.0] and bal.counts.tolist() == [[0] * 4] * 2
    assert native.route_balanced_bwd(probs, topi, w, None, True, bal, torch.ones(2, device="cuda")).shape == (0, 4)
    native.check_status()


@pytest.mark.gpu
def test_kernels_on_unaligned_rows(native):
    """Rows that start off their vectors take single loads."""
    buf = torch.randn(1 + 50 * 16, device="cuda")
    for off, dtype in ((1, torch.float32), (1, torch.bfloat16), (0, torch.bfloat16)):
        l = buf.to(dtype)[off:off + 800].view(50, 16)
        v = inputs(50, 16, 3, [20, 30], 0.7, dtype, device="cuda")
        v["logits"] = l
        check(native, v, 3, True)


@pytest.mark.gpu
def test_kernels_under_capture_and_on_another_stream(native):
    v = inputs(700, 48, 4, [300, 400], 0.7, torch.bfloat16, device="cuda")

    def run():
        probs, topi, w, bal = native.route_balanced(v["logits"], 4, True, v["cu"], v["counted"])
        return probs, topi, w, bal.loss, bal.z_loss, bal.counts, native.route_balanced_bwd(probs, topi, w, v["dw"], True, bal, v["dloss"], v["dz"])
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(want, other, held):
        assert torch.equal(a, b) and torch.equal(a, c)
    v["logits"].copy_(v["logits"].flip(0))   # other data, the same graph
    graph.replay()
    for a, c in zip(run(), held):
        assert torch.equal(a, c)


@pytest.mark.gpu
def test_an_expert_that_is_none(native):
    """Indexes outside the experts have no gradient and are reported; one that is named twice has both."""
    v = inputs(9, 8, 2, device="cuda")
    probs, topi, w, bal = native.route_balanced(v["logits"], 2, False)
    twice = topi.clone()
    twice[:, 1] = twice[:, 0]
    got = native.route_balanced_bwd(probs, twice, w, v["dw"], False, bal, dtype=torch.float32)
    g = torch.zeros_like(probs).scatter_add_(1, twice, v["dw"])
    assert torch.allclose(got, probs * (g - (g * probs).sum(1, keepdim=True)), atol=1e-6)
    native.check_status()
    out = topi.clone()
    out[3, 1] = 8
    out[4, 0] = -1
    got = native.route_balanced_bwd(probs, out, w, v["dw"], False, bal, dtype=torch.float32)
    d = v["dw"].clone()
    d[3, 1] = d[4, 0] = 0
    g = torch.zeros_like(probs).scatter_add_(1, out.clamp(0, 7), d)
    assert torch.allclose(got, probs * (g - (g * probs).sum(1, keepdim=True)), atol=1e-6)
    with pytest.raises(RuntimeError, match="chosen expert"):
        native.check_status()


@pytest.mark.gpu
def test_many_tokens(native):
    """More than 2^31 probabilities: offsets in 64 bits."""
    T, E, k = (1 << 31) // 512 + 1000, 512, 2
    logits = torch.zeros(T, E, dtype=torch.bfloat16, device="cuda")
    logits[-700:] = torch.randn(700, E, device="cuda").bfloat16()
    cu = torch.tensor([0, T - 700, T], dtype=torch.int32, device="cuda")
    probs, topi, w, bal = native.route_balanced(logits, k, True, cu)
    p2, t2, w2, b2 = native.route_balanced(logits[-700:].contiguous(), k, True)
    assert torch.equal(probs[-700:], p2) and torch.equal(topi[-700:], t2) and torch.allclose(bal.loss[1:], b2.loss, rtol=1e-5)
    assert bal.counts[0].tolist() == [T - 700] * 2 + [0] * 510 and abs(float(bal.loss[0]) - 2.0) < 1e-4
    one = torch.ones(2, device="cuda")
    g = native.route_balanced_bwd(probs, topi, w, None, True, bal, one, one)
    g2 = native.route_balanced_bwd(p2, t2, w2, None, True, b2, one[:1].contiguous(), one[:1].contiguous())
    assert torch.equal(g[-700:], g2)
