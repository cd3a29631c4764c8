"""Norms around a branch (``residual_norm`` and its gradient), on the CPU and by the kernels, against 64 bits.

Tolerances count roundings: U = 2^-8 for one to bf16. h and z are rounded once, z is also off by what h's rounding does to it, which stays below
another U of it and U of |h| r |w| where the sum cancels; the gradients are rounded once, weight gradients once after a sum in fp32, and
``dgate`` is fp32. An fp32 sum of N terms is off by at most N / 2 roundings of 2^-24 of the terms' absolute values along a chain; the kernels add in
chains of at most H / 32 + 48 per row and T per block and column."""
import itertools

import pytest
import torch

from mini_trainer_b200.ops.torch_ref import TorchOps

U = torch.finfo(torch.bfloat16).eps / 2
E = 2.0 ** -17   # an fp32 chain of up to 8192 / 32 + 48 terms, and the reciprocal root
EPS = 1e-5


def inputs(T, H, post=True, pre=True, gated=False, seed=0, device="cpu", size=1.0):
    g = torch.Generator().manual_seed(seed)

    def t(*shape, mean=0.0, gain=1.0):
        return (torch.randn(*shape, generator=g) * gain + mean).bfloat16().to(device)

    return {"x": t(T, H, gain=2 * size), "y": t(T, H, gain=size), "w_post": t(H, mean=0.7, gain=0.3) if post else None, "w_pre": t(H, mean=1.0, gain=0.3) if pre else None,
            "gate": torch.randn(T, generator=g).to(device) if gated else None, "dh": t(T, H), "dz": t(T, H) if pre else None}


def rms(x, w):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def f64(v):
    return {k: None if t is None else t.double().cpu() for k, t in v.items()}


def check_forward(v, scale, got):
    d = f64(v)
    b = scale * (1.0 if d["gate"] is None else d["gate"][:, None])
    n = d["y"] if d["w_post"] is None else rms(d["y"], d["w_post"])
    h, (gh, gz, (ry, rh)) = d["x"] + b * n, got
    assert ((gh.double().cpu() - h).abs() <= U * h.abs() + E * (d["x"].abs() + (b * n).abs()) + 1e-30).all()
    if d["w_post"] is not None:
        r = 1 / torch.sqrt((d["y"] ** 2).mean(-1) + EPS)
        assert ((ry.double().cpu() - r).abs() <= E * r).all()
    if d["w_pre"] is None:
        assert gz is None and rh is None
        return
    stored = gh.double().cpu()   # the norm is of what is stored
    z, r = rms(stored, d["w_pre"]), 1 / torch.sqrt((stored ** 2).mean(-1) + EPS)
    assert ((gz.double().cpu() - z).abs() <= (U + E) * z.abs() + 1e-30).all() and ((rh.double().cpu() - r).abs() <= E * r).all()


def check_backward(v, scale, h, stats, got, dws):
    d = f64(v)
    h = h.double().cpu()
    y, wp, wq, gate = (None if t is None else t.clone().requires_grad_() for t in (d["y"], d["w_post"], d["w_pre"], d["gate"]))
    b = scale * (1.0 if gate is None else gate[:, None])
    branch = b * (y if wp is None else rms(y, wp))
    dx = torch.zeros_like(d["y"]) if d["dh"] is None else d["dh"]
    size = dx.abs()
    if wq is not None:
        hl = h.clone().requires_grad_()
        more, dwq = torch.autograd.grad(rms(hl, wq), (hl, wq), d["dz"])
        r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
        g, hh = (d["dz"] * d["w_pre"]).abs(), (h * r).abs()
        size = size + r * (g + hh * (g * hh).mean(-1, keepdim=True))
        dx = dx + more
        terms = (d["dz"].abs() * hh).sum(0)
        assert ((dws[1].double().cpu() - dwq).abs() <= U * dwq.abs() + (E + 2.0 ** -24 * h.shape[0]) * terms + 1e-30).all()
    there = [t for t in (y, gate, wp) if t is not None]
    grads = dict(zip(map(id, there), torch.autograd.grad(branch, there, dx)))
    dy, dgate, dwp = (grads.get(id(t)) for t in (y, gate, wp))
    gx, gy, gg = got
    assert ((gx.double().cpu() - dx).abs() <= U * dx.abs() + E * size + 1e-30).all()
    ab = (scale * (1.0 if d["gate"] is None else d["gate"][:, None])) * torch.ones_like(dx[:, :1])
    n = d["y"].abs()
    if wp is not None:
        r = 1 / torch.sqrt((d["y"] ** 2).mean(-1, keepdim=True) + EPS)
        yh = d["y"].abs() * r
        n, g = yh * d["w_post"].abs(), ab.abs() * size * d["w_post"].abs()
        esize = r * (g + yh * (g * yh).mean(-1, keepdim=True))
        terms = (ab.abs() * size * yh).sum(0)
        assert ((dws[0].double().cpu() - dwp).abs() <= U * dwp.abs() + (2 * E + 2.0 ** -24 * h.shape[0]) * terms + 1e-30).all()
    else:
        esize = ab.abs() * size
    assert ((gy.double().cpu() - dy).abs() <= U * dy.abs() + 3 * E * esize + 1e-30).all()
    assert (gg is None) == (gate is None)
    if gate is not None:
        assert ((gg.double().cpu() - dgate).abs() <= 3 * E * abs(scale) * (size * n).sum(-1) + 1e-30).all()


def forward_and_backward(ops, v, scale, with_dh=True):
    out = ops.residual_norm(v["x"], v["y"], v["w_post"], v["w_pre"], EPS, scale=scale, gate=v["gate"])
    dws = [None if w is None else torch.full_like(w, float("nan")) for w in (v["w_post"], v["w_pre"])]
    if not with_dh:
        v = {**v, "dh": None}
    got = ops.residual_norm_bwd(v["dh"], v["dz"], v["y"], out[0], out[2], v["w_post"], v["w_pre"], *dws, scale=scale, gate=v["gate"])
    if v["y"].shape[0]:
        check_forward(v, scale, out)
        check_backward(v, scale, out[0], out[2], got, dws)
    return out, got, dws


FORMS = [(True, True), (True, False), (False, True)]


# ------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize("post,pre", FORMS)
@pytest.mark.parametrize("gated", [False, True])
def test_plain_backend_against_64_bits(post, pre, gated):
    for T, H, scale in ((1, 8, 1.0), (7, 72, 0.22), (33, 264, -1.5)):
        forward_and_backward(TorchOps(), inputs(T, H, post, pre, gated, seed=T), scale)
    if pre:
        forward_and_backward(TorchOps(), inputs(5, 40, post, pre, gated), 1.0, with_dh=False)


def test_formula_against_differences():
    """dh and dz along a direction of x and y, by central differences in 64 bits: the step's square, 2^-40, is what they are off."""
    v = f64(inputs(6, 48, gated=True))
    u = torch.randn(6, 48, generator=torch.Generator().manual_seed(3), dtype=torch.float64)

    def f(e):
        y, x = v["y"] + e * u, v["x"] - e * u
        h = x + 0.5 * v["gate"][:, None] * rms(y, v["w_post"])
        return (h * v["dh"]).sum() + (rms(h, v["w_pre"]) * v["dz"]).sum()

    h = v["x"] + 0.5 * v["gate"][:, None] * rms(v["y"], v["w_post"])
    ops, dw = TorchOps(), [torch.empty(48, dtype=torch.float64) for _ in range(2)]
    stats = tuple(1 / torch.sqrt((t * t).mean(-1) + EPS) for t in (v["y"], h))
    dx, dy, _ = ops.residual_norm_bwd(v["dh"], v["dz"], v["y"], h, stats, v["w_post"], v["w_pre"], *dw, scale=0.5, gate=v["gate"])
    slope = (f(2.0 ** -20) - f(-2.0 ** -20)) / 2.0 ** -19
    assert abs(slope - ((dy - dx) * u).sum()) <= 2.0 ** -16 * ((dy - dx) * u).abs().sum()


def host_ops():
    from .test_native_host import make_ops
    ops = make_ops(mtb200_residual_norm_bwd_blocks=lambda T, H: 3)
    ops._index = None
    return ops


def test_calls_of_the_kernels_and_their_refusals():
    ops = host_ops()
    v = inputs(5, 64, gated=True)
    h, z, stats = ops.residual_norm(v["x"], v["y"], v["w_post"], v["w_pre"], EPS, scale=0.5, gate=v["gate"])
    assert ops.calls[-1][0] == "mtb200_residual_norm_fwd" and ops.calls[-1][1][9:13] == (0.5, EPS, 5, 64)
    dws = [torch.empty_like(v["w_post"]), torch.empty_like(v["w_pre"])]
    dx, dy, dgate = ops.residual_norm_bwd(v["dh"], v["dz"], v["y"], h, stats, v["w_post"], v["w_pre"], *dws, scale=0.5, gate=v["gate"])
    assert ops.calls[-1][0] == "mtb200_residual_norm_bwd" and ops.calls[-1][1][15:18] == (0.5, 5, 64) and dgate.shape == (5,)
    empty = inputs(0, 64)
    ops.residual_norm_bwd(empty["dh"], empty["dz"], empty["y"], empty["y"], (torch.empty(0), torch.empty(0)), empty["w_post"], empty["w_pre"], *dws)
    assert not dws[0].any() and not dws[1].any()
    n = len(ops.calls)
    bad = [dict(x=v["x"].float()), dict(x=v["x"][:4]), dict(y=v["y"][:, :60]), dict(y=v["y"].t().contiguous().t()), dict(w_post=v["w_post"][:32]), dict(w_pre=v["w_pre"].float()),
           dict(gate=v["gate"].bfloat16()), dict(gate=v["gate"][:, None]), dict(w_post=None, w_pre=None), dict(y=torch.zeros(5, 8200, dtype=torch.bfloat16)),
           dict(x=torch.zeros(5 * 64 + 4, dtype=torch.bfloat16)[4:].view(5, 64))]
    for change in bad:
        a = {**v, **change}
        with pytest.raises(ValueError):
            ops.residual_norm(a["x"], a["y"], a["w_post"], a["w_pre"], EPS, gate=a["gate"])
    bad = [dict(dz=None), dict(stats=(stats[0], None)), dict(stats=(stats[0].double(), stats[1])), dict(dws=[dws[0], None]), dict(dws=[None, dws[1]]), dict(h=h[:3]),
           dict(dh=v["dh"].float()), dict(w_pre=None), dict(w_pre=None, dz=None, dh=None, stats=(stats[0], None), dws=[dws[0], None])]
    for change in bad:
        a = {**v, "h": h, "stats": stats, "dws": dws, **change}
        for o in (ops, TorchOps()) if set(change) & {"dz", "w_pre"} else (ops,):
            with pytest.raises(ValueError):
                o.residual_norm_bwd(a["dh"], a["dz"], a["y"], a["h"], a["stats"], a["w_post"], a["w_pre"], *a["dws"], gate=a["gate"])
    assert len(ops.calls) == n


# ------------------------------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def ops():
    from mini_trainer_b200.ops.native import NativeOps
    return NativeOps("cuda:0")


@pytest.mark.gpu
@pytest.mark.parametrize("post,pre", FORMS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T,H", [(1, 8), (3, 24), (5, 512), (130, 264), (33, 1000), (67, 1032), (19, 2056), (300, 4096), (5, 4104), (9, 8192), (1, 8192)])
def test_kernels_against_64_bits(ops, T, H, post, pre, gated):
    forward_and_backward(ops, inputs(T, H, post, pre, gated, seed=T + H, device="cuda"), 0.75)
    if pre:
        forward_and_backward(ops, inputs(T, H, post, pre, gated, seed=H, device="cuda"), 1.0, with_dh=False)
    ops.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", [(20011, 64), (9973, 512), (8003, 1536), (4097, 4096), (2501, 8192)])
def test_more_rows_than_resident_blocks(ops, T, H):
    """Persistent blocks and rows by bulk copies, several sets per block and an odd last one."""
    for post, pre in FORMS:
        forward_and_backward(ops, inputs(T, H, post, pre, True, seed=H, device="cuda"), 0.22)
    ops.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("T,H", [(7003, 256), (4501, 640), (2371, 768), (601, 2816), (1201, 5120), (301, 6144), (149, 6152), (2369, 8)])
def test_both_layouts_of_a_row_over_threads(ops, T, H):
    """One and two vectors of a row per thread, as many rows under way as an SM holds and one more, several turns of the partial rows' sum."""
    for post, pre in FORMS:
        forward_and_backward(ops, inputs(T, H, post, pre, H % 512 == 0, seed=T, device="cuda"), 1.5)
    ops.check_status()


@pytest.mark.gpu
def test_sizes_of_the_values(ops):
    """Rows of zeros (eps alone holds the root), of tiny and of large values."""
    for size in (0.0, 2.0 ** -40, 2.0 ** 30):
        v = inputs(70, 256, gated=True, device="cuda", size=size)
        forward_and_backward(ops, v, 1.0)
    ops.check_status()


@pytest.mark.gpu
def test_agrees_with_norm_and_sum_apart(ops):
    v = inputs(500, 2048, device="cuda")
    h, z, (ry, rh) = ops.residual_norm(v["x"], v["y"], v["w_post"], v["w_pre"], EPS)
    n, r = ops.rmsnorm(v["y"], v["w_post"], EPS)
    assert torch.allclose(r, ry, rtol=1e-6)
    two = n.float() + v["x"].float()
    assert ((h.float() - two).abs() <= U * h.float().abs() + 2.1 * U * n.float().abs()).all()   # n is rounded twice there, the sum once here
    z2, r2 = ops.rmsnorm(h, w=v["w_pre"], eps=EPS)
    assert torch.allclose(r2, rh, rtol=1e-6) and ((z.float() - z2.float()).abs() <= 3.1 * U * z2.float().abs()).all()


@pytest.mark.gpu
def test_two_streams_captured_and_twice(ops):
    """Calls on two streams at once share no scratch, a captured call replays on new inputs, and equal calls are equal bit for bit."""
    shapes = [(3000, 1024), (777, 4096)]
    vs = [inputs(T, H, gated=True, seed=T, device="cuda") for T, H in shapes]
    want = [forward_and_backward(ops, v, 0.5) for v in vs]
    streams = [torch.cuda.Stream() for _ in vs]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, v in zip(streams, vs):
            with torch.cuda.stream(s):
                out = ops.residual_norm(v["x"], v["y"], v["w_post"], v["w_pre"], EPS, scale=0.5, gate=v["gate"])
                dws = [torch.empty_like(v["w_post"]), torch.empty_like(v["w_pre"])]
                got.append((out, ops.residual_norm_bwd(v["dh"], v["dz"], v["y"], out[0], out[2], v["w_post"], v["w_pre"], *dws, scale=0.5, gate=v["gate"]), dws))
    torch.cuda.synchronize()
    for (a, b, c), (x, y, z) in zip(itertools.cycle(want), got):
        for p, q in zip((a[0], a[1], *a[2], *b, *c), (x[0], x[1], *x[2], *y, *z)):
            assert torch.equal(p, q)
    v, graph = vs[0], torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.residual_norm(v["x"], v["y"], v["w_post"], v["w_pre"], EPS, scale=0.5, gate=v["gate"])
        dws = [torch.empty_like(v["w_post"]), torch.empty_like(v["w_pre"])]
        back = ops.residual_norm_bwd(v["dh"], v["dz"], v["y"], out[0], out[2], v["w_post"], v["w_pre"], *dws, scale=0.5, gate=v["gate"])
    new = inputs(*shapes[0], gated=True, seed=99, device="cuda")
    for k in v:
        v[k].copy_(new[k])
    graph.replay()
    torch.cuda.synchronize()
    check_forward(new, 0.5, out)
    check_backward(new, 0.5, out[0], out[2], back, dws)
    ops.check_status()
