"""Matrices orthogonalised by Newton-Schulz products and updates by an orthogonalised momentum, on the CPU and by the kernels, against 64 bits.

The plain form is fp32: a rounding of X (2^-24 of its entries) grows by at most 3.4445^5 = 485 on the way and products of up to n terms add n / 8 of them, so 485 * 32 * 2^-24 = 2^-10 of the norm
is far above it. The kernels hold X to 22 bits up to the last step, and M and the polynomial to 11: a rounding of those, 2^-12 of their entries, of uniform and independent sign, moves X by
at most 2^-12 * 2 * 4.8 * |X| in a step through b (their spectral norm is at most that of a random matrix with such entries, and |M|, |polynomial| <= 3.5), and what a step has moved is carried on by at most the polynomial's slope
at values near one, 1.5 on either side, and 3.9 at the largest (1.2): five steps add up to less than 2^-12 * 9.6 * (1 + 1.5 + 1.5^2 + 1.5^3 + 1.5^4) / sqrt(3) < 0.018 were all of it in
one direction. It is spread over as many as the matrix has: TOL below is a third of that. Where the few entries that are not zero meet in no row or column, each of them is a singular
value and the products are diagonal: every rounding is in one direction, and the whole 0.018 = 3 TOL is what holds. The result is rounded by U = 2^-8 of an entry at most."""
import math

import pytest
import torch

from mini_trainer_b200.ops.torch_ref import TorchOps

U = torch.finfo(torch.bfloat16).eps / 2
TOL = 0.006
A, B, C = 3.4445, -4.7750, 2.0315


def matrices(kind, *shape, seed=0, dtype=torch.float32, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    *lead, m, n = shape

    def normal(*s):
        return torch.randn(*s, generator=g)
    if kind == "normal":
        x = normal(*shape) * 1e-3
    elif kind == "features":   # a gradient's: sums of outer products whose features differ in size
        t = max(1, min(m, n) // 2)
        x = (normal(*lead, t, m) * normal(*lead, 1, m).exp()).mT @ (normal(*lead, t, n) * normal(*lead, 1, n).exp())
    elif kind == "low_rank":
        x = normal(*lead, m, 8) @ normal(*lead, 8, n) + 0.01 * normal(*shape)
    elif kind == "rank_one":
        x = normal(*lead, m, 1) @ normal(*lead, 1, n)
    elif kind == "sparse":
        x = normal(*shape) * (torch.rand(*shape, generator=g) < 0.01)
    elif kind == "tiny":
        x = normal(*shape) * 1e-12
    elif kind == "one":
        x = torch.zeros(*shape)
        x[..., m // 2, n // 3] = -3.0
    return x.to(dtype).to(device)


def exact(g, steps=5):
    """By the singular values: each goes through the polynomial."""
    u, s, v = torch.linalg.svd(g.double(), full_matrices=False)
    s = s / (s.square().sum(-1, keepdim=True).sqrt() + 1e-7)
    for _ in range(steps):
        s = A * s + B * s ** 3 + C * s ** 5
    return u @ (s.unsqueeze(-1) * v)


def check(got, g, tol, steps=5):
    want = exact(g, steps)
    assert got.shape == g.shape and got.dtype == torch.bfloat16
    d, size = torch.linalg.matrix_norm(got.double() - want), torch.linalg.matrix_norm(want)
    assert (d <= (tol + U / math.sqrt(3)) * size + 1e-30).all(), (d / size).max()
    # no entry is off by more than a rounding and what a row may hold of the rest
    rows = torch.linalg.vector_norm(want, dim=-1, keepdim=True) + size[..., None, None] / math.sqrt(g.shape[-2])
    assert ((got.double() - want).abs() <= U * want.abs() + 3 * tol * rows).all()


KINDS = ["normal", "features", "low_rank", "rank_one", "sparse", "tiny", "one"]
SHAPES = [(1, 1), (1, 40), (40, 1), (13, 30), (30, 13), (64, 64), (129, 257), (200, 72), (3, 17, 40), (2, 2, 40, 24), (2, 130, 130)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", KINDS)
def test_plain_form(shape, kind):
    g = matrices(kind, *shape)
    check(TorchOps().orthogonalise(g), g, 2.0 ** -10)
    b = matrices(kind, *shape, dtype=torch.bfloat16)
    check(TorchOps().orthogonalise(b, steps=3), b, 2.0 ** -10, 3)


def test_orthogonal_rows():
    """A well-conditioned matrix comes out with singular values near one; more steps keep them there."""
    g = torch.randn(40, 200, generator=torch.Generator().manual_seed(0))
    for steps in (5, 8):
        s = torch.linalg.svdvals(TorchOps().orthogonalise(g, steps).double())
        assert 0.65 < s.min() and s.max() < 1.25


def muon_exact(v, lr, mu, wd, coef, nesterov, scale):
    g, m, w = (v[k].double() for k in ("grad", "moment", "master"))
    g = g * coef
    m = mu * m + g
    stored = m.to(v["moment"].dtype).double()
    return m, lambda m_stored: (1 - lr * wd) * w - lr * scale * exact(g + mu * m_stored if nesterov else m_stored)


def check_muon(ops, shape, moment_dtype, grad_dtype, nesterov, wd, coef, scale, tol, device="cpu", unaligned=False):
    v = {"grad": matrices("features", *shape, seed=1, dtype=grad_dtype, device=device), "moment": matrices("features", *shape, seed=2, dtype=moment_dtype, device=device),
         "master": matrices("normal", *shape, seed=3, device=device) * 20}
    if unaligned:
        for k, t in list(v.items()):
            b = torch.empty(t.numel() + 1, dtype=t.dtype, device=device)[1:].view(t.shape)
            v[k] = b.copy_(t)
    before = {k: t.clone() for k, t in v.items()}
    param = torch.empty(shape, dtype=torch.bfloat16, device=device)
    lr, mu = 0.02, 0.95
    c = torch.tensor([coef], device=device) if coef != 1.0 else coef
    ops.muon_step(v["master"], v["moment"], v["grad"], param, lr, mu, wd, c, nesterov=nesterov, scale=scale)
    full = 0.2 * math.sqrt(max(shape[-2:])) if scale is None else scale
    m, rest = muon_exact(before, lr, mu, wd, torch.tensor(coef, dtype=torch.float32).double().item(), nesterov, full)
    unit = U if moment_dtype is torch.bfloat16 else 2.0 ** -23
    g = (before["grad"].double() * coef).abs()
    assert torch.equal(v["grad"], before["grad"])
    assert ((v["moment"].double() - m).abs() <= unit * m.abs() + 2.0 ** -22 * (g + before["moment"].double().abs())).all()
    want = rest(v["moment"].double())   # the momentum counts as it is stored
    size = torch.linalg.matrix_norm(exact((before["grad"].double() * coef + mu * v["moment"].double()) if nesterov else v["moment"].double()))[..., None, None] * lr * full
    d = torch.linalg.matrix_norm(v["master"].double() - want)[..., None, None]
    assert (d <= tol * size + 2.0 ** -22 * torch.linalg.matrix_norm(want)[..., None, None]).all()
    assert torch.equal(param, v["master"].to(torch.bfloat16))


MUON = [((24, 40), torch.float32, torch.float32, True, 0.1, 1.0, None), ((3, 40, 24), torch.bfloat16, torch.bfloat16, True, 0.0, 0.37, None), ((65, 33), torch.float32, torch.bfloat16, False, 0.1, 0.5, 0.7)]


@pytest.mark.parametrize("shape,moment,grad,nesterov,wd,coef,scale", MUON)
def test_plain_muon(shape, moment, grad, nesterov, wd, coef, scale):
    check_muon(TorchOps(), shape, moment, grad, nesterov, wd, coef, scale, 2.0 ** -10)


@pytest.mark.parametrize("backend", ["plain", "native"])
def test_refusals(backend):
    from .test_native_host import make_ops
    ops = TorchOps() if backend == "plain" else make_ops()
    g = torch.ones(6, 8)
    for bad in (dict(g=g[0]), dict(g=g.double()), dict(g=g.t()), dict(g=g.half()), dict(g=g, steps=0), dict(g=g, steps=2.0), dict(g=g, steps=True), dict(g=g, steps=65),
                dict(g=torch.empty(1, 1 << 24, device="meta")), dict(g=torch.empty((1 << 16) + 1, (1 << 16) + 1, device="meta"))):
        with pytest.raises(ValueError):
            ops.orthogonalise(**bad)
    good = dict(master=g.clone(), moment=g.clone(), grad=g, param_out=g.bfloat16(), lr=0.1, momentum=0.9, weight_decay=0.0)
    for bad in (dict(master=g.bfloat16()), dict(moment=g.double()), dict(moment=g), dict(master=good["moment"]), dict(grad=g[:5]), dict(param_out=g.half()), dict(param_out=torch.ones(8, 6).t()),
                dict(lr=float("nan")), dict(momentum=float("inf")), dict(grad_coef=torch.ones(2)), dict(steps=0), dict(grad=g.t())):
        with pytest.raises(ValueError):
            ops.muon_step(**{**good, **bad})
    if backend == "native":
        with pytest.raises(ValueError, match="made for"):
            ops.orthogonalise(g)
        with pytest.raises(ValueError, match="made for"):
            ops.muon_step(**good)
        ops.check_device = lambda t: None
        with pytest.raises(ValueError, match="bf16"):
            ops.muon_step(**{**good, "param_out": torch.ones(6, 8)})
        assert not ops.calls


# ------------------------------------------------------------------------------------------ kernels
@pytest.fixture(scope="module")
def native():
    from mini_trainer_b200.ops import get_ops
    return get_ops(torch.device("cuda:0"))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES + [(256, 688), (688, 256), (512, 512), (300, 1001), (1001, 300), (1100, 1300), (1300, 1032), (5, 260, 520), (20, 136, 64), (70, 264, 264),
                                            (128, 2048), (2048, 128), (100, 2049), (2100, 40), (128, 4096), (3, 3001, 70), (100, 4100), (64, 128), (32, 129), (20, 257), (257, 64), (50, 513), (33, 8192), (8192, 64), (32, 16384), (17, 9000), (16385, 30), (8193, 48), (5, 31, 3000), (128, 300), (33, 1030), (90, 64, 700), (40, 700, 128), (160, 24, 24), (9, 128, 1025)])
@pytest.mark.parametrize("kind", KINDS)
def test_kernels(native, shape, kind):
    g = matrices(kind, *shape, device="cuda")
    got = native.orthogonalise(g)
    check(got, g, 3 * TOL if kind in ("sparse", "one") else TOL)
    assert torch.equal(got, native.orthogonalise(g))
    native.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(40, 12440), (12440, 40), (200, 8201), (8201, 200), (700, 4100), (4100, 700), (3, 600, 1000), (2, 1000, 600), (40, 520, 640), (1281, 1290)])
@pytest.mark.parametrize("kind", ["features", "rank_one", "one"])
def test_long_reductions_and_blocks_above_the_diagonal(native, shape, kind):
    """A reduction in up to eight parts; symmetric operands whose blocks above the diagonal are read from below it."""
    g = matrices(kind, *shape, device="cuda")
    got = native.orthogonalise(g)
    check(got, g, 3 * TOL if kind in ("sparse", "one") else TOL)
    assert torch.equal(got, native.orthogonalise(g))
    native.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(130, 250), (250, 130), (520, 512)])
@pytest.mark.parametrize("steps", [1, 2, 6])
def test_kernels_by_steps(native, shape, steps):
    g = matrices("features", *shape, dtype=torch.bfloat16, device="cuda")
    check(native.orthogonalise(g, steps), g, TOL, steps)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(40, 72), (72, 40), (264, 520), (520, 264), (140, 301)])
def test_matrices_that_start_off_16_bytes(native, shape):
    for dtype in (torch.float32, torch.bfloat16):
        g = matrices("features", *shape, dtype=dtype, device="cuda")
        b = torch.empty(g.numel() + 3, dtype=dtype, device="cuda")[3:].view(shape).copy_(g)
        assert torch.equal(native.orthogonalise(b), native.orthogonalise(g))


@pytest.mark.gpu
def test_large_matrices(native):
    """Tiles by single CTAs and by pairs, either side the longer, against products in 64 bits."""
    for shape in ((2048, 2048), (4096, 1040), (1040, 4096), (2500, 6000)):
        g = matrices("features", *shape, device="cuda")
        x = g.double() / (g.double().norm() + 1e-7)
        for _ in range(5):
            if shape[0] > shape[1]:
                k = x.T @ x
                x = A * x + x @ (B * k + C * k @ k)
            else:
                k = x @ x.T
                x = A * x + (B * k + C * k @ k) @ x
        got = native.orthogonalise(g)
        assert float((got.double() - x).norm() / x.norm()) <= TOL + U / math.sqrt(3)
    native.check_status()


@pytest.mark.gpu
def test_a_matrix_that_is_not_finite_is_alone(native):
    g = matrices("normal", 5, 72, 136, device="cuda")
    want = native.orthogonalise(g)
    bad = g.clone()
    bad[1, 3, 5], bad[3, 0, 0], bad[4] = float("nan"), float("inf"), 0.0
    got = native.orthogonalise(bad)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and (got[4] == 0).all()
    assert torch.isnan(got[1]).any()
    assert native.orthogonalise(torch.empty(0, 4, 8, device="cuda")).shape == (0, 4, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,moment,grad,nesterov,wd,coef,scale", MUON + [((520, 1032), torch.float32, torch.float32, True, 0.1, 0.9, None), ((4, 264, 129), torch.bfloat16, torch.float32, True, 0.1, 1.0, None),
                                                                                   ((2, 100, 600), torch.bfloat16, torch.bfloat16, False, 0.1, 0.7, None), ((700, 72), torch.float32, torch.bfloat16, True, 0.1, 0.9, None)])
@pytest.mark.parametrize("unaligned", [False, True])
def test_muon_kernels(native, shape, moment, grad, nesterov, wd, coef, scale, unaligned):
    check_muon(native, shape, moment, grad, nesterov, wd, coef, scale, TOL, "cuda", unaligned)
    native.check_status()


@pytest.mark.gpu
def test_under_capture_and_on_another_stream(native):
    g = matrices("features", 2, 264, 520, device="cuda")
    want = native.orthogonalise(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = native.orthogonalise(g)
    torch.cuda.synchronize()
    assert torch.equal(other, want)
    master, moment, param = torch.zeros_like(g), torch.zeros_like(g), torch.empty_like(g, dtype=torch.bfloat16)
    coef = torch.full((1,), 0.5, device="cuda")
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = native.orthogonalise(g)
    with torch.cuda.graph(second):
        native.muon_step(master, moment, g, param, 0.1, 0.9, 0.1, coef)
    for _ in range(2):
        graph.replay()
        second.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, want)
    m2, w2, p2 = torch.zeros_like(g), torch.zeros_like(g), torch.empty_like(param)
    for _ in range(2):
        native.muon_step(w2, m2, g, p2, 0.1, 0.9, 0.1, 0.5)
    assert torch.equal(master, w2) and torch.equal(moment, m2) and torch.equal(param, p2)


@pytest.mark.gpu
def test_stacks_behind_2_31_elements(native):
    """A stack of more than 2^31 elements: its last matrices as a stack of their own."""
    small = torch.zeros((1 << 31) // (128 * 1024) + 5, 1024, 128, dtype=torch.bfloat16, device="cuda")
    small[-3:] = matrices("normal", 3, 1024, 128, dtype=torch.bfloat16, device="cuda")
    got = native.orthogonalise(small)   # (how many slabs a matrix has goes by the stack, and with it the order of sums)
    alone = native.orthogonalise(small[-3:].contiguous())
    assert (got[:-3] == 0).all() and ((got[-3:].double() - alone.double()).norm() <= TOL * alone.double().norm())
    del small, got
    g = torch.zeros((1 << 31) // (2048 * 1024) + 3, 2048, 1024, dtype=torch.bfloat16, device="cuda")
    g[-4:] = matrices("normal", 4, 2048, 1024, dtype=torch.bfloat16, device="cuda")
    got = native.orthogonalise(g)
    assert torch.equal(got[-4:], native.orthogonalise(g[-4:].contiguous())) and (got[:-4] == 0).all()
    native.check_status()
