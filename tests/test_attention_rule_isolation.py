"""Numbers that are not finite stay in their sample, in the gradients too: tiles of 128 rows hold rows of the next sample, and the other samples' gradients are those of finite neighbours."""
import pytest
import torch

from mini_trainer_b200.ops.torch_ref import TorchOps

from .test_attention_rule import exact, make, rule_of, starts, within

# samples that end inside a tile, at its end and a row behind it; heads in pairs and not, shared key blocks, every kind of score
CASES = [
    ([200, 77, 300], 4, 2, 64, None, 90, None, False),
    ([129, 1, 130], 3, 1, 128, 30.0, None, [60, 1, 130], True),
    ([100, 140, 383], 4, 1, 128, 25.0, 150, None, False),
    ([300, 300, 300], 6, 2, 64, None, None, [0, 9, 299], True),
    ([128, 255, 70], 2, 2, 128, None, None, None, False),
    ([40, 30, 20], 8, 1, 64, 20.0, 16, [0, 30, 5], True),
]
BAD = [float("nan"), float("inf"), -float("inf")]


def poisoned(case, qkv, dout, sample, what, bad, rows):
    """Copies with ``bad`` in ``what`` of one sample: all of its rows, its first or its last."""
    lens, hq, hkv, d = case[:4]
    a = sum(lens[:sample])
    at = {"all": slice(a, a + lens[sample]), "first": slice(a, a + 1), "last": slice(a + lens[sample] - 1, a + lens[sample])}[rows]
    q, g = qkv.clone(), dout.clone()
    column = {"q": slice(0, hq * d), "k": slice(hq * d, (hq + hkv) * d), "v": slice((hq + hkv) * d, None), "qkv": slice(None)}
    if what == "dout":
        g[at] = bad
    elif rows == "all":
        q[at, column[what]] = bad
    else:   # a single number of a row
        q[at, column[what].start or 0] = bad
    return q, g


def check(ops, case, what, rows, device):
    lens, hq, hkv, d = case[:4]
    qkv, dout = make(lens, hq, hkv, d, device=device)
    cu, rule = starts(lens), rule_of(case, device)
    want, bound = exact(qkv, cu, hq, hkv, d, rule_of(case), dout)
    for bad in BAD:
        for s in range(len(lens)):
            q, g = poisoned(case, qkv, dout, s, what, bad, rows)
            o, l = ops.attention(q, None, cu, max(lens), hq, hkv, d, rule=rule)
            grad = ops.attention_bwd(g, q, o, l, None, cu, max(lens), hq, hkv, d, rule=rule)
            for k in set(range(len(lens))) - {s}:
                r = slice(cu[k], cu[k + 1])
                for x, w, b in ((o, want[0], bound[0]), (l.t(), want[1].t(), bound[1].t()), (grad, want[2], bound[2])):
                    within(x[r], w[r], b[r])


@pytest.mark.parametrize("what", ["qkv", "dout"])
def test_plain_backend(what):
    check(TorchOps(), CASES[1], what, "all", "cpu")


@pytest.fixture(scope="module")
def ops():
    from mini_trainer_b200.ops.native import NativeOps
    return NativeOps("cuda:0")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ["all", "first", "last"])
@pytest.mark.parametrize("what", ["qkv", "q", "k", "v", "dout"])
@pytest.mark.parametrize("case", CASES)
def test_gradients_of_the_other_samples(ops, case, what, rows):
    check(ops, case, what, rows, "cuda")
    ops.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("splits,whole", [(2, 1), (4, 5)])
def test_with_key_blocks_that_ctas_share(ops, splits, whole, monkeypatch):
    from mini_trainer_b200.ops import attention_plan
    monkeypatch.setattr(attention_plan, "rule_shares", lambda *a: (splits, whole))
    ops._attn_plan_cache.clear()
    case = ([333, 200, 201], 8, 2, 64, 30.0, 100, [200, 0, 7], True)
    for what in ("qkv", "dout"):
        check(ops, case, what, "all", "cuda")
    ops._attn_plan_cache.clear()
    ops.check_status()


@pytest.mark.gpu
def test_in_a_graph_and_after_it(ops):
    """A replay on inputs that are not finite, one on inputs that are, and eager calls between them."""
    case = CASES[2]
    lens, hq, hkv, d = case[:4]
    qkv, dout = make(lens, hq, hkv, d, device="cuda")
    cu, rule = starts(lens), rule_of(case, "cuda")
    want, bound = exact(qkv, cu, hq, hkv, d, rule_of(case), dout)
    x, g = qkv.clone(), dout.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, l = ops.attention(x, None, cu, max(lens), hq, hkv, d, rule=rule)
        grad = ops.attention_bwd(g, x, o, l, None, cu, max(lens), hq, hkv, d, rule=rule)
    for bad in (None, 1, None):
        x.copy_(qkv), g.copy_(dout)
        if bad is not None:
            x[cu[bad]: cu[bad + 1]] = float("inf")
        for run in range(2):
            graph.replay()
            eo, el = ops.attention(x, None, cu, max(lens), hq, hkv, d, rule=rule)
            eager = ops.attention_bwd(g, x, eo, el, None, cu, max(lens), hq, hkv, d, rule=rule)
            for k in {0, 1, 2} - {bad}:
                r = slice(cu[k], cu[k + 1])
                within(grad[r], want[2][r], bound[2][r])
                within(eager[r], want[2][r], bound[2][r])
    ops.check_status()
