"""Attention under a rule (score cap, bias by distance, window, prefix): the plain backend on the CPU and the kernels, against 64 bits.

Tolerances count roundings. A rounding to bf16 is off by at most U = 2^-8 of the value. out = sum p v: every p is rounded once and the sum once;
an exponential is off by at most 1.0e-4 (the cubic), a capped score by 5.1e-7 of itself within the cap and 2^-21 of the cap beyond it. dS = p (dP - delta) c is rounded once, its delta is formed
with the rounded out; dQ, dK and dV are rounded once. ``bounds`` adds these up entry by entry."""
import math
import random

import pytest
import torch

from mini_trainer_b200.ops import attention_plan as A
from mini_trainer_b200.ops.attention_rule import AttentionRule
from mini_trainer_b200.ops.torch_ref import TorchOps

U = torch.finfo(torch.bfloat16).eps / 2
EXP = 1.0e-4 + 2.0 ** -20
CAP = 5.1e-7


def starts(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def make(lens, hq, hkv, d, gain=2.0, seed=0, tail=0, device="cpu", dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens) + tail
    qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=g)
    qkv[:, : hq * d] *= gain
    return qkv.to(dtype).to(device), torch.randn(T, hq * d, generator=g).to(dtype).to(device)


def slopes_of(hq, device="cpu"):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / hq) for h in range(hq)], device=device)


def sees(n, window, prefix):
    """Written from the definition, pair by pair of index grids."""
    i = torch.arange(n).view(n, 1).expand(n, n)
    j = i.t()
    return ((j <= i) & ((i - j) < (window or n + 1))) | (j < prefix)


def exact(qkv, cu, hq, hkv, d, rule, dout=None, scale=None):
    """``(values, bounds)`` of out, lse and (with ``dout``) dqkv in 64 bits; rows behind the last sample are zero."""
    x = qkv.double().cpu().view(qkv.shape[0], hq + 2 * hkv, d)
    T, g = x.shape[0], hq // hkv
    scale = d ** -0.5 if scale is None else scale
    out, lse, grad = torch.zeros(T, hq, d, dtype=torch.float64), torch.zeros(hq, T, dtype=torch.float64), torch.zeros_like(x)
    bo, bl, bg = torch.zeros_like(out), torch.zeros_like(lse), torch.zeros_like(x)
    for s, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
        n = b - a
        if n == 0:
            continue
        see = sees(n, rule.window, rule.prefix[s] if rule.prefix is not None else 0)
        dist = (torch.arange(n)[:, None] - torch.arange(n)[None]).abs().double()
        for h in range(hq):
            q, k, v = x[a:b, h], x[a:b, hq + h // g], x[a:b, hq + hkv + h // g]
            z = (q @ k.t()) * scale
            c = torch.ones_like(z)
            if rule.cap:
                t = torch.tanh(z / rule.cap)
                z, c = rule.cap * t, 1 - t * t
            size = z.abs()
            if rule.slopes is not None:
                z = z - rule.slopes[h].double().cpu() * dist
                size = size + rule.slopes[h].double().cpu() * dist
            z = z.masked_fill(~see, -math.inf)
            l = torch.logsumexp(z, 1)
            p = torch.exp(z - l[:, None])
            o = p @ v
            # a score's own error: the product of rows in fp32, the cap's polynomial, its place in the bias
            dz = (2.0 ** -18 * (q.abs() @ k.abs().t()) * scale + CAP * size + 2.0 ** -21 * (rule.cap or 0.0) + 2.0 ** -21 * size).masked_fill(~see, 0.0)
            rel = EXP + dz + (p * (dz + EXP)).sum(1, keepdim=True)   # of p, normalised
            out[a:b, h], lse[h, a:b] = o, l
            eo = (p * (U + rel)) @ v.abs() + U * o.abs()
            bo[a:b, h], bl[h, a:b] = 1.1 * eo + 1e-7, (p * (dz + EXP)).sum(1) + 2.0 ** -20 * l.abs() + 1e-6
            if dout is None:
                continue
            do = dout.double().cpu().view(T, hq, d)[a:b, h]
            dp, delta = do @ v.t(), (do * o).sum(1, keepdim=True)
            ds = p * (dp - delta) * c * scale
            edelta = (do.abs() * 1.1 * eo).sum(1, keepdim=True) + 2.0 ** -18 * (do.abs() * o.abs()).sum(1, keepdim=True)
            eds = (U + 2 * rel) * ds.abs() + p * c * scale * (edelta + 2.0 ** -18 * (do.abs() @ v.abs().t())) + (3 * CAP + 2.0 ** -20) * p * (dp - delta).abs() * scale
            grad[a:b, h] += ds @ k
            grad[a:b, hq + h // g] += ds.t() @ q
            grad[a:b, hq + hkv + h // g] += p.t() @ do
            bg[a:b, h] += eds @ k.abs()
            bg[a:b, hq + h // g] += eds.t() @ q.abs()
            bg[a:b, hq + hkv + h // g] += (p * (U + 2 * rel)).t() @ do.abs()
    bg = 1.1 * bg + U * grad.abs() + 1e-6
    return (out.view(T, -1), lse, grad.view(T, -1)), (bo.view(T, -1), bl, bg.view(T, -1))


def within(got, want, bound):
    over = (got.double().cpu() - want).abs() - bound
    assert torch.isfinite(got).all()
    assert over.max() <= 0, f"{int((over > 0).sum())} of {over.numel()} entries off by more than the roundings, the worst by {over.max():.3g} (bound {bound.flatten()[over.argmax()]:.3g})"


# (lengths, query heads, kv heads, head_dim, cap, window, prefixes, bias)
CASES = [
    ([1], 1, 1, 64, 30.0, None, None, False),
    ([5], 2, 1, 128, None, 1, None, False),
    ([127], 4, 1, 128, 50.0, None, None, False),
    ([128, 1, 129], 2, 2, 64, None, 2, None, True),
    ([0, 130, 0, 257, 1], 4, 2, 64, 20.0, 64, None, False),
    ([300], 3, 1, 64, None, 127, None, False),
    ([300], 3, 1, 128, None, 128, None, True),
    ([513], 2, 2, 128, None, 129, None, False),
    ([700], 6, 2, 64, 25.0, 200, None, True),
    ([400, 260], 2, 1, 128, None, None, [0, 260], False),
    ([400, 260], 2, 1, 64, None, None, [1, 127], True),
    ([391, 129], 3, 3, 64, 30.0, None, [128, 129], True),
    ([650, 70], 4, 1, 128, 30.0, 100, [300, 3], True),
    ([900], 2, 2, 64, None, 40, [129], False),
    ([640], 5, 1, 64, 40.0, 1000, [640], False),
    ([385, 511], 1, 1, 128, 15.0, 256, [200, 0], False),
]


def rule_of(case, device="cpu"):
    lens, hq, hkv, d, cap, window, prefix, bias = case
    return AttentionRule(cap=cap, window=window, prefix=prefix, slopes=slopes_of(hq, device) if bias else None)


# ------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize("case", CASES[:13])
def test_plain_backend_against_64_bits(case):
    lens, hq, hkv, d = case[:4]
    rule, cu = rule_of(case), starts(lens)
    qkv, dout = make(lens, hq, hkv, d, tail=3)
    (out, lse, grad), (bo, bl, bg) = exact(qkv, cu, hq, hkv, d, rule, dout)
    ops = TorchOps()
    o, l = ops.attention(qkv, None, cu, max(lens), hq, hkv, d, rule=rule)
    within(o, out, bo)
    within(l, lse, bl)
    within(ops.attention_bwd(dout, qkv, o, l, None, cu, max(lens), hq, hkv, d, rule=rule), grad, bg)


def test_formula_of_the_gradient_against_differences():
    """The derivative along a direction, by differences in 64 bits: 2^-17 apart the formula's third derivative is below 1e-8 of it."""
    case = CASES[12]
    lens, hq, hkv, d = case[:4]
    rule, cu = rule_of(case), starts(lens)
    qkv, dout = make(lens, hq, hkv, d, gain=1.0, dtype=torch.float64)
    u = torch.randn(qkv.shape, generator=torch.Generator().manual_seed(5), dtype=torch.float64)
    (_, _, grad), _ = exact(qkv, cu, hq, hkv, d, rule, dout)
    h = 2.0 ** -17
    f = [(exact(qkv + e * u, cu, hq, hkv, d, rule)[0][0] * dout).sum() for e in (h, -h)]
    assert abs((f[0] - f[1]) / (2 * h) - (grad * u).sum()) <= 1e-6 * (grad.abs() * u.abs()).sum()


def test_without_options_a_rule_is_the_causal_form():
    lens, hq, hkv, d = [70, 1, 130], 4, 2, 64
    qkv, dout = make(lens, hq, hkv, d)
    ops, cu = TorchOps(), starts(lens)
    a, b = ops.attention(qkv, None, cu, 130, hq, hkv, d), ops.attention(qkv, None, cu, 130, hq, hkv, d, rule=AttentionRule())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(ops.attention_bwd(dout, qkv, *a, None, cu, 130, hq, hkv, d), ops.attention_bwd(dout, qkv, *a, None, cu, 130, hq, hkv, d, rule=AttentionRule(window=131)))


@pytest.mark.parametrize("bad,needle", [
    (dict(cap=0.0), "positive"), (dict(cap=-3.0), "positive"), (dict(cap=float("inf")), "positive"), (dict(cap=float("nan")), "positive"),
    (dict(window=0), "window"), (dict(window=-5), "window")])
def test_rules_that_mean_nothing_are_refused(bad, needle):
    with pytest.raises(ValueError, match=needle):
        AttentionRule(**bad)


def test_prefixes_and_starts_are_checked_against_the_batch():
    qkv, _ = make([5, 6], 2, 1, 64)
    ops = TorchOps()
    for prefix in ([5], [6, 6], [-1, 0], [5, 7]):
        with pytest.raises(ValueError, match="prefix"):
            ops.attention(qkv, None, [0, 5, 11], 6, 2, 1, 64, rule=AttentionRule(prefix=prefix))
    for cu in ([0, 5, 12], [1, 5, 11], [0, 6, 5], []):
        with pytest.raises(ValueError, match="sequence starts"):
            ops.attention(qkv, None, cu, 6, 2, 1, 64, rule=AttentionRule(window=3))
    for slopes in (torch.ones(3), torch.ones(2, dtype=torch.float64), torch.ones(4)[::2], torch.ones(2, 1)):
        with pytest.raises(ValueError, match="slopes"):
            ops.attention(qkv, None, [0, 5, 11], 6, 2, 1, 64, rule=AttentionRule(slopes=slopes))


@pytest.mark.parametrize("seed", range(40))
def test_work_tables_hold_every_pair_that_is_seen(seed):
    """The tiles that the kernels derive from a row of the table cover exactly the blocks with a visible pair (forward: those of a pair of row blocks
    may be one more), and every tile called whole is."""
    import random
    r = random.Random(seed)
    n = r.randint(1, 900)
    window, prefix = r.choice([1, 2, 127, 128, 129, r.randint(1, 1000), 1 << 30]), r.choice([0, 0, 1, 127, 128, 129, r.randint(0, n), n])
    prefix = min(prefix, n)
    see = sees(n, window, prefix)
    blocks = -(-n // 128)
    tile = [[bool(see[128 * i: 128 * i + 128, 128 * j: 128 * j + 128].any()) for j in range(blocks)] for i in range(blocks)]
    for i in range(blocks):
        tiles = -(-prefix // 128)
        frm = max(tiles, max(0, 128 * i + 1 - window) // 128)
        mine = list(range(tiles)) + list(range(frm, i + 1))
        assert len(mine) == A.key_tiles(128 * i, window, prefix) == len(set(mine)) and sorted(mine) == [j for j in range(blocks) if tile[i][j]]
        assert A.query_blocks(128 * i, n, window, prefix) == sum(tile[k][i] for k in range(blocks))
    for block, backward in ((128, False), (256, False), (128, True)):
        items = A.rule_items([0, 0, n, n], [0, prefix, 0], window, block, backward)
        assert sorted(it[3] for it in items) == list(range(0, n, block)) and all(it[1:3] == (0, n) and it[4] == prefix and it[0] > 0 for it in items)
        assert [it[0] for it in items] == sorted((it[0] for it in items), reverse=True)


def test_backward_of_a_rule_without_edges_is_planned_as_the_causal_one():
    for lens, hq, hkv, d in (([5987], 12, 2, 128), ([128] * 16, 32, 8, 128), ([4313], 32, 8, 128), ([300] * 41, 16, 4, 64)):
        cu = starts(lens)
        work = [it[0] for it in A.rule_items(cu, [0] * len(lens), 1 << 30, 128, True)]
        blocks = A.blocks_per_sequence(cu)
        splits = A.backward_splits(blocks, hq, hkv, 148, hq // hkv)
        assert A.rule_splits(work, hq, hkv, 148, hq // hkv) == splits
        assert A.rule_in_order(work, hq, hkv, d, splits) == A.backward_in_order(blocks, hq, hkv, d, splits)
    assert A.rule_splits([], 4, 1, 148, 4) == 1


def test_only_the_last_part_of_a_launch_is_shared():
    four = lambda blocks: 4
    assert A.rule_shares([9] * 64, 32, 8, 148, four) == (2, 55)          # 512 key blocks of one length: three times the GPU, and 68 shared by two
    assert A.rule_shares([9] * 64, 32, 8, 148, lambda blocks: 1) == (1, 0)   # without room for partials
    assert A.rule_shares([9] * 74, 32, 8, 148, four) == (1, 0)           # four times the GPU exactly
    assert A.rule_shares([9] * 64, 8, 8, 148, four) == (1, 0)            # a head has nothing to share
    assert A.rule_shares([], 32, 8, 148, four) == (1, 0)
    for seed in range(40):
        r = random.Random(seed)
        work = sorted((r.randint(1, 40) for _ in range(r.randint(1, 120))), reverse=True)
        hkv, group = r.choice([1, 2, 4, 8]), r.choice([1, 2, 3, 4, 8])
        most = r.randint(1, 8)
        splits, whole = A.rule_shares(work, hkv * group, hkv, 148, lambda blocks: min(group, most))
        assert 1 <= splits <= min(group, most) and 0 <= whole < len(work) and (splits > 1 or whole == 0)
        if whole == 0:
            assert splits == A.rule_splits(work, hkv * group, hkv, 148, min(group, most))


def test_forward_of_a_rule_without_edges_takes_the_causal_form():
    for lens, hq, hkv, d in (([2048], 16, 4, 64), ([16384], 2, 1, 128), ([300] * 41, 16, 4, 64), ([128] * 100, 32, 8, 128), ([5000] * 4, 9, 3, 128), ([1024], 14, 2, 128), ([700] * 30, 3, 1, 64)):
        cu = starts(lens)
        work = [it[0] for it in A.rule_items(cu, [0] * len(lens), 1 << 30, 128, False)]
        pairs = [(it[0], it[3] + 128 < it[2]) for it in A.rule_items(cu, [0] * len(lens), 1 << 30, 256, False)]
        assert A.rule_in_pairs(work, lambda: pairs, hq, hkv, d, 148) == A.forward_in_pairs(A.blocks_per_sequence(cu), hq, hkv, d, 148)
    assert A.rule_in_pairs([], list, 4, 1, 64, 148)


def host_ops():
    from .test_native_host import make_ops
    ops = make_ops()
    ops.attention_impl, ops._captured = "native", []
    ops._move_table = lambda rows: torch.tensor(rows, dtype=torch.int32)
    ops._index = None
    return ops


def test_kernel_calls_get_the_rule_and_its_table(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    ops = host_ops()
    qkv, dout = make([200, 130], 4, 2, 64, tail=6)
    cu = [0, 200, 330]
    rule = AttentionRule(cap=30.0, window=50, prefix=[3, 0], slopes=slopes_of(4))
    out, lse = ops.attention(qkv, None, cu, 200, 4, 2, 64, rule=rule)
    name, args = ops.calls[-1]
    assert name == "mtb200_attn_rule_fwd_one" and args[6:12] == (4, 336, 330, 4, 2, 64) and args[13:15] == (30.0, 50) and args[15] == rule.slopes.data_ptr()
    assert not out[330:].any() and not lse[:, 330:].any()
    table = ops._cached(cu, (False, 4, 2, 64, 0.125, rule.key, False, 0))[0]
    assert sorted(map(tuple, table.tolist())) == [(0, 200, 0, 3), (0, 200, 128, 3), (200, 130, 0, 0), (200, 130, 128, 0)]
    ops.attention(qkv, None, cu, 200, 4, 2, 64, rule=AttentionRule(window=50, prefix=[4, 0]))   # another prefix is another table
    assert ops.calls[-1][1][5] != args[5]
    ops.attention_bwd(dout, qkv, out, lse, None, cu, 200, 4, 2, 64, rule=rule)
    assert ops.calls[-1][0] == "mtb200_attn_rule_bwd" and ops.calls[-1][1][12:18] == (4, 336, 330, 4, 2, 64)
    n = len(ops.calls)
    out, lse = ops.attention(qkv, None, [0, 0], 0, 4, 2, 64, rule=rule.__class__(window=2))   # samples without tokens
    assert len(ops.calls) == n and not out.any() and not ops.attention_bwd(dout, qkv, out, lse, None, [0], 0, 4, 2, 64, rule=AttentionRule(cap=2.0)).any()


def test_kernel_calls_refuse_what_they_cannot_address(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    ops = host_ops()
    qkv, dout = make([64], 4, 2, 64)
    rule, cu = AttentionRule(cap=30.0), [0, 64]
    out, lse = ops.attention(qkv, None, cu, 64, 4, 2, 64, rule=rule)

    def refused(needle, call):
        n = len(ops.calls)
        with pytest.raises(ValueError, match=needle):
            call()
        assert len(ops.calls) == n

    wide = torch.zeros(64, 516, dtype=torch.bfloat16)
    for bad in (qkv.float(), qkv[:, :-64], wide[:, 1:513], wide[:, :512], qkv.t().contiguous().t(), qkv[None], torch.zeros(64 * 512 + 4, dtype=torch.bfloat16)[4:].view(64, 512)):
        refused("expected bf16 rows|sequence starts", lambda: ops.attention(bad, None, cu, 64, 4, 2, 64, rule=rule))
    refused("head dimensions", lambda: ops.attention(qkv, None, cu, 64, 2, 1, 128 + 128, rule=rule))
    refused("share", lambda: ops.attention(qkv, None, cu, 64, 4, 3, 64, rule=rule))
    refused("scale", lambda: ops.attention(qkv, None, cu, 64, 4, 2, 64, scale=0.0, rule=rule))
    refused("scale", lambda: ops.attention(qkv, None, cu, 64, 4, 2, 64, scale=-1.0, rule=AttentionRule(window=4)))
    refused("caps of", lambda: ops.attention(qkv, None, cu, 64, 4, 2, 64, rule=AttentionRule(cap=1e6)))
    refused("caps of", lambda: ops.attention(qkv, None, cu, 64, 4, 2, 64, rule=AttentionRule(cap=1e-6)))
    refused("sequence starts", lambda: ops.attention(qkv, None, [0, 65], 64, 4, 2, 64, rule=rule))
    refused("prefix", lambda: ops.attention(qkv, None, cu, 64, 4, 2, 64, rule=AttentionRule(prefix=[65])))
    refused("slopes", lambda: ops.attention(qkv, None, cu, 64, 4, 2, 64, rule=AttentionRule(slopes=torch.ones(2))))
    refused("expected bf16 rows", lambda: ops.attention_bwd(dout[:32], qkv, out, lse, None, cu, 64, 4, 2, 64, rule=rule))
    refused("expected bf16 rows", lambda: ops.attention_bwd(dout, qkv, out.float(), lse, None, cu, 64, 4, 2, 64, rule=rule))
    refused("lse", lambda: ops.attention_bwd(dout, qkv, out, lse.double(), None, cu, 64, 4, 2, 64, rule=rule))
    refused("lse", lambda: ops.attention_bwd(dout, qkv, out, lse[:2], None, cu, 64, 4, 2, 64, rule=rule))
    ops.attention_impl = "flash_attn"
    refused("library attention", lambda: ops.attention(qkv, None, cu, 64, 4, 2, 64, rule=rule))


# ------------------------------------------------------------------------------------------ GPU
@pytest.fixture(scope="module")
def ops():
    from mini_trainer_b200.ops.native import NativeOps
    return NativeOps("cuda:0")


def run(ops, case, qkv, dout, scale=None):
    lens, hq, hkv, d = case[:4]
    rule, cu = rule_of(case, "cuda"), starts(lens)
    o, l = ops.attention(qkv, None, cu, max(lens), hq, hkv, d, scale=scale, rule=rule)
    g = ops.attention_bwd(dout, qkv, o, l, None, cu, max(lens), hq, hkv, d, scale=scale, rule=rule)
    ops.check_status()
    return o, l, g


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["pairs", "one"])
@pytest.mark.parametrize("gain", [1.0, 40.0])   # scores within the cap, and far beyond it
@pytest.mark.parametrize("case", CASES)
def test_kernels_against_64_bits(ops, case, gain, form, monkeypatch):
    monkeypatch.setattr(A, "rule_in_pairs", lambda *a: form == "pairs")
    ops._attn_plan_cache.clear()
    lens, hq, hkv, d = case[:4]
    qkv, dout = make(lens, hq, hkv, d, gain=gain, tail=5, device="cuda")
    want, bound = exact(qkv, starts(lens), hq, hkv, d, rule_of(case), dout)
    for g, w, b in zip(run(ops, case, qkv, dout), want, bound):
        within(g, w, b)


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["pairs", "one"])
@pytest.mark.parametrize("d", [64, 128])
def test_every_combination_on_ragged_samples(ops, d, form, monkeypatch):
    import itertools
    monkeypatch.setattr(A, "rule_in_pairs", lambda *a: form == "pairs")
    ops._attn_plan_cache.clear()
    for cap, window, prefix, bias, (hq, hkv) in itertools.product([None, 35.0], [None, 77], [None, [0, 140, 9]], [False, True], [(4, 2), (3, 1)]):
        case = ([201, 333, 45], hq, hkv, d, cap, window, prefix, bias)
        qkv, dout = make(case[0], hq, hkv, d, seed=hq, device="cuda")
        want, bound = exact(qkv, starts(case[0]), hq, hkv, d, rule_of(case), dout)
        for g, w, b in zip(run(ops, case, qkv, dout), want, bound):
            within(g, w, b)


@pytest.mark.gpu
@pytest.mark.parametrize("splits,whole", [(2, 0), (2, 1), (3, 4), (4, 5), (2, 6)])
@pytest.mark.parametrize("d", [64, 128])
def test_key_blocks_shared_from_some_on(ops, d, splits, whole, monkeypatch):
    """The first key blocks of a table with a CTA each, the others' heads divided over several, with every kind of score."""
    monkeypatch.setattr(A, "rule_shares", lambda *a: (splits, whole))
    ops._attn_plan_cache.clear()
    for cap, window, prefix, bias in ((None, 150, None, False), (30.0, None, [7, 130], False), (None, None, None, True), (30.0, 100, [200, 0], True)):
        case = ([333, 401], 8, 2, d, cap, window, prefix, bias)   # seven key blocks, two kv heads
        qkv, dout = make(case[0], 8, 2, d, seed=splits, device="cuda")
        want, bound = exact(qkv, starts(case[0]), 8, 2, d, rule_of(case), dout)
        for g, w, b in zip(run(ops, case, qkv, dout), want, bound):
            within(g, w, b)
    ops._attn_plan_cache.clear()


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["pairs", "one"])
@pytest.mark.parametrize("cap", [None, 25.0, 120.0])
def test_slopes_of_every_size_and_sign(ops, cap, form, monkeypatch):
    """Zero, so steep that only the query itself counts, and negative ones, which favour the far end; a prefix with keys behind the query."""
    monkeypatch.setattr(A, "rule_in_pairs", lambda *a: form == "pairs")
    ops._attn_plan_cache.clear()
    lens, hq, hkv, d = [400, 131], 6, 2, 64
    cu, qkv_dout = starts(lens), make(lens, hq, hkv, d, gain=3.0, device="cuda")
    for prefix, window in ((None, None), ([390, 7], 50)):
        slopes = torch.tensor([0.0, 1e-4, 0.6, 4.0, 60.0, -0.05], device="cuda")
        rule = AttentionRule(cap=cap, window=window, prefix=prefix, slopes=slopes)
        qkv, dout = qkv_dout
        o, l = ops.attention(qkv, None, cu, 400, hq, hkv, d, rule=rule)
        g = ops.attention_bwd(dout, qkv, o, l, None, cu, 400, hq, hkv, d, rule=rule)
        want, bound = exact(qkv, cu, hq, hkv, d, rule, dout)
        for x, w, b in zip((o, l, g), want, bound):
            within(x, w, b)
    ops.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [0.02, 1.0, 60.0, 300.0])
def test_caps_of_every_size(ops, cap):
    """Around the border between the polynomials, the exact form, and caps beyond the polynomials' coefficients."""
    lens, hq, hkv, d = [200, 129], 2, 1, 128
    for gain in (0.2, 4.0, 14.0):
        case = (lens, hq, hkv, d, cap, None, None, False)
        qkv, dout = make(lens, hq, hkv, d, gain=gain, device="cuda")
        want, bound = exact(qkv, starts(lens), hq, hkv, d, rule_of(case), dout)
        for x, w, b in zip(run(ops, case, qkv, dout), want, bound):
            within(x, w, b)


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(ops):
    """One batch, the same host list, on streams that do not wait for each other: each fills a work table of its own."""
    case = ([900, 77, 300], 6, 2, 128, 30.0, 300, [100, 0, 300], True)
    qkv, dout = make(case[0], 6, 2, 128, device="cuda")
    rule, cu = rule_of(case, "cuda"), starts(case[0])
    want = ops.attention(qkv, None, cu, 900, 6, 2, 128, rule=rule)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                o, l = ops.attention(qkv, None, cu, 900, 6, 2, 128, rule=rule)
                got.append((o, l, ops.attention_bwd(dout, qkv, o, l, None, cu, 900, 6, 2, 128, rule=rule)))
    torch.cuda.synchronize()
    exactly, bound = exact(qkv, cu, 6, 2, 128, rule_of(case), dout)
    for o, l, g in got:
        assert torch.equal(o, want[0]) and torch.equal(l, want[1])
        within(g, exactly[2], bound[2])
    ops.check_status()


@pytest.mark.gpu
def test_gradient_along_a_direction_against_differences(ops):
    case = CASES[12]
    lens, hq, hkv, d = case[:4]
    rule, cu = rule_of(case), starts(lens)
    qkv, dout = make(lens, hq, hkv, d, gain=1.0, device="cuda")
    _, _, grad = run(ops, case, qkv, dout)
    u = torch.randn(qkv.shape, generator=torch.Generator().manual_seed(5), dtype=torch.float64)
    h, x = 2.0 ** -17, qkv.double().cpu()
    f = [(exact(x + e * u, cu, hq, hkv, d, rule)[0][0] * dout.double().cpu()).sum() for e in (h, -h)]
    _, (_, _, bg) = exact(qkv, cu, hq, hkv, d, rule, dout)
    assert abs((f[0] - f[1]) / (2 * h) - (grad.double().cpu() * u).sum()) <= (bg * u.abs()).sum()


@pytest.mark.gpu
def test_without_options_a_rule_agrees_with_the_causal_kernels(ops):
    for lens, hq, hkv, d in (([700, 3, 150], 4, 2, 128), ([513, 129], 3, 1, 64)):
        qkv, dout = make(lens, hq, hkv, d, device="cuda")
        cu = starts(lens)
        a = ops.attention(qkv, None, cu, max(lens), hq, hkv, d)
        case = (lens, hq, hkv, d, None, None, None, False)
        o, l, g = run(ops, case, qkv, dout)
        want, bound = exact(qkv, cu, hq, hkv, d, AttentionRule(), dout)
        for x, y, b in zip((*a, ops.attention_bwd(dout, qkv, *a, None, cu, max(lens), hq, hkv, d)), (o, l, g), bound):
            assert ((x.double() - y.double()).abs().cpu() <= 2 * b).all()
        ops.check_status()


@pytest.mark.gpu
def test_long_sample_through_a_window(ops):
    """Behind the first window every row sees as many keys: against the plain form on the samples' ends, where a shorter sample gives the same rows."""
    n, w, hq, hkv, d = 20000, 500, 2, 1, 128
    case = ([n], hq, hkv, d, 30.0, w, None, True)
    qkv, dout = make([n], hq, hkv, d, device="cuda")
    dout[: n - 700] = 0
    o, l, g = run(ops, case, qkv, dout)
    m = 700 + w + 128   # rows that the last 700 see, and some more
    short = ([m], hq, hkv, d, 30.0, w, None, True)
    want, bound = exact(qkv[-m:], [0, m], hq, hkv, d, rule_of(short), dout[-m:])
    for a, t, b, sl in ((o, want[0], bound[0], slice(-700, None)), (g, want[2], bound[2], slice(-700 - w + 1, None))):
        within(a[sl], t[sl], b[sl])
    within(l[:, -700:], want[1][:, -700:], bound[1][:, -700:])
    assert not g[: n - 700 - w].any()   # no query with a gradient sees these keys


@pytest.mark.gpu
def test_strided_rows_and_rows_behind_the_last_sample(ops):
    """Activations and gradients in the middle of wider buffers; what lies behind the last sample is garbage that nothing reads."""
    case = ([130, 260], 4, 2, 64, 30.0, 90, [5, 200], True)
    lens, hq, hkv, d = case[:4]
    qkv, dout = make(lens, hq, hkv, d, tail=41, device="cuda")
    qkv[390:], dout[390:] = float("nan"), float("inf")
    big, bigd = torch.full((431, 8 * 64 + 24), float("nan"), dtype=torch.bfloat16, device="cuda"), torch.zeros(431, 4 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    big[:, 16:528], bigd[:, :256] = qkv, dout
    o, l, g = run(ops, case, big[:, 16:528], bigd[:, :256])
    rule, cu = rule_of(case), starts(lens)
    want, bound = exact(qkv[:390], cu, hq, hkv, d, rule, dout[:390])
    for a, w, b in ((o, want[0], bound[0]), (l.t(), want[1].t(), bound[1].t()), (g, want[2], bound[2])):
        within(a[:390], w, b)
        assert not a[390:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["pairs", "one"])
@pytest.mark.parametrize("case", [([200, 77, 300], 4, 2, 64, None, 90, None, False), ([129, 1, 130], 3, 1, 128, 30.0, None, [60, 1, 130], True),
                                  ([100, 140, 383], 4, 1, 128, 25.0, 150, None, False), ([300, 300, 300], 6, 2, 64, None, None, [0, 9, 299], True)])
def test_infinities_of_one_sample_stay_there(ops, case, form, monkeypatch):
    """Tiles at a sample's end hold rows of the next one: the other samples' outputs are those of finite neighbours."""
    monkeypatch.setattr(A, "rule_in_pairs", lambda *a: form == "pairs")
    ops._attn_plan_cache.clear()
    lens, hq, hkv, d = case[:4]
    qkv, _ = make(lens, hq, hkv, d, device="cuda")
    cu = starts(lens)
    want, bound = exact(qkv, cu, hq, hkv, d, rule_of(case))
    for bad in (float("nan"), float("inf"), -float("inf")):
        for s in range(3):
            q = qkv.clone()
            q[cu[s]: cu[s + 1]] = bad
            o, l = ops.attention(q, None, cu, max(lens), hq, hkv, d, rule=rule_of(case, "cuda"))
            ops.check_status()
            for k in {0, 1, 2} - {s}:
                rows = slice(cu[k], cu[k + 1])
                for x, w, b in ((o, want[0], bound[0]), (l.t(), want[1].t(), bound[1].t())):
                    within(x[rows], w[rows], b[rows])


@pytest.mark.gpu
def test_rules_on_side_streams_and_in_captured_graphs(ops):
    """Two graphs captured from one backend, replayed in turn with eager calls between them, on other inputs than they were captured with."""
    cases = [CASES[8], CASES[12]]
    graphs, held = [], []
    for case in cases:
        lens, hq, hkv, d = case[:4]
        qkv, dout = make(lens, hq, hkv, d, device="cuda")
        rule, cu = rule_of(case, "cuda"), starts(lens)
        run(ops, case, qkv, dout)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, l = ops.attention(qkv, None, cu, max(lens), hq, hkv, d, rule=rule)
            g = ops.attention_bwd(dout, qkv, o, l, None, cu, max(lens), hq, hkv, d, rule=rule)
        graphs.append(graph)
        held.append((case, qkv, dout, o, l, g, rule))   # a graph reads its inputs where they were: the slopes live as long as it does
    ops._attn_plan_cache.clear()
    for seed in (3, 4):
        side = torch.cuda.Stream()
        for graph, (case, qkv, dout, o, l, g, _) in zip(graphs, held):
            lens, hq, hkv, d = case[:4]
            a, b = make(lens, hq, hkv, d, seed=seed, device="cuda")
            qkv.copy_(a)
            dout.copy_(b)
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                eager = run(ops, case, a, b)
            graph.replay()
            torch.cuda.synchronize()
            want, bound = exact(a, starts(lens), hq, hkv, d, rule_of(case), b)
            for x, y, w, t in zip((o, l, g), eager, want, bound):
                within(x, w, t)
                within(y, w, t)


@pytest.mark.gpu
def test_forward_is_the_same_bit_for_bit_twice(ops):
    case = ([900, 77], 6, 2, 128, 30.0, 300, [100, 0], True)
    qkv, dout = make(case[0], 6, 2, 128, device="cuda")
    a, b = run(ops, case, qkv, dout), run(ops, case, qkv, dout)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    k = (6 + 2) * 128   # dK and dV have one writer; dQ's tiles are added in the order they arrive
    assert torch.equal(a[2][:, 6 * 128:], b[2][:, 6 * 128:]) and k


@pytest.mark.gpu
def test_a_table_that_does_not_fit_the_batch_is_reported(ops):
    qkv, dout = make([64], 2, 1, 64, device="cuda")
    out, lse = torch.zeros(64, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 64, device="cuda")
    for row in ([0, 65, 0, 0], [-1, 64, 0, 0], [0, 64, 64, 0], [0, 64, 0, 65], [0, 64, 0, -1]):
        plan = torch.tensor([row], dtype=torch.int32, device="cuda")
        for name, tail in (("mtb200_attn_rule_fwd", (0,)), ("mtb200_attn_rule_fwd_one", ())):
            ops._call(name, qkv.data_ptr(), qkv.stride(0), out.data_ptr(), out.stride(0), lse.data_ptr(), plan.data_ptr(), 1, 64, 64, 2, 1, 64, *tail,
                      0.125, 0.0, 5, None, ops.status.data_ptr(), ops._st())
            with pytest.raises(RuntimeError, match="work item"):
                ops.check_status()
    assert not out.any() and not lse.any()
