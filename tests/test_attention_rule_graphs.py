"""Attention under a rule in captured graphs: a graph holds its work tables itself, and the backend keeps nothing for it."""
import gc

import pytest
import torch

from mini_trainer_b200.ops.attention_rule import AttentionRule

from .test_attention_rule import exact, host_ops, make, rule_of, slopes_of, starts, within


def test_captured_calls_leave_nothing_behind(monkeypatch):
    from mini_trainer_b200.ops import attention_plan
    made = []
    items = attention_plan.rule_items
    monkeypatch.setattr(attention_plan, "rule_items", lambda *a: made.append(a) or items(*a))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    ops = host_ops()
    qkv, dout = make([200, 130], 4, 2, 64)
    cu, rule = [0, 200, 330], AttentionRule(cap=30.0, window=50, prefix=[3, 0], slopes=slopes_of(4))
    held = None
    for k in range(3):
        out, lse = ops.attention(qkv, None, cu, 200, 4, 2, 64, rule=rule)
        ops.attention_bwd(dout, qkv, out, lse, None, cu, 200, 4, 2, 64, rule=rule)
        names = [n for n, _ in ops.calls[-4:]]
        assert names == ["mtb200_write_ints", "mtb200_attn_rule_fwd_one", "mtb200_write_ints", "mtb200_attn_rule_bwd"]
        assert ops.calls[-4][1][2] == 16 and ops.calls[-3][1][5] == ops.calls[-4][1][0] and ops.calls[-1][1][11] == ops.calls[-2][1][0]   # four blocks, and the launch reads what was written
        kept = {name: len(v) for name, v in vars(ops).items() if isinstance(v, (dict, list)) and name != "calls"}
        assert held is None or kept == held
        held = kept
    assert len(made) == 2   # planned once each way
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    ops.attention(qkv, None, cu, 200, 4, 2, 64, rule=rule)   # an eager call gets a table that is filled now, from the same plan
    assert len(made) == 2 and sorted(map(tuple, ops._cached(cu, (False, 4, 2, 64, 0.125, rule.key, False, 0))[0].tolist())) == [(0, 200, 0, 3), (0, 200, 128, 3), (200, 130, 0, 0), (200, 130, 128, 0)]
    n = len(ops.calls)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert not ops.attention(qkv, None, [0, 0], 0, 4, 2, 64, rule=AttentionRule(window=3))[0].any() and len(ops.calls) == n
    with pytest.raises(ValueError, match="sequence starts"):
        ops.attention(qkv[:300], None, cu, 200, 4, 2, 64, rule=rule)


@pytest.fixture(scope="module")
def ops():
    from mini_trainer_b200.ops.native import NativeOps
    return NativeOps("cuda:0")


def both(ops, case, qkv, dout, rule, cu):
    lens, hq, hkv, d = case[:4]
    o, l = ops.attention(qkv, None, cu, max(lens), hq, hkv, d, rule=rule)
    return o, l, ops.attention_bwd(dout, qkv, o, l, None, cu, max(lens), hq, hkv, d, rule=rule)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 1007, 1008, 1009, 5000])
def test_integers_written_by_launches(ops, n):
    src = torch.randint(-2 ** 31, 2 ** 31, (n,), dtype=torch.int64).int()
    dst = torch.full((n + 8,), 7, dtype=torch.int32, device="cuda")
    ops._call("mtb200_write_ints", dst.data_ptr(), src.data_ptr(), n, ops._st())
    assert torch.equal(dst[:n].cpu(), src) and (dst[n:] == 7).all()


@pytest.mark.gpu
def test_a_graph_outlives_the_plans_it_was_captured_with(ops):
    """Warmed up on the stream that captures, so that there are eager tables for it; they, the plans and the list of starts are gone when the graph runs, and their memory is others'."""
    case = ([391, 129, 640], 4, 2, 64, 30.0, 100, [128, 129, 0], True)
    lens, hq, hkv, d = case[:4]
    qkv, dout = make(lens, hq, hkv, d, device="cuda")
    rule, cu = rule_of(case, "cuda"), starts(lens)
    want, bound = exact(qkv, cu, hq, hkv, d, rule_of(case), dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(ops, case, qkv, dout, rule, cu)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = both(ops, case, qkv, dout, rule, cu)
    with torch.cuda.stream(side):
        again = both(ops, case, qkv, dout, rule, cu)
    side.synchronize()
    ops._attn_plan_cache.clear()
    del cu
    gc.collect()
    with torch.cuda.stream(side):
        junk = [torch.full((k,), -3, dtype=torch.int32, device="cuda") for k in (32, 64, 128, 1024) for _ in range(64)]
    host = [torch.full((k,), -3, dtype=torch.int32).pin_memory() for k in (32, 64, 128, 1024) for _ in range(16)]
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for x, y, w, b in zip(got, again, want, bound):
        within(x, w, b)
        within(y, w, b)
    ops.check_status()
    assert junk and host


@pytest.mark.gpu
def test_captured_again_and_again_holds_no_memory(ops):
    """Tables of more rows than one launch carries; what is allocated, on the device and pinned on the host, is the same after every capture but the first."""
    lens = [70] * 600
    case = (lens, 2, 1, 64, None, 50, None, False)
    qkv, dout = make(lens, 2, 1, 64, device="cuda")
    cu, rule = starts(lens), AttentionRule(window=50)
    eager = both(ops, case, qkv, dout, rule, cu)
    pinned = []
    for _ in range(3):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = both(ops, case, qkv, dout, rule, cu)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])
        k = (2 + 1) * 64
        assert torch.equal(got[2][:, 128:], eager[2][:, 128:]) and (got[2][:, :128].float() - eager[2][:, :128].float()).abs().max() <= 2 ** -7 * eager[2][:, :128].float().abs().max() and k
        del graph, got
        gc.collect()
        torch.cuda.empty_cache()
        pinned.append((torch.cuda.memory_allocated(), torch.cuda.host_memory_stats().get("allocated_bytes.current", 0)))
    assert pinned[0] == pinned[1] == pinned[2]
    ops.check_status()
