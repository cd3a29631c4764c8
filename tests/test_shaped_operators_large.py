"""The operators for shaped scores on minibatches of the framework's own size (60 000 tokens and more), and where offsets pass 2^31 elements: what comes last is compared with 64 bits."""
import pytest
import torch

from mini_trainer_b200.ops.attention_rule import AttentionRule

from . import test_capped_head, test_residual_norm
from .test_attention_rule import exact, make, slopes_of, starts, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from mini_trainer_b200.ops.native import NativeOps
    return NativeOps("cuda:0")


@pytest.fixture(autouse=True)
def memory_given_back():
    yield
    torch.cuda.empty_cache()


def both(ops, qkv, dout, cu, hq, hkv, d, rule):
    longest = max(b - a for a, b in zip(cu[:-1], cu[1:]))
    o, l = ops.attention(qkv, None, cu, longest, hq, hkv, d, rule=rule)
    g = ops.attention_bwd(dout, qkv, o, l, None, cu, longest, hq, hkv, d, rule=rule)
    ops.check_status()
    return o, l, g


def check_samples(got, qkv, dout, cu, hq, hkv, d, rule, which):
    for s in which:
        r = slice(cu[s], cu[s + 1])
        one = AttentionRule(cap=rule.cap, window=rule.window, slopes=rule.slopes, prefix=None if rule.prefix is None else [rule.prefix[s]])
        want, bound = exact(qkv[r], [0, cu[s + 1] - cu[s]], hq, hkv, d, one, dout[r])
        for x, w, b in zip((got[0][r], got[1][:, r], got[2][r]), want, bound):
            within(x, w, b)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cap,window,prefix,bias", [(50.0, 4096, False, False), (None, 1000, True, True), (30.0, None, True, True)])
def test_attention_over_sixty_thousand_tokens(ops, cap, window, prefix, bias, d):
    hq, hkv = 4, 2
    lens = [22000, 129, 18000, 1, 300, 9000, 10001, 128, 441]
    cu = starts(lens)
    qkv, dout = make(lens, hq, hkv, d, device="cuda")
    rule = AttentionRule(cap=cap, window=window, prefix=[n // 3 for n in lens] if prefix else None, slopes=slopes_of(hq, "cuda") if bias else None)
    check_samples(both(ops, qkv, dout, cu, hq, hkv, d, rule), qkv, dout, cu, hq, hkv, d, rule, (1, 3, 4, 7, 8))


def test_attention_behind_two_to_the_31_elements(ops):
    """360 000 rows of 6144: 4.4 GB of q, k and v, of which the last samples lie past 32 bits."""
    hq, hkv, d = 32, 8, 128
    lens = [3999] * 90 + [77, 13]
    cu = starts(lens)
    g = torch.Generator("cuda").manual_seed(1)
    qkv = torch.empty(cu[-1], (hq + 2 * hkv) * d, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    dout = torch.empty(cu[-1], hq * d, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    assert qkv.numel() > 1 << 31
    rule = AttentionRule(cap=30.0, window=200)
    check_samples(both(ops, qkv, dout, cu, hq, hkv, d, rule), qkv, dout, cu, hq, hkv, d, rule, (90, 91))


@pytest.mark.parametrize("T,H", [(70001, 64), (60000, 264)])
def test_norms_over_sixty_thousand_tokens(ops, T, H):
    v = test_residual_norm.inputs(T, H, gated=True, device="cuda")
    test_residual_norm.forward_and_backward(ops, v, 0.5)
    ops.check_status()


def test_norms_behind_two_to_the_31_elements(ops):
    T, H, last = 270000, 8192, 40
    g = torch.Generator("cuda").manual_seed(1)
    x, y = (torch.empty(T, H, dtype=torch.bfloat16, device="cuda").normal_(generator=g) for _ in range(2))
    w = torch.rand(H, device="cuda", generator=g).bfloat16()
    h, z, stats = ops.residual_norm(x, y, w, w, test_residual_norm.EPS)
    v = {"x": x[-last:], "y": y[-last:], "w_post": w, "w_pre": w, "gate": None, "dh": None, "dz": None}
    test_residual_norm.check_forward(v, 1.0, (h[-last:], z[-last:], tuple(s[-last:] for s in stats)))
    dws = [torch.empty_like(w), torch.empty_like(w)]
    dz = x   # any gradient; the weights' sums of all rows are other tests'
    dx, dy, _ = ops.residual_norm_bwd(None, dz, y, h, stats, w, w, *dws)
    few = [torch.empty_like(w), torch.empty_like(w)]
    part = ops.residual_norm_bwd(None, dz[-last:], y[-last:], h[-last:], tuple(s[-last:] for s in stats), w, w, *few)
    assert torch.equal(dx[-last:], part[0]) and torch.equal(dy[-last:], part[1])
    ops.check_status()


def test_head_over_three_chunks(ops):
    x, w, t = test_capped_head.inputs(20000, 64, 1000, device="cuda")
    test_capped_head.check(ops, x, w, t, 30.0, 1.0, 1.0 / 20000)
    ops.check_status()


def test_head_behind_two_to_the_31_elements(ops):
    """A chunk of 8192 rows by 270 000 columns: the last rows against the same rows alone in 64 bits."""
    T, V, last = 8192, 270000, 8
    x, w, t = test_capped_head.inputs(T, 64, V, device="cuda", ignored=0.0)
    t[-1], t[-2] = V - 1, 0
    loss, dx, dw = test_capped_head.run(ops, x, w, t, 30.0, 1.0, 1.0)
    want, bound = test_capped_head.exact(x[-last:], w, t[-last:], 30.0, 1.0, 1.0)
    for got, v, b in ((loss, want[0], bound[0]), (dx, want[1], bound[1])):
        assert ((got[-last:].double().cpu() - v).abs() <= b).all()
    assert torch.isfinite(dw).all()
    ops.check_status()
