"""How small values may be. The exponentials' reference is a bound of the largest score, not that score, and must not use up the range of the products behind it: scaled by a power of two V gives an
output that is scaled by it, bit for bit, as long as no product falls below the normal numbers of fp32 (2^-126). Probabilities are at least 2^-62 where they count (scores without a bias) or 2^-45."""
import pytest
import torch

from mini_trainer_b200.ops import attention_plan as A
from mini_trainer_b200.ops.attention_rule import AttentionRule

from .test_attention_rule import exact, starts, within


@pytest.fixture(scope="module")
def ops():
    from mini_trainer_b200.ops.native import NativeOps
    return NativeOps("cuda:0")


def opposed(lens, hq, hkv, d, score, seed=0):
    """Queries against the keys' common direction: all products are near ``-score`` times the default scale's inverse."""
    g = torch.Generator().manual_seed(seed)
    T = sum(lens)
    a = torch.ones(d) * (2 * (torch.rand(d, generator=g) < 0.5) - 1)
    x = torch.randn(T, hq + 2 * hkv, d, generator=g)
    x[:, :hq] = -score * d ** -0.5 * a * (1 + 0.02 * torch.randn(T, hq, 1, generator=g))
    x[:, hq: hq + hkv] = a * (1 + 0.02 * torch.randn(T, hkv, 1, generator=g))
    return x.reshape(T, -1).bfloat16()


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["pairs", "one"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("cap,score", [(48.0, 19.0), (42.0, 20.0), (100.0, 20.0), (30.0, 14.0), (48.0, 30.0), (None, 20.0)])
@pytest.mark.parametrize("bias", [False, True])
def test_small_values_under_scores_that_are_all_negative(ops, bias, cap, score, d, form, monkeypatch):
    monkeypatch.setattr(A, "rule_in_pairs", lambda *a: form == "pairs")
    ops._attn_plan_cache.clear()
    lens, hq, hkv = [513, 300], 4, 1
    cu, width = starts(lens), (hq + hkv) * d
    # just under where the bias of 32 keys is too steep for a bound, on both sides; level; and between
    slopes = torch.tensor([0.89, -0.89, 0.0, 0.3], device="cuda") if bias else None
    for prefix, window in ((None, None), ([300, 7], 200)):
        rule = AttentionRule(cap=cap, slopes=slopes, prefix=prefix, window=window)
        qkv = opposed(lens, hq, hkv, d, score).cuda()
        o, l = ops.attention(qkv, None, cu, 513, hq, hkv, d, rule=rule)
        want, bound = exact(qkv, cu, hq, hkv, d, rule)
        within(o, want[0], bound[0])
        within(l, want[1], bound[1])
        small = qkv.clone()
        small[:, width:] *= 2.0 ** (-70 if bias else -40)
        o2, l2 = ops.attention(small, None, cu, 513, hq, hkv, d, rule=rule)
        assert torch.equal(l2, l) and torch.equal(o2.double() * 2.0 ** (70 if bias else 40), o.double())
    ops._attn_plan_cache.clear()
    ops.check_status()


# ------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize("bad", [2.7, float("inf"), "3", torch.tensor(2.5), [4]])
def test_windows_and_prefixes_count_tokens(bad):
    """A part of a token was cut off without a word."""
    with pytest.raises(ValueError, match="counts tokens"):
        AttentionRule(window=bad)
    with pytest.raises(ValueError, match="counts tokens"):
        AttentionRule(prefix=[1, bad])


def test_whole_numbers_of_any_kind_are_taken():
    import numpy
    for k in (5, 5.0, numpy.int32(5), torch.tensor(5)):
        rule = AttentionRule(window=k, prefix=torch.tensor([5, 0]) if torch.is_tensor(k) else [k, 0])
        assert rule.window == rule.keys == 5 and rule.prefix == (5, 0) and rule.key == AttentionRule(window=5, prefix=(5, 0)).key
    assert AttentionRule(window=1 << 40).keys == 1 << 30
