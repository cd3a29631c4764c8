"""Which form of the attention kernels a packed batch runs on, from the lengths of its sequences alone.

A launch is a list of units (CTAs, or pairs of query tiles of a persistent CTA) of known length, dealt to the SMs longest first.
``finish_time`` bounds when the last one is done; the forms and splits are compared by it. The unit times of the forward are measured
on a B200 (microseconds; 630 batches of one to 300 sequences of 16 to 16384 tokens, 1 to 32 heads): over these the choice costs 0.2 % on
average against the better form, always pairs would cost 19 % (at most 90 %), always one tile 14 % (at most 125 %).
"""
from __future__ import annotations

from collections import Counter

BLOCK = 128   # rows of a query block, keys of a key block

# Forward, per head_dim. one: launch, a CTA, a key tile of it. two: launch; a pair of heads, a key tile of both; a pair of row
# blocks, a key tile of both; a row block without partner, a key tile of it.
_ONE = {64: (1.87, 4.1, 0.84), 128: (1.88, 5.55, 0.94)}
_TWO = {64: (3.98, 2.81, 1.65, 3.4, 1.75, 1.89, 1.61), 128: (3.32, 5.27, 1.72, 4.83, 1.66, 3.47, 1.66)}

# Backward, in iterations (one query block of one head, 1.5 us at head_dim 64 and 2.7 at 128): a CTA's start and end (loads of K and V,
# stores of dK and dV), and what a partial sum of dK and dV adds to it.
_BWD_CTA, _BWD_PARTIAL = 5.0, 2.0


def finish_time(units: list, workers: int) -> float:
    """Lower bound, and in practice about the value, of the finish time of ``units`` [(time, count)] on ``workers``: the longest
    unit, the mean load, and k units on one worker as soon as there are more than (k - 1) * workers of at least that length."""
    units = sorted(units, reverse=True)
    t = max(units[0][0], sum(c * n for c, n in units) / workers)
    seen, k = 0, 2
    for c, n in units:
        seen += n
        while k <= 8 and seen > (k - 1) * workers:
            t = max(t, k * c)
            k += 1
    return t


def blocks_per_sequence(cu_host) -> list:
    return [-(-(b - a) // BLOCK) for a, b in zip(cu_host[:-1], cu_host[1:]) if b > a]


def _with_at_least(blocks: list) -> list:
    """``out[n]``: sequences of at least ``n`` blocks (``out[0]`` unused)."""
    out = [0] * (max(blocks) + 2)
    for b in blocks:
        out[b] += 1
    for n in range(len(out) - 2, 0, -1):
        out[n] += out[n + 1]
    return out


def forward_in_pairs(blocks: list, hq: int, hkv: int, d: int, sms: int) -> bool:
    """Forward: pairs of query tiles (``attention_fwd.cuh``) or one tile per CTA (``attention_fwd_one.cuh``). A unit with ``n`` key
    tiles exists once per sequence of at least ``n`` blocks."""
    if not blocks:
        return True
    if sum(blocks) * hq <= sms:   # one tile per CTA is done after the longest tile, and pairs take longer over theirs
        return False
    return _forward_in_pairs(blocks, hq, hkv, d, sms)


def _forward_in_pairs(blocks: list, hq: int, hkv: int, d: int, sms: int) -> bool:
    at = _with_at_least(blocks)
    longest = len(at) - 2
    launch, a, b = _ONE[d]
    one = launch + finish_time([(a + b * n, at[n] * hq) for n in range(1, longest + 1)], sms)
    launch, a, b, ra, rb, la, lb = _TWO[d]
    if (hq // hkv) % 2 == 0:
        units = [(a + b * n, at[n] * hq // 2) for n in range(1, longest + 1)]
    else:
        units = [(ra + rb * n, at[n] * hq) for n in range(2, longest + 1, 2)]
        units += [(la + lb * n, (at[n] - at[n + 1]) * hq) for n in range(1, longest + 1, 2) if at[n] > at[n + 1]]
    return launch + finish_time(units, sms) <= one


def backward_splits(blocks: list, hq: int, hkv: int, sms: int, most: int) -> int:
    """Backward: CTAs (at most ``most``) that share the query heads of a key block. A key block of a kv head is one CTA's work; with few
    kv heads and a short batch that leaves SMs idle and the longest CTA decides (5987 tokens, 12/2 heads: 437 -> 137 us with
    the heads divided). But every CTA loads K and V again and adds a partial sum, so short samples are not divided
    (16 of 128 tokens, 32/8 heads of 128: 47 us whole, 86 when divided until there were two CTAs per SM)."""
    group = hq // hkv
    if not blocks or group == 1 or most <= 1:
        return 1
    if sum(blocks) * hq <= sms and most >= group:   # however divided, everything runs at once: the longest CTA decides
        return group if _BWD_PARTIAL < (group - 1) * max(blocks) else 1
    return _backward_splits(blocks, hq, hkv, sms, most)


def _backward_splits(blocks: list, hq: int, hkv: int, sms: int, most: int) -> int:
    at = _with_at_least(blocks)
    longest, group, units = len(at) - 2, hq // hkv, sum(blocks) * hkv
    best, splits = float("inf"), 1
    for s in range(1, min(group, most) + 1):
        if s > 1 and units * (s - 1) >= 2 * sms:   # two CTAs per SM already
            break
        cta = _BWD_CTA + (_BWD_PARTIAL if s > 1 else 0.0)
        t = finish_time([(cta + group / s * n, at[n] * hkv * s) for n in range(1, longest + 1)], sms)
        t = max(t, cta + -(-group // s) * longest)
        if t < best:
            best, splits = t, s
    return splits


# Iterations of a CTA, on average, from which the backward is launched behind its predecessor's end and not under its tail (csrc/attention_bwd.cuh). 85 batches at head_dim 128
# (16/4, 32/8, 12/2, 16/16 and 8/1 heads, one to 148 sequences), early over in order, with the forward and with a product in front of it: from 20 on 0.99 to 1.15, 1.03 on
# average (8 of 2048 tokens, 16/4: 675 and 586 us; one of 4096, 32/8: 601 and 569), below 12 0.95 to 1.04, 0.99 (37 of 128, 12/2: 53 and 54), between them
# 0.97 to 1.05. At head_dim 64 early is the faster or level throughout (0.95 to 1.00 in 13 batches).
IN_ORDER_ITERATIONS = 20


def backward_in_order(blocks: list, hq: int, hkv: int, d: int, splits: int) -> bool:
    """Backward: whether CTAs go round the chip in order, or come early to whatever SMs are free."""
    return d == 128 and sum(b * (b + 1) for b in blocks) * (hq // hkv) >= 2 * IN_ORDER_ITERATIONS * splits * sum(blocks) > 0


# Under a rule (attention_rule.py) a unit's length no longer follows from its block's place alone.

def key_tiles(q0: int, window: int, prefix: int) -> int:
    """Key tiles that the query rows ``[q0, q0 + BLOCK)`` of a sample look at: the prefix's and the window's."""
    tiles = -(-prefix // BLOCK)
    return tiles + max(0, q0 // BLOCK + 1 - max(tiles, max(0, q0 + 1 - window) // BLOCK))


def query_blocks(k0: int, n: int, window: int, prefix: int) -> int:
    """Query blocks of a sample of ``n`` tokens that see one of the keys ``[k0, k0 + BLOCK)``."""
    blocks = -(-n // BLOCK)
    return blocks if k0 < prefix else min(blocks, (k0 + BLOCK - 2 + window) // BLOCK + 1) - k0 // BLOCK


def rule_items(cu_host, prefixes, window: int, block: int, backward: bool) -> list:
    """Work table of a batch under a rule: rows ``(seq_start, seq_len, block_start, prefix)``, most work first, and that work."""
    items = []
    for a, b, p in zip(cu_host[:-1], cu_host[1:], prefixes):
        for s0 in range(0, b - a, block):
            last = s0 + block - BLOCK
            work = query_blocks(s0, b - a, window, p) if backward else key_tiles(last if last < b - a else s0, window, p)
            items.append((work, a, b - a, s0, p))
    items.sort(key=lambda it: -it[0])
    return items


# Forward, a key tile of one and of two query tiles with (cap, bias) over one without: batches of two to forty samples at both head dimensions.
_RULE_TILE = {(False, False): (1.0, 1.0), (True, False): (1.27, 1.27), (False, True): (1.12, 1.17), (True, True): (1.45, 1.65)}


def rule_in_pairs(work: list, pair_work, hq: int, hkv: int, d: int, sms: int, cap: bool = False, bias: bool = False) -> bool:
    """``forward_in_pairs`` for row blocks of these numbers of key tiles. ``pair_work()``: where heads do not pair up, ``(tiles, has a partner)`` of every pair
    of row blocks."""
    if not work:
        return True
    if len(work) * hq <= sms:
        return False
    one_tile, two_tiles = _RULE_TILE[cap, bias]
    launch, a, b = _ONE[d]
    one = launch + finish_time([(a + one_tile * b * n, c * hq) for n, c in Counter(work).items()], sms)
    launch, a, b, ra, rb, la, lb = _TWO[d]
    if (hq // hkv) % 2 == 0:
        units = [(a + two_tiles * b * n, c * hq // 2) for n, c in Counter(work).items()]
    else:
        units = [((ra + two_tiles * rb * n) if two else (la + two_tiles * lb * n), c * hq) for (n, two), c in Counter(pair_work()).items()]
    return launch + finish_time(units, sms) <= one


def rule_splits(work: list, hq: int, hkv: int, sms: int, most: int) -> int:
    """``backward_splits`` for key blocks of these numbers of query blocks."""
    group = hq // hkv
    if not work or group == 1 or most <= 1:
        return 1
    if len(work) * hq <= sms and most >= group:
        return group if _BWD_PARTIAL < (group - 1) * max(work) else 1
    counts = Counter(work)
    best, splits = float("inf"), 1
    for s in range(1, min(group, most) + 1):
        if s > 1 and len(work) * hkv * (s - 1) >= 2 * sms:
            break
        cta = _BWD_CTA + (_BWD_PARTIAL if s > 1 else 0.0)
        t = max(finish_time([(cta + group / s * n, c * hkv * s) for n, c in counts.items()], sms), cta + -(-group // s) * max(work))
        if t < best:
            best, splits = t, s
    return splits


def rule_shares(work: list, hq: int, hkv: int, sms: int, most) -> tuple:
    """``(CTAs that share a key block, key blocks in front that have one each)`` for these numbers of query blocks, the largest first. ``most(blocks)``: CTAs
    that so many key blocks may be shared by. Where whole key blocks fill the GPU a few times and a part of a time, only those of the last part are shared, which then takes a part of a
    block's time: one sample of 8192 tokens through a window of 1024, 32/8 heads of 128, 480 -> 443 us, 16384 through 2048, 16/4 of 64, 478 -> 435, 5000 and 3000 through 512 311 -> 298
    (four of 4096 through 256 231 -> 233). It does not pay where key blocks differ, as their order evens their sum out: a causal batch of three, 608 -> 611, 40 samples of 300 103 -> 104."""
    splits = rule_splits(work, hq, hkv, sms, most(len(work)))
    group, rounds = hq // hkv, len(work) * hkv // sms
    if group == 1 or rounds == 0 or splits > 1:
        return splits, 0

    def finish(whole, s):
        units = [(_BWD_CTA + group * n, c * hkv) for n, c in Counter(work[:whole]).items()]
        units += [(_BWD_CTA + _BWD_PARTIAL + group / s * n, c * hkv * s) for n, c in Counter(work[whole:]).items()]
        return finish_time(units, sms)
    best, choice = finish(len(work), 1) * 0.97, (1, 0)
    for whole in {rounds * sms // hkv, max(0, rounds - 1) * sms // hkv} - {0}:
        for s in range(2, min(group, most(len(work) - whole)) + 1) if whole < len(work) else ():
            t = finish(whole, s)
            if t < best:
                best, choice = t, (s, whole)
    return choice


def rule_in_order(work: list, hq: int, hkv: int, d: int, splits: int) -> bool:
    """``backward_in_order`` for key blocks of these numbers of query blocks."""
    return d == 128 and sum(work) * (hq // hkv) >= IN_ORDER_ITERATIONS * splits * len(work) > 0
