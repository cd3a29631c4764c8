// What the attention kernels do to a score between Q K^T and the softmax when they run under a rule (ops/attention_rule.py):
//   s   = scale q.k
//   s  -> cap tanh(s / cap)                        (CAP)
//   s  -> s - slope[head] |i - j|                  (BIAS; i, j: positions of query and key in their sample)
//   query i sees key j  iff  (j <= i and i - j < window) or j < prefix         (the diagonal is always seen: no row is empty)
// The kernels are instances of the same templates as the plain causal ones, whose own instances (NoRule) have the registers and, to 1 %, the times they had before. Masks need no parameter of
// the template: which tiles exist, and which of them are crossed by an edge of the mask, is found per tile. The cap is in cap.cuh.
//
// P and, in the backward, dS are rounded to bf16 as operands of their products, as in the causal kernels: operands of 32 bits (tf32) have half the rate and twice the tensor memory, which is
// full. That is what the gradients are off by (2.8e-3 of their norm against 64 bits, where fp32 rounded once is off by 1.7e-3); statistics, scores and accumulators are fp32.
//
// Bound as the plain causal kernels are, by the chain of hand-offs between the softmax warps and the tensor core, and then by what the softmax warps have to do to a
// score: a cap adds five to seven packed instructions a pair, and the reference's comparisons of absolute values, a bias three. 8192 tokens in three samples, 32/8 heads of 128
// (188 GFLOP forward, 471 backward), scores with a standard deviation of 1 and of 3, a cap of 50, us:
//   forward   causal kernel 183, 204   a rule without either 193, 215   cap 237, 256   bias 213, 225   both 274, 283
//   backward                583, 586                         588, 591       619, 622        579, 583        614, 618
// Scores that fill the cap (16; one in five hundred is beyond it, so nearly every tile has some) and that pass it (60): forward capped 458, 420, both 630, 626; backward 695, 695, both 705, 706.
// At a deviation of 1 the tensor core is busy for 57, 45, 50 and about 37 % of the forward's cycles, issue slots for 44, 42, 48 and 42 %: no pipe is full, a row's instructions depend on each other.
// Windows and prefixes cost what their tiles do: one sample of 8192 tokens with a window of 1024 takes 0.63 ms both ways, without one 1.9.
#pragma once
#include <stdint.h>

#include "cap.cuh"
#include "ptx.cuh"

namespace mtb {

struct AttRuleArgs {
  int window;            // keys a query sees, itself among them; 1 << 30 for all
  const float* slopes;   // [Hq]
  int whole;             // backward: key blocks times kv heads, from the first on, that have one CTA each; only those behind them are shared by p.splits
  // Backward: *odd is `number` or more where something of this launch's batch is not finite that samples share a tile with (numbers grow from launch to launch, so nothing has to be reset; a
  // number that an overlapping launch left there costs time and nothing else; so does that of any launch behind a captured one, whose replays keep the number they were captured with).
  unsigned long long* odd;
  unsigned long long number;
  CapArgs cap;           // of raw products
};

template <bool CAP_, bool BIAS_>
struct Rule { static constexpr bool ON = true, CAP = CAP_, BIAS = BIAS_; static constexpr int ROW = 4; using Args = AttRuleArgs; };   // ROW: ints of a row of the work table
struct NoRule { static constexpr bool ON = false, CAP = false, BIAS = false; static constexpr int ROW = 3; struct Args {}; };

inline AttRuleArgs att_rule_args(float scale, float cap, int window, const float* slopes) {
  AttRuleArgs r{};
  r.window = window > 0 && window < (1 << 30) ? window : 1 << 30;
  r.slopes = slopes;
  if (cap > 0.f) r.cap = cap_args(scale, cap, static_cast<double>(cap) * 1.4426950408889634);
  return r;
}

// Bits 0 .. n - 1.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// Key tiles of 128 that a tile of query rows [q0, q0 + 128) looks at: the prefix's, then those from `skip` on behind them.
struct AttTiles {
  int prefix_tiles, skip;
  // The j-th of n. With a bias from the diagonal back: near keys have the larger scores, so the reference maximum is found at once and the accumulator hardly ever
  // rescaled (the other way round it was in nearly every tile: 280 us where it takes 210, 8192 tokens in three samples, 32/8 heads of 128).
  template <class R>
  __device__ __forceinline__ int tile(int j, int n) const {
    if (R::BIAS) j = n - 1 - j;
    return j >= prefix_tiles ? j + skip : j;
  }
};
// Whether every row of [q0, q0 + 128) sees every key of [k0, k0 + 128).
__device__ __forceinline__ bool att_all_seen(const AttRuleArgs& r, int q0, int k0, int prefix) {
  return k0 + 128 <= prefix || (k0 + 127 <= q0 && q0 + 127 - k0 < r.window);
}
// Of 32 keys from k on, the ones that query i sees.
__device__ __forceinline__ uint32_t att_keys_seen(const AttRuleArgs& r, int i, int k, int prefix) {
  return low_bits(prefix - k) | (low_bits(i + 1 - k) & ~low_bits(i + 1 - r.window - k));
}
// Of 32 queries from i on, the ones that see key j.
__device__ __forceinline__ uint32_t att_queries_seen(const AttRuleArgs& r, int j, int i, int prefix) {
  return j < prefix ? 0xffffffffu : low_bits(j + r.window - i) & ~low_bits(j - i);
}


// One query's scores against C x 32 keys from `key` on, raw products in registers, on their way to probabilities.
//
// The reference of the exponentials does not have to be the largest score, only near it and the same throughout. A cap is monotonic, so the largest product capped is
// the largest capped score; a bias is not, but within 32 keys it changes by 31 slopes: the largest product of each 32, capped, with the bias of the nearer
// end is near it, too high by at most that, or too low by the little that a cap is told by its slope (2^2.3, below). Where capped scores without a bias are small, up to 2^+-30 as exponentials,
// their largest absolute value, which has to be known for the cap's polynomial anyhow, is bound enough: 2^60 too high at most, which leaves the smallest probability that counts beside the
// largest, 2^-24 of it, at 2^-84, 42 bits above fp32's last. With a bias the largest product is taken with its sign: 2^60 and the 2^40 of a bias together left nothing. So the scores themselves are only formed on their way into the exponentials, which
// keeps the FMA pipe and the special-function unit busy at once; formed in place first, capped scores took 286 us where they take 232 (8192 tokens in three samples,
// 32/8 heads of 128; 192 without a cap). They are formed in place, and their largest taken, where this does not hold (`formed`):
// products beyond the cap, slopes so steep that the bound could be 2^40 too high for them alone, and biased keys on the diagonal.
constexpr float ATT_STEEP = 40.f / 31.f;
// Rows [first, 128) of a [128, 64 KB] tile in shared memory (128B swizzle: a row's bytes stay together) set to zero by `n` threads, for reads by the tensor core behind
// the caller's next arrival. A tile at a sample's end holds rows of the next sample, which meet probabilities and gradients of zero; a product
// with zero is only zero for finite numbers, and one sample's infinities are not another's. The forward takes the same time with it. The backward, which has three such tiles and more to do to them, took
// 7 to 15 % longer with every one's rows zeroed, so it looks for numbers that are not finite beforehand (AttLook of attention_bwd.cuh) and only takes the trouble when there are any.
template <int KB>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int first, int thread, int n) {
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll 8
    for (int at = first * 128 + thread * 16; at < 128 * 128; at += n * 16) *reinterpret_cast<uint4*>(tile + kb * 16384 + at) = make_uint4(0u, 0u, 0u, 0u);
  fence_proxy_async_smem();
}

// Which way a tile takes is decided once for all of it: branches for every 32 keys kept the compiler from mixing their instructions (a biased forward took 279 us with them and 247 without).
enum { ATT_RAW = 0, ATT_LOW = 1, ATT_FORMED = 2 };   // from products; the same within half of the cap; scores formed in place
// EDGE: an edge of the mask crosses the tile. Left for the exponentials: `seen`, `any` (whether one of the warp's rows sees a key of 32), the bias.
template <class R, bool EDGE, int C>
struct AttScores {
  uint32_t sv[C][32], seen[C];
  bool any[C];
  int way;
  float slope2, from, sl2;   // slope in units of log2 e (negated where keys are behind the queries), first key minus query

  __device__ __forceinline__ float2 pair(int c, int i) const { return make_float2(__uint_as_float(sv[c][2 * i]), __uint_as_float(sv[c][2 * i + 1])); }
  __device__ __forceinline__ bool sees(int c, int i) const { return !EDGE || (seen[c] >> i & 1u); }

  // This thread's scores capped by the exact form.
  __device__ __forceinline__ void exact(const AttRuleArgs& r, uint32_t taddr) {
    cap_in_place(r.cap, taddr, 2 * C);
#pragma unroll
    for (int c = 0; c < C; ++c) tmem_ld_32x32(taddr + c * 32, sv[c]);
    tmem_ld_wait();
  }
  // Forms the scores, masked ones -inf, and returns their maximum. `low`: they are to be capped yet, and within half of the cap.
  __device__ __forceinline__ float form(const AttRuleArgs& r, bool low) {
    float m[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      m[c] = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float2 v = pair(c, i);
        if constexpr (R::CAP) { if (R::BIAS && low) v = fmul2(v, cap_half_part(r.cap, v)); }
        else v = fmul2(v, splat(sl2));
        if constexpr (R::BIAS) {
          const float x = from + (c * 32 + 2 * i), y = from + (c * 32 + 2 * i + 1);
          v = ffma2(splat(-slope2), make_float2(fabsf(x), fabsf(y)), v);
        }
        if (!sees(c, 2 * i)) v.x = -INFINITY;
        if (!sees(c, 2 * i + 1)) v.y = -INFINITY;
        sv[c][2 * i] = __float_as_uint(v.x); sv[c][2 * i + 1] = __float_as_uint(v.y);
        m[c] = fmax3(m[c], v.x, v.y);
      }
    }
    float most = fmaxf(m[0], m[1]);
#pragma unroll
    for (int c = 2; c < C; c += 2) most = fmax3(most, m[c], m[c + 1]);
    return most;
  }

  // The reference: largest score, or the bound, in units of log2 e; -inf where nothing is seen. The tile: 128 queries from q0, keys from k0 on, of which this thread
  // has those from `key` on.
  __device__ __forceinline__ float reference(const AttRuleArgs& r, int query, int key, int q0, int k0, int prefix, uint32_t taddr) {
    from = static_cast<float>(key - query);
    bool small = true, low = false;
    float big[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      seen[c] = EDGE ? att_keys_seen(r, query, key + c * 32, prefix) : 0xffffffffu;
      any[c] = !EDGE || __any_sync(0xffffffffu, seen[c] != 0u);
    }
    if constexpr (R::CAP) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        big[c] = 0.f;
#pragma unroll
        for (int i = 0; i < 32; i += 2) big[c] = fmax3(big[c], fabsf(__uint_as_float(sv[c][i])), fabsf(__uint_as_float(sv[c][i + 1])));
      }
      float most = big[0];
#pragma unroll
      for (int c = 1; c < C; ++c) most = fmaxf(most, big[c]);
      low = __all_sync(0xffffffffu, most <= r.cap.low);
      small = low || __all_sync(0xffffffffu, most <= r.cap.most);
      if (!R::BIAS && !small) exact(r, taddr);
    }
    way = low ? ATT_LOW : ATT_RAW;
    if constexpr (R::CAP || R::BIAS) {
      bool formed = !small;
      if constexpr (R::BIAS) {
        // The tile on the diagonal comes first and mostly has the largest score: found exactly, that score's probability is 1, which rounds without an error
        // (gradients 3.3e-3 off instead of 4.0e-3). It is also the one that can have keys on both sides of a query; behind it they are only seen in a prefix.
        formed = formed || k0 == q0 || fabsf(slope2) > ATT_STEEP;
        if (k0 > q0 && !formed) slope2 = -slope2;
      }
      if (formed) {
        way = ATT_FORMED;
        // the exact form for all of a biased tile that has larger scores, so that the polynomial of degree eleven is not in `form` too (8192 tokens 296 -> 284 us, 41 short samples
        // 109 -> 102; with scores up to the cap, which are rarer, 398 -> 388 and 126 -> 135)
        if (R::CAP && R::BIAS && !low) exact(r, taddr);
        return form(r, low);
      }
    }
    float mc[C];   // independent chains
#pragma unroll
    for (int c = 0; c < C; ++c) {
      mc[c] = -INFINITY;
      if (EDGE && !any[c]) continue;
      if (EDGE && !R::CAP) {   // (a masked product that stayed infinite would be NaN when it is capped)
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (!sees(c, i)) sv[c][i] = 0xff800000u;   // -inf
      }
    }
    if (R::CAP && !R::BIAS && !EDGE && low) {
#pragma unroll
      for (int c = 0; c < C; ++c) mc[c] = big[c];
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (EDGE && !any[c]) continue;
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float x = __uint_as_float(sv[c][i]), y = __uint_as_float(sv[c][i + 1]);
          if (R::CAP && !sees(c, i)) x = -INFINITY;
          if (R::CAP && !sees(c, i + 1)) y = -INFINITY;
          mc[c] = fmax3(mc[c], x, y);
        }
      }
    }
    if constexpr (R::BIAS) {
      if (R::CAP && low) {   // of scores within half of the cap what they are uncapped is near enough: 2^2.3 too high at most, or too low where all are negative (exactly 284 us where it takes 269)
#pragma unroll
        for (int c = 0; c < C; ++c) mc[c] *= r.cap.b[0].x;
      } else if (R::CAP) {
#pragma unroll
        for (int c = 0; c < C; ++c) mc[c] = mc[c] > -INFINITY ? cap_exact(r.cap, mc[c]) : mc[c];
      }
#pragma unroll
      for (int c = 0; c < C; ++c) {   // of 32 keys the nearest has the larger bias unless the slope is negative
        const float near = fmaxf(slope2 * (from + (c * 32)), slope2 * (from + (c * 32 + 31)));
        mc[c] = R::CAP ? mc[c] + near : fmaf(mc[c], sl2, near);
      }
    }
    float m = fmaxf(mc[0], mc[1]);
#pragma unroll
    for (int c = 2; c < C; c += 2) m = fmax3(m, mc[c], mc[c + 1]);
    if constexpr (!R::BIAS) m = m == -INFINITY ? m : R::CAP ? cap_exact(r.cap, m) : m * sl2;
    return m;
  }

  // 32 probabilities, exp2(score - ref), of piece c: rounded to bf16 pairs, and their sum. Every FMA_EVERY-th pair is formed on the FMA pipe, where nothing is
  // masked, which wants exact zeros, and the cap's polynomial does not fill that pipe as it is.
  template <int FMA_EVERY, int WAY>
  __device__ __forceinline__ void probabilities(const AttRuleArgs& r, int c, float ref, uint32_t (&pk)[16], float2 (&l2)[2]) const {
    if (EDGE && !any[c]) {
#pragma unroll
      for (int i = 0; i < 16; ++i) pk[i] = 0u;
      return;
    }
    constexpr int FMA = EDGE || R::CAP ? 32 : FMA_EVERY;
    [[maybe_unused]] float2 off[4] = {};   // of the bias, within 8 keys
    if constexpr (R::BIAS) {
#pragma unroll
      for (int i = 0; i < 4; ++i) off[i] = make_float2(slope2 * (2 * i), slope2 * (2 * i + 1));
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float2 x;
      if constexpr (WAY == ATT_FORMED) x = fadd2(pair(c, i), splat(-ref));
      else {
        const float2 b = R::BIAS ? fadd2(off[i & 3], splat(fmaf(slope2, from + (c * 32 + (i >> 2) * 8), -ref))) : splat(-ref);
        x = WAY == ATT_LOW ? cap_half(r.cap, pair(c, i), b) : R::CAP ? cap_pair(r.cap, pair(c, i), b) : ffma2(pair(c, i), splat(sl2), b);
        if (R::CAP && !sees(c, 2 * i)) x.x = -INFINITY;
        if (R::CAP && !sees(c, 2 * i + 1)) x.y = -INFINITY;
      }
      const float2 e = (i % FMA == FMA - 1) ? ex2_fma2(x) : make_float2(ex2_mufu(x.x), ex2_mufu(x.y));
      l2[i & 1] = fadd2(l2[i & 1], e);
      pk[i] = pack_bf16(e.x, e.y);
    }
  }
};
template <int W> struct AttWay { static constexpr int value = W; };
// emit(AttWay) for the way a tile takes.
template <class R, typename Emit>
__device__ __forceinline__ void att_by_way(int way, Emit emit) {
  if constexpr (R::CAP) {
    if (way == ATT_LOW) { emit(AttWay<ATT_LOW>{}); return; }
  }
  if constexpr (R::CAP || R::BIAS) {
    if (way == ATT_FORMED) { emit(AttWay<ATT_FORMED>{}); return; }
  }
  emit(AttWay<ATT_RAW>{});
}

}  // namespace mtb
