// Router of a mixture-of-experts layer with the losses that keep its experts in use, and the gradient of its logits.
//
// For a token's logits l [E]: p = softmax(l), the k largest logits (the lower expert of equal ones), w = their p, renormalised over the chosen ones
// when `renorm`, lse = log sum exp(l). For a packed sample s with n counted tokens, c_e pairs that chose e and P_e = sum of p_e:
//   balance = E / n^2 sum_e c_e P_e        z = 1/n sum lse^2
// and with factors db, dz of the two and dw of the weights
//   dl_e = p_e (g_e - sum_j p_j g_j + 2 lse dz / n),    g_e = [e chosen] dtop_e + db E c_e / n^2
// where dtop is dw through the renormalisation. Counts are whole numbers and constants of the gradient.
//
// One pass over the logits and one over the probabilities. A warp has a token, a lane PER neighbouring experts, so that rows move as vectors, and ties go to
// the lower expert by lane and by place. A lane sorts its own experts; a choice is then the warp's largest head and the lane that has it, two instructions of the whole warp (with PER above 4 the
// lanes look for their next one instead). A block has a run of tokens; its part of a sample's sums goes to row (block + sample) of a scratch table,
// which is another one for every (block, sample) that meet, since either number grows along the tokens: no atomics, no host table, one order of sums. A second
// kernel sums a sample's rows.
//
// Exponentials, logarithms and quotients are the approximate instructions in fp32: two units of the last place each, so that probabilities, weights and losses are 7e-8 to 9e-8 of their norm off where the exact functions leave 8e-8; a probability
// below 2^-126 is zero.
//
// Bound by instructions: 64000 tokens, 128 experts, 8 chosen, fp32 logits, 41 samples: 38 us forward with the sums behind it (75 % of the issue slots; its 75 MB would take 11), 19 backward (0.61 of the copy rate). With maxima by
// shuffles, divisions, tokens loaded when they are needed and the samples' starts searched in the backward 71 and 55. A call of few tokens is bound by the host, which takes 20 us forward and 13 backward.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "per_device.h"
#include "ptx.cuh"

namespace mtb {
namespace rb {

typedef __nv_bfloat16 bf16;
constexpr int WARPS = 16, THREADS = 32 * WARPS;            // of the forward
constexpr int BWD_WARPS = 8, BWD_THREADS = 32 * BWD_WARPS;
constexpr int BLOCKS_PER_SM = 2;                           // as many as are resident (but one at PER = 16): one round of them
constexpr int bwd_blocks(int per) { return per <= 4 ? 5 : per == 8 ? 3 : 2; }   // the same of the backward
constexpr int MOST_EXPERTS = 512, MOST_CHOSEN = 32;
constexpr int FINISH_THREADS = 1024;

struct Sample { int s, lo, hi; };   // number, and its tokens

// Bounds of sample s; whatever the table holds they are inside [0, T].
__device__ __forceinline__ int bound(const int* cu, int i, int S, int T) {
  if (cu == nullptr) return i == 0 ? 0 : T;
  return min(max(cu[min(i, S)], 0), T);
}
// First sample that ends behind token t, or S.
__device__ __forceinline__ int sample_of(const int* cu, int t, int S, int T) {
  int lo = 0, hi = S;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (bound(cu, mid + 1, S, T) > t) hi = mid; else lo = mid + 1;
  }
  return lo;
}

template <typename T, int PER, bool VEC>
__device__ __forceinline__ void load_row(const T* row, int E, int lane, float (&x)[PER]) {
  const int e0 = lane * PER;
  if constexpr (VEC) {
    if (e0 < E) {
      if constexpr (sizeof(T) == 2) {
        if constexpr (PER >= 8) {
#pragma unroll
          for (int i = 0; i < PER; i += 8) {
            const uint4 u = *reinterpret_cast<const uint4*>(row + e0 + i);
            const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z), d = unpack_bf16(u.w);
            x[i] = a.x; x[i + 1] = a.y; x[i + 2] = b.x; x[i + 3] = b.y; x[i + 4] = c.x; x[i + 5] = c.y; x[i + 6] = d.x; x[i + 7] = d.y;
          }
        } else if constexpr (PER == 4) {
          const uint2 u = *reinterpret_cast<const uint2*>(row + e0);
          const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y);
          x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
        } else if constexpr (PER == 2) {
          const float2 a = unpack_bf16(*reinterpret_cast<const uint32_t*>(row + e0));
          x[0] = a.x; x[1] = a.y;
        } else {
          x[0] = __bfloat162float(row[e0]);
        }
      } else {
        if constexpr (PER >= 4) {
#pragma unroll
          for (int i = 0; i < PER; i += 4) {
            const float4 u = *reinterpret_cast<const float4*>(row + e0 + i);
            x[i] = u.x; x[i + 1] = u.y; x[i + 2] = u.z; x[i + 3] = u.w;
          }
        } else if constexpr (PER == 2) {
          const float2 u = *reinterpret_cast<const float2*>(row + e0);
          x[0] = u.x; x[1] = u.y;
        } else {
          x[0] = row[e0];
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] = -INFINITY;
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = e0 + i < E ? static_cast<float>(row[e0 + i]) : -INFINITY;
  }
}
template <typename T, int PER, bool VEC>
__device__ __forceinline__ void store_row(T* row, int E, int lane, const float (&x)[PER]) {
  const int e0 = lane * PER;
  if constexpr (VEC) {
    if (e0 >= E) return;
    if constexpr (sizeof(T) == 2) {
      if constexpr (PER >= 8) {
#pragma unroll
        for (int i = 0; i < PER; i += 8)
          *reinterpret_cast<uint4*>(row + e0 + i) = make_uint4(pack_bf16(x[i], x[i + 1]), pack_bf16(x[i + 2], x[i + 3]), pack_bf16(x[i + 4], x[i + 5]), pack_bf16(x[i + 6], x[i + 7]));
      } else if constexpr (PER == 4) {
        *reinterpret_cast<uint2*>(row + e0) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
      } else if constexpr (PER == 2) {
        *reinterpret_cast<uint32_t*>(row + e0) = pack_bf16(x[0], x[1]);
      } else {
        row[e0] = __float2bfloat16(x[0]);
      }
    } else {
      if constexpr (PER >= 4) {
#pragma unroll
        for (int i = 0; i < PER; i += 4) *reinterpret_cast<float4*>(row + e0 + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
      } else if constexpr (PER == 2) {
        *reinterpret_cast<float2*>(row + e0) = make_float2(x[0], x[1]);
      } else {
        row[e0] = x[0];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (e0 + i < E) {
        if constexpr (sizeof(T) == 2) row[e0 + i] = __float2bfloat16(x[i]);
        else row[e0 + i] = x[i];
      }
  }
}

// A number's place in the order of logits as an unsigned one above 0: equal for equal numbers, of either zero (x + 0 has one zero, and one form of what is not a number, which is
// the highest, as in a sort).
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ (static_cast<uint32_t>(static_cast<int>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_order(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ float reciprocal(float x) {   // within a unit of the last place
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float log2_mufu(float x) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Sum over lanes 0 .. k - 1, zero elsewhere, in those lanes.
__device__ __forceinline__ float sum_first(float v, int k) {
  if (k > 8) return warp_sum(v);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// {sum of p_e, pairs} of a (block, sample) and expert, and {sum of lse^2, tokens} of a (block, sample)
struct Part { float p; int c; };

template <typename T, int PER, bool VEC>
__global__ void __launch_bounds__(THREADS, PER == 16 ? 1 : BLOCKS_PER_SM) route_kernel(const T* __restrict__ logits, const int* __restrict__ cu, const uint8_t* __restrict__ counted, int tokens, int E,
                                                        int k, int S, int renorm, int run, float* __restrict__ probs, long long* __restrict__ topi,
                                                        float* __restrict__ w, float* __restrict__ lse, float* __restrict__ inverse, int* __restrict__ sample, Part* __restrict__ part,
                                                        Part* __restrict__ part_z) {
  __shared__ __align__(16) float row_sh[WARPS][PER * 32];   // a token's probabilities; at the end of a sample's tokens, the warps' sums
  __shared__ int count_sh[PER * 32];
  __shared__ int choice_sh[WARPS][MOST_CHOSEN];
  __shared__ Part z_sh[WARPS];
  constexpr bool SORTED = PER <= 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t below = (1u << lane) - 1u;
  pdl_wait();
  const int t0 = blockIdx.x * run, t1 = min(tokens, t0 + run);
  int s = sample_of(cu, t0, S, tokens);
  for (int a = t0; a < t1;) {
    // tokens [a, b) are of sample s, or of none
    const int first = s < S ? max(a, bound(cu, s, S, tokens)) : t1;
    const bool inside = first <= a && s < S;
    const int b = min(t1, inside ? bound(cu, s + 1, S, tokens) : first);
    float sum[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) sum[i] = 0.f;
    float z = 0.f;
    int n = 0;
    if (inside) {
      for (int i = threadIdx.x; i < E; i += THREADS) count_sh[i] = 0;
      __syncthreads();
    }
    float next[PER];
    if (a + warp < b) load_row<T, PER, VEC>(logits + static_cast<long long>(a + warp) * E, E, lane, next);
    for (int t = a + warp; t < b; t += WARPS) {
      float x[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] = next[i];
      if (t + WARPS < b) load_row<T, PER, VEC>(logits + static_cast<long long>(t + WARPS) * E, E, lane, next);
      const bool in_loss = inside && (counted == nullptr || counted[t] != 0);
      const long long at = static_cast<long long>(t) * E;
      uint32_t key[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) key[i] = (VEC ? lane * PER : lane * PER + i) < E ? order_of(x[i]) : 0u;
      uint32_t head = key[0], places = 0xE4u;   // SORTED: places of the sorted experts in the lane, two bits each
      if constexpr (SORTED) {   // neighbours only, and only where the later one is larger: equal ones keep their order
        int place[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) place[i] = i;
#pragma unroll
        for (int r = 0; r < PER; ++r)
#pragma unroll
          for (int i = r & 1; i + 1 < PER; i += 2) {
            const bool turn = key[i + 1] > key[i];
            const uint32_t hk = max(key[i], key[i + 1]), lk = min(key[i], key[i + 1]);
            const int hp = turn ? place[i + 1] : place[i], lp = turn ? place[i] : place[i + 1];
            key[i] = hk; key[i + 1] = lk; place[i] = hp; place[i + 1] = lp;
          }
        head = key[0];
        places = 0u;
#pragma unroll
        for (int i = 0; i < PER; ++i) places |= static_cast<uint32_t>(place[i]) << (2 * i);
      } else {
#pragma unroll
        for (int i = 1; i < PER; ++i) head = max(head, key[i]);
      }
      uint32_t top = __reduce_max_sync(0xffffffffu, head);
      const float m = from_order(top);   // (not a number where a logit is none, and so is all that follows)
      float total = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        x[i] = ex2_mufu((x[i] - m) * 1.4426950408889634f);
        total += (VEC ? lane * PER : lane * PER + i) < E ? x[i] : 0.f;
      }
      total = warp_sum(total);
      const float inv = reciprocal(total), l = fmaf(log2_mufu(total), 0.69314718055994531f, m);
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] *= inv;
      store_row<float, PER, VEC>(probs + at, E, lane, x);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < PER; ++i) row_sh[warp][lane * PER + i] = x[i];
      int c = 0;
#pragma unroll 2
      while (true) {   // the lowest of the lanes that have the largest head writes its expert down and goes on to its next
        const bool has = head == top;
        const uint32_t all = __ballot_sync(0xffffffffu, has);   // of every lane, so before the condition
        const bool own = has && (all & below) == 0u;
        if constexpr (SORTED) {
          if (own) choice_sh[warp][c] = lane * PER + static_cast<int>(places & 3u);
          places = own ? places >> 2 : places;
#pragma unroll
          for (int i = 0; i + 1 < PER; ++i) key[i] = own ? key[i + 1] : key[i];
          key[PER - 1] = own ? 0u : key[PER - 1];
          head = key[0];
        } else if (own) {
          int at_i = 0;
#pragma unroll
          for (int i = PER - 1; i >= 0; --i) if (key[i] == head) at_i = i;
          choice_sh[warp][c] = lane * PER + at_i;
          head = 0u;
#pragma unroll
          for (int i = 0; i < PER; ++i) { if (i == at_i) key[i] = 0u; head = max(head, key[i]); }
        }
        if (++c == k) break;
        top = __reduce_max_sync(0xffffffffu, head);
      }
      __syncwarp();
      const int mine_at = lane < k ? choice_sh[warp][lane] : 0;   // lane c has the c-th choice
      const float mine = lane < k ? row_sh[warp][mine_at] : 0.f;
      float scale = 1.f;
      if (renorm) scale = reciprocal(sum_first(mine, k));
      const float share = mine * scale;
      if (lane < k) {
        topi[static_cast<long long>(t) * k + lane] = mine_at;
        w[static_cast<long long>(t) * k + lane] = share;
      }
      if (lane == 0) { lse[t] = l; inverse[t] = scale; sample[t] = in_loss ? s : -1; }
      if (in_loss) {
#pragma unroll
        for (int i = 0; i < PER; ++i) sum[i] += x[i];
        if (lane < k) atomicAdd(&count_sh[mine_at], 1);
        z = fmaf(l, l, z);
        ++n;
      }
    }
    if (inside) {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < PER; ++i) row_sh[warp][lane * PER + i] = sum[i];
      if (lane == 0) z_sh[warp] = Part{z, n};
      __syncthreads();
      const long long row = static_cast<long long>(blockIdx.x) + s;
      for (int e = threadIdx.x; e < E; e += THREADS) {
        float p = 0.f;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) p += row_sh[i][e];
        part[row * E + e] = Part{p, count_sh[e]};
      }
      if (threadIdx.x == 0) {
        Part q{0.f, 0};
        for (int i = 0; i < WARPS; ++i) { q.p += z_sh[i].p; q.c += z_sh[i].c; }
        part_z[row] = q;
      }
      __syncthreads();
    }
    // the next sample with tokens behind b
    a = b;
    while (s < S && bound(cu, s + 1, S, tokens) <= a) ++s;
  }
  pdl_trigger();
}

// One block per sample: sums of its rows, in 64 bits, and the losses.
__global__ void __launch_bounds__(FINISH_THREADS) finish_kernel(const int* __restrict__ cu, int tokens, int E, int S, int run, const Part* __restrict__ part,
                                                                const Part* __restrict__ part_z, float* __restrict__ balance, float* __restrict__ zloss,
                                                                int* __restrict__ counts, int* __restrict__ ns, float* __restrict__ usage) {
  __shared__ double p_sh[FINISH_THREADS];
  __shared__ int c_sh[FINISH_THREADS];
  __shared__ double3 total_sh[FINISH_THREADS / 32];
  __shared__ double per_sh;
  pdl_wait();
  const int s = blockIdx.x, lo = bound(cu, s, S, tokens), hi = bound(cu, s + 1, S, tokens);
  const int row0 = lo / run + s, rows = hi > lo ? (hi - 1) / run - lo / run + 1 : 0;
  // the rows in `groups` parts, a power of two, an expert's one behind the other
  int groups = 1;
  while (2 * groups * E <= FINISH_THREADS) groups *= 2;
  const int g = threadIdx.x / E, e = threadIdx.x - g * E;
  double p = 0.0, z = 0.0, n = 0.0;
  int c = 0;
  if (g < groups) {
#pragma unroll 8
    for (int r = g; r < rows; r += groups) {
      const Part q = part[static_cast<long long>(row0 + r) * E + e];
      p += q.p;
      c += q.c;
    }
  }
  for (int r = threadIdx.x; r < rows; r += FINISH_THREADS) { z += part_z[row0 + r].p; n += part_z[row0 + r].c; }
  p_sh[threadIdx.x] = p;
  c_sh[threadIdx.x] = c;
  for (int h = groups / 2; h > 0; h /= 2) {
    __syncthreads();
    if (g < h) {
      p_sh[threadIdx.x] = p += p_sh[threadIdx.x + h * E];
      c_sh[threadIdx.x] = c += c_sh[threadIdx.x + h * E];
    }
  }
  if (g == 0) counts[static_cast<long long>(s) * E + e] = c;
  double3 v = make_double3(g == 0 ? p * c : 0.0, z, n);
  auto add = [&](int o) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    v.z += __shfl_xor_sync(0xffffffffu, v.z, o);
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) add(o);
  if ((threadIdx.x & 31) == 0) total_sh[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    v = total_sh[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) add(o);
    if (threadIdx.x == 0) {
      const bool some = v.z > 0.0;
      balance[s] = some ? static_cast<float>(E * v.x / (v.z * v.z)) : 0.f;
      zloss[s] = some ? static_cast<float>(v.y / v.z) : 0.f;
      ns[s] = static_cast<int>(v.z);
      per_sh = some ? E / (v.z * v.z) : 0.0;
    }
  }
  __syncthreads();
  if (g == 0) usage[static_cast<long long>(s) * E + e] = static_cast<float>(c * per_sh);
}
static_assert(FINISH_THREADS == 1024 && MOST_EXPERTS <= FINISH_THREADS, "a warp per 32 threads' sums, a thread to an expert at least");

// What a token's gradient is made of; loaded one token ahead.
template <int PER>
struct Token {
  float p[PER], d, w, l, inverse;
  long long e;
  int s;
};
template <typename T, int PER, bool VEC>
__global__ void __launch_bounds__(BWD_THREADS, bwd_blocks(PER)) route_bwd_kernel(const float* __restrict__ probs, const long long* __restrict__ topi, const float* __restrict__ w,
                                                                const float* __restrict__ dw, const float* __restrict__ lse, const float* __restrict__ inverse, const int* __restrict__ sample,
                                                                const float* __restrict__ usage, const int* __restrict__ ns, const float* __restrict__ dbalance,
                                                                const float* __restrict__ dz, int tokens, int E, int k, int S, int renorm, T* __restrict__ dlogits, int* status) {
  __shared__ __align__(16) float top_sh[BWD_WARPS][PER * 32];   // dtop of the token's chosen experts, zero elsewhere
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < PER; ++i) top_sh[warp][lane * PER + i] = 0.f;
  __syncwarp();
  pdl_wait();
  const int stride = gridDim.x * BWD_WARPS;
  auto load = [&](Token<PER>& o, int t) {
    load_row<float, PER, VEC>(probs + static_cast<long long>(t) * E, E, lane, o.p);
    o.e = -1; o.d = o.w = 0.f;
    if (dw != nullptr && lane < k) {
      const long long pair = static_cast<long long>(t) * k + lane;
      o.e = topi[pair];
      o.d = dw[pair];
      if (renorm) o.w = w[pair];
    }
    o.s = sample[t];
    o.l = dz != nullptr ? lse[t] : 0.f;
    o.inverse = inverse[t];
  };
  Token<PER> next;
  int t = blockIdx.x * BWD_WARPS + warp;
  if (t < tokens) load(next, t);
  for (; t < tokens; t += stride) {
    const Token<PER> o = next;
    if (t + stride < tokens) load(next, t + stride);
    const bool in_loss = o.s >= 0 && o.s < S;
    float g[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) g[i] = 0.f;
    float zt = 0.f;
    if (in_loss) {
      if (dbalance != nullptr) {
        const float f = dbalance[o.s];
        load_row<float, PER, VEC>(usage + static_cast<long long>(o.s) * E, E, lane, g);
#pragma unroll
        for (int i = 0; i < PER; ++i) g[i] = (VEC ? lane * PER : lane * PER + i) < E ? g[i] * f : 0.f;
      }
      if (dz != nullptr) zt = 2.f * o.l * dz[o.s] * reciprocal(static_cast<float>(ns[o.s]));
    }
    if (dw != nullptr) {
      float d = o.d;
      const bool named = lane < k && o.e >= 0 && o.e < E;
      if (lane < k && !named) atomicExch(status, 62);   // no expert: its pair has no gradient
      if (renorm) d = (d - sum_first(named ? d * o.w : 0.f, k)) * o.inverse;
      if (named) atomicAdd(&top_sh[warp][o.e], d);   // of an expert that is named twice, both
      __syncwarp();
#pragma unroll
      for (int i = 0; i < PER; ++i) g[i] += top_sh[warp][lane * PER + i];
      __syncwarp();
      if (named) top_sh[warp][o.e] = 0.f;
      __syncwarp();
    }
    float inner = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) inner += (VEC ? lane * PER : lane * PER + i) < E ? o.p[i] * g[i] : 0.f;
    inner = warp_sum(inner);
#pragma unroll
    for (int i = 0; i < PER; ++i) g[i] = o.p[i] * (g[i] - inner + zt);
    store_row<T, PER, VEC>(dlogits + static_cast<long long>(t) * E, E, lane, g);
  }
  pdl_trigger();
}

// Tokens of a block: at most BLOCKS_PER_SM blocks to an SM, and whole rounds of the warps.
inline int run_of(int tokens, int sms) {
  const int run = (tokens + BLOCKS_PER_SM * sms - 1) / (BLOCKS_PER_SM * sms);
  return (run + WARPS - 1) / WARPS * WARPS;
}
inline bool sizes_ok(int T, int E, int k, int S) { return T > 0 && E > 0 && E <= MOST_EXPERTS && k > 0 && k <= MOST_CHOSEN && k <= E && S > 0; }
inline int ok() { return cudaGetLastError() == cudaSuccess ? 0 : -5; }

}  // namespace rb
}  // namespace mtb

extern "C" {
using namespace mtb::rb;

#define ROUTE_PER(CALL) \
  if (E <= 32) { CALL(1); } else if (E <= 64) { CALL(2); } else if (E <= 128) { CALL(4); } else if (E <= 256) { CALL(8); } else { CALL(16); }

// part [rows, E] and part_z [rows] are scratch of 8 bytes an entry, rows at least S and BLOCKS_PER_SM (2) an SM. logits [T, E], bf16 or (fp32) fp32; cu [S + 1] int32 ascending, or null for one sample of all tokens (S = 1); counted [T] bytes, or null. probs [T, E], w [T, k], lse [T],
// balance [S], zloss [S]: fp32; topi [T, k]: int64; counts [S, E], ns [S], sample [T] (whose losses a token is in, or -1): int32; inverse [T] (of the sum
// of a token's chosen probabilities where renorm, else 1), usage [S, E] (E counts / n^2): fp32, for the gradient.
int mtb200_route_balanced(const void* logits, int fp32, const int* cu, const void* counted, int T, int E, int k, int S, int renorm, float* probs, long long* topi, float* w,
                          float* lse, float* inverse, int* sample, void* part, void* part_z, int rows, float* balance, float* zloss, int* counts, int* ns, float* usage, cudaStream_t st) {
  if (!sizes_ok(T, E, k, S) || (cu == nullptr && S != 1)) return -10;
  const int run = run_of(T, mtb::sms_here()), blocks = (T + run - 1) / run;
  if (rows < blocks + S) return -11;
  const int per = E <= 32 ? 1 : E <= 64 ? 2 : E <= 128 ? 4 : E <= 256 ? 8 : 16;
  const bool vec = E % per == 0 && ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(probs)) & 15) == 0;
#define FWD(T_, PER, VEC) mtb::launch_pdl(route_kernel<T_, PER, VEC>, blocks, THREADS, 0, st, (const T_*)logits, cu, (const uint8_t*)counted, T, E, k, S, renorm, run, probs, topi, w, lse, inverse, sample, (Part*)part, (Part*)part_z)
#define FWD_TYPE(PER) if (fp32) { if (vec) FWD(float, PER, true); else FWD(float, PER, false); } else { if (vec) FWD(bf16, PER, true); else FWD(bf16, PER, false); }
  ROUTE_PER(FWD_TYPE)
#undef FWD_TYPE
#undef FWD
  mtb::launch_pdl(finish_kernel, S, FINISH_THREADS, 0, st, cu, T, E, S, run, (const Part*)part, (const Part*)part_z, balance, zloss, counts, ns, usage);
  return ok();
}

// dw [T, k], dbalance [S], dz [S]: fp32, any of them null. dlogits [T, E]: bf16 or (fp32) fp32.
int mtb200_route_balanced_bwd(const float* probs, const long long* topi, const float* w, const float* dw, const float* lse, const float* inverse, const int* sample, const float* usage, const int* ns, const float* dbalance, const float* dz, int T, int E, int k, int S, int renorm, void* dlogits, int fp32,
                              int* status, cudaStream_t st) {
  if (!sizes_ok(T, E, k, S)) return -10;
  const int per = E <= 32 ? 1 : E <= 64 ? 2 : E <= 128 ? 4 : E <= 256 ? 8 : 16;
  int blocks = (T + BWD_WARPS - 1) / BWD_WARPS;
  if (blocks > bwd_blocks(per) * mtb::sms_here()) blocks = bwd_blocks(per) * mtb::sms_here();
  const bool vec = E % per == 0 && ((reinterpret_cast<uintptr_t>(dlogits) | reinterpret_cast<uintptr_t>(probs) | reinterpret_cast<uintptr_t>(usage)) & 15) == 0;
#define BWD(T_, PER, VEC) mtb::launch_pdl(route_bwd_kernel<T_, PER, VEC>, blocks, BWD_THREADS, 0, st, probs, topi, w, dw, lse, inverse, sample, usage, ns, dbalance, dz, T, E, k, S, renorm, (T_*)dlogits, status)
#define BWD_TYPE(PER) if (fp32) { if (vec) BWD(float, PER, true); else BWD(float, PER, false); } else { if (vec) BWD(bf16, PER, true); else BWD(bf16, PER, false); }
  ROUTE_PER(BWD_TYPE)
#undef BWD_TYPE
#undef BWD
  return ok();
}

}  // extern "C"
