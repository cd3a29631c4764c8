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
// the lower expert by lane and by place. A block has a run of tokens; its part of a sample's sums goes to row (block + sample) of a scratch table,
// which is another one for every (block, sample) that meet, since either number grows along the tokens: no atomics, no host table, one order of sums. A second
// kernel sums a sample's rows.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx.cuh"

namespace mtb {
namespace rb {

typedef __nv_bfloat16 bf16;
constexpr int WARPS = 8, THREADS = 32 * WARPS;
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

// A number's place in the order of logits as an unsigned one above 0: equal for equal numbers (of either zero), highest for what is not a number, as in a sort.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// {sum of p_e, pairs} of a (block, sample) and expert, and {sum of lse^2, tokens} of a (block, sample)
struct Part { float p; int c; };

template <typename T, int PER, bool VEC>
__global__ void __launch_bounds__(THREADS) route_kernel(const T* __restrict__ logits, const int* __restrict__ cu, const uint8_t* __restrict__ counted, int tokens, int E,
                                                        int k, int S, int renorm, int run, float* __restrict__ probs, long long* __restrict__ topi,
                                                        float* __restrict__ w, float* __restrict__ lse, Part* __restrict__ part, Part* __restrict__ part_z) {
  __shared__ float sum_sh[WARPS][PER * 32];
  __shared__ int count_sh[PER * 32];
  __shared__ Part z_sh[WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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
    for (int t = a + warp; t < b; t += WARPS) {
      float x[PER];
      const long long at = static_cast<long long>(t) * E;
      load_row<T, PER, VEC>(logits + at, E, lane, x);
      uint32_t key[PER];
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        key[i] = lane * PER + i < E ? order_of(x[i]) : 0u;
        m = fmaxf(m, x[i]);
      }
      m = warp_max(m);
      float total = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) { x[i] = expf(x[i] - m); total += lane * PER + i < E ? x[i] : 0.f; }
      total = warp_sum(total);
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] /= total;
      store_row<float, PER, VEC>(probs + at, E, lane, x);
      const float l = m + logf(total);
      float mine = 0.f, chosen = 0.f;   // lane c holds the c-th probability
      int mine_at = 0;
      for (int c = 0; c < k; ++c) {
        uint32_t best = 0;
        int at_i = 0;
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) if (key[i] > best) { best = key[i]; at_i = i; v = x[i]; }
        const uint32_t top = __reduce_max_sync(0xffffffffu, best);
        const int owner = __ffs(__ballot_sync(0xffffffffu, best == top)) - 1;
        v = __shfl_sync(0xffffffffu, v, owner);
        const int e = __shfl_sync(0xffffffffu, lane * PER + at_i, owner);
        if (lane == owner) {
#pragma unroll
          for (int i = 0; i < PER; ++i) if (i == at_i) key[i] = 0u;
        }
        if (lane == c) { mine = v; mine_at = e; }
        chosen += v;
      }
      if (lane < k) {
        topi[static_cast<long long>(t) * k + lane] = mine_at;
        w[static_cast<long long>(t) * k + lane] = renorm ? mine / chosen : mine;
      }
      if (lane == 0) lse[t] = l;
      if (inside && (counted == nullptr || counted[t] != 0)) {
#pragma unroll
        for (int i = 0; i < PER; ++i) sum[i] += x[i];
        if (lane < k) atomicAdd(&count_sh[mine_at], 1);
        z += l * l;
        ++n;
      }
    }
    if (inside) {
#pragma unroll
      for (int i = 0; i < PER; ++i) sum_sh[warp][lane * PER + i] = sum[i];
      if (lane == 0) z_sh[warp] = Part{z, n};
      __syncthreads();
      const long long row = static_cast<long long>(blockIdx.x) + s;
      for (int e = threadIdx.x; e < E; e += THREADS) {
        float p = 0.f;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) p += sum_sh[i][e];
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
                                                                int* __restrict__ counts, int* __restrict__ ns) {
  __shared__ double p_sh[FINISH_THREADS];
  __shared__ int c_sh[FINISH_THREADS];
  __shared__ double total_sh[FINISH_THREADS / 32];
  pdl_wait();
  const int s = blockIdx.x, lo = bound(cu, s, S, tokens), hi = bound(cu, s + 1, S, tokens);
  const int row0 = lo / run + s, rows = hi > lo ? (hi - 1) / run - lo / run + 1 : 0;
  // the rows in `groups` parts, an expert's one behind the other
  const int groups = FINISH_THREADS / E, g = threadIdx.x / E, e = threadIdx.x - g * E;
  double p = 0.0;
  int c = 0;
  if (g < groups) {
#pragma unroll 8
    for (int r = g; r < rows; r += groups) {
      const Part q = part[static_cast<long long>(row0 + r) * E + e];
      p += q.p;
      c += q.c;
    }
  }
  p_sh[threadIdx.x] = p;
  c_sh[threadIdx.x] = c;
  __syncthreads();
  double prod = 0.0;
  if (threadIdx.x < E) {
    for (int i = 1; i < groups; ++i) { p += p_sh[i * E + e]; c += c_sh[i * E + e]; }
    counts[static_cast<long long>(s) * E + e] = c;
    prod = p * c;
  }
  auto sum_block = [&](double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) total_sh[threadIdx.x >> 5] = v;
    __syncthreads();
    double all = 0.0;
    for (int i = 0; i < FINISH_THREADS / 32; ++i) all += total_sh[i];
    return all;
  };
  const double all = sum_block(prod);
  double z = 0.0, n = 0.0;
  for (int r = threadIdx.x; r < rows; r += FINISH_THREADS) { z += part_z[row0 + r].p; n += part_z[row0 + r].c; }
  z = sum_block(z);
  n = sum_block(n);
  if (threadIdx.x == 0) {
    const bool some = n > 0.0;
    balance[s] = some ? static_cast<float>(E * all / (n * n)) : 0.f;
    zloss[s] = some ? static_cast<float>(z / n) : 0.f;
    ns[s] = static_cast<int>(n);
  }
}

template <typename T, int PER, bool VEC>
__global__ void __launch_bounds__(THREADS) route_bwd_kernel(const float* __restrict__ probs, const long long* __restrict__ topi, const float* __restrict__ w,
                                                            const float* __restrict__ dw, const float* __restrict__ lse, const int* __restrict__ cu,
                                                            const uint8_t* __restrict__ counted, const int* __restrict__ counts, const int* __restrict__ ns,
                                                            const float* __restrict__ dbalance, const float* __restrict__ dz, int tokens, int E, int k, int S,
                                                            int renorm, int run, T* __restrict__ dlogits, int* status) {
  __shared__ float top_sh[WARPS][PER * 32];   // dtop of the token's chosen experts, zero elsewhere
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int i = 0; i < PER; ++i) top_sh[warp][lane * PER + i] = 0.f;
  __syncwarp();
  pdl_wait();
  const int t0 = blockIdx.x * run, t1 = min(tokens, t0 + run);
  int s = sample_of(cu, min(t0 + warp, tokens - 1), S, tokens);
  for (int t = t0 + warp; t < t1; t += WARPS) {
    while (s < S && bound(cu, s + 1, S, tokens) <= t) ++s;
    const bool in_loss = s < S && bound(cu, s, S, tokens) <= t && (counted == nullptr || counted[t] != 0);
    const long long at = static_cast<long long>(t) * E, pair = static_cast<long long>(t) * k;
    float p[PER], g[PER];
    load_row<float, PER, VEC>(probs + at, E, lane, p);
#pragma unroll
    for (int i = 0; i < PER; ++i) g[i] = 0.f;
    if (dw != nullptr) {
      long long e = -1;
      float d = 0.f, wt = 0.f, pt = 0.f;
      if (lane < k) {
        e = topi[pair + lane];
        d = dw[pair + lane];
        if (e < 0 || e >= E) { atomicExch(status, 62); e = -1; }   // no expert: its pair has no gradient
        else if (renorm) { wt = w[pair + lane]; pt = probs[at + e]; }
      }
      if (renorm) {
        const float dot = warp_sum(d * wt), chosen = warp_sum(pt);
        d = (d - dot) / chosen;
      }
      if (e >= 0) atomicAdd(&top_sh[warp][e], d);   // of an expert that is named twice, both
      __syncwarp();
#pragma unroll
      for (int i = 0; i < PER; ++i) g[i] = top_sh[warp][lane * PER + i];
      __syncwarp();
      if (e >= 0) top_sh[warp][e] = 0.f;
      __syncwarp();
    }
    float zt = 0.f;
    if (in_loss) {
      const float n = static_cast<float>(ns[s]);
      if (dbalance != nullptr) {
        const float f = dbalance[s] * (static_cast<float>(E) / n) / n;
        const int* c = counts + static_cast<long long>(s) * E + lane * PER;
#pragma unroll
        for (int i = 0; i < PER; ++i) if (lane * PER + i < E) g[i] += f * static_cast<float>(c[i]);
      }
      if (dz != nullptr) zt = 2.f * lse[t] * dz[s] / n;
    }
    float inner = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) inner += lane * PER + i < E ? p[i] * g[i] : 0.f;
    inner = warp_sum(inner);
#pragma unroll
    for (int i = 0; i < PER; ++i) g[i] = p[i] * (g[i] - inner + zt);
    store_row<T, PER, VEC>(dlogits + at, E, lane, g);
  }
  pdl_trigger();
}

// Tokens of a block: about four blocks to an SM, and whole rounds of the warps.
inline int run_of(int tokens, int sms) {
  const int run = (tokens + 4 * sms - 1) / (4 * sms);
  return (run + WARPS - 1) / WARPS * WARPS;
}
inline bool sizes_ok(int T, int E, int k, int S) { return T > 0 && E > 0 && E <= MOST_EXPERTS && k > 0 && k <= MOST_CHOSEN && k <= E && S > 0; }
inline int ok() { return cudaGetLastError() == cudaSuccess ? 0 : -5; }
inline int sms_of() {
  static int sms = 0;
  if (sms == 0) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) sms = 148;
  }
  return sms;
}

}  // namespace rb
}  // namespace mtb

extern "C" {
using namespace mtb::rb;

// Rows of the scratch tables of mtb200_route_balanced: part [rows, E] and part_z [rows], 8 bytes each.
int mtb200_route_balanced_rows(int T, int S) {
  if (T <= 0) return S;
  const int run = run_of(T, sms_of());
  return (T + run - 1) / run + S;
}

#define ROUTE_PER(CALL) \
  if (E <= 32) { CALL(1); } else if (E <= 64) { CALL(2); } else if (E <= 128) { CALL(4); } else if (E <= 256) { CALL(8); } else { CALL(16); }

// logits [T, E], bf16 or (fp32) fp32; cu [S + 1] int32 ascending, or null for one sample of all tokens (S = 1); counted [T] bytes, or null. probs [T, E], w [T, k], lse [T],
// balance [S], zloss [S]: fp32; topi [T, k]: int64; counts [S, E], ns [S]: int32.
int mtb200_route_balanced(const void* logits, int fp32, const int* cu, const void* counted, int T, int E, int k, int S, int renorm, float* probs, long long* topi, float* w,
                          float* lse, void* part, void* part_z, float* balance, float* zloss, int* counts, int* ns, cudaStream_t st) {
  if (!sizes_ok(T, E, k, S) || (cu == nullptr && S != 1)) return -10;
  const int run = run_of(T, sms_of()), blocks = (T + run - 1) / run;
  const int per = E <= 32 ? 1 : E <= 64 ? 2 : E <= 128 ? 4 : E <= 256 ? 8 : 16;
  const bool vec = E % per == 0 && ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(probs)) & 15) == 0;
#define FWD(T_, PER, VEC) mtb::launch_pdl(route_kernel<T_, PER, VEC>, blocks, THREADS, 0, st, (const T_*)logits, cu, (const uint8_t*)counted, T, E, k, S, renorm, run, probs, topi, w, lse, (Part*)part, (Part*)part_z)
#define FWD_TYPE(PER) if (fp32) { if (vec) FWD(float, PER, true); else FWD(float, PER, false); } else { if (vec) FWD(bf16, PER, true); else FWD(bf16, PER, false); }
  ROUTE_PER(FWD_TYPE)
#undef FWD_TYPE
#undef FWD
  mtb::launch_pdl(finish_kernel, S, FINISH_THREADS, 0, st, cu, T, E, S, run, (const Part*)part, (const Part*)part_z, balance, zloss, counts, ns);
  return ok();
}

// dw [T, k], dbalance [S], dz [S]: fp32, any of them null. dlogits [T, E]: bf16 or (fp32) fp32.
int mtb200_route_balanced_bwd(const float* probs, const long long* topi, const float* w, const float* dw, const float* lse, const int* cu, const void* counted,
                              const int* counts, const int* ns, const float* dbalance, const float* dz, int T, int E, int k, int S, int renorm, void* dlogits, int fp32,
                              int* status, cudaStream_t st) {
  if (!sizes_ok(T, E, k, S) || (cu == nullptr && S != 1)) return -10;
  const int run = run_of(T, sms_of()), blocks = (T + run - 1) / run;
  const int per = E <= 32 ? 1 : E <= 64 ? 2 : E <= 128 ? 4 : E <= 256 ? 8 : 16;
  const bool vec = E % per == 0 && ((reinterpret_cast<uintptr_t>(dlogits) | reinterpret_cast<uintptr_t>(probs)) & 15) == 0;
#define BWD(T_, PER, VEC) mtb::launch_pdl(route_bwd_kernel<T_, PER, VEC>, blocks, THREADS, 0, st, probs, topi, w, dw, lse, cu, (const uint8_t*)counted, counts, ns, dbalance, dz, T, E, k, S, renorm, run, (T_*)dlogits, status)
#define BWD_TYPE(PER) if (fp32) { if (vec) BWD(float, PER, true); else BWD(float, PER, false); } else { if (vec) BWD(bf16, PER, true); else BWD(bf16, PER, false); }
  ROUTE_PER(BWD_TYPE)
#undef BWD_TYPE
#undef BWD
  return ok();
}

}  // extern "C"
