// Likelihoods from what a product over the vocabulary has left of its logits (gemm_act.cuh, ACT_LSE): of every 128 columns the largest z log2 e and the sum of the exponentials below it, without
// the row's target, and the target's z. With the others' log-partition o the loss is log(1 + e^(o - z)), which keeps its digits where the target is nearly certain, and lse = z + loss.
// A row's statistics are 8 bytes per 128 columns (8192 x 128256: 66 MB beside a product of 5 ms): a block per row, memory-bound.
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx.cuh"

namespace mtb {
namespace nll {

constexpr int THREADS = 128;

__global__ void __launch_bounds__(THREADS) nll_kernel(const float2* __restrict__ stats, const float* __restrict__ at_target, const long long* __restrict__ targets, int pieces,
                                                      long long columns, long long ignore, float* __restrict__ loss, float* __restrict__ lse, int* status) {
  __shared__ float2 sh[THREADS / 32];
  pdl_wait();
  const long long row = blockIdx.x;
  const float2* st = stats + row * pieces;
  float m = -INFINITY, s = 0.f;
  auto add = [&](float2 v) {
    const float n = fmaxf(m, v.x), base = n == -INFINITY ? 0.f : n;
    s = s * ex2_mufu(m - base) + v.y * ex2_mufu(v.x - base);
    m = n;
  };
#pragma unroll 4
  for (int i = threadIdx.x; i < pieces; i += THREADS) add(st[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float2 v = make_float2(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
    add(v);
  }
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) add(sh[i]);
    const long long t = targets[row];
    const float others = (m + log2f(s)) * 0.69314718055994531f;   // natural again; -infinity where there are none
    const bool has = t >= 0 && t < columns;   // a column's number may be what is ignored, too: the partition is of all columns then as well
    if (t != ignore && !has) atomicExch(status, 63);
    float l = 0.f, z = others;
    if (has) {
      const float at = at_target[row], d = others - at;
      l = fmaxf(d, 0.f) + log1pf(expf(-fabsf(d)));
      if (d != d) l = d;
      z = at + l;
    }
    loss[row] = t != ignore ? l : 0.f;
    lse[row] = z;
  }
  pdl_trigger();
}

}  // namespace nll
}  // namespace mtb

extern "C" {

int mtb200_gemm_lse(const void* A, long long lda, const void* W, float2* stats, float* at_target, const long long* targets, int M, int N, int K, float alpha, int form, int* status,
                    cudaStream_t stream);

// loss, lse [T] fp32 of the logits alpha x[T, H] * w[columns, H]^T, row-major without padding. stats [T, ceil(columns / 128)] and at_target [T] are scratch; `form` as in mtb200_gemm_lse. A target that is
// neither a column nor `ignore` is recorded and counts as ignored.
int mtb200_linear_nll(const void* x, const void* w, const long long* targets, float2* stats, float* at_target, int T, int columns, int H, float alpha, long long ignore, int form, float* loss, float* lse,
                      int* status, cudaStream_t st) {
  using namespace mtb;
  if (T <= 0) return 0;
  if (columns <= 0) return -10;
  if (const int rc = mtb200_gemm_lse(x, H, w, stats, at_target, targets, T, columns, H, alpha, form, status, st)) return rc;
  launch_pdl(nll::nll_kernel, T, nll::THREADS, 0, st, stats, at_target, targets, (columns + 127) / 128, static_cast<long long>(columns), ignore, loss, lse, status);
  return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

}  // extern "C"
