// Varlen causal GQA attention backward for sm_100a.
//
// One CTA owns one (sequence, 128-key block, kv head): K and V of that block stay in shared memory
// and dK, dV accumulate in tensor memory over every query head of the GQA group and every query
// block at or below the causal diagonal, so they are written once, without atomics. Per
// (query head, query block) the CTA runs five tcgen05 GEMMs on TRANSPOSED scores (keys on the lanes):
//   S^T = K Q^T        dP^T = V dO^T                        (TMEM, 128 columns each)
//   P^T = exp(S^T*scale - lse), dS^T = P^T * (dP^T - delta) * scale   (8 warps)
//   dV += P^T dO       dK += dS^T Q       dQ = dS K
// With keys on the lanes, P^T and dS^T are the A operands of dV and dK as they stand: they are written back over the
// columns of tensor memory they were computed from and never become shared-memory tiles (a 128 x 128 product with both
// operands in shared memory already reads the 128 bytes per clock that shared memory has). Only dS has a shared-memory
// tile, for dQ, where it is read MN-major. The room that frees holds a second Q tile.
//
// The MMAs of neighbouring iterations interleave so that the softmax of one runs under the products of another. Issue order:
//   ... dK(i) dQ(i) | dP(i+1) dV(i+1) S(i+2) | dK(i+1) dQ(i+1) | ...            (D = 64: dQ in front of dK)
// P(i+1) is computed while dK(i), dQ(i) run and dQ(i) is drained, dS(i+1) while dV(i+1) and S(i+2) run. The chain that bounds
// an iteration is dS -> dK dQ -> drain -> dP -> dS, where the form with everything in one chain (S dP | softmax | dK dV dQ |
// drain) had five products, the whole softmax and the drain. At D = 128 an iteration takes about 4950 clocks for 2560 of MMA,
// the same for every order of the products tried: the chain's hand-offs and latencies, and dQ's tensor reduces of 64 KB.
// 1 x 16384 tokens, 32/8 heads: 6.5 -> 5.5 ms at D = 128 (main kernel),
// 5.3 -> 3.2 ms at D = 64 (all passes; 3.6 with dV in front of dP and the shared columns).
//
// dQ shares the columns of dP at D = 128 (it is read out before the next dP is issued) and has its own at D = 64. Its tiles
// (several key blocks contribute to one query block) go through a 32 KB staging buffer, 64 columns at a time, into an fp32
// [T, Hq*D] accumulator with TMA tensor reduces (cp.reduce.async.bulk.tensor .add, one 32-column x 128-row box each,
// 128B-swizzled so the staging stores are free of bank conflicts); a small kernel rounds the accumulator to bf16 afterwards.
// Four warps of their own drain, one more issues the reduces, so the softmax warps see nothing of dQ.
//
// Rows past the end of the sequence contribute nothing: a query's lse is staged as +infinity, a key's dS is zero. That holds for finite numbers; under a rule also for others, which
// stay in their sample: the next sample's rows of Q, dO and K in a tile at this one's end, met by zeros, and what this sample's own K adds to the next one's rows of dQ. The first kernel looks
// for them (AttLook); where there are any, the TMA warp zeroes those rows before the tile counts as landed, and dQ of rows that are not there leaves as zeros.
//
// With short samples a CTA has few iterations, and its first loads and its stores count: the loads go out before tensor memory is allocated, and dK and dV
// leave by tensor stores. 148 samples of 128 tokens, 16/4 heads: 106 -> 102 us at D = 64, 193 -> 182 at 128 (all passes); 37 of 1024 492 -> 482, 879 -> 871.
// The rest of it is dQ's accumulator, which is written, added to and read in fp32: 78 MB of it in 101 us.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "attention_rule.cuh"
#include "entries.h"
#include "gemm_epilogue.cuh"
#include "ptx.cuh"

namespace mtb {

int make_tmap_2d_bf16(CUtensorMap* out, const void* base, uint64_t inner, uint64_t outer, uint64_t ld,
                      uint32_t box_inner, uint32_t box_outer);
int make_tmap_2d_f32(CUtensorMap* out, const void* base, uint64_t inner, uint64_t outer, uint64_t ld,
                     uint32_t box_inner, uint32_t box_outer);

constexpr int AB_B = 128;          // block edge (queries and keys)
// four warpgroups: {TMA, MMA, dQ reduce, row statistics}, 2 x softmax (two threads per key row), dQ drain
constexpr int AB_THREADS = 512;
// Registers per thread after the split; over the four warpgroups they add up to the 4 x 128 of the launch.
constexpr int AB_REGS_IO = 104, AB_REGS_SOFTMAX = 152, AB_REGS_DRAIN = 104;
static_assert(AB_REGS_IO + 2 * AB_REGS_SOFTMAX + AB_REGS_DRAIN == 4 * 128, "register split");

template <int D>
struct AttBwdSmem {
  static constexpr int TILE = AB_B * D * 2;         // a [128, D] bf16 tile
  static constexpr int OFF_K = 0, OFF_V = TILE, OFF_DO = 2 * TILE, OFF_Q = 3 * TILE;   // Q: 2 buffers
  static constexpr int OFF_DS = 5 * TILE;           // dS as [key, query], 128 x 128 bf16
  static constexpr int OFF_ST = OFF_DS + AB_B * AB_B * 2;    // dQ staging: 2 boxes of 128 rows x 32 fp32 columns
  static constexpr int OFF_STAT = OFF_ST + 2 * 16384;        // 2 buffers x {-lse * log2 e, -delta * scale} x 128 queries
  static constexpr int OFF_BAR = OFF_STAT + 2 * 2 * 128 * 4;
  // D = 128 fills the shared memory of an SM, so there is no slack to align with: the kernel checks that the window
  // starts on a 1024-byte boundary (swizzle atom).
  static constexpr int TOTAL = OFF_BAR + 256;
};

struct AbTrue { static constexpr bool value = true; };
struct AbFalse { static constexpr bool value = false; };

template <class R>
struct AttBwdParams {
  __nv_bfloat16* dqkv;
  long long ldq;
  const float* lse;
  const float* delta;
  float* dq_acc;        // [T, Hq*D] fp32, zeroed by attn_delta_kernel
  const int* plan;      // [n_items, 3] = seq_start, seq_len, k0; under a rule [n_items, 4], with the sample's prefix
  int T, Hq, Hkv;
  int G;                // Hq / Hkv
  unsigned hkv_inv;     // (2^32 - 1) / Hkv
  int splits;           // CTAs that share a key block's query heads (under a rule one's behind r.whole)
  float* ws;            // splits > 1: fp32 partials of dK and dV
  unsigned long long* counters;   // splits > 1: one arrival counter per (key block, warp); last_arrival in gemm_epilogue.cuh
  unsigned long long epoch;
  float scale;
  int* status;
  typename R::Args r;
};


template <int D, class R>
__global__ void __launch_bounds__(AB_THREADS, 1)
attn_bwd_kernel(const __grid_constant__ CUtensorMap tm_qkv, const __grid_constant__ CUtensorMap tm_do,
                const __grid_constant__ CUtensorMap tm_dq, const __grid_constant__ CUtensorMap tm_dkv, AttBwdParams<R> p) {
  using L = AttBwdSmem<D>;
  constexpr int KB = D / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw;
  if (smem_u32(smem) & 1023u) {   // uniform over the CTA: nothing has been allocated or armed yet
    if (threadIdx.x == 0) atomicExch(p.status, 20);
    return;
  }
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* kv_full = bars;          // K and V resident
  uint64_t* q_full = bars + 1;       // [2] Q landed
  uint64_t* q_free = bars + 3;       // [2] dK has read Q
  uint64_t* do_full = bars + 5;      // dO landed
  uint64_t* do_free = bars + 6;      // dV and dP have read dO
  uint64_t* s_full = bars + 7;       // S^T complete
  uint64_t* dp_full = bars + 8;      // dP^T complete; every earlier MMA too, so the dS tile is writable
  uint64_t* p_ready = bars + 9;      // P^T in tensor memory (8 arrivals)
  uint64_t* ds_ready = bars + 10;    // dS^T in tensor memory and dS in shared memory (8 arrivals)
  uint64_t* dq_full = bars + 11;     // dQ complete
  uint64_t* dq_read = bars + 12;     // dQ read out of tensor memory (4 arrivals): dP columns reusable
  uint64_t* stage_full = bars + 13;  // 64 columns of dQ staged (4 arrivals)
  uint64_t* stage_free = bars + 14;  // the tensor reduces have read the staging buffer
  uint64_t* stat_full = bars + 15;   // [2] lse / delta of a query block staged
  uint64_t* stat_free = bars + 17;   // [2] consumed (8 arrivals)
  uint64_t* all_done = bars + 19;    // dK and dV complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 20);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  [[maybe_unused]] uint64_t* tail_full = bars + 21;   // a tile whose last rows are to be zeroed landed

  pdl_wait();   // the work table comes first
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  bool careful = false;
  if constexpr (R::ON) careful = *static_cast<const volatile unsigned long long*>(p.r.odd) >= p.r.number;
  // units: the first r.whole have a CTA each, p.splits share those behind them, of which `shared` is the number
  int unit, sub, shared, own_splits = 1;
  if constexpr (R::ON) {
    unit = blockIdx.x; sub = shared = 0;
    if (unit >= p.r.whole && p.splits > 1) {
      own_splits = p.splits;
      shared = (unit - p.r.whole) / p.splits;
      sub = unit - p.r.whole - shared * p.splits;
      unit = p.r.whole + shared;
    }
  } else {
    unit = shared = p.splits == 1 ? blockIdx.x : blockIdx.x / p.splits;
    sub = blockIdx.x - unit * p.splits;
  }
  const int splits = R::ON ? own_splits : p.splits;
  int item = static_cast<int>(__umulhi(static_cast<unsigned>(unit), p.hkv_inv));   // unit / Hkv, or one less
  if (unit - item * p.Hkv >= p.Hkv) ++item;
  const int hk = unit - item * p.Hkv;
  const int G = p.G;
  const int h_first = hk * G + (splits == 1 ? 0 : G * sub / splits), heads = splits == 1 ? G : G * (sub + 1) / splits - G * sub / splits;
  const int seq_start = p.plan[item * R::ROW + 0], seq_len = p.plan[item * R::ROW + 1], k0 = p.plan[item * R::ROW + 2];
  // query blocks [jblk, nq) of the sequence: those at or below the diagonal; under a rule those that see a key of this block
  int prefix = 0, jblk = k0 / AB_B, nq = (seq_len + AB_B - 1) / AB_B;
  if constexpr (R::ON) {
    prefix = p.plan[item * R::ROW + 3];
    if (k0 < prefix) jblk = 0;
    else if (p.r.window < seq_len) nq = min(nq, (k0 + AB_B - 2 + p.r.window) / AB_B + 1);
  }
  const int per_head = nq - jblk;
  const int n_iters = heads * per_head;
  // bounds check of the host-built work item (uniform over the CTA; nothing allocated or armed yet)
  if (seq_start < 0 || seq_len <= 0 || k0 < 0 || k0 >= seq_len || prefix < 0 || prefix > seq_len || static_cast<long long>(seq_start) + seq_len > p.T) {
    if (threadIdx.x == 0) atomicExch(p.status, 61);
    return;
  }

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1); mbar_init(do_full, 1); mbar_init(do_free, 1); mbar_init(s_full, 1); mbar_init(dp_full, 1);
    mbar_init(p_ready, 8); mbar_init(ds_ready, 8); mbar_init(dq_full, 1); mbar_init(dq_read, 4);
    mbar_init(stage_full, 4); mbar_init(stage_free, 1); mbar_init(all_done, 1);
    for (int b = 0; b < 2; ++b) { mbar_init(&q_full[b], 1); mbar_init(&q_free[b], 1); mbar_init(&stat_full[b], 1); mbar_init(&stat_free[b], 8); }
    *abort_flag = 0;
    if constexpr (R::ON) mbar_init(tail_full, 1);
    fence_mbar_init();
    if (!careful) {   // the first loads go out before anything else is set up
      mbar_arrive_expect_tx(kv_full, 2 * L::TILE);
      mbar_arrive_expect_tx(&q_full[0], L::TILE);
      mbar_arrive_expect_tx(do_full, L::TILE);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        tma_load_2d(smem + L::OFF_K + kb * 16384, &tm_qkv, kv_full, (p.Hq + hk) * D + kb * 64, seq_start + k0);
        tma_load_2d(smem + L::OFF_Q + kb * 16384, &tm_qkv, &q_full[0], h_first * D + kb * 64, seq_start + jblk * AB_B);
        tma_load_2d(smem + L::OFF_V + kb * 16384, &tm_qkv, kv_full, (p.Hq + p.Hkv + hk) * D + kb * 64, seq_start + k0);
        tma_load_2d(smem + L::OFF_DO + kb * 16384, &tm_do, do_full, h_first * D + kb * 64, seq_start + jblk * AB_B);
      }
    }
    tma_prefetch_desc(&tm_dq);
    tma_prefetch_desc(&tm_dkv);
  }
  if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t t_s = tmem_base, t_dp = tmem_base + 128, t_dv = tmem_base + 256, t_dk = tmem_base + 256 + D;
  // dQ has columns of its own where they are left over (D = 64); at D = 128 it shares those of dP
  constexpr bool DQ_OWN = 2 * 128 + 3 * D <= 512;
  const uint32_t t_dq = DQ_OWN ? tmem_base + 256 + 2 * D : t_dp;

  if (warp < 4) {
    setmaxnreg_dec<AB_REGS_IO>();
    if (warp == 0) {
      // ------------------------------------------------------------------ TMA producer
      if (R::ON && careful) {
        if (elect_one()) {
          uint32_t tails = 0;
          auto request = [&](uint8_t* tile, const CUtensorMap* map, uint64_t* bar, int column, int first) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) tma_load_2d(tile + kb * 16384, map, bar, column + kb * 64, seq_start + first);
          };
          // the tile from row `first` on, landed and the rows behind the sequence zeroed
          auto tail = [&](uint8_t* tile, const CUtensorMap* map, int column, int first) -> bool {
            mbar_arrive_expect_tx(tail_full, L::TILE);
            request(tile, map, tail_full, column, first);
            if (!mbar_wait(tail_full, tails++ & 1, abort_flag)) return false;
            zero_rows<KB>(tile, seq_len - first, 0, 1);
            return true;
          };
          auto load = [&](uint8_t* tile, const CUtensorMap* map, uint64_t* full, int column, int first) -> bool {
            if (first + AB_B > seq_len) {
              if (!tail(tile, map, column, first)) return false;
              mbar_arrive(full);
              return true;
            }
            mbar_arrive_expect_tx(full, L::TILE);
            request(tile, map, full, column, first);
            return true;
          };
          const bool k_tail = k0 + AB_B > seq_len;   // K and V share a barrier: the arrival comes with V's bytes
          if (k_tail && !tail(smem + L::OFF_K, &tm_qkv, (p.Hq + hk) * D, k0)) { atomicExch(p.status, 21); goto done; }
          mbar_arrive_expect_tx(kv_full, k_tail ? L::TILE : 2 * L::TILE);
          if (!k_tail) request(smem + L::OFF_K, &tm_qkv, kv_full, (p.Hq + hk) * D, k0);
          request(smem + L::OFF_V, &tm_qkv, kv_full, (p.Hq + p.Hkv + hk) * D, k0);
          int h = h_first, i = jblk;
          for (int it = 0; it < n_iters; ++it) {
            const int b = it & 1;
            if (it > 1 && !mbar_wait(&q_free[b], ((it - 2) >> 1) & 1, abort_flag)) { atomicExch(p.status, 21); goto done; }
            if (!load(smem + L::OFF_Q + b * L::TILE, &tm_qkv, &q_full[b], h * D, i * AB_B)) { atomicExch(p.status, 21); goto done; }
            if (it > 0 && !mbar_wait(do_free, (it - 1) & 1, abort_flag)) { atomicExch(p.status, 21); goto done; }
            if (!load(smem + L::OFF_DO, &tm_do, do_full, h * D, i * AB_B)) { atomicExch(p.status, 21); goto done; }
            if (++i == nq) { i = jblk; ++h; }
          }
          pdl_trigger();
        }
      } else if (elect_one()) {
        int h = h_first, i = jblk;
        if (++i == nq) { i = jblk; ++h; }
        for (int it = 1; it < n_iters; ++it) {   // the first iteration's tiles have been asked for above
          const int b = it & 1;
          if (it > 1 && !mbar_wait(&q_free[b], ((it - 2) >> 1) & 1, abort_flag)) { atomicExch(p.status, 21); goto done; }
          mbar_arrive_expect_tx(&q_full[b], L::TILE);
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
            tma_load_2d(smem + L::OFF_Q + b * L::TILE + kb * 16384, &tm_qkv, &q_full[b], h * D + kb * 64, seq_start + i * AB_B);
          if (it > 0 && !mbar_wait(do_free, (it - 1) & 1, abort_flag)) { atomicExch(p.status, 21); goto done; }
          mbar_arrive_expect_tx(do_full, L::TILE);
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
            tma_load_2d(smem + L::OFF_DO + kb * 16384, &tm_do, do_full, h * D + kb * 64, seq_start + i * AB_B);
          if (++i == nq) { i = jblk; ++h; }
        }
        pdl_trigger();   // what is left is the last iteration and the stores of dK and dV
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------ MMA issuer
      if (elect_one()) {
        constexpr uint32_t id_nt = make_idesc_bf16(AB_B, AB_B, false, false);   // S^T, dP^T
        constexpr uint32_t id_ts = make_idesc_bf16(AB_B, D, false, true);       // dV, dK (A in tensor memory)
        constexpr uint32_t id_dq = make_idesc_bf16(AB_B, D, true, true);        // dQ = dS K
        // every tile lives at a fixed shared-memory address, so the descriptors are built once; inside
        // the loop a k-step is one add (start-address field, in 16-byte units)
        const uint32_t sk = smem_u32(smem + L::OFF_K), sq = smem_u32(smem + L::OFF_Q), sdo = smem_u32(smem + L::OFF_DO);
        const uint32_t dKk = smem_desc_lo(sk, 16), dVk = smem_desc_lo(smem_u32(smem + L::OFF_V), 16);
        const uint32_t dQk = smem_desc_lo(sq, 16), dDOk = smem_desc_lo(sdo, 16);
        const uint32_t dDSm = smem_desc_lo(smem_u32(smem + L::OFF_DS), 16384), dKm = smem_desc_lo(sk, 16384);
        const uint32_t dQm = smem_desc_lo(sq, 16384), dDOm = smem_desc_lo(sdo, 16384);
        auto kstep = [](int k) { return static_cast<uint32_t>((k >> 2) * 1024 + (k & 3) * 2); };   // K-major: 32 B per step, 16 KB per 64
        auto mstep = [](int k) { return static_cast<uint32_t>(k * 128); };                           // MN-major: 2048 B per step
        auto astep = [](int k) { return static_cast<uint32_t>(k < 4 ? k * 8 : 64 + (k - 4) * 8); };   // bf16 A operand in tensor memory
        auto qbuf = [&](int it) { return static_cast<uint32_t>((it & 1) * (L::TILE >> 4)); };
        auto issue_s = [&](int it) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) umma_bf16_lo(t_s, dKk + kstep(k), dQk + qbuf(it) + kstep(k), id_nt, k != 0);
          umma_commit(s_full);
        };
        auto issue_dp = [&]() {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) umma_bf16_lo(t_dp, dVk + kstep(k), dDOk + kstep(k), id_nt, k != 0);
          umma_commit(dp_full);
        };
        auto issue_dv = [&](int it) {   // dP of the same iteration has been issued: dO is free when both are done
#pragma unroll
          for (int k = 0; k < AB_B / 16; ++k) umma_bf16_ts_lo(t_dv, t_s + astep(k), dDOm + mstep(k), id_ts, it != 0 || k != 0);
          umma_commit(do_free);
        };
        if (!mbar_wait(kv_full, 0, abort_flag)) { atomicExch(p.status, 22); goto done; }
        if (!mbar_wait(&q_full[0], 0, abort_flag)) { atomicExch(p.status, 23); goto done; }
        tc_fence_after();
        issue_s(0);
        if (!mbar_wait(do_full, 0, abort_flag)) { atomicExch(p.status, 23); goto done; }
        tc_fence_after();
        issue_dp();
        if (!mbar_wait(p_ready, 0, abort_flag)) { atomicExch(p.status, 25); goto done; }
        tc_fence_after();
        issue_dv(0);
        if (n_iters > 1) {
          if (!mbar_wait(&q_full[1], 0, abort_flag)) { atomicExch(p.status, 23); goto done; }
          tc_fence_after();
          issue_s(1);
        }
        auto issue_dk = [&](int it) {
#pragma unroll
          for (int k = 0; k < AB_B / 16; ++k) umma_bf16_ts_lo(t_dk, t_dp + astep(k), dQm + qbuf(it) + mstep(k), id_ts, it != 0 || k != 0);
          umma_commit(&q_free[it & 1]);
        };
        auto issue_dq = [&]() {
#pragma unroll
          for (int k = 0; k < AB_B / 16; ++k) umma_bf16_lo(t_dq, dDSm + mstep(k), dKm + mstep(k), id_dq, k != 0);
          umma_commit(dq_full);
        };
        for (int it = 0; it < n_iters; ++it) {
          if (!mbar_wait(ds_ready, it & 1, abort_flag)) { atomicExch(p.status, 25); goto done; }
          if (DQ_OWN && it > 0 && !mbar_wait(dq_read, (it - 1) & 1, abort_flag)) { atomicExch(p.status, 24); goto done; }
          tc_fence_after();
          if (DQ_OWN) { issue_dq(); issue_dk(it); }
          else { issue_dk(it); issue_dq(); }     // dK reads dS^T from the columns that dQ overwrites
          if (it + 1 < n_iters) {
            if (!mbar_wait(do_full, (it + 1) & 1, abort_flag)) { atomicExch(p.status, 23); goto done; }
            if (!DQ_OWN && !mbar_wait(dq_read, it & 1, abort_flag)) { atomicExch(p.status, 24); goto done; }
            tc_fence_after();
            issue_dp();
            if (!mbar_wait(p_ready, (it + 1) & 1, abort_flag)) { atomicExch(p.status, 25); goto done; }
            tc_fence_after();
            issue_dv(it + 1);
            if (it + 2 < n_iters) {
              if (!mbar_wait(&q_full[it & 1], ((it + 2) >> 1) & 1, abort_flag)) { atomicExch(p.status, 23); goto done; }
              tc_fence_after();
              issue_s(it + 2);
            }
          }
        }
        umma_commit(all_done);
      }
    } else if (warp == 2) {
      // ------------------------------------------------------------------ dQ reduce warp
      if (elect_one()) {
        const uint32_t stage = smem_u32(smem + L::OFF_ST);
        int h = h_first, i = jblk, n = 0;
        for (int it = 0; it < n_iters; ++it) {
          for (int part = 0; part < KB; ++part, ++n) {
            if (!mbar_wait(stage_full, n & 1, abort_flag)) { atomicExch(p.status, 30); goto done; }
#pragma unroll
            for (int c = 0; c < 2; ++c)
              asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.bulk_group [%0, {%2, %3}], [%1];"
                           ::"l"(reinterpret_cast<uint64_t>(&tm_dq)), "r"(stage + c * 16384), "r"(h * D + part * 64 + c * 32),
                             "r"(seq_start + i * AB_B) : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            mbar_arrive(stage_free);
          }
          if (++i == nq) { i = jblk; ++h; }
        }
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");   // every add has been performed before the CTA exits
      }
    } else {
      // ------------------------------------------------------------------ row statistics of the query blocks
      float* stat = reinterpret_cast<float*>(smem + L::OFF_STAT);
      int h = h_first, i = jblk;
      for (int it = 0; it < n_iters; ++it) {
        const int b = it & 1;
        if (it > 1 && !mbar_wait(&stat_free[b], ((it - 2) >> 1) & 1, abort_flag)) { atomicExch(p.status, 32); goto done; }
        const long long base = static_cast<long long>(h) * p.T + seq_start;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int x = j * 32 + lane, qpos = i * AB_B + x;
          const bool ok = qpos < seq_len;
          float nl = ok ? p.lse[base + qpos] * -1.4426950408889634f : -INFINITY;
          // the part of a bias that goes by the query alone, within the block; where queries see keys behind them the softmax warps form all of it
          if constexpr (R::BIAS)
            if (!(k0 < prefix && i * AB_B < k0 + AB_B - 1)) nl -= p.r.slopes[h] * 1.4426950408889634f * x;
          stat[b * 256 + x] = nl;
          stat[b * 256 + 128 + x] = ok ? p.delta[base + qpos] * -p.scale : 0.f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&stat_full[b]);
        if (++i == nq) { i = jblk; ++h; }
      }
    }
  } else if (warp >= 12) {
    // ------------------------------------------------------------------ dQ drain (one thread per query row)
    setmaxnreg_dec<AB_REGS_DRAIN>();
    const int r = (warp & 3) * 32 + lane;
    const uint32_t src = t_dq + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    uint8_t* rowp = smem + L::OFF_ST + r * 128;
    int n = 0;
    [[maybe_unused]] int i = jblk;
    for (int it = 0; it < n_iters; ++it) {
      if (!mbar_wait(dq_full, it & 1, abort_flag)) { atomicExch(p.status, 28); goto done; }
      tc_fence_after();
#pragma unroll 1
      for (int part = 0; part < KB; ++part, ++n) {
        uint32_t v[2][32];
        tmem_ld_32x32(src + part * 64, v[0]);
        tmem_ld_32x32(src + part * 64 + 32, v[1]);
        tmem_ld_wait();
        if (part == KB - 1) {   // the last columns are in registers: the next dP may overwrite them
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(dq_read);
        }
        if constexpr (R::ON) {
          if (careful && i * AB_B + r >= seq_len) {
#pragma unroll
            for (int x = 0; x < 32; ++x) v[0][x] = v[1][x] = 0u;
          }
        }
        if (n > 0 && !mbar_wait(stage_free, (n - 1) & 1, abort_flag)) { atomicExch(p.status, 31); goto done; }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int g = 0; g < 8; ++g)
            *reinterpret_cast<uint4*>(rowp + c * 16384 + ((g ^ (r & 7)) << 4)) = make_uint4(v[c][g * 4], v[c][g * 4 + 1], v[c][g * 4 + 2], v[c][g * 4 + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(stage_full);
      }
      if constexpr (R::ON) { if (++i == nq) i = jblk; }
    }
  } else {
    // ------------------------------------------------------------------ softmax (two threads per key row)
    setmaxnreg_inc<AB_REGS_SOFTMAX>();
    const int q = warp & 3;
    const int half = (warp >> 2) - 1;      // which 64 queries (softmax) / which half of the D columns (epilogue)
    const int r = q * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t ts = t_s + lane_addr + half * 64, tp = t_dp + lane_addr + half * 64;
    const float sl2 = p.scale * 1.4426950408889634f;
    const float2 sl2v = make_float2(sl2, sl2), scv = make_float2(p.scale, p.scale);
    uint8_t* ds_row = smem + L::OFF_DS + half * 16384 + r * 128;
    int i = jblk;
    [[maybe_unused]] int h = h_first;
    for (int it = 0; it < n_iters; ++it) {
      const int b = it & 1;
      const float* stat = reinterpret_cast<const float*>(smem + L::OFF_STAT) + b * 256 + half * 64;
      if (!mbar_wait(&stat_full[b], (it >> 1) & 1, abort_flag)) { atomicExch(p.status, 26); goto done; }
      if (!mbar_wait(s_full, it & 1, abort_flag)) { atomicExch(p.status, 26); goto done; }
      tc_fence_after();
      float2 pr[32];      // probabilities of this thread's 64 (key, query) pairs; with a cap times its derivative, 1 - tanh^2
      if constexpr (R::ON) {
        uint32_t sv[2][32];
        tmem_ld_32x32(ts, sv[0]);
        tmem_ld_32x32(ts + 32, sv[1]);
        tmem_ld_wait();
        const int key = k0 + r, q0 = i * AB_B;
        float slope2 = 0.f;
        if constexpr (R::BIAS) slope2 = p.r.slopes[h] * 1.4426950408889634f;
        if constexpr (R::CAP) {   // capped scores in place of the products
          float big[2] = {0.f, 0.f};
#pragma unroll
          for (int cc = 0; cc < 2; ++cc)
#pragma unroll
            for (int x = 0; x < 32; x += 2) big[cc] = fmax3(big[cc], fabsf(__uint_as_float(sv[cc][x])), fabsf(__uint_as_float(sv[cc][x + 1])));
          auto form = [&](auto low) {
#pragma unroll
            for (int cc = 0; cc < 2; ++cc)
#pragma unroll
              for (int x = 0; x < 32; x += 2) {
                const float2 s = make_float2(__uint_as_float(sv[cc][x]), __uint_as_float(sv[cc][x + 1]));
                const float2 v = decltype(low)::value ? fmul2(s, cap_half_part(p.r.cap, s)) : cap_pair(p.r.cap, s);
                sv[cc][x] = __float_as_uint(v.x); sv[cc][x + 1] = __float_as_uint(v.y);
              }
          };
          if (__all_sync(0xffffffffu, fmaxf(big[0], big[1]) <= p.r.cap.low)) form(AbTrue{});
          else if (__all_sync(0xffffffffu, fmaxf(big[0], big[1]) <= p.r.cap.most)) form(AbFalse{});
          else {
            cap_in_place(p.r.cap, ts, 4);
            tmem_ld_32x32(ts, sv[0]);
            tmem_ld_32x32(ts + 32, sv[1]);
            tmem_ld_wait();
          }
        }
        // EDGE: an edge of the mask crosses the tile; RIGHT (with a bias): queries see keys behind them
        auto probabilities = [&](auto edge, auto right) {
          [[maybe_unused]] constexpr bool EDGE = decltype(edge)::value, RIGHT = decltype(right)::value;
          [[maybe_unused]] const float behind = static_cast<float>(q0 + half * 64 - key);
          [[maybe_unused]] const float2 row = splat(-slope2 * static_cast<float>(q0 - key));
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            uint32_t pk[16];
            const uint32_t seen = EDGE ? att_queries_seen(p.r, key, q0 + half * 64 + cc * 32, prefix) : 0u;
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              const float2 nl = *reinterpret_cast<const float2*>(stat + cc * 32 + x);
              const float2 s = make_float2(__uint_as_float(sv[cc][x]), __uint_as_float(sv[cc][x + 1]));
              float2 a = R::CAP ? fadd2(s, nl) : ffma2(s, sl2v, nl);
              if constexpr (R::BIAS)
                a = fadd2(a, RIGHT ? make_float2(-slope2 * fabsf(behind + (cc * 32 + x)), -slope2 * fabsf(behind + (cc * 32 + x + 1))) : row);
              if constexpr (EDGE) {
                if (!(seen >> x & 1u)) a.x = -INFINITY;
                if (!(seen >> (x + 1) & 1u)) a.y = -INFINITY;
              }
              const float2 e = make_float2(ex2_mufu(a.x), !EDGE && (x & 2) ? ex2_fma(a.y) : ex2_mufu(a.y));   // masked scores want exact zeros
              pk[x >> 1] = pack_bf16(e.x, e.y);
              pr[cc * 16 + (x >> 1)] = R::CAP ? fmul2(e, ffma2(fmul2(s, splat(p.r.cap.inv2)), s, splat(1.f))) : e;
            }
            tmem_st_32x16(ts + cc * 16, pk);
          }
        };
        const bool edge = !att_all_seen(p.r, q0, k0, prefix);
        if (R::BIAS && k0 < prefix && q0 < k0 + AB_B - 1) {
          if (edge) probabilities(AbTrue{}, AbTrue{}); else probabilities(AbFalse{}, AbTrue{});
        } else if (edge) probabilities(AbTrue{}, AbFalse{});
        else probabilities(AbFalse{}, AbFalse{});
      } else {
        uint32_t sv[2][32];
        tmem_ld_32x32(ts, sv[0]);
        tmem_ld_32x32(ts + 32, sv[1]);
        tmem_ld_wait();
        if (i == jblk) {   // diagonal block: of the queries, 32 at a time, a warp's keys are seen by none before piece q, by those from the lane on in it
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            if (half * 2 + cc <= q) {
#pragma unroll
              for (int x = 0; x < 32; ++x)
                if (half * 2 + cc < q || lane > x) sv[cc][x] = 0xff800000u;   // exp2(-inf) = 0
            }
          }
        }
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          uint32_t pk[16];
#pragma unroll
          for (int x = 0; x < 32; x += 4) {
            const float4 nl = *reinterpret_cast<const float4*>(stat + cc * 32 + x);
            // packed fp32 pairs: one FMA scales and shifts two scores
            const float2 a0 = ffma2(make_float2(__uint_as_float(sv[cc][x]), __uint_as_float(sv[cc][x + 1])), sl2v, make_float2(nl.x, nl.y));
            const float2 a1 = ffma2(make_float2(__uint_as_float(sv[cc][x + 2]), __uint_as_float(sv[cc][x + 3])), sl2v, make_float2(nl.z, nl.w));
            // a quarter of the exponentials runs on the FMA pipe: the special-function unit bounds this phase
            const float2 e0 = make_float2(ex2_mufu(a0.x), ex2_mufu(a0.y)), e1 = make_float2(ex2_mufu(a1.x), ex2_fma(a1.y));
            pr[cc * 16 + (x >> 1)] = e0;
            pr[cc * 16 + (x >> 1) + 1] = e1;
            pk[x >> 1] = pack_bf16(e0.x, e0.y);
            pk[(x >> 1) + 1] = pack_bf16(e1.x, e1.y);
          }
          tmem_st_32x16(ts + cc * 16, pk);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready);
      if (!mbar_wait(dp_full, it & 1, abort_flag)) { atomicExch(p.status, 27); goto done; }
      tc_fence_after();
      uint32_t dv[2][32];
      tmem_ld_32x32(tp, dv[0]);
      tmem_ld_32x32(tp + 32, dv[1]);
      tmem_ld_wait();
#pragma unroll
      for (int cc = 0; cc < 2; ++cc) {
        uint32_t dk[16];
#pragma unroll
        for (int x = 0; x < 32; x += 4) {
          const float4 nd = *reinterpret_cast<const float4*>(stat + 128 + cc * 32 + x);
          // one FMA forms (dP - delta) * scale for two entries
          const float2 d0 = ffma2(make_float2(__uint_as_float(dv[cc][x]), __uint_as_float(dv[cc][x + 1])), scv, make_float2(nd.x, nd.y));
          const float2 d1 = ffma2(make_float2(__uint_as_float(dv[cc][x + 2]), __uint_as_float(dv[cc][x + 3])), scv, make_float2(nd.z, nd.w));
          const float2 s0 = fmul2(pr[cc * 16 + (x >> 1)], d0), s1 = fmul2(pr[cc * 16 + (x >> 1) + 1], d1);
          dk[x >> 1] = pack_bf16(s0.x, s0.y);
          dk[(x >> 1) + 1] = pack_bf16(s1.x, s1.y);
        }
        if (k0 + AB_B > seq_len) {   // last key block: keys past the sequence give nothing to dQ (their rows of dK and dV are not stored)
#pragma unroll
          for (int x = 0; x < 16; ++x) dk[x] = k0 + r < seq_len ? dk[x] : 0u;
        }
        tmem_st_32x16(tp + cc * 16, dk);
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<uint4*>(ds_row + (((cc * 4 + g) ^ (r & 7)) << 4)) = make_uint4(dk[g * 4], dk[g * 4 + 1], dk[g * 4 + 2], dk[g * 4 + 3]);
      }
      tmem_st_wait();
      fence_proxy_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) { mbar_arrive(ds_ready); mbar_arrive(&stat_free[b]); }
      if (++i == nq) {
        i = jblk;
        if constexpr (R::BIAS) ++h;
      }
    }
    // epilogue: dK, dV (rows = keys)
    if (!mbar_wait(all_done, 0, abort_flag)) { atomicExch(p.status, 29); goto done; }
    tc_fence_after();
    const int kpos = k0 + r;
    const bool ok = kpos < seq_len;
    const bool whole = kpos - lane + 31 < seq_len;   // uniform over the warp
    __nv_bfloat16* rowp = p.dqkv + (static_cast<long long>(seq_start) + kpos) * p.ldq;
    // A warp has 64 columns of one gradient (D = 64: dK or dV) or of both (D = 128), in pieces of 32; rows that all exist leave by tensor stores, staged
    // where Q was (stored 16 bytes at a time to rows that are far apart, they took 3500 clocks per CTA at D = 64 and 9000 at 128).
    constexpr int PIECES = D / 32, BOXES = D / 64;
    constexpr int PART = PIECES * 1024;   // floats of a warp's partial
    uint8_t* box = smem + L::OFF_Q + (warp - 4) * BOXES * 4096;
    auto gradient = [&](int x) { return D == 64 ? half : x >> 1; };                          // 0: dK, 1: dV
    auto column = [&](int x) { return D == 64 ? x * 32 : half * 64 + (x & 1) * 32; };
    auto store = [&](int x, const float (&f)[32]) {   // piece x of this thread's row
      const int col = (gradient(x) == 0 ? p.Hq + hk : p.Hq + p.Hkv + hk) * D + column(x);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint4 d = make_uint4(pack_bf16(f[g * 8], f[g * 8 + 1]), pack_bf16(f[g * 8 + 2], f[g * 8 + 3]),
                                   pack_bf16(f[g * 8 + 4], f[g * 8 + 5]), pack_bf16(f[g * 8 + 6], f[g * 8 + 7]));
        if (whole) *reinterpret_cast<uint4*>(box + (x >> 1) * 4096 + lane * 128 + ((((x & 1) * 4 + g) ^ (lane & 7)) << 4)) = d;
        else if (ok) *reinterpret_cast<uint4*>(rowp + col + g * 8) = d;
      }
      if (whole && (x & 1)) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&tm_dkv, box + (x >> 1) * 4096, col - 32, seq_start + kpos);
          bulk_commit();
        }
      }
    };
    float* base = p.ws + (static_cast<long long>(shared) * splits * 8 + (warp - 4)) * PART + lane * 4;   // split s: + s * 8 * PART
#pragma unroll 1
    for (int x = 0; x < PIECES; ++x) {
      uint32_t v[32];
      tmem_ld_32x32((gradient(x) == 0 ? t_dk : t_dv) + lane_addr + column(x), v);
      tmem_ld_wait();
      float f[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(v[j]);
      if (splits == 1) store(x, f);
      else {   // lane-interleaved 16-byte pieces: every access is one contiguous 512 bytes
#pragma unroll
        for (int j = 0; j < 8; ++j)
          __stcg(reinterpret_cast<float4*>(base + static_cast<long long>(sub) * 8 * PART + x * 1024 + j * 128), make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]));
      }
    }
    if (splits > 1) {   // the warp that arrives last adds the partials, in split order whoever that is; nobody waits
      unsigned long long* counter = p.counters + shared * 8 + (warp - 4);
      __threadfence();
      __syncwarp();
      unsigned last = 0;
      if (lane == 0) last = last_arrival(counter, p.epoch, splits);
      last = __shfl_sync(0xffffffffu, last, 0);
      if (last) {
        __threadfence();
#pragma unroll 1
        for (int x = 0; x < PIECES; ++x) {
          float f[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) f[j] = 0.f;
#pragma unroll 2
          for (int s = 0; s < splits; ++s) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float4 t = __ldcg(reinterpret_cast<const float4*>(base + static_cast<long long>(s) * 8 * PART + x * 1024 + j * 128));
              f[4 * j] += t.x; f[4 * j + 1] += t.y; f[4 * j + 2] += t.z; f[4 * j + 3] += t.w;
            }
          }
          store(x, f);
        }
        if (lane == 0) *counter = 0;
      }
    }
    if (lane == 0) bulk_wait_read<0>();   // before the shared memory goes away
  }
done:
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Under a rule the first kernel also looks for what is not finite where samples share a tile. A row of dO, O, V or Q shows in its delta, as O is not finite with them, but for infinities of Q under
// a cap, which bounds the scores they make; a row of K need not show (its score may be -infinity). So K is read along, and with a cap the rows of Q behind a sample's end that share a tile with
// it, by blocks of their own: LOOK_BLOCKS to a row of the work table (a key block of 128), a warp to two rows.
// 8192 tokens in three samples, 32/8 heads of 128, capped: the first kernel 42.8 -> 47.1 us (of 655), 41 short samples at D = 64 without a cap 17.0 -> 18.5 (of 148), 148 samples of about 100 tokens, 16/4 heads of
// 128, capped, where those rows are most of Q, 39 -> 49 (of 242); the kernel that works on the tiles is as fast as it was. Zeroing every such row instead took 7 to 15 % of the whole, seeing them in the products 3 to 10 %.
constexpr int LOOK_BLOCKS = 8;
struct AttLook {
  static constexpr bool ON = true;
  const __nv_bfloat16* qkv;
  long long ld;
  const int* plan;
  int G, blocks;   // blocks: the first of the launch, for Q (none without a cap)
  unsigned long long *odd, number;
  __device__ __forceinline__ void report(bool bad) const { if (bad) atomicMax(odd, number); }
};
struct AttNoLook { static constexpr bool ON = false; };
// Zero of a finite 16 bytes, NaN of others.
__device__ __forceinline__ float2 att_times_zero(const uint4& u, float2 z) {
  const float2 none = make_float2(0.f, 0.f);
  z = ffma2(unpack_bf16(u.x), none, z); z = ffma2(unpack_bf16(u.y), none, z); z = ffma2(unpack_bf16(u.z), none, z);
  return ffma2(unpack_bf16(u.w), none, z);
}
__device__ __forceinline__ void att_look_behind(const AttLook& a, int n, int HqD) {
  const int b = blockIdx.x, item = b / LOOK_BLOCKS;
  const int seq_start = a.plan[item * 4], seq_len = a.plan[item * 4 + 1], k0 = a.plan[item * 4 + 2];
  if (seq_start < 0 || seq_len <= 0 || k0 < 0 || k0 >= seq_len || static_cast<long long>(seq_start) + seq_len > n) return;   // reported by the kernel that works on it
  const int r0 = k0 + (b % LOOK_BLOCKS) * 16 + static_cast<int>(threadIdx.x >> 5) * 2;
  if (r0 + 1 < seq_len) return;
  float2 z = make_float2(0.f, 0.f);
  for (int c = static_cast<int>(threadIdx.x & 31) * 8; c < HqD; c += 2 * 256) {
    uint4 u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = r0 + (k & 1), x = c + (k >> 1) * 256;
      u[k] = r >= seq_len && seq_start + r < n && x < HqD ? *reinterpret_cast<const uint4*>(a.qkv + static_cast<long long>(seq_start + r) * a.ld + x) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) z = att_times_zero(u[k], z);
  }
  a.report(!(z.x + z.y == 0.f));
}

// delta[h, t] = sum_d dO[t, h, d] * O[t, h, d], and zeros into the dQ accumulator, for the first n of T rows; D / 8 lanes per (t, h), one 16-byte load of each operand per
// lane and row, two rows in flight. Bound by reading dO and O and writing the accumulator once (as a launch of its own the zeroing
// took 9 us next to 14 us for 12 345 tokens x 16 heads of 64, forward and backward together 177 us, now 168).
template <class Look>
static __global__ void __launch_bounds__(256, Look::ON ? 6 : 0) attn_delta_kernel(const __nv_bfloat16* __restrict__ o, long long ldo, const __nv_bfloat16* __restrict__ dout,
                                                        long long lddo, float* __restrict__ delta, float* __restrict__ dq_acc, int T, int n, int Hq, int D, [[maybe_unused]] Look look) {
  pdl_trigger();
  pdl_wait();
  if constexpr (Look::ON) {
    if (static_cast<int>(blockIdx.x) < look.blocks) { att_look_behind(look, n, Hq * D); return; }
  }
  int look_blocks = 0;
  if constexpr (Look::ON) look_blocks = look.blocks;
  const int lanes = D >> 3;   // 8 or 16: a power of two that divides the warp
  const int per_block = 256 / lanes, sub = threadIdx.x / lanes, c = (threadIdx.x & (lanes - 1)) * 8;
  const long long rows = static_cast<long long>(n) * Hq, first = static_cast<long long>(static_cast<int>(blockIdx.x) - look_blocks) * 2 * per_block + sub;
  uint4 a[2], b[2];
  [[maybe_unused]] uint4 kv[2];
  int t[2], h[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const long long row = first + k * per_block;
    a[k] = b[k] = make_uint4(0u, 0u, 0u, 0u);
    t[k] = rows <= 0xffffffffLL ? static_cast<int>(static_cast<unsigned>(row) / static_cast<unsigned>(Hq)) : static_cast<int>(row / Hq);
    h[k] = static_cast<int>(row - static_cast<long long>(t[k]) * Hq);
    if (row < rows) {
      a[k] = *reinterpret_cast<const uint4*>(o + static_cast<long long>(t[k]) * ldo + h[k] * D + c);
      b[k] = *reinterpret_cast<const uint4*>(dout + static_cast<long long>(t[k]) * lddo + h[k] * D + c);
    }
    if constexpr (Look::ON) {
      kv[k] = make_uint4(0u, 0u, 0u, 0u);
      const int head = h[k] / look.G;
      if (row < rows && head * look.G == h[k]) kv[k] = *reinterpret_cast<const uint4*>(look.qkv + static_cast<long long>(t[k]) * look.ld + (Hq + head) * D + c);
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const long long row = first + k * per_block;
    const uint32_t av[4] = {a[k].x, a[k].y, a[k].z, a[k].w}, bv[4] = {b[k].x, b[k].y, b[k].z, b[k].w};
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 u = unpack_bf16(av[i]), v = unpack_bf16(bv[i]);
      s += u.x * v.x + u.y * v.y;
    }
    for (int m = lanes >> 1; m > 0; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
    if (row < rows) {
      if (c == 0) delta[static_cast<long long>(h[k]) * T + t[k]] = s;
      if constexpr (Look::ON) {
        const float2 z = att_times_zero(kv[k], make_float2(0.f, 0.f));
        look.report(!(fabsf(s) <= 3.4e38f && z.x + z.y == 0.f));
      }
      float4* z = reinterpret_cast<float4*>(dq_acc + row * D + c);
      z[0] = z[1] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
}

// dqkv[t, 0:Hq*D] = bf16(dq_acc[t, :])
static __global__ void __launch_bounds__(256) attn_dq_store_kernel(const float* __restrict__ acc, __nv_bfloat16* __restrict__ dqkv, long long ldq,
                                                           long long T, int HqD) {
  pdl_trigger();
  pdl_wait();
  // grid = (tokens, column blocks): no 64-bit division per thread
  const long long t = blockIdx.x;
  const int c = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
  if (c >= HqD) return;
  const float4 a = *reinterpret_cast<const float4*>(acc + t * HqD + c), b = *reinterpret_cast<const float4*>(acc + t * HqD + c + 4);
  *reinterpret_cast<uint4*>(dqkv + t * ldq + c) =
      make_uint4(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w), pack_bf16(b.x, b.y), pack_bf16(b.z, b.w));
}

template <int D, class R>
static int launch_bwd(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& c, const CUtensorMap& d, const AttBwdParams<R>& p, int n_items, bool in_order, cudaStream_t st) {
  static bool configured = false;
  auto kern = attn_bwd_kernel<D, R>;
  if (!configured) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, AttBwdSmem<D>::TOTAL) != cudaSuccess) return -4;
    configured = true;
  }
  // Blocks that come under their predecessor's tail stand on whatever SMs are free first; launched behind its end (in_order), consecutive ones (the kv heads of a
  // key block) go round the chip in order. Where a block has many iterations that decides more than the 3 us of an early launch: the kernel alone, D = 128, 4313 tokens,
  // 32/8 heads, 174 us in order and 195 early with 4 samples, 370 and 406 with one. The rule is attention_plan.backward_in_order.
  int whole = 0;
  if constexpr (R::ON) whole = p.r.whole;
  const unsigned grid = whole + (n_items * p.Hkv - whole) * p.splits;
  if (in_order) kern<<<grid, AB_THREADS, AttBwdSmem<D>::TOTAL, st>>>(a, b, c, d, p);
  else launch_pdl(kern, grid, AB_THREADS, AttBwdSmem<D>::TOTAL, st, a, b, c, d, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

template <class R>
static int bwd(const void* qkv, long long ld, const void* out, long long ldo, const void* dout, long long lddo, int rows, int n_items, int D, long long part_bytes,
               bool in_order, float* delta, const AttBwdParams<R>& p, cudaStream_t st) {
  const int T = p.T, Hq = p.Hq, Hkv = p.Hkv;
  if ((D != 64 && D != 128) || Hkv <= 0 || Hq % Hkv || ld % 8 || ldo % 8 || lddo % 8 || p.ldq % 8 || p.splits < 1 || p.splits > Hq / Hkv) return -10;
  long long units = static_cast<long long>(n_items) * Hkv;   // that CTAs share
  if constexpr (R::ON) {
    if (p.r.whole < 0 || p.r.whole > units) return -10;
    units -= p.r.whole;
  }
  if (p.splits > 1 && (p.ws == nullptr || p.counters == nullptr || units * 8 > SPLIT_COUNTERS || p.splits * units * 2 * AB_B * D * 4 > part_bytes)) return -11;
  CUtensorMap tq, tdo, tdq, tdkv;
  int rc = make_tmap_2d_bf16(&tq, qkv, static_cast<uint64_t>(ld), static_cast<uint64_t>(rows), static_cast<uint64_t>(ld), 64, 128);
  if (rc) return rc;
  rc = make_tmap_2d_bf16(&tdo, dout, static_cast<uint64_t>(Hq) * D, static_cast<uint64_t>(rows), static_cast<uint64_t>(lddo), 64, 128);
  if (rc) return rc - 10;
  rc = make_tmap_2d_f32(&tdq, p.dq_acc, static_cast<uint64_t>(Hq) * D, static_cast<uint64_t>(T), static_cast<uint64_t>(Hq) * D, 32, 128);
  if (rc) return rc - 20;
  rc = make_tmap_2d_bf16(&tdkv, p.dqkv, (static_cast<uint64_t>(Hq) + 2 * Hkv) * D, static_cast<uint64_t>(T), static_cast<uint64_t>(p.ldq), 64, 32);
  if (rc) return rc - 30;
  const int per_block = 2 * 256 / (D / 8);
  const long long blocks = (static_cast<long long>(rows) * Hq + per_block - 1) / per_block;
  const __nv_bfloat16 *o = reinterpret_cast<const __nv_bfloat16*>(out), *d_o = reinterpret_cast<const __nv_bfloat16*>(dout);
  if constexpr (R::ON) {
    const long long behind = R::CAP ? static_cast<long long>(n_items) * LOOK_BLOCKS : 0;
    if (blocks + behind >= 1ll << 31) return -10;
    const AttLook look{reinterpret_cast<const __nv_bfloat16*>(qkv), ld, p.plan, Hq / Hkv, static_cast<int>(behind), p.r.odd, p.r.number};
    launch_pdl(attn_delta_kernel<AttLook>, static_cast<unsigned>(blocks + behind), 256, 0, st, o, ldo, d_o, lddo, delta, p.dq_acc, T, rows, Hq, D, look);
  } else {
    launch_pdl(attn_delta_kernel<AttNoLook>, static_cast<unsigned>(blocks), 256, 0, st, o, ldo, d_o, lddo, delta, p.dq_acc, T, rows, Hq, D, AttNoLook{});
  }
  rc = D == 128 ? launch_bwd<128, R>(tq, tdo, tdq, tdkv, p, n_items, in_order, st) : launch_bwd<64, R>(tq, tdo, tdq, tdkv, p, n_items, in_order, st);
  if (rc) return rc;
  launch_pdl(attn_dq_store_kernel, dim3(static_cast<unsigned>(rows), (Hq * D / 8 + 255) / 256), 256, 0, st, p.dq_acc, p.dqkv, p.ldq, rows, Hq * D);
  return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

}  // namespace mtb
