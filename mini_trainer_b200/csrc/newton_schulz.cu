// Matrices orthogonalised by Newton-Schulz products, one or a stack of them, and the update of a parameter by its orthogonalised momentum.
//
//   X0 = G / (|G| + 1e-7)  (Frobenius norm)        X <- (a I + b A + c A^2) X,  A = X X^T        steps times
// takes every singular value x of X to a x + b x^3 + c x^5, so those above 1e-3 of the norm or so end near one. A matrix with more rows than columns is multiplied from the right
// instead, X (a I + b A + c A^2) with A = X^T X: operands of the tensor cores may have either dimension innermost, so nothing is ever transposed. With r the shorter side
// and n the longer a step is the products r r n, r r r and r r n; the first two are symmetric: only the tiles on and below the diagonal are computed. Of large ones no others are stored, and who reads a block of 64 columns
// above it loads the rows below instead, the other dimension innermost: the transposes passed through the shared memory that the operands need (they took 3 to 5 % of a call: 64 x 2048 x 1024 3.00 -> 2.88 ms, 4096 x 4096 1.26 -> 1.22, loops at the power cap). 3 r^2 n + r^3 operations a step instead of 4 r^2 n + 2 r^3.
//
// The second product's epilogue adds b A and a I to c A^2, so that the third has the linear term in it.
//
// Numbers. Operands are fp16, X 2^p with 2^p about the root of the longer side, and A and the polynomial about 2^12: entries of all three then lie in the middle of the type's
// range (|X| <= 1.3, |A| <= 1.6 and |polynomial| <= 3.5 in norm, whatever G is). Its 11 bits are eight times finer than bf16's 8. That alone is not enough: a rounding of X is noise
// in all directions, and a direction in which X has next to nothing grows by a = 3.44 in each step, 485 times in five. So X is held as two numbers, hi and lo = 2^11 (X - hi), and the
// last product's epilogue adds a lo to the polynomial times hi: what is left of the rounding is what b A and c A^2 would have made of it, which is small
// in just those directions. What is rounded in the last two steps grows little more; their X goes without. Error of the result, relative, simulated with the roundings (in brackets: X without lo, and
// bf16 throughout): normal 512 x 1376 1.3e-3 (1.3e-3, 1.1e-2), sums of outer products of features that differ in size 1.3e-3 (2.2e-3, 1.7e-2), rank 8 and a hundredth of noise 2.5e-3 (3.7e-2, 0.3), rank 1 3.4e-3
// (0.15, 1.2); half of bf16's step, to which the result is rounded, is 1.7e-3 in the mean. Sums are fp32 in tensor memory. Measured, the result's rounding included: 2.0e-3 to 3.7e-3 in the mean from a shorter side of 1 to 200, whatever the longer one;
// single matrices scatter where few roundings make an error, with a shorter side of 16 up to 6e-3 and of five and less up to 1.7e-2 (the worst of some thousand of each size).
//
// The products: persistent, warp-specialised, 3-D TMA maps over the stack, tcgen05.mma of fp16 into two accumulators in tensor memory, by single CTAs (tiles of 128 x 128, for few tiles) or CTA pairs
// (256 x 256). All launches of a call are queued by one host call, each under its predecessor's tail. A large call is bound by its products: 4096 x 4096 (1.37 TFLOP in five steps) 1.22 ms in a row under the power cap:
// its gram product and square 57 us each at 80 % of the tensor pipe (136 tiles on 74 pairs), its last product 103 us at 88 %. A launch of one round is bound by its chain, about 3.4 us beside its reduction (first
// operands 1.0, sums to stores 1.5, end to the next one's start 1.4), and on single CTAs by L2, from which an SM takes 64 bytes a clock: 0.25 us for 64 of the reduction. More epilogue warps (sixteen of
// 32 columns) made it longer, 688 x 256 by 8 % and 1024 x 1024 by 5 (77 and 109 us with eight, replayed).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "per_device.h"
#include "ptx.cuh"

namespace mtb {

int make_tmap_3d_16(CUtensorMap* out, const void* base, uint64_t inner, uint64_t outer, uint64_t n, uint64_t ld, uint64_t stride, uint32_t box_inner, uint32_t box_outer);

namespace ns {

constexpr double NS_A = 3.4445, NS_B = -4.7750, NS_C = 2.0315;
// Factors of A and of the polynomial in fp16, about 2^12; the second such that the polynomial's value where A is next to nothing, a, is a number of the type.
constexpr double SCALE_A = 4096.0, SCALE_P = 14112.0 / NS_A;
constexpr int LO_BITS = 11;
constexpr int BM = 128, BK = 64, STAGES = 5;
constexpr int OP_BYTES = BM * BK * 2;                    // an operand's part of a stage: 128 rows (or columns) of 64
constexpr int STAGE_BYTES = 2 * OP_BYTES;
constexpr int EPI_WARPS = 8;                             // two to a quarter of the rows
constexpr int BOX = 32 * 128;                            // a warp's staging: 32 rows of 128 bytes, or 64 of 64; and as much for what is added
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr int SMEM = STAGES * STAGE_BYTES + EPI_WARPS * 2 * BOX + 1024 + 256;
constexpr int GROUP_M = 8;
constexpr int WHOLE_BITS = 8;                            // large symmetric matrices are stored in blocks of 256, the largest tile: those on the diagonal whole, none above it
constexpr uint32_t PEER_MASK = 0xFEFFFFFFu;              // of a shared::cluster address: the same place in CTA 0
static_assert(SMEM <= 227 * 1024, "shared memory");

// SYM: a symmetric product. APPLY: the step's last one, its result hi (and lo).
enum { SYM = 0, APPLY = 1 };

struct Params {
  int M, N, K, stack;
  int workers, group_m;
  float alpha, diag;             // D = alpha product + beta res (SYM: + diag on the diagonal)
  uint16_t* d;                   // fp16, or (bf16_out) bf16; rows padded to whole 16 bytes
  uint16_t* lo;                  // APPLY: 2^11 of what D's rounding has left, or null
  const __half* res;             // or null
  float beta;
  long long ld, stride;          // of d, lo and res
  int bf16_out;                  // APPLY
  int whole_bits;                // SYM: of D's blocks that are stored whole on the diagonal, and not above it
  int sym_a, sym_b;              // TURN: whether the operand is a symmetric matrix, of which map_s has the transpose
  int* status;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <int CTAS>
__device__ __forceinline__ void load_box(void* dst, const void* map, uint32_t bar, int c0, int c1, int c2) {
  if constexpr (CTAS == 2)
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
  else
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2) : "memory");
}
// 128 rows (from `row`) x 64 of the reduction (from `k`) of an operand whose innermost dimension is the reduction, or (MN) the rows.
template <int CTAS, bool MN>
__device__ __forceinline__ void load_operand(uint8_t* dst, const void* map, uint32_t bar, int row, int k, int z) {
  if constexpr (MN) {
    load_box<CTAS>(dst, map, bar, row, k, z);
    load_box<CTAS>(dst + OP_BYTES / 2, map, bar, row + 64, k, z);
  } else {
    load_box<CTAS>(dst, map, bar, k, row, z);
  }
}
// First block of 64 of the reduction in which 128 rows of a symmetric operand, from `row` on, are above what is stored; the same in both CTAs of a pair.
__device__ __forceinline__ int turn_at(int sym, int row) { return sym ? ((row >> WHOLE_BITS) + 1) << (WHOLE_BITS - 6) : 0x7fffffff; }
template <int CTAS, bool MN>
__device__ __forceinline__ void load_side(uint8_t* dst, const void* map, const void* map_s, bool turned, uint32_t bar, int row, int k, int z) {
  if (!MN && turned) load_operand<CTAS, true>(dst, map_s, bar, row, k, z);
  else load_operand<CTAS, MN>(dst, map, bar, row, k, z);
}
template <int CTAS>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CTAS == 2)
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
template <int CTAS>
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t leader = 0) {   // `leader`: number of the pair's first CTA in its cluster
  if constexpr (CTAS == 2) {
    const uint16_t mask = static_cast<uint16_t>(3u << leader);
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"(mask) : "memory");
  } else {
    umma_commit(bar);
  }
}
template <int CTAS>
__device__ __forceinline__ void arrive_leader(uint64_t* bar) {
  if constexpr (CTAS == 2) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(smem_u32(bar) & PEER_MASK) : "memory");
  else mbar_arrive(bar);
}
// One stage, 64 of the reduction.
template <int CTAS>
__device__ __forceinline__ void mma_stage(uint32_t d, uint32_t sa, uint32_t sb, uint32_t idesc, bool a_mn, bool b_mn, bool first) {
#pragma unroll
  for (int k = 0; k < BK / 16; ++k) {
    const uint64_t da = a_mn ? make_smem_desc(sa + k * 2048, 8192, 1024) : make_smem_desc(sa + k * 32, 16, 1024);
    const uint64_t db = b_mn ? make_smem_desc(sb + k * 2048, 8192, 1024) : make_smem_desc(sb + k * 32, 16, 1024);
    mma<CTAS>(d, da, db, idesc, !first || k != 0);
  }
}
// fp16 x fp16 -> fp32
__host__ __device__ constexpr uint32_t idesc_f16(uint32_t m, uint32_t n, bool a_mn, bool b_mn) {
  return make_idesc_bf16(m, n, a_mn, b_mn) & ~((1u << 7) | (1u << 10));
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_f16(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }

// A producer that gave up: until the last of its `issued` loads have landed, or a while has passed.
__device__ __forceinline__ void settle_loads(uint64_t* full_bar, uint32_t issued) {
  for (uint32_t i = issued > STAGES ? issued - STAGES : 0; i < issued; ++i)
    for (uint32_t n = 0; n < (1u << 22) && !mbar_try_wait(&full_bar[i % STAGES], (i / STAGES) & 1); ++n) {}
}

// Tile `t` of a matrix: on and below the diagonal row by row, or in bands of group_m row-tiles.
template <int KIND>
__device__ __forceinline__ void tile_at(int t, int tiles_m, int tiles_n, int group_m, int& tm, int& tn) {
  if constexpr (KIND == SYM) {
    int i = static_cast<int>((sqrtf(8.f * t + 1.f) - 1.f) * 0.5f);
    while (i * (i + 1) / 2 > t) --i;
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    tm = i;
    tn = t - i * (i + 1) / 2;
  } else {
    const int band = t / (group_m * tiles_n), first = band * group_m, rows = min(group_m, tiles_m - first), local = t - first * tiles_n;
    tm = first + local % rows;
    tn = local / rows;
  }
}

// A warp's 32 rows of 64 columns between memory and registers go by its staging in shared memory: eight lanes to a row there, a lane to a row here. (TMA stores of the staged boxes queue
// behind the operands' loads, and a tile has four to wait for: the last product of 64 x 2048 x 1024 with hi and lo 303 us with them, 260 so.)
__device__ __forceinline__ uint4* staged(uint8_t* box, int row, int piece) { return reinterpret_cast<uint4*>(box + row * 128 + ((piece ^ (row & 7)) << 4)); }
// What is added to the sums, into the second box, asked for ahead of them, so that it arrives under their wait.
__device__ __forceinline__ void ask(const Params& p, uint8_t* box, int y0, int col, int z, int lane) {
  if (p.res == nullptr) return;
  const __half* src = p.res + z * p.stride + static_cast<long long>(y0 + (lane >> 3)) * p.ld + col + (lane & 7) * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i)   // (what is past the matrix stays as it was, and what it is added to is not stored)
    if (y0 + (lane >> 3) + 4 * i < p.M && col + (lane & 7) * 8 < p.N)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(staged(box + BOX, (lane >> 3) + 4 * i, lane & 7))), "l"(src + 4 * i * p.ld) : "memory");
}
__device__ __forceinline__ void arrived() { asm volatile("cp.async.wait_all;" ::: "memory"); __syncwarp(); }
// `h`: this lane's row, to rows [y0, y0 + 32) and columns [col, col + 64) of a matrix of which [rows, cols] exist.
__device__ __forceinline__ void put(uint16_t* to, long long ld, int rows, int cols, int y0, int col, uint8_t* box, const uint32_t (&h)[32], int lane) {
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) *staged(box, lane, i) = make_uint4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
  __syncwarp();
  uint16_t* dst = to + static_cast<long long>(y0 + (lane >> 3)) * ld + col + (lane & 7) * 8;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (y0 + (lane >> 3) + 4 * i < rows && col + (lane & 7) * 8 < cols) *reinterpret_cast<uint4*>(dst + 4 * i * ld) = *staged(box, (lane >> 3) + 4 * i, lane & 7);
}
// 64 columns of a warp's 32 rows (a lane has a row), from the product's sums `f` to the stores.
template <int KIND>
__device__ __forceinline__ void finish64(const Params& p, float* f, uint8_t* box, bool diagonal, int y0, int col, int z, int lane, bool more = false) {   // `more`: the next 64 columns come after these
#pragma unroll
  for (int j = 0; j < 64; ++j) f[j] *= p.alpha;
  if (p.res != nullptr) {
    arrived();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4 u = *staged(box + BOX, lane, i);
      const float2 a = unpack_f16(u.x), b = unpack_f16(u.y), d = unpack_f16(u.z), e = unpack_f16(u.w);
      f[8 * i] += p.beta * a.x; f[8 * i + 1] += p.beta * a.y; f[8 * i + 2] += p.beta * b.x; f[8 * i + 3] += p.beta * b.y;
      f[8 * i + 4] += p.beta * d.x; f[8 * i + 5] += p.beta * d.y; f[8 * i + 6] += p.beta * e.x; f[8 * i + 7] += p.beta * e.y;
    }
    __syncwarp();
    if (more) ask(p, box, y0, col + 64, z, lane);
  }
  uint32_t h[32];
  uint16_t* d = p.d + z * p.stride;
  if constexpr (KIND == SYM) {
    if (diagonal) {
#pragma unroll
      for (int j = 0; j < 64; ++j) if (col + j == y0 + lane) f[j] += p.diag;
    }
#pragma unroll
    for (int j = 0; j < 32; ++j) h[j] = pack_f16(f[2 * j], f[2 * j + 1]);
    put(d, p.ld, p.M, p.N, y0, col, box, h, lane);
    if (!diagonal && (y0 >> p.whole_bits) == (col >> p.whole_bits)) {
      // In a block on the diagonal, which is stored whole, the transpose: 64 rows (this tile's columns) of 32 (its rows). Neighbouring lanes exchange a word, so that each writes two rows' entries of one column.
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const uint32_t o = __shfl_xor_sync(0xffffffffu, h[j], 1);
        const uint32_t word = lane & 1 ? __byte_perm(o, h[j], 0x7632) : __byte_perm(h[j], o, 0x5410);
        *reinterpret_cast<uint32_t*>(box + (2 * j + (lane & 1)) * 64 + (lane >> 1) * 4) = word;
      }
      __syncwarp();
      uint16_t* dst = d + static_cast<long long>(col + (lane >> 2)) * p.ld + y0 + (lane & 3) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (col + (lane >> 2) + 8 * i < p.N && y0 + (lane & 3) * 8 < p.M)
          *reinterpret_cast<uint4*>(dst + 8 * i * p.ld) = *reinterpret_cast<const uint4*>(box + ((lane >> 2) + 8 * i) * 64 + (lane & 3) * 16);
    }
  } else {
    if (p.bf16_out) {
#pragma unroll
      for (int j = 0; j < 32; ++j) h[j] = pack_bf16(f[2 * j], f[2 * j + 1]);
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j) h[j] = pack_f16(f[2 * j], f[2 * j + 1]);
    }
    put(d, p.ld, p.M, p.N, y0, col, box, h, lane);
    if (p.lo != nullptr) {
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const float2 hi = unpack_f16(h[j]);
        h[j] = pack_f16((f[2 * j] - hi.x) * (1 << LO_BITS), (f[2 * j + 1] - hi.y) * (1 << LO_BITS));
      }
      put(p.lo + z * p.stride, p.ld, p.M, p.N, y0, col, box, h, lane);
    }
  }
}

// TURN: an operand that is not MN may be symmetric, with more than a block of 256.
template <int CTAS, bool A_MN, bool B_MN, int KIND, bool TURN>
__global__ void __cluster_dims__(CTAS, 1, 1) __launch_bounds__(THREADS, 1)
product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_s, const Params p) {
  constexpr int TILE = BM * CTAS;      // rows and columns of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES + EPI_WARPS * 2 * BOX);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CTAS == 2 ? cluster_rank() : 0;
  const int worker = blockIdx.x / CTAS;
  const int tiles_m = (p.M + TILE - 1) / TILE, tiles_n = (p.N + TILE - 1) / TILE;
  const int tiles = KIND == SYM ? tiles_m * (tiles_m + 1) / 2 : tiles_m * tiles_n;
  const int items = tiles * p.stack, kblocks = (p.K + BK - 1) / BK;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tfull_bar[a], 1); mbar_init(&tempty_bar[a], CTAS * EPI_WARPS); }
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
    if (TURN) tma_prefetch_desc(&map_s);
  }
  __syncwarp();   // (whatever is .aligned is for whole warps: here and below they come together again behind what one thread, or each for itself, has done)
  if (warp == 1) {
    if constexpr (CTAS == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(2 * TILE) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(tmem_slot, 2 * TILE);
      tmem_relinquish();
    }
  }
  tc_fence_before();   // (who touches global memory waits for the launch in front before it does: all this passes under that one's tail)
  __syncthreads();
  if constexpr (CTAS == 2) cluster_barrier();   // the partner's barriers are there before anything is sent to them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (elect_one()) {
      uint32_t it = 0;
      for (int w = worker; w < items; w += p.workers) {
        int tm, tn;
        const int z = w / tiles;
        tile_at<KIND>(w - z * tiles, tiles_m, tiles_n, p.group_m, tm, tn);
        const int row = tm * TILE + static_cast<int>(rank) * BM, col = tn * TILE + static_cast<int>(rank) * BM;
        const int turn_a = turn_at(p.sym_a, row), turn_b = turn_at(p.sym_b, col);
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&empty_bar[s], ((it / STAGES) & 1) ^ 1, abort_flag)) { atomicExch(p.status, 71); if (rank == 0) settle_loads(full_bar, it); goto done; }
          uint8_t* sa = smem + s * STAGE_BYTES;
          const uint32_t bar = CTAS == 2 ? smem_u32(&full_bar[s]) & PEER_MASK : smem_u32(&full_bar[s]);
          const bool once = KIND == SYM && tm == tn;   // the same rows twice
          if (rank == 0) mbar_arrive_expect_tx(&full_bar[s], CTAS * (once ? OP_BYTES : STAGE_BYTES));
          if (it == 0) pdl_wait();
          load_side<CTAS, A_MN>(sa, &map_a, &map_s, TURN && kb >= turn_a, bar, row, kb * BK, z);
          if (!once) load_side<CTAS, B_MN>(sa + OP_BYTES, &map_b, &map_s, TURN && kb >= turn_b, bar, col, kb * BK, z);
        }
      }
      pdl_trigger();
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      pdl_wait();   // (so that its bounded waits are for this launch's loads alone)
      uint32_t it = 0, n = 0;
      for (int w = worker; w < items; w += p.workers, ++n) {
        int tm = 0, tn = 1;
        if constexpr (KIND == SYM || TURN) tile_at<KIND>(w % tiles, tiles_m, tiles_n, p.group_m, tm, tn);
        const bool once = KIND == SYM && tm == tn;
        const int turn_a = turn_at(p.sym_a, tm * TILE), turn_b = turn_at(p.sym_b, tn * TILE);
        if (!mbar_wait(&tempty_bar[n & 1], ((n >> 1) & 1) ^ 1, abort_flag)) { atomicExch(p.status, 72); goto done; }
        tc_fence_after();
        const uint32_t d = tmem_base + (n & 1) * TILE;
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = it % STAGES;
          if (!mbar_wait(&full_bar[s], (it / STAGES) & 1, abort_flag)) { atomicExch(p.status, 73); goto done; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + s * STAGE_BYTES), sb = once ? sa : sa + OP_BYTES;
          const bool a_mn = A_MN || (TURN && kb >= turn_a), b_mn = B_MN || (TURN && kb >= turn_b);
          mma_stage<CTAS>(d, sa, sb, idesc_f16(TILE, TILE, a_mn, b_mn), a_mn, b_mn, kb == 0);
          commit<CTAS>(&empty_bar[s]);
        }
        commit<CTAS>(&tfull_bar[n & 1]);
      }
    }
  } else {
    // epilogue: quarter q of the rows, half of the columns, 64 at a time
    const int q = warp & 3, half = (warp - 2) >> 2;
    uint8_t* box = smem + STAGES * STAGE_BYTES + (warp - 2) * 2 * BOX;
    uint32_t n = 0;
    for (int w = worker; w < items; w += p.workers, ++n) {
      int tm, tn;
      const int z = w / tiles;
      tile_at<KIND>(w - z * tiles, tiles_m, tiles_n, p.group_m, tm, tn);
      const int y0 = tm * TILE + static_cast<int>(rank) * BM + q * 32, c0 = half * (TILE / 2);
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + (n & 1) * TILE;
      if (n == 0) pdl_wait();
      ask(p, box, y0, tn * TILE + c0, z, lane);
      if (!__all_sync(0xffffffffu, mbar_wait(&tfull_bar[n & 1], (n >> 1) & 1, abort_flag))) { atomicExch(p.status, 74); goto done; }
      tc_fence_after();
#pragma unroll 1
      for (int c = c0; c < c0 + TILE / 2; c += 64) {
        const int col = tn * TILE + c;
        if (y0 >= p.M || col >= p.N) break;
        __syncwarp();
        uint32_t v[2][32];
        tmem_ld_32x32(taddr + c, v[0]);
        tmem_ld_32x32(taddr + c + 32, v[1]);
        tmem_ld_wait();
        finish64<KIND>(p, reinterpret_cast<float*>(&v[0][0]), box, tm == tn, y0, col, z, lane, c + 64 < c0 + TILE / 2 && col + 64 < p.N);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_leader<CTAS>(&tempty_bar[n & 1]);
    }
  }
done:
  tc_fence_before();
  __syncthreads();
  if constexpr (CTAS == 2) cluster_barrier();   // nobody tears down while the partner may still signal or read
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CTAS == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * TILE) : "memory");
    else tmem_dealloc(tmem_base, 2 * TILE);
  }
}

// The same product with its reduction divided over the CTAs (or pairs) of a cluster, for launches of few tiles: one tile to a cluster. An SM takes a tile's operands from L2 at 64 bytes a clock, 512 clocks for
// 64 of the reduction, which is what a launch of one round lasts for; `splits` SMs take it in parts. When all have multiplied, each sends every other the sums that one finishes, fp32 through
// the cluster's shared memory (over the operands' stages), and finishes its own: units of 32 rows and 64 columns, added in the order of the parts.
constexpr int MOST_SPLITS = 8;   // of single CTAs; 4 of pairs (a cluster has eight CTAs at most)
// The place of this CTA's shared memory at `addr` in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t remote_address(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void store_cluster4(uint32_t to, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}
template <int CTAS, bool A_MN, bool B_MN, int KIND, bool TURN>
__global__ void __launch_bounds__(THREADS, 1)
split_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_s, const Params p, const int splits) {
  constexpr int TILE = BM * CTAS;
  static_assert(STAGES * STAGE_BYTES >= TILE * 128 * 4, "the sums of a tile's rows fit over the stages");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES + EPI_WARPS * 2 * BOX);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfull_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t in_cluster = cluster_rank(), rank = in_cluster % CTAS;
  const int split = in_cluster / CTAS, item = blockIdx.x / (CTAS * splits);
  const int tiles_m = (p.M + TILE - 1) / TILE, tiles_n = (p.N + TILE - 1) / TILE;
  const int tiles = KIND == SYM ? tiles_m * (tiles_m + 1) / 2 : tiles_m * tiles_n;
  const int kblocks = (p.K + BK - 1) / BK, kb0 = kblocks * split / splits, n = kblocks * (split + 1) / splits - kb0;
  const int z = item / tiles;
  int tm, tn;
  tile_at<KIND>(item - z * tiles, tiles_m, tiles_n, p.group_m, tm, tn);
  const bool once = KIND == SYM && tm == tn;   // the same rows twice

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    mbar_init(tfull_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&map_a);
    tma_prefetch_desc(&map_b);
    if (TURN) tma_prefetch_desc(&map_s);
  }
  __syncwarp();   // (whatever is .aligned is for whole warps: here and below they come together again behind what one thread, or each for itself, has done)
  if (warp == 1) {
    if constexpr (CTAS == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TILE) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(tmem_slot, TILE);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_barrier();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (elect_one()) {
      pdl_wait();
      const int row = tm * TILE + static_cast<int>(rank) * BM, col = tn * TILE + static_cast<int>(rank) * BM;
      const int turn_a = turn_at(p.sym_a, row), turn_b = turn_at(p.sym_b, col);
      for (int it = 0; it < n; ++it) {
        const int s = it % STAGES;
        if (!mbar_wait(&empty_bar[s], ((it / STAGES) & 1) ^ 1, abort_flag)) { atomicExch(p.status, 71); if (rank == 0) settle_loads(full_bar, it); break; }
        uint8_t* sa = smem + s * STAGE_BYTES;
        const uint32_t bar = CTAS == 2 ? smem_u32(&full_bar[s]) & PEER_MASK : smem_u32(&full_bar[s]);
        if (rank == 0) mbar_arrive_expect_tx(&full_bar[s], CTAS * (once ? OP_BYTES : STAGE_BYTES));
        load_side<CTAS, A_MN>(sa, &map_a, &map_s, TURN && kb0 + it >= turn_a, bar, row, (kb0 + it) * BK, z);
        if (!once) load_side<CTAS, B_MN>(sa + OP_BYTES, &map_b, &map_s, TURN && kb0 + it >= turn_b, bar, col, (kb0 + it) * BK, z);
      }
      pdl_trigger();
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      pdl_wait();
      const int turn_a = turn_at(p.sym_a, tm * TILE), turn_b = turn_at(p.sym_b, tn * TILE);
      for (int it = 0; it < n; ++it) {
        const int s = it % STAGES;
        if (!mbar_wait(&full_bar[s], (it / STAGES) & 1, abort_flag)) { atomicExch(p.status, 73); break; }
        tc_fence_after();
        const uint32_t sa = smem_u32(smem + s * STAGE_BYTES), sb = once ? sa : sa + OP_BYTES;
        const bool a_mn = A_MN || (TURN && kb0 + it >= turn_a), b_mn = B_MN || (TURN && kb0 + it >= turn_b);
        mma_stage<CTAS>(tmem_base, sa, sb, idesc_f16(TILE, TILE, a_mn, b_mn), a_mn, b_mn, it == 0);
        commit<CTAS>(&empty_bar[s], in_cluster);
      }
      commit<CTAS>(tfull_bar, in_cluster);
    }
  } else {
    pdl_wait();
    if (!mbar_wait(tfull_bar, 0, abort_flag) && lane == 0) atomicExch(p.status, 74);
  }
  __syncthreads();
  cluster_barrier();   // every CTA has multiplied: nothing reads the stages any more
  tc_fence_after();
  // [part][unit of the one that finishes it][4 columns][row] of 16 bytes
  constexpr int ACROSS = TILE / 64;   // units side by side
  const int per_owner = 4 * ACROSS / splits;
  if (warp >= 2) {
    const int q = warp & 3, half = (warp - 2) >> 2;
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll 1
    for (int c = half * (TILE / 2); c < (half + 1) * (TILE / 2); c += 32) {
      const int unit = q * ACROSS + c / 64;
      const uint32_t at = remote_address(smem_u32(smem) + (split * per_owner + unit % per_owner) * 8192 + (c % 64) / 4 * 512 + lane * 16, static_cast<uint32_t>(unit / per_owner) * CTAS + rank);
      uint32_t v[32];
      tmem_ld_32x32(taddr + c, v);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; j += 4)
        store_cluster4(at + j / 4 * 512, __uint_as_float(v[j]), __uint_as_float(v[j + 1]), __uint_as_float(v[j + 2]), __uint_as_float(v[j + 3]));
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_barrier();   // ... and every part has arrived
  if (warp >= 2) {
    uint8_t* box = smem + STAGES * STAGE_BYTES + (warp - 2) * 2 * BOX;
    for (int u = warp - 2; u < per_owner; u += EPI_WARPS) {
      const int unit = split * per_owner + u, y0 = tm * TILE + static_cast<int>(rank) * BM + unit / ACROSS * 32, col = tn * TILE + unit % ACROSS * 64;
      if (y0 >= p.M || col >= p.N) continue;
      ask(p, box, y0, col, z, lane);
      float f[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) f[j] = 0.f;
      for (int s = 0; s < splits; ++s) {
        const uint8_t* src = smem + (s * per_owner + u) * 8192 + lane * 16;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float4 v = *reinterpret_cast<const float4*>(src + j * 512);
          f[4 * j] += v.x; f[4 * j + 1] += v.y; f[4 * j + 2] += v.z; f[4 * j + 3] += v.w;
        }
      }
      finish64<KIND>(p, f, box, tm == tn, y0, col, z, lane);
    }
  }
  __syncthreads();
  if constexpr (CTAS == 2) cluster_barrier();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CTAS == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TILE) : "memory");
    else tmem_dealloc(tmem_base, TILE);
  }
}

// ------------------------------------------------------------------------------------------ in front of the products, and behind them
constexpr int LIN_THREADS = 256;
constexpr int MOST_CHUNKS = 2048;   // of a stack, in the sums of squares

// What is orthogonalised: a gradient, or a momentum that takes the gradient in first.
struct Source {
  const void* g; int g_bf16;
  void* m; int m_bf16;             // null: g itself
  const float* coef;               // factor of the gradient, on the device, or null
  float mu; int nesterov;
};
__device__ __forceinline__ float load16or32(const void* p, int is16, long long i) {
  return is16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}
// Eight elements; those past `n` are zero.
__device__ __forceinline__ void load8(const void* p, int is16, long long i, int n, bool vec, float (&x)[8]) {
  if (vec) {
    if (is16) {
      const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p) + i);
      const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z), d = unpack_bf16(u.w);
      x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
    } else {
      const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i), b = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i + 4);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = j < n ? load16or32(p, is16, i + j) : 0.f;
  }
}
__device__ __forceinline__ void store8(void* p, int is16, long long i, int n, bool vec, const float (&x)[8]) {
  if (vec) {
    if (is16) {
      *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p) + i) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
    } else {
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i + 4) = make_float4(x[4], x[5], x[6], x[7]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) {
        if (is16) reinterpret_cast<__nv_bfloat16*>(p)[i + j] = __float2bfloat16(x[j]);
        else reinterpret_cast<float*>(p)[i + j] = x[j];
      }
  }
}
// Eight elements of what is orthogonalised. `update`: the momentum takes the gradient in; else it has. The momentum counts as it is stored.
__device__ __forceinline__ void source8(const Source& s, float coef, long long i, int n, bool vec, bool update, float (&u)[8]) {
  load8(s.g, s.g_bf16, i, n, vec, u);
  if (s.m == nullptr) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) u[j] *= coef;
  float m[8];
  load8(s.m, s.m_bf16, i, n, vec, m);
  if (update) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m[j] = fmaf(s.mu, m[j], u[j]);
      if (s.m_bf16) m[j] = __bfloat162float(__float2bfloat16(m[j]));
    }
    store8(s.m, s.m_bf16, i, n, vec, m);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) u[j] = s.nesterov ? fmaf(s.mu, m[j], u[j]) : m[j];
}

// Sum of eight squares. In fp32, but where that is past its range the numbers themselves need not be (from 1.8e19 on): those again in 64 bits.
__device__ __forceinline__ double squares8(const float (&u)[8]) {
  float q = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) q = fmaf(u[j], u[j], q);
  double sum = q;
  if (!(q <= 3.4028234e38f)) {
    sum = 0.0;
#pragma unroll
    for (int j = 0; j < 8; ++j) { const double x = u[j]; sum = fma(x, x, sum); }
  }
  return sum;
}
// What takes a matrix with these squares to X0 2^p, as two factors: one alone would be too small a number of the type for the largest matrices.
struct Factor { float first, second; };
__device__ __forceinline__ Factor factor_of(double squares, int p2) {
  const double norm = sqrt(squares) + 1e-7;
  const bool large = norm > 0x1p100;
  return Factor{large ? 0x1p-64f : 1.f, static_cast<float>(ldexp(1.0, large ? p2 + 64 : p2) / norm)};
}

// Sums of squares of the chunks of each matrix, [stack, chunks]; the momentum's update on the way.
__global__ void __launch_bounds__(LIN_THREADS) squares_kernel(Source s, long long numel, int chunks, long long per_chunk, int vec, double* __restrict__ sums) {
  __shared__ double sh[LIN_THREADS / 32];
  pdl_wait();
  const int z = blockIdx.x / chunks, c = blockIdx.x - z * chunks;
  const long long lo = c * per_chunk, hi = min(numel, lo + per_chunk), base = z * numel;
  const float coef = s.coef != nullptr ? *s.coef : 1.f;
  double total = 0.0;
  auto add = [&](const float (&u)[8]) { total += squares8(u); };
  constexpr int STEP = LIN_THREADS * 8, AHEAD = 4;
  long long i = lo + threadIdx.x * 8;
  for (; i + (AHEAD - 1) * STEP + 8 <= hi; i += AHEAD * STEP) {   // several loads under way
    float u[AHEAD][8];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) source8(s, coef, base + i + a * STEP, 8, vec != 0, true, u[a]);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) add(u[a]);
  }
  for (; i < hi; i += STEP) {
    float u[8];
    source8(s, coef, base + i, static_cast<int>(min(8ll, hi - i)), vec != 0, true, u);
    add(u);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < LIN_THREADS / 32; ++i) total += sh[i];
    sums[blockIdx.x] = total;
  }
  pdl_trigger();
}

// X0 2^p as hi and lo, rows padded to ld. `lo` null: hi alone.
__global__ void __launch_bounds__(LIN_THREADS) scale_kernel(Source s, int rows, int cols, int ld, int chunks, int blocks_per, int vec, int p2, const double* __restrict__ sums,
                                                           __half* __restrict__ hi, __half* __restrict__ lo) {
  __shared__ double sh[LIN_THREADS / 32];
  __shared__ Factor factor_sh;
  pdl_wait();
  const int z = blockIdx.x / blocks_per, blk = blockIdx.x - z * blocks_per;
  double total = 0.0;
  for (int i = threadIdx.x; i < chunks; i += LIN_THREADS) total += sums[static_cast<long long>(z) * chunks + i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < LIN_THREADS / 32; ++i) total += sh[i];
    factor_sh = factor_of(total, p2);
  }
  __syncthreads();
  const Factor f = factor_sh;
  const float coef = s.coef != nullptr ? *s.coef : 1.f;
  const int per_row = (cols + 7) / 8;   // (what pads a row is never read)
  const long long units = static_cast<long long>(rows) * per_row, base = static_cast<long long>(z) * rows * cols, out = static_cast<long long>(z) * rows * ld;
  for (long long u = static_cast<long long>(blk) * LIN_THREADS + threadIdx.x; u < units; u += static_cast<long long>(blocks_per) * LIN_THREADS) {
    const long long row = u / per_row;
    const int col = static_cast<int>(u - row * per_row) * 8;
    float x[8];
    source8(s, coef, base + row * cols + col, min(8, cols - col), vec != 0, false, x);
    uint32_t h[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a = x[2 * j] * f.first * f.second, b = x[2 * j + 1] * f.first * f.second;
      h[j] = pack_f16(a, b);
      const float2 r = unpack_f16(h[j]);
      l[j] = pack_f16((a - r.x) * (1 << LO_BITS), (b - r.y) * (1 << LO_BITS));
    }
    *reinterpret_cast<uint4*>(hi + out + row * ld + col) = make_uint4(h[0], h[1], h[2], h[3]);
    if (lo != nullptr) *reinterpret_cast<uint4*>(lo + out + row * ld + col) = make_uint4(l[0], l[1], l[2], l[3]);
  }
  pdl_trigger();
}

// bf16 rows without their padding.
__global__ void __launch_bounds__(LIN_THREADS) unpad_kernel(const __nv_bfloat16* __restrict__ x, int ld, long long rows, int cols, __nv_bfloat16* __restrict__ out) {
  pdl_wait();
  const long long n = rows * cols;
  for (long long i = static_cast<long long>(blockIdx.x) * LIN_THREADS + threadIdx.x; i < n; i += static_cast<long long>(gridDim.x) * LIN_THREADS) {
    const long long row = i / cols;
    out[i] = x[row * ld + (i - row * cols)];
  }
  pdl_trigger();
}

// w <- keep w - step o 2^-p of the padded fp16 rows o, and the working copy. (A rounding of o to fp16, 2^-11 of an entry at most, is an eighth of the one to bf16 that an orthogonalised matrix is returned with, and below
// what the products' own operands leave, 2e-3 of its norm; in fp32 the last product would write, and this read, twice the bytes.)
__global__ void __launch_bounds__(LIN_THREADS) update_kernel(float* __restrict__ master, __nv_bfloat16* __restrict__ param, const __half* __restrict__ o, int ld, long long rows,
                                                            int cols, int vec, float keep, float step) {
  pdl_wait();
  const int per_row = (cols + 7) / 8;   // (what pads a row is never read)
  const long long units = rows * per_row;
  for (long long u = static_cast<long long>(blockIdx.x) * LIN_THREADS + threadIdx.x; u < units; u += static_cast<long long>(gridDim.x) * LIN_THREADS) {
    const long long row = u / per_row, at = row * cols;
    const int col = static_cast<int>(u - row * per_row) * 8, n = min(8, cols - col);
    const uint4 q = *reinterpret_cast<const uint4*>(o + row * ld + col);
    const float2 a = unpack_f16(q.x), b = unpack_f16(q.y), c = unpack_f16(q.z), d = unpack_f16(q.w);
    const float x[8] = {a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
    float w[8];
    load8(master, 0, at + col, n, vec != 0, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = fmaf(-step, x[j], keep * w[j]);
    store8(master, 0, at + col, n, vec != 0, w);
    if (param != nullptr) store8(param, 1, at + col, n, vec != 0, w);
  }
  pdl_trigger();
}

// ------------------------------------------------------------------------------------------ a whole call in one launch
// Where the shorter side is at most 128 a call may be one launch: a cluster of up to sixteen CTAs has a matrix, each a slab of the longer side (256, 512 or 1024 columns where the shorter one is up to 128, 64 or 32),
// which stays in shared memory as hi and lo from the first step to the last. In a slab's 64 columns rows are 128 bytes apart, which is an operand with the columns as the reduction (the gram product) and with the
// rows as the reduction (the last product) alike; a matrix with more rows than columns is turned when it is read. Per step: the gram product of the slab; its sums to the CTA that finishes those rows and columns (shared
// memory of the cluster), which adds them in the order of the slabs and gives A to all; its square, every CTA for itself; the polynomial over A; the last product and the slab's new hi and lo.
// A slab of at most 64 (32) rows goes through the last product in two (four) parts side by side: the polynomial stands two (four) times on the diagonal of a 128 x 128 operand, the reduction runs over
// the parts one behind the other, and each part's columns come out in rows of their own, so that all warps have some. Bound by the chain of
// those, a step takes 2.5 us for 64 x 64, 2.9 for 32 x 256 and 5.3 for 128 x 256 (the other form's launches 9 to 16). In the other form and so, by rows of launches: 64 x 64 50 and 17 us, 128 x 256 59 and 37 (46 in two slabs), 128 x 512 64 and
// 52, 32 x 2048 74 and 35, 64 x 8192 85 and 61.
constexpr int SMALL_R = 128, SMALL_PARTS = 16, SMALL_THREADS = 512, SMALL_ENTRIES = 128 * 256;   // most of a slab
constexpr int SMALL_A = 2 * SMALL_R * 128, SMALL_RECV = 16 * 4096;
constexpr int small_smem(int entries) { return 4 * entries + SMALL_A + SMALL_RECV + 1024 + 256; }
static_assert(small_smem(SMALL_ENTRIES) <= 227 * 1024, "shared memory");

struct Small {
  int rows, cols, r, n, tall;    // r: the shorter side, n: the longer one; tall: it is the rows
  int w, parts, R;               // columns of a slab, slabs; rows of a slab in shared memory, 32, 64 or 128
  int steps, kept, p2, vec;
  __nv_bfloat16* out;            // what is orthogonalised, or null: the update
  float* master;
  __nv_bfloat16* param;
  float keep, step;              // master <- keep master - step (O 2^p2)
  int* status;
};
// Eight entries of row `row` of the (turned) matrix from column `col` on; `at`: where its stack entry starts.
__device__ __forceinline__ void gather8(const Source& s, const Small& p, float coef, long long at, int row, int col, bool update, float (&u)[8]) {
  const int n = row < p.r ? max(0, min(8, p.n - col)) : 0;
  if (n == 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = 0.f;
  } else if (!p.tall) {
    source8(s, coef, at + static_cast<long long>(row) * p.cols + col, n, p.vec != 0, update, u);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      u[j] = 0.f;
      if (j < n) {
        const long long i = at + static_cast<long long>(col + j) * p.cols + row;
        u[j] = load16or32(s.g, s.g_bf16, i);
        if (s.m != nullptr) {
          u[j] *= coef;
          float m = load16or32(s.m, s.m_bf16, i);
          if (update) {
            m = fmaf(s.mu, m, u[j]);
            if (s.m_bf16) { const __nv_bfloat16 b = __float2bfloat16(m); reinterpret_cast<__nv_bfloat16*>(s.m)[i] = b; m = __bfloat162float(b); }
            else reinterpret_cast<float*>(s.m)[i] = m;
          }
          u[j] = s.nesterov ? fmaf(s.mu, m, u[j]) : m;
        }
      }
    }
  }
}
__device__ __forceinline__ uint4* piece_at(uint8_t* x, int row, int piece, int R = SMALL_R) { return reinterpret_cast<uint4*>(x + (piece >> 3) * (R * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4)); }
// Bounded, as mbar_wait, for what other CTAs of the cluster have sent.
__device__ __forceinline__ bool wait_sent(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  for (uint32_t i = 0; i < SPIN_LIMIT; ++i) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
    if (ok) return true;
    if ((i & 1023u) == 1023u && *abort_flag) return false;
  }
  *abort_flag = 1;
  return false;
}
// To another CTA of the cluster, whose barrier counts the bytes.
__device__ __forceinline__ void send8(uint32_t to, uint2 v, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(to), "r"(v.x), "r"(v.y), "r"(bar) : "memory");
}
__device__ __forceinline__ void send16(uint32_t to, uint4 v, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "r"(bar) : "memory");
}

__global__ void __launch_bounds__(SMALL_THREADS, 1) small_kernel(const Source src, const Small p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* hi = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int R = p.R, copies = SMALL_R / R, cw = p.w / copies;   // parts of a slab in the last product, and their columns
  uint8_t* lo = hi + p.w * 2 * R;
  uint8_t* a = lo + p.w * 2 * R;               // A, then the polynomial in its place: 128 x 128, two blocks of 64 columns
  uint8_t* recv = a + SMALL_A;                 // sums from the other slabs
  double* norm = reinterpret_cast<double*>(recv + SMALL_RECV);
  uint64_t* done_bar = reinterpret_cast<uint64_t*>(norm + SMALL_PARTS);
  uint64_t *sums_bar = done_bar + 1, *a_bar = done_bar + 2;   // of the sums that are finished here, and of A from the others
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done_bar + 3);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  Factor* factor = reinterpret_cast<Factor*>(tmem_slot + 2);
  __shared__ double warp_sums[SMALL_THREADS / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = warp & 3, sub = warp >> 2;   // a quarter of the rows, a quarter of the columns
  const int parts = p.parts, rank = parts > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int z = blockIdx.x / parts, n0 = rank * p.w;
  const long long at = static_cast<long long>(z) * p.rows * p.cols;
  const int pieces = p.w / 8, tasks = p.r * pieces;
  const float per = 1.f / (p.tall ? p.r : pieces);
  auto task = [&](int i, int& row, int& piece) {   // neighbouring threads have neighbours in memory
    const int d = p.tall ? p.r : pieces;
    int a = __float2int_rz(static_cast<float>(i) * per);   // i below 2^12: off by one at most
    int b = i - a * d;
    if (b >= d) { ++a; b -= d; }
    if (b < 0) { --a; b += d; }
    row = p.tall ? b : a;
    piece = p.tall ? a : b;
  };

  if (threadIdx.x == 0) {
    mbar_init(done_bar, 1);
    mbar_init(sums_bar, 1);
    mbar_init(a_bar, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  __syncwarp();
  if (warp == 0) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
  pdl_wait();
  const float coef = src.coef != nullptr ? *src.coef : 1.f;
  double total = 0.0;
  for (int i0 = threadIdx.x; i0 < tasks; i0 += 2 * SMALL_THREADS) {   // as they are, fp32, over where hi and lo will be; two pieces under way
    float u[2][8];
    int row[2], piece[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      task(min(i0 + b * SMALL_THREADS, tasks - 1), row[b], piece[b]);
      if (b == 0 || i0 + SMALL_THREADS < tasks) gather8(src, p, coef, at, row[b], n0 + piece[b] * 8, true, u[b]);
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      if (b == 1 && i0 + SMALL_THREADS >= tasks) break;
      total += squares8(u[b]);
      *piece_at(hi, row[b], piece[b], R) = make_uint4(__float_as_uint(u[b][0]), __float_as_uint(u[b][1]), __float_as_uint(u[b][2]), __float_as_uint(u[b][3]));
      *piece_at(lo, row[b], piece[b], R) = make_uint4(__float_as_uint(u[b][4]), __float_as_uint(u[b][5]), __float_as_uint(u[b][6]), __float_as_uint(u[b][7]));
    }
  }
  for (int i = threadIdx.x; i < (R - p.r) * pieces; i += SMALL_THREADS) {   // rows that are not there
    const int row = p.r + i / pieces;
    uint4* x = piece_at(hi, row, i - (row - p.r) * pieces, R);
    *x = *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(x) + (lo - hi)) = make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) warp_sums[warp] = total;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (threadIdx.x == 0) {
    total = 0.0;
    for (int i = 0; i < SMALL_THREADS / 32; ++i) total += warp_sums[i];
    norm[rank] = total;
  }
  __syncwarp();
  if (parts > 1) {
    cluster_barrier();   // every CTA of the cluster is there
    if (threadIdx.x == 0) for (int t = 0; t < parts; ++t) if (t != rank) asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote_address(smem_u32(norm + rank), t)), "d"(total) : "memory");
    __syncwarp();
    cluster_barrier();
  }
  if (threadIdx.x == 0) {
    total = 0.0;
    for (int t = 0; t < parts; ++t) total += norm[t];
    *factor = factor_of(total, p.p2);
  }
  __syncthreads();
  const Factor f0 = *factor;
  for (int i = threadIdx.x; i < tasks; i += SMALL_THREADS) {
    int row, piece;
    task(i, row, piece);
    const uint4 x = *piece_at(hi, row, piece, R), y = *piece_at(lo, row, piece, R);
    const uint32_t u[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    uint32_t h[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float c = __uint_as_float(u[2 * j]) * f0.first * f0.second, d = __uint_as_float(u[2 * j + 1]) * f0.first * f0.second;
      h[j] = pack_f16(c, d);
      const float2 b = unpack_f16(h[j]);
      l[j] = pack_f16((c - b.x) * (1 << LO_BITS), (d - b.y) * (1 << LO_BITS));
    }
    *piece_at(hi, row, piece, R) = make_uint4(h[0], h[1], h[2], h[3]);
    *piece_at(lo, row, piece, R) = make_uint4(l[0], l[1], l[2], l[3]);
  }

  const float alpha_a = static_cast<float>(ldexp(SCALE_A, -2 * p.p2)), alpha_p = static_cast<float>(SCALE_P * NS_C / (SCALE_A * SCALE_A)), beta_p = static_cast<float>(SCALE_P * NS_B / SCALE_A);
  constexpr float diag_p = static_cast<float>(SCALE_P * NS_A), beta_x = static_cast<float>(NS_A / (1 << LO_BITS));
  const uint32_t idesc_sq = idesc_f16(SMALL_R, (p.r + 31) / 32 * 32, false, false);   // columns of the warps' parts that are there
  const int ksteps = (p.r + 15) / 16;
  const uint32_t idesc_last = idesc_f16(SMALL_R, cw, false, true);
  const uint32_t quarter = tmem + (static_cast<uint32_t>(q * 32) << 16), d3 = SMALL_R;   // D3 behind the square's columns
  const int row = q * 32 + lane;
  const bool there = q * 32 < p.r && sub * 32 < p.r;   // whether this warp's part of the square matrices is; the others stay zero
#pragma unroll
  for (int i = 0; i < 4; ++i) *piece_at(a, row, sub * 4 + i) = make_uint4(0, 0, 0, 0);
  uint32_t sums_bytes = 0, a_bytes = 0;   // what comes from other CTAs in a step
  for (int u = 0; u < 16; ++u)
    if ((u >> 2) * 32 < p.r && (u & 3) * 32 < p.r) {
      if (u % parts == rank) sums_bytes += (parts - 1) * 4096;
      else a_bytes += 2048;
    }
  uint32_t phase = 0;
  // What all have written to shared memory is multiplied by one thread; all wait for the sums.
  auto multiply = [&](auto issue) {
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    if (warp == 0 && elect_one()) {
      tc_fence_after();
      issue();
      umma_commit(done_bar);
    }
    __syncwarp();   // (lanes that wait would hold up the one that issues)
    if (!mbar_wait(done_bar, phase, abort_flag) && lane == 0) atomicExch(p.status, 75);
    phase ^= 1;
    __syncwarp();
    tc_fence_after();
  };
  for (int step = 0; step < p.steps; ++step) {
    multiply([&]() {
      for (int k = 0; k < p.w / 16; ++k) {
        const uint64_t d = make_smem_desc(smem_u32(hi) + (k >> 2) * (R * 128) + (k & 3) * 32, 16, 1024);   // (rows past R are the next columns', and what they give is not read)
        umma_bf16(tmem, d, d, idesc_sq, k != 0);
      }
    });
    if (parts == 1) {
      if (there) {
        uint32_t v[32];
        tmem_ld_32x32(quarter + sub * 32, v);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t h[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) h[j] = pack_f16(__uint_as_float(v[8 * i + 2 * j]) * alpha_a, __uint_as_float(v[8 * i + 2 * j + 1]) * alpha_a);
          *piece_at(a, row, sub * 4 + i) = make_uint4(h[0], h[1], h[2], h[3]);
        }
      }
    } else {
      // unit (quarter, quarter) is finished by CTA unit % parts, as its unit / parts-th; [unit there][slab][4 columns][row] of 16 bytes
      if (there) {
        const int unit = q * 4 + sub, owner = unit % parts, place = ((unit / parts) * parts + rank) * 4096 + lane * 16;
        uint32_t v[32];
        tmem_ld_32x32(quarter + sub * 32, v);
        tmem_ld_wait();
        // Nothing that is sent overtakes: sums of the next step come from a CTA that has all of this step's A, and A from one that has all of its sums.
        if (owner == rank) {
#pragma unroll
          for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(recv + place + i * 512) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        } else {
          const uint32_t to = remote_address(smem_u32(recv) + place, owner), bar = remote_address(smem_u32(sums_bar), owner);
#pragma unroll
          for (int i = 0; i < 8; ++i) send16(to + i * 512, make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]), bar);
        }
      }
      if (threadIdx.x == 0) {
        mbar_arrive_expect_tx(sums_bar, sums_bytes);
        mbar_arrive_expect_tx(a_bar, a_bytes);
      }
      __syncthreads();   // this CTA's own sums
      if (!wait_sent(sums_bar, step & 1, abort_flag) && lane == 0) atomicExch(p.status, 76);
      __syncwarp();
      // sixteen warps share what is finished here: 32 / parts columns of a unit each, four at least
      const int share = min(parts, 8), mine = warp / share, u = rank + mine * parts, per = 8 / share;
      if (u < 16 && (u >> 2) * 32 < p.r && (u & 3) * 32 < p.r) {
        for (int c = 0; c < per; ++c) {
          const int four = (warp % share) * per + c;   // columns 4 four .. of the unit
          float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
          for (int t = 0; t < parts; ++t) {
            const float4 x = *reinterpret_cast<const float4*>(recv + (mine * parts + t) * 4096 + four * 512 + lane * 16);
            s[0] += x.x; s[1] += x.y; s[2] += x.z; s[3] += x.w;
          }
          const uint2 h = make_uint2(pack_f16(s[0] * alpha_a, s[1] * alpha_a), pack_f16(s[2] * alpha_a, s[3] * alpha_a));
          uint8_t* dst = reinterpret_cast<uint8_t*>(piece_at(a, (u >> 2) * 32 + lane, (u & 3) * 4 + four / 2)) + (four & 1) * 8;
          *reinterpret_cast<uint2*>(dst) = h;
          for (int t = 1; t < parts; ++t) send8(remote_address(smem_u32(dst), (rank + t) % parts), h, remote_address(smem_u32(a_bar), (rank + t) % parts));
        }
      }
      if (!wait_sent(a_bar, step & 1, abort_flag) && lane == 0) atomicExch(p.status, 77);
      __syncwarp();
    }
    multiply([&]() {
      for (int k = 0; k < ksteps; ++k) {
        const uint64_t d = make_smem_desc(smem_u32(a) + (k >> 2) * (SMALL_R * 128) + (k & 3) * 32, 16, 1024);
        umma_bf16(tmem, d, d, idesc_sq, k != 0);
      }
    });
    if (there) {
      uint32_t v[32];
      tmem_ld_32x32(quarter + sub * 32, v);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 old = *piece_at(a, row, sub * 4 + i);
        const uint32_t o[4] = {old.x, old.y, old.z, old.w};
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 b = unpack_f16(o[j]);
          const int col = sub * 32 + 8 * i + 2 * j;
          float x = fmaf(__uint_as_float(v[8 * i + 2 * j]), alpha_p, beta_p * b.x), y = fmaf(__uint_as_float(v[8 * i + 2 * j + 1]), alpha_p, beta_p * b.y);
          if (col == row) x += diag_p;
          if (col + 1 == row) y += diag_p;
          h[j] = pack_f16(x, y);
        }
        for (int c = 0; c < copies; ++c) *piece_at(a, row + c * R, sub * 4 + i + c * (R / 8)) = make_uint4(h[0], h[1], h[2], h[3]);
      }
    }
    multiply([&]() {
      for (int c = 0; c < copies; ++c)
        for (int k = 0; k < ksteps; ++k) {
          const int at_k = c * R + k * 16;
          const uint64_t da = make_smem_desc(smem_u32(a) + (at_k >> 6) * (SMALL_R * 128) + (at_k & 63) * 2, 16, 1024);
          const uint64_t db = make_smem_desc(smem_u32(hi) + c * (cw / 64) * (R * 128) + k * 2048, R * 128, 1024);
          umma_bf16(tmem + d3, da, db, idesc_last, (c | k) != 0);
        }
    });
    const bool end = step + 1 == p.steps, to_out = end && p.out != nullptr;
    const float alpha_x = static_cast<float>(ldexp(1.0 / SCALE_P, to_out ? -p.p2 : 0));
    const int xrow = (q * 32) % R + lane, xcol = q * 32 / R * cw;   // of the slab: this lane's row, the first column of its part
    if (xrow - lane < p.r) {
      const float2 alpha2 = make_float2(alpha_x, alpha_x), beta2 = make_float2(beta_x, beta_x), up2 = make_float2(1 << LO_BITS, 1 << LO_BITS);
#pragma unroll 1
      for (int c = sub * (cw / 4); c < (sub + 1) * (cw / 4); c += 16) {
        uint32_t v[16];
        tmem_ld_32x16(quarter + d3 + c, v);
        uint8_t *hp = reinterpret_cast<uint8_t*>(piece_at(hi, xrow, (xcol + c) / 8, R)), *lp = lo + (hp - hi);
        const int second = xrow & 1 ? -16 : 16;   // c is a multiple of 16: its second piece differs in the lowest bit
        uint32_t o[8];
        if (step < p.kept) {
          const uint4 x = *reinterpret_cast<const uint4*>(lp), y = *reinterpret_cast<const uint4*>(lp + second);
          o[0] = x.x; o[1] = x.y; o[2] = x.z; o[3] = x.w; o[4] = y.x; o[5] = y.y; o[6] = y.z; o[7] = y.w;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = 0u;
        }
        tmem_ld_wait();
        uint32_t h[8], l[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 f = ffma2(make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), alpha2, fmul2(unpack_f16(o[j]), beta2));
          h[j] = to_out ? pack_bf16(f.x, f.y) : pack_f16(f.x, f.y);
          const float2 b = unpack_f16(h[j]), d = fmul2(fadd2(f, make_float2(-b.x, -b.y)), up2);
          l[j] = pack_f16(d.x, d.y);
        }
        *reinterpret_cast<uint4*>(hp) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(hp + second) = make_uint4(h[4], h[5], h[6], h[7]);
        if (step + 1 < p.kept) {
          *reinterpret_cast<uint4*>(lp) = make_uint4(l[0], l[1], l[2], l[3]);
          *reinterpret_cast<uint4*>(lp + second) = make_uint4(l[4], l[5], l[6], l[7]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  pdl_trigger();
  for (int i = threadIdx.x; i < tasks; i += SMALL_THREADS) {
    int row, piece;
    task(i, row, piece);
    const int col = n0 + piece * 8, n = row < p.r ? max(0, min(8, p.n - col)) : 0;
    if (n == 0) continue;
    const uint4 x = *piece_at(hi, row, piece, R);
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) { const float2 b = p.out != nullptr ? unpack_bf16(u[j]) : unpack_f16(u[j]); f[2 * j] = b.x; f[2 * j + 1] = b.y; }
    const long long first = at + (p.tall ? static_cast<long long>(col) * p.cols + row : static_cast<long long>(row) * p.cols + col);
    if (p.out != nullptr) {
      if (!p.tall) { store8(p.out, 1, first, n, p.vec != 0, f); continue; }
#pragma unroll
      for (int j = 0; j < 8; ++j) if (j < n) p.out[first + static_cast<long long>(j) * p.cols] = __float2bfloat16(f[j]);
      continue;
    }
    if (!p.tall) {
      float w[8];
      load8(p.master, 0, first, n, p.vec != 0, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = fmaf(-p.step, f[j], p.keep * w[j]);
      store8(p.master, 0, first, n, p.vec != 0, w);
      if (p.param != nullptr) store8(p.param, 1, first, n, p.vec != 0, w);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) {
          const long long e = first + static_cast<long long>(j) * p.cols;
          const float w = fmaf(-p.step, f[j], p.keep * p.master[e]);
          p.master[e] = w;
          if (p.param != nullptr) p.param[e] = __float2bfloat16(w);
        }
    }
  }
  __syncthreads();
  if (parts > 1) cluster_barrier();   // nobody leaves while another may still write to it
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------------------------ host
struct Matrix {            // stack of fp16 matrices with padded rows
  uint16_t* p;
  long long rows, cols, ld, stack;
  CUtensorMap k, mn;       // loads with the columns as the reduction, or with the rows
  int make() {
    const uint64_t stride = static_cast<uint64_t>(rows) * ld;
    const int rc = make_tmap_3d_16(&k, p, cols, rows, stack, ld, stride, BK, BM);
    return rc ? rc : make_tmap_3d_16(&mn, p, cols, rows, stack, ld, stride, 64, 64);
  }
};

// Clusters of a split product that can be resident at once; 0 where the device has none of that size.
template <int CTAS>
static int resident_clusters(int splits) {
  static PerDevice<int> known[MOST_SPLITS + 1];   // and one more than them; 0: not asked yet
  int& here = known[splits].here();
  if (here == 0) {
    auto kern = split_kernel<CTAS, false, false, SYM, false>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(CTAS * splits);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = CTAS * splits; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
    here = n + 1;
  }
  return here - 1;
}
struct Form { int ctas, splits; };
// The form of a product by what its rounds of tiles take, in us: 64 of the reduction 0.28 on a single CTA (its operands from L2 at 64 bytes a clock) and 0.30 on a pair, up to 0.36 and 0.43
// where all SMs multiply at once; and what stands in front of and behind them. Fitted to stacks of 1 to 64 matrices of 64 to 4096 when each launch took half a microsecond longer than now, so it is the order of the forms that holds: whole calls take 113 us for 1024 x 1024 in
// single CTAs and 175 in pairs, 4096 x 4096 1512 and 1220, 512 x 512 85 and 151, in parts of a half 106 and 148; 1001 x 4097 209 and 269, 197 with the gram product on pairs in four parts; 1536 x 8960 498 and 495, 426 with the gram
// product on pairs in two parts and the last on pairs, 470 with it on single CTAs in two; 64 x 28672 188 with it on single CTAs in four parts and 138 in eight, 256 x 14336 154 and 131.
static Form choose(long long M, long long N, long long K, long long stack, bool sym, int pairs, int sms) {
  constexpr double base[2][4] = {{3.0, 6.0, 6.8, 7.6}, {8.0, 8.7, 9.1, 0.0}};
  auto tiles = [&](long long tile) {
    const long long tm = (M + tile - 1) / tile, tn = (N + tile - 1) / tile;
    return (sym ? tm * (tm + 1) / 2 : tm * tn) * stack;
  };
  const long long kb = (K + BK - 1) / BK;
  Form best{1, 1};
  double least = 1e30;
  for (int ctas = 1; ctas <= 2; ++ctas)
    for (int s = 0; 1 << s <= MOST_SPLITS; ++s) {
      const int splits = 1 << s;
      if ((ctas == 2 && (pairs <= 0 || splits * 2 > MOST_SPLITS)) || (s && kb < 2 * splits)) continue;
      const int room = s == 0 ? (ctas == 2 ? pairs : sms) : ctas == 2 ? resident_clusters<2>(splits) : resident_clusters<1>(splits);
      if (room <= 0) continue;
      const long long n = tiles(BM * ctas), whole = n / room, rest = n % room;   // rounds of all workers, and what is left
      const double parts = static_cast<double>((kb + splits - 1) / splits);
      auto part = [&](long long at_once) {
        const double busy = at_once * splits * ctas >= sms ? 1.0 : static_cast<double>(at_once * splits * ctas) / sms;
        return parts * (ctas == 2 ? 0.30 + 0.13 * busy : 0.28 + 0.08 * busy);
      };
      const double each = s == 0 ? 0.0 : base[ctas - 1][s];   // a split product has nothing of the next round under its epilogue
      const double t = whole * (part(room) + each) + (rest ? part(rest) + each : 0.0) + (s == 0 ? base[ctas - 1][0] : 0.0);
      if (t < least) { least = t; best = Form{ctas, splits}; }
    }
  return best;
}
template <int CTAS, bool A_MN, bool B_MN, int KIND, bool TURN>
static int launch(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& s, Params p, int splits, int workers, cudaStream_t st) {
  auto kern = product_kernel<CTAS, A_MN, B_MN, KIND, TURN>;
  auto split = split_kernel<CTAS, A_MN, B_MN, KIND, TURN>;
  static PerDevice<bool> configured;
  if (bool& done = configured.here(); !done) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess ||
        cudaFuncSetAttribute(split, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess) return -4;
    done = true;
  }
  const long long tile = BM * CTAS, tm = (p.M + tile - 1) / tile, tn = (p.N + tile - 1) / tile;
  const long long items = (KIND == SYM ? tm * (tm + 1) / 2 : tm * tn) * p.stack;
  if (items >= 1ll << 27) return -10;
  p.group_m = GROUP_M;
  if (splits > 1) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = CTAS * splits; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(items * CTAS * splits)); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM; cfg.stream = st;
    cfg.attrs = attr; cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, split, a, b, s, p, splits) == cudaSuccess ? 0 : -5;
  }
  p.workers = static_cast<int>(items < workers ? items : workers);
  launch_pdl(kern, p.workers * CTAS, THREADS, SMEM, st, a, b, s, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

static long long up(long long x, long long to) { return (x + to - 1) / to * to; }
struct Layout { long long ld, r, ldr, xbytes, gbytes, chunks, total; };
static Layout layout(long long rows, long long cols, long long stack) {
  Layout l;
  l.ld = up(cols, 64);   // rows of whole 128 bytes: ones that start off 32 cost a TMA load up to twice the requests
  l.r = rows < cols ? rows : cols;
  l.ldr = up(l.r, 64);
  l.xbytes = up(stack * rows * l.ld * 2, 256);
  l.gbytes = up(stack * l.r * l.ldr * 2, 256);
  const long long numel = rows * cols;
  long long most = MOST_CHUNKS / stack;
  if (most < 1) most = 1;
  l.chunks = (numel + 4095) / 4096;   // (16384 each took 3 us longer for a step of 576 x 576, now 94, and 5 for 16 x 512 x 512, now 142; 2048: level)
  if (l.chunks > most) l.chunks = most;
  l.total = 4 * l.xbytes + 2 * l.gbytes + up(stack * l.chunks * 8, 256);
  return l;
}

// Clusters of `parts` CTAs that can be resident at once, 0 where the device takes none of that size.
static int small_room(int parts) {
  static PerDevice<int> known[SMALL_PARTS + 1];   // and one more than them; 0: not asked yet
  int& here = known[parts].here();
  if (here == 0) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = parts; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(parts); cfg.blockDim = dim3(SMALL_THREADS); cfg.dynamicSmemBytes = small_smem(SMALL_ENTRIES);
    cfg.attrs = &attr; cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(small_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, small_smem(SMALL_ENTRIES)) != cudaSuccess ||
        cudaFuncSetAttribute(small_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, small_kernel, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
    here = n + 1;
  }
  return here - 1;
}
// Whether a call is one launch, and how that divides a matrix: false where it does not fit one, or would take longer so. By sizes and the device alone.
static bool small_form(Small& p, long long stack) {
  p.tall = p.rows > p.cols;
  p.r = p.tall ? p.cols : p.rows;
  p.n = p.tall ? p.rows : p.cols;
  if (p.r > SMALL_R || stack > 1 << 20) return false;
  p.R = p.r <= 32 && p.n > 128 ? 32 : p.r <= 64 && p.n > 64 ? 64 : 128;   // a slab's parts have 64 columns at least
  p.kept = p.steps > 2 ? p.steps - 2 : p.steps - 1;
  const int most = SMALL_ENTRIES / p.R, step = 64 * (SMALL_R / p.R);
  // Rounds of clusters, of what a slab's size takes and what its exchange does, in us, against fifteen launches that pass over the matrices six times a step: 32 x 2048 48 as two slabs and 35 as eight, 128 x 128 28 as
  // one and 41 as two, 64 x 128 x 1024 (two rounds of clusters of four) 132 and 123 in the other form.
  double least = 75.0 + static_cast<double>(stack) * p.r * p.n * 6.5e-6;
  p.parts = 0;
  for (int parts = 1; parts <= SMALL_PARTS; parts *= 2) {
    const int w = static_cast<int>(up((p.n + parts - 1) / parts, step));
    if (w > most) continue;
    const int room = small_room(parts);
    if (room <= 0) continue;
    const double e = w * p.R / 8192.0, wide = p.r > 64 ? 1.0 : 0.0;
    const double t = (stack > room ? 1.3 : 1.0) * ((stack + room - 1) / room) * (3.0 + 2.3 * e + p.steps * (2.1 + 0.5 * wide + 0.78 * e + (parts > 1 ? 1.9 + 2.6 * wide + 0.1 * parts : 0.0)));
    if (t < least) { least = t; p.parts = parts; p.w = w; }
  }
  return p.parts != 0;
}
static int small_call(const Source& src, const Small& p, long long stack, cudaStream_t st) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.parts; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(stack * p.parts)); cfg.blockDim = dim3(SMALL_THREADS); cfg.dynamicSmemBytes = small_smem(p.w * p.R); cfg.stream = st;
  cfg.attrs = attr; cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, small_kernel, src, p) == cudaSuccess ? 0 : -5;
}

// Everything up to the last product, which leaves hi 2^p in *result (fp16, padded), or bf16 in `out` (padded rows of out_ld).
static int orthogonalise(const Source& src, long long rows, long long cols, long long stack, int steps, void* out, long long out_ld, int p2, uint8_t* ws, int pairs, int* status, cudaStream_t st) {
  const Layout l = layout(rows, cols, stack);
  const bool right = rows > cols;
  __half* x[2][2] = {{(__half*)ws, (__half*)(ws + l.xbytes)}, {(__half*)(ws + 2 * l.xbytes), (__half*)(ws + 3 * l.xbytes)}};
  uint8_t* g = ws + 4 * l.xbytes;
  double* sums = (double*)(g + 2 * l.gbytes);
  const long long numel = rows * cols;
  const bool plain = ((reinterpret_cast<uintptr_t>(src.g) | reinterpret_cast<uintptr_t>(src.m)) & 15) == 0;
  const int vec_flat = plain && numel % 8 == 0, vec_rows = plain && cols % 8 == 0;
  const long long per_chunk = up((numel + l.chunks - 1) / l.chunks, 8 * LIN_THREADS);
  if (stack * l.chunks >= 1ll << 31) return -10;
  launch_pdl(squares_kernel, static_cast<unsigned>(stack * l.chunks), LIN_THREADS, 0, st, src, numel, static_cast<int>(l.chunks), per_chunk, vec_flat, sums);
  const int kept = steps > 2 ? steps - 2 : steps - 1;   // steps whose X is held as two numbers
  long long blocks = (rows * ((cols + 7) / 8) + LIN_THREADS - 1) / LIN_THREADS, most = (sms_here() * 8 + stack - 1) / stack;
  if (blocks > most) blocks = most;
  launch_pdl(scale_kernel, static_cast<unsigned>(stack * blocks), LIN_THREADS, 0, st, src, static_cast<int>(rows), static_cast<int>(cols), static_cast<int>(l.ld), static_cast<int>(l.chunks),
             static_cast<int>(blocks), vec_rows, p2, sums, x[0][0], kept > 0 ? x[0][1] : nullptr);
  if (cudaGetLastError() != cudaSuccess) return -5;

  Matrix xh[2], gram{(uint16_t*)g, l.r, l.r, l.ldr, stack}, poly{(uint16_t*)(g + l.gbytes), l.r, l.r, l.ldr, stack};
  for (int i = 0; i < 2; ++i) {
    xh[i] = Matrix{(uint16_t*)x[i][0], rows, cols, l.ld, stack};
    if (const int rc = xh[i].make()) return rc - 20;
  }
  int rc = gram.make();
  if (!rc) rc = poly.make();
  if (rc) return rc - 30;

  const int sms = sms_here();
  const int r = static_cast<int>(l.r), K = static_cast<int>(right ? rows : cols);
  const Form fg = choose(r, r, K, stack, true, pairs, sms), fp = choose(r, r, r, stack, true, pairs, sms), fa = choose(rows, cols, r, stack, false, pairs, sms);
#define PRODUCT(F, A_MN, B_MN, KIND, TURN, ...) (F.ctas == 2 ? launch<2, A_MN, B_MN, KIND, TURN>(__VA_ARGS__, F.splits, pairs, st) : launch<1, A_MN, B_MN, KIND, TURN>(__VA_ARGS__, F.splits, sms, st))
#define PRODUCT_SYM(F, A_MN, B_MN, KIND, ...) (turn ? PRODUCT(F, A_MN, B_MN, KIND, true, __VA_ARGS__) : PRODUCT(F, A_MN, B_MN, KIND, false, __VA_ARGS__))
  // Where the matrix is two blocks wide the launches are short, and the transposes cost less than what each of them has to think about: 8 x 2048 x 512 175 us with the transposes and 179 without, 4 x 512 x 1376 120 and 122; larger
  // ones, in loops at the power cap: 64 x 2048 x 1024 3.00 ms and 2.88, 4096 x 4096 1.26 and 1.22, 5120 x 5120 2.36 and 2.28.
  const bool turn = r > 2 << WHOLE_BITS;
  for (int i = 0; i < steps; ++i) {
    const Matrix& X = xh[i & 1];
    Params p{r, r, K, static_cast<int>(stack), 0, 0, static_cast<float>(ldexp(SCALE_A, -2 * p2)), 0.f, gram.p, nullptr, nullptr, 0.f, l.ldr, l.r * l.ldr, 0, turn ? WHOLE_BITS : 24, 0, 0, status};
    rc = right ? PRODUCT(fg, true, true, SYM, false, X.mn, X.mn, gram.mn, p) : PRODUCT(fg, false, false, SYM, false, X.k, X.k, gram.mn, p);
    if (rc) return rc;
    p.K = r;
    p.alpha = static_cast<float>(SCALE_P * NS_C / (SCALE_A * SCALE_A));
    p.diag = static_cast<float>(SCALE_P * NS_A);
    p.d = poly.p;
    p.res = reinterpret_cast<const __half*>(gram.p);
    p.beta = static_cast<float>(SCALE_P * NS_B / SCALE_A);
    p.sym_a = p.sym_b = 1;
    rc = PRODUCT_SYM(fp, false, false, SYM, gram.k, gram.k, gram.mn, p);
    if (rc) return rc;
    const bool to_out = i + 1 == steps && out != nullptr;
    const long long ld = to_out ? out_ld : l.ld;   // (the last step has no residual, whose rows would be another matrix's)
    Params a{static_cast<int>(rows), static_cast<int>(cols), r, static_cast<int>(stack), 0, 0, static_cast<float>(ldexp(1.0 / SCALE_P, to_out ? -p2 : 0)), 0.f,
             to_out ? (uint16_t*)out : xh[(i + 1) & 1].p, i + 1 < kept ? (uint16_t*)x[(i + 1) & 1][1] : nullptr, i < kept ? x[i & 1][1] : nullptr, static_cast<float>(ldexp(NS_A, -LO_BITS)),
             ld, rows * ld, to_out, 0, !right, right, status};
    rc = right ? PRODUCT_SYM(fa, false, false, APPLY, X.k, poly.k, poly.mn, a) : PRODUCT_SYM(fa, false, true, APPLY, poly.k, X.mn, poly.mn, a);
    if (rc) return rc;
  }
#undef PRODUCT_SYM
#undef PRODUCT
  return 0;
}
static int exponent(long long rows, long long cols) { return static_cast<int>(lround(0.5 * log2(static_cast<double>(rows > cols ? rows : cols)))); }
static bool sizes_ok(long long rows, long long cols, long long stack, int steps) {
  return rows > 0 && cols > 0 && stack > 0 && rows < 1 << 24 && cols < 1 << 24 && stack < 1 << 24 && steps >= 1 && steps <= 64 && (rows < cols ? rows : cols) <= 1 << 16;
}

}  // namespace ns
}  // namespace mtb

extern "C" {

int mtb200_gemm2_pairs();

// Bytes of the workspace of the two calls below, which starts on 256 bytes; 0 where they are one launch on the current device, and take none.
long long mtb200_newton_schulz_workspace(long long rows, long long cols, long long stack, int steps) {
  using namespace mtb::ns;
  if (!sizes_ok(rows, cols, stack, steps)) return -1;
  Small one{static_cast<int>(rows), static_cast<int>(cols)};
  one.steps = steps;
  return small_form(one, stack) ? 0 : layout(rows, cols, stack).total;
}
// Launches of a call: sums and scaling, three products a step, one behind them.
// out [stack, rows, cols] bf16 = g [stack, rows, cols] (bf16 or fp32) orthogonalised.
int mtb200_newton_schulz(const void* g, int g_bf16, void* out, long long rows, long long cols, long long stack, int steps, void* ws, long long ws_bytes, int* status, cudaStream_t st) {
  using namespace mtb::ns;
  if (!sizes_ok(rows, cols, stack, steps)) return -10;
  const Source src{g, g_bf16, nullptr, 0, nullptr, 0.f, 0};
  Small one{static_cast<int>(rows), static_cast<int>(cols)};
  one.steps = steps; one.p2 = exponent(rows, cols); one.out = (__nv_bfloat16*)out; one.status = status;
  one.vec = cols % 8 == 0 && ((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  if (small_form(one, stack)) return small_call(src, one, stack, st);
  const Layout l = layout(rows, cols, stack);
  if (ws_bytes < l.total || (reinterpret_cast<uintptr_t>(ws) & 255)) return -11;
  const bool direct = cols % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  uint8_t* w = reinterpret_cast<uint8_t*>(ws);
  void* to = direct ? out : w + 2 * (steps & 1) * l.xbytes;   // the buffer that the last step writes
  int rc = orthogonalise(src, rows, cols, stack, steps, to, direct ? cols : l.ld, exponent(rows, cols), w, mtb200_gemm2_pairs(), status, st);
  if (rc || direct) return rc;
  const long long n = stack * rows * cols;
  long long blocks = (n + LIN_THREADS - 1) / LIN_THREADS;
  if (blocks > mtb::sms_here() * 16) blocks = mtb::sms_here() * 16;
  mtb::launch_pdl(unpad_kernel, static_cast<unsigned>(blocks), LIN_THREADS, 0, st, (const __nv_bfloat16*)to, static_cast<int>(l.ld), stack * rows, static_cast<int>(cols), (__nv_bfloat16*)out);
  return cudaGetLastError() == cudaSuccess ? 0 : -5;
}
// m <- mu m + coef g;  master <- keep master - step O(nesterov ? coef g + mu m : m);  param <- master. g bf16 or fp32, m fp32 or bf16, master fp32, param bf16 or null, coef on the device or null.
int mtb200_muon_step(float* master, void* m, int m_bf16, const void* g, int g_bf16, void* param, const float* coef, long long rows, long long cols, long long stack, int steps, float mu,
                     int nesterov, float keep, float step, void* ws, long long ws_bytes, int* status, cudaStream_t st) {
  using namespace mtb::ns;
  if (!sizes_ok(rows, cols, stack, steps) || m == nullptr) return -10;
  const Source src{g, g_bf16, m, m_bf16, coef, mu, nesterov};
  Small one{static_cast<int>(rows), static_cast<int>(cols)};
  one.steps = steps; one.p2 = exponent(rows, cols); one.master = master; one.param = (__nv_bfloat16*)param; one.keep = keep; one.step = static_cast<float>(ldexp(step, -one.p2)); one.status = status;
  one.vec = cols % 8 == 0 && ((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(master) | reinterpret_cast<uintptr_t>(param)) & 15) == 0;
  if (small_form(one, stack)) return small_call(src, one, stack, st);
  const Layout l = layout(rows, cols, stack);
  if (ws_bytes < l.total || (reinterpret_cast<uintptr_t>(ws) & 255)) return -11;
  uint8_t* w = reinterpret_cast<uint8_t*>(ws);
  const int p2 = exponent(rows, cols);
  int rc = orthogonalise(src, rows, cols, stack, steps, nullptr, 0, p2, w, mtb200_gemm2_pairs(), status, st);
  if (rc) return rc;
  const __half* o = reinterpret_cast<const __half*>(w + 2 * (steps & 1) * l.xbytes);
  const int vec = cols % 8 == 0 && ((reinterpret_cast<uintptr_t>(master) | reinterpret_cast<uintptr_t>(param)) & 15) == 0;
  long long blocks = (stack * rows * ((cols + 7) / 8) + LIN_THREADS - 1) / LIN_THREADS;
  if (blocks > mtb::sms_here() * 8) blocks = mtb::sms_here() * 8;
  mtb::launch_pdl(update_kernel, static_cast<unsigned>(blocks), LIN_THREADS, 0, st, master, (__nv_bfloat16*)param, o, static_cast<int>(l.ld), stack * rows, static_cast<int>(cols), vec, keep,
                  static_cast<float>(ldexp(step, -p2)));
  return cudaGetLastError() == cudaSuccess ? 0 : -5;
}

}  // extern "C"
