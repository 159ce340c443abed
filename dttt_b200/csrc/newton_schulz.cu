// Newton-Schulz orthogonalisation of batches of matrices on the tensor cores.
//
//   x_0 = g / |g|_F                                     g [rows, cols], d the smaller side
//   G_k = x_k x_k^T  (x_k^T x_k when rows > cols)       [d, d]
//   P_k = b G_k + c G_k G_k                             [d, d], symmetric
//   x_{k+1} = a x_k + P_k x_k  (a x_k + x_k P_k)        y = x_steps in bf16
//
// y is a polynomial of the matrix times g / |g|; its derivative is taken with the polynomial and the norm held constant (the map
// is then linear and self-adjoint), so the backward applies the same a r + P_k r in reverse order to the cotangent.
//
// Operands are f16, not bf16: the same tensor-core rate with three more bits.  Roundings of G, of P and of x inside P x stay within the
// row or the column space of x: they turn singular vectors by about as much as they are, and nothing amplifies that.  What x loses when
// it is stored lies mostly outside both, where an iteration multiplies by a = 3.4445 (five of them by 485), and the gradient of a
// write, of as many tokens as a chunk has, fills at most a part of either space.  So x is kept in two f16 halves: the products take the
// upper one, and the lower one is added with what the map does outside the spaces, alpha + s (below).  Only the last group does
// without.  Five steps, off by (2-norm, the bf16 result's own 1.66e-3 included; in brackets with the upper half alone):
//   512 x 2048 (paired iterations)  rank 1 3.9e-3 (0.145), rank 64 3.8e-3 (1.6e-2), rank 256 3.4e-3 (7.1e-3), full 2.06e-3 (2.06e-3)
//   509 x 1283                      rank 1 2.3e-3 (0.147), rank 63 2.1e-3 (2.0e-2), rank 254 2.0e-3 (7.9e-3), full 1.9e-3 (1.9e-3)
//   128 x 256                       rank 1 2.5e-3 (0.145), rank 16 2.1e-3 (3.5e-2), rank 64 2.1e-3 (1.3e-2), full 2.07e-3 (1.98e-3)
// It costs 4 x 2048 x 8192 1807 -> 1834 us, 8192 x 2048 with its derivative 823 -> 839, 3 x 509 x 1283 likewise 221 -> 230, 128 x 512 in
// one launch 53 -> 66.  Keeping G and P in two halves as well would leave the bf16 result's rounding alone, at three times the products.
// Everything that is stored has singular values below 1.21 (x), 1.47 (G) and 2.82 (P), so fixed powers of two keep it inside f16: 2^12
// for those (the lower half ends at 2^-25 of that scale).  The cotangent, which grows 3.4445-fold per iteration where the matrix has no
// singular value, is scaled to norm 2^5 and stays inside f16 for six products; the seventh leaves as f32, and further ones start again
// from that.  Sums are f32 (tensor memory), the norms f64.
//
// Every product is C = alpha A B + beta D (+ s I) on CTA pairs: tiles of 256 rows and 256 or 128 columns, tcgen05.mma.cta_group::2,
// plain per-CTA TMA loads, symmetric results formed for the tiles on and below the diagonal and stored twice.  What bounds it:
//   * large matrices: the tensor cores.  4 x 2048 x 8192 f32, five steps: 1.84 ms for 2.23 TFLOP (symmetric halves counted once) =
//     1210 TFLOP/s; tensor pipe 92 % busy in a product with x alone, 86 % and 78 % where the lower half is read, and read and written;
//     8192 x 2048 with its derivative 0.84 ms = 1075 TFLOP/s.
//   * middle ones: the chain of products, each of which is one round of tiles whose first loads, store and mirrored store are
//     not hidden: 3 x 509 x 1283, five steps 177 us and its derivative 53 us, 8 to 11 us a product; programmatic launches start a
//     product's prologue under the one before (263 -> 230 us).  All of them in one cooperative launch gained nothing.
//   * d <= 128 and L <= 4096, most of them (`is_small`): one CTA or cluster and one launch, 23 us for 2 x 128 x 256 and two steps.
#include "host_check.h"
#include "ptx_sm100.cuh"

#include <cuda_fp16.h>

#include <cstring>
#include <mutex>

namespace dttt {
namespace ns {

constexpr int BM = 128;        // rows of A per CTA (256 per pair)
constexpr int BK = 64;
constexpr int UMMA_K = 16;
constexpr int A_BYTES = BM * BK * 2;
constexpr int EPI_WARPS = 8;   // two per quarter of the accumulator's rows, half of the columns each
constexpr int THREADS = (2 + EPI_WARPS) * 32;
constexpr int STAGING_BYTES = EPI_WARPS * 4096;                // epilogue: 32 rows x 128 bytes per warp

// What a product's epilogue does beside alpha A B + beta D: a kernel of its own each.
enum { MODE_PLAIN = 0, MODE_SUM = 1, MODE_DIAG = 2, MODE_SPLIT = 3 };      // + beta2 D2 + diag I | + diag I | + beta2 D2, in two halves

// BN: output columns per pair (256 or 128); each CTA loads BN / 2 of them.  With a second summand a second staging area takes the place
// of one stage.
template <int BN, int MODE>
struct Tile {
  static constexpr int B_BYTES = (BN / 2) * BK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr bool TWO = MODE == MODE_SUM || MODE == MODE_SPLIT;
  static constexpr int STAGES = (BN == 256 ? 6 : 8) - (TWO ? (STAGING_BYTES + STAGE_BYTES - 1) / STAGE_BYTES : 0);
  static constexpr int SMEM = STAGES * STAGE_BYTES + 1024 + (TWO ? 2 : 1) * STAGING_BYTES + 1024;
  static_assert(SMEM <= 227 * 1024, "shared memory of an SM");
};

constexpr int MAX_STEPS = 32;
constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr float X_SCALE = 4096.f;           // of x, G and P
constexpr float R_SCALE = 32.f;             // of the cotangent
constexpr int PART_STEPS = 7;               // of the derivative between two f32 results: 32 3.4445^6 < 65504

enum { OUT_F16 = 0, OUT_BF16 = 1, OUT_F32 = 2 };

struct Params {
  int M, N, K, batch;
  int a_mn_major, b_mn_major;
  float alpha, beta;
  const __half* D;             // or null; same shape as C
  const __half* D2;            // a second one
  long long ldd, d_batch;      // of both
  float beta2, diag;
  __half* lo;                  // what the f16 rounding of C leaves, with the layout of C; may be D2
  void* C;
  int out;
  long long ldc, c_batch;
  const double* num;           // per-batch factors of the output, or null
  const double* den;
  int* status;
  int symmetric;               // C is symmetric: tiles on and below the diagonal, those below are stored a second time transposed
  int tiles_m, tiles_n;
};

// A symmetric C takes the tiles that reach the diagonal or lie below it: with tiles `w` = 256 / BN to a square block, block row tm has
// w (tm + 1) of them.
__host__ __device__ inline int tiles_per_matrix(const Params& p, int w) {
  return p.symmetric ? w * (p.tiles_m * (p.tiles_m + 1) / 2) : p.tiles_m * p.tiles_n;
}

template <int BN>
__device__ __forceinline__ void tile_coords(int tile, const Params& p, int& b, int& tm, int& tn) {
  constexpr int w = 256 / BN;
  const int per_batch = tiles_per_matrix(p, w);
  b = tile / per_batch;
  const int t = tile - b * per_batch;
  if (p.symmetric) {
    const int q = t / w;                                       // counts square blocks row by row
    tm = (int)((sqrtf(8.f * (float)q + 1.f) - 1.f) * 0.5f);
    while (tm * (tm + 1) / 2 > q) --tm;                        // the root may round across a whole number
    while ((tm + 1) * (tm + 2) / 2 <= q) ++tm;
    tn = t - w * (tm * (tm + 1) / 2);
    return;
  }
  constexpr int GROUP = 8;                                     // bands of 8 pair rows, n fastest inside a band
  const int band = t / (GROUP * p.tiles_n);
  const int first_m = band * GROUP;
  const int rows = min(GROUP, p.tiles_m - first_m);
  const int r = t - band * GROUP * p.tiles_n;
  tm = first_m + (r % rows);
  tn = r / rows;
}

// ------------------------------------------------------------------ the epilogue's pieces
// A warp handles 32 rows x 64 columns of 16-bit values at a time.  Global memory sees whole 128-byte lines, eight lanes to a row;
// the threads see a row each (as tcgen05.ld delivers the accumulator).  A 4 KB staging area with 16-byte pieces XOR-swizzled
// by row turns one into the other.  `rows`, `cols`: what is left of the matrix from here on (may be negative); stored f16 matrices
// have rows of a multiple of 8, so a piece is there or not as a whole, and what is in the padding is never read.
__device__ __forceinline__ void load_rows(const __half* d, long long ld, int rows, int cols, int lane, uint4 (&v)[8]) {
  const int piece = lane & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int rr = i * 4 + (lane >> 3);
    v[i] = d && rr < rows && piece * 8 < cols ? __ldcg(reinterpret_cast<const uint4*>(d + rr * ld + piece * 8)) : make_uint4(0, 0, 0, 0);
  }
}
__device__ __forceinline__ void stage_in(uint8_t* stg, int lane, const uint4 (&v)[8]) {
  const int piece = lane & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int rr = i * 4 + (lane >> 3);
    *reinterpret_cast<uint4*>(stg + rr * 128 + ((piece ^ (rr & 7)) * 16)) = v[i];
  }
}
template <class T2> __device__ __forceinline__ T2 pack2(float a, float b);
template <> __device__ __forceinline__ __half2 pack2<__half2>(float a, float b) { return __floats2half2_rn(a, b); }
template <> __device__ __forceinline__ __nv_bfloat162 pack2<__nv_bfloat162>(float a, float b) { return __floats2bfloat162_rn(a, b); }
// What is left of two values beside `h`, their f16 roundings.
__device__ __forceinline__ __half2 left_over(__half2 h, float a, float b) {
  const float2 f = __half22float2(h);
  return __floats2half2_rn(a - f.x, b - f.y);
}
template <class T2>
__device__ __forceinline__ uint4 pack8(const uint32_t* r) {
  uint4 v;
  T2* h = reinterpret_cast<T2*>(&v);
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = pack2<T2>(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]));
  return v;
}
__device__ __forceinline__ void flush_lines(const uint8_t* stg, int lane, uint16_t* out, long long ld, int rows, int cols) {
  const int piece = lane & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int rr = i * 4 + (lane >> 3);
    const uint4 v = *reinterpret_cast<const uint4*>(stg + rr * 128 + ((piece ^ (rr & 7)) * 16));
    if (rr < rows && piece * 8 < cols) *reinterpret_cast<uint4*>(out + rr * ld + piece * 8) = v;
  }
}
// rows that start at any element: 32 neighbouring elements per instruction
__device__ __forceinline__ void flush_ragged(const uint8_t* stg, int lane, uint16_t* out, long long ld, int rows, int cols) {
#pragma unroll 4
  for (int rr = 0; rr < 32; ++rr) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int j = h * 32 + lane;
      const uint16_t v = *reinterpret_cast<const uint16_t*>(stg + rr * 128 + (((j >> 3) ^ (rr & 7)) * 16) + (j & 7) * 2);
      if (rr < rows && j < cols) out[rr * ld + j] = v;
    }
  }
}
// 32 columns
__device__ __forceinline__ void store_f32(float* out, long long ld, int rows, int cols, int lane, const uint32_t (&r)[32]) {
  if (lane >= rows) return;
  float* o = out + lane * ld;
  if ((ld & 3) == 0) {
#pragma unroll
    for (int j = 0; j < 32; j += 4)
      if (j < cols) *reinterpret_cast<float4*>(o + j) = make_float4(__uint_as_float(r[j]), __uint_as_float(r[j + 1]), __uint_as_float(r[j + 2]),
                                                                    __uint_as_float(r[j + 3]));
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < cols) o[j] = __uint_as_float(r[j]);
  }
}
// The transpose of 32 rows x 32 columns: column j becomes a row.  Neighbouring lanes (rows 2i, 2i + 1 of the piece) trade one value per
// pair of columns, so that each stores two neighbours: an instruction writes 64 bytes of two rows.
__device__ __forceinline__ void store_transposed(__half* out, long long ld, int rows, int cols, int lane, const uint32_t (&r)[32]) {
  const bool odd = lane & 1;
  const int at = lane & ~1;
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    const float mine = __uint_as_float(odd ? r[j + 1] : r[j]);
    const float theirs = __shfl_xor_sync(0xffffffffu, __uint_as_float(odd ? r[j] : r[j + 1]), 1);
    const __half2 v = odd ? __floats2half2_rn(theirs, mine) : __floats2half2_rn(mine, theirs);
    const int jr = j + odd;
    if (jr < rows && at < cols) *reinterpret_cast<__half2*>(out + jr * ld + at) = v;
  }
}

template <int BN, int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
ns_product_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB, const Params p) {
  constexpr int STAGES = Tile<BN, MODE>::STAGES, STAGE_BYTES = Tile<BN, MODE>::STAGE_BYTES;
  constexpr bool TWO = Tile<BN, MODE>::TWO;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);      // the leader's count both CTAs' bytes
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;                          // the leader's: both CTAs' epilogues have drained it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_word = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair_id = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
  const int num_tiles = p.batch * tiles_per_matrix(p, 256 / BN);
  const int kblocks = (p.K + BK - 1) / BK;
  constexpr uint32_t TMEM_COLS = 2 * BN;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&acc_full[a], 1); mbar_init(&acc_empty[a], 2 * EPI_WARPS * 32); }
    *abort_word = 0;
    fence_mbar_init();
    tma_prefetch_desc(&mapA);
    tma_prefetch_desc(&mapB);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // launched while the product before it still runs (programmatic dependence): up to here nothing touched global memory
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();

  if (warp == 0) {
    if (elect_one()) {
      uint32_t it = 0;
      bool ok = true;
      for (int tile = pair_id; tile < num_tiles && ok; tile += n_pairs) {
        int b, tm, tn;
        tile_coords<BN>(tile, p, b, tm, tn);
        const int m0 = tm * 2 * BM + (int)rank * BM;
        const int n0 = tn * BN + (int)rank * (BN / 2);
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1;
          if (!mbar_wait_bounded(&empty[s], ph ^ 1, abort_word, p.status, ERR_WAIT_EMPTY)) { ok = false; break; }
          uint8_t* sA = smem + s * STAGE_BYTES;
          uint8_t* sB = sA + A_BYTES;
          if (rank == 0) mbar_expect_tx(&full[s], 2 * STAGE_BYTES);
          const uint32_t bar = mapa_u32(&full[s], 0);
          const int k0 = kb * BK;
          if (!p.a_mn_major) {
            tma_load_3d_pair(sA, &mapA, bar, k0, m0, b);
          } else {
#pragma unroll
            for (int j = 0; j < BM / 64; ++j) tma_load_3d_pair(sA + j * (BK * 128), &mapA, bar, m0 + j * 64, k0, b);
          }
          if (!p.b_mn_major) {
            tma_load_3d_pair(sB, &mapB, bar, k0, n0, b);
          } else {
#pragma unroll
            for (int j = 0; j < (BN / 2) / 64; ++j) tma_load_3d_pair(sB + j * (BK * 128), &mapB, bar, n0 + j * 64, k0, b);
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = make_idesc_f16(2 * BM, BN, p.a_mn_major, p.b_mn_major);
      const uint32_t a_lbo = p.a_mn_major ? BK * 128 : 16, b_lbo = p.b_mn_major ? BK * 128 : 16;
      const uint32_t a_kstep = p.a_mn_major ? UMMA_K * 128 : UMMA_K * 2;
      const uint32_t b_kstep = p.b_mn_major ? UMMA_K * 128 : UMMA_K * 2;
      uint32_t it = 0, local_tile = 0;
      bool ok = true;
      for (int tile = pair_id; tile < num_tiles && ok; tile += n_pairs, ++local_tile) {
        const int acc = local_tile & 1;
        const uint32_t acc_ph = (local_tile >> 1) & 1;
        if (!mbar_wait_bounded(&acc_empty[acc], acc_ph ^ 1, abort_word, p.status, ERR_WAIT_TMEM_EMPTY)) { ok = false; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = it % STAGES;
          const uint32_t ph = (it / STAGES) & 1;
          if (!mbar_wait_bounded(&full[s], ph, abort_word, p.status, ERR_WAIT_FULL)) { ok = false; break; }
          tc_fence_after();
          const uint32_t sA = smem_u32(smem + s * STAGE_BYTES);
          const uint32_t sB = sA + A_BYTES;
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k)
            umma_f16_pair(d_tmem, make_smem_desc(sA + k * a_kstep, a_lbo, 1024), make_smem_desc(sB + k * b_kstep, b_lbo, 1024), idesc,
                          (kb | k) ? 1u : 0u);
          umma_commit_pair(&empty[s], 3);
        }
        if (ok) umma_commit_pair(&acc_full[acc], 3);
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, c0 = ((warp - 2) >> 2) * (BN / 2);      // tensor memory lanes belong to warps by their number mod 4
    uint32_t local_tile = 0;
    for (int tile = pair_id; tile < num_tiles; tile += n_pairs, ++local_tile) {
      int b, tm, tn;
      tile_coords<BN>(tile, p, b, tm, tn);
      const int acc = local_tile & 1;
      const uint32_t acc_ph = (local_tile >> 1) & 1;
      const int row0 = tm * 2 * BM + (int)rank * BM + quarter * 32, n0 = tn * BN + c0;
      const int rows = p.M - row0;                             // of this warp's 32 (may be negative)
      float alpha = p.alpha, beta = p.beta;
      bool none = false;                                       // a zero matrix has a zero derivative, whatever the cotangent
      if (p.num || p.den) {
        const double den = p.den ? p.den[b] : 1.0;
        const float f = (float)((p.num ? p.num[b] : 1.0) / den);
        none = den == 0.0;
        alpha *= f; beta *= f;
      }
      const __half* d0 = p.D ? p.D + (long long)b * p.d_batch + (long long)row0 * p.ldd + n0 : nullptr;
      uint4 dnext[8];                                          // 64 columns of D, eight lanes to a row's 128 bytes
      load_rows(d0, p.ldd, rows, (int)p.ldd - n0, lane, dnext);
      uint4 lnext[8];                                          // and of D2
      if (TWO) load_rows(p.D2 + (d0 - p.D), p.ldd, rows, (int)p.ldd - n0, lane, lnext);
      int got = 1;
      if (lane == 0) got = mbar_wait_bounded(&acc_full[acc], acc_ph, abort_word, p.status, ERR_WAIT_TMEM_FULL) ? 1 : 0;
      got = __shfl_sync(0xffffffffu, got, 0);
      if (!got) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + acc * BN + c0 + ((uint32_t)(quarter * 32) << 16);
      uint8_t* stg = smem + STAGES * STAGE_BYTES + 1024 + (warp - 2) * 4096;
      uint8_t* stg2 = stg + STAGING_BYTES;                     // of D2 and `lo`
#pragma unroll 1
      for (int c = 0; c < BN / 2; c += 64) {
        if (d0) {
          stage_in(stg, lane, dnext);
          if (c + 64 < BN / 2) load_rows(d0 + c + 64, p.ldd, rows, (int)p.ldd - n0 - c - 64, lane, dnext);
        }
        if (TWO) {
          stage_in(stg2, lane, lnext);
          if (c + 64 < BN / 2) load_rows(p.D2 + (d0 - p.D) + c + 64, p.ldd, rows, (int)p.ldd - n0 - c - 64, lane, lnext);
        }
        __syncwarp();
        // 32 columns at a time: 64 of them spill beside the rows that are on their way, and next to this much shared memory there is no L1
        // for that (4 x 2048 x 8192 1826 instead of 1578 us, both at the burst clock); in narrow tiles they fit and are no gain (2 x 300 x
        // 700 145 instead of 130 us).  A lane's row of the staging areas is its own until the flush: results take the place of the summands
        // that they were made of.
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          uint32_t r[32];
          tmem_ld_32x32(taddr + c + 32 * h, r);
          tmem_ld_wait();
          const int col = n0 + c + 32 * h;
          const int on = MODE == MODE_SUM || MODE == MODE_DIAG ? row0 + lane - col : -1;      // the diagonal among the 32
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int at = lane * 128 + (((4 * h + q) ^ (lane & 7)) * 16);
            uint4 dv = make_uint4(0, 0, 0, 0), lv = make_uint4(0, 0, 0, 0);
            if (d0) dv = *reinterpret_cast<const uint4*>(stg + at);
            if (TWO) lv = *reinterpret_cast<const uint4*>(stg2 + at);
            const __half2 *dh = reinterpret_cast<const __half2*>(&dv), *lh = reinterpret_cast<const __half2*>(&lv);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float2 df = __half22float2(dh[e >> 1]), lf = __half22float2(lh[e >> 1]);
              float x = fmaf(beta, e & 1 ? df.y : df.x, alpha * __uint_as_float(r[8 * q + e]));
              if (TWO) x = fmaf(p.beta2, e & 1 ? lf.y : lf.x, x);
              if (MODE == MODE_SUM || MODE == MODE_DIAG) x += on == 8 * q + e ? p.diag : 0.f;
              r[8 * q + e] = none ? 0u : __float_as_uint(x);
            }
            if (MODE == MODE_SPLIT) {
              const uint4 o = pack8<__half2>(r + 8 * q);
              const __half2* hi = reinterpret_cast<const __half2*>(&o);
              uint4 w;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                reinterpret_cast<__half2*>(&w)[e] = left_over(hi[e], __uint_as_float(r[8 * q + 2 * e]), __uint_as_float(r[8 * q + 2 * e + 1]));
              *reinterpret_cast<uint4*>(stg + at) = o;
              *reinterpret_cast<uint4*>(stg2 + at) = w;
            } else if (p.out == OUT_F16) {
              *reinterpret_cast<uint4*>(stg + at) = pack8<__half2>(r + 8 * q);
            } else if (p.out == OUT_BF16) {
              *reinterpret_cast<uint4*>(stg + at) = pack8<__nv_bfloat162>(r + 8 * q);
            }
          }
          if (p.out == OUT_F32)
            store_f32(reinterpret_cast<float*>(p.C) + (long long)b * p.c_batch + (long long)row0 * p.ldc + col, p.ldc, rows, p.N - col, lane, r);
          if (p.symmetric && tn < tm * (256 / BN))             // the result's other half
            store_transposed(reinterpret_cast<__half*>(p.C) + (long long)b * p.c_batch + (long long)col * p.ldc + row0, p.ldc, p.N - col,
                             (int)p.ldc - row0, lane, r);
          __syncwarp();                                        // the next load is one of the whole warp
        }
        if (p.out != OUT_F32) {
          const long long at = (long long)b * p.c_batch + (long long)row0 * p.ldc + n0 + c;
          uint16_t* out = reinterpret_cast<uint16_t*>(p.C) + at;
          if ((p.ldc & 7) == 0) flush_lines(stg, lane, out, p.ldc, rows, (int)p.ldc - n0 - c);
          else flush_ragged(stg, lane, out, p.ldc, rows, p.N - n0 - c);
          if (MODE == MODE_SPLIT) flush_lines(stg2, lane, reinterpret_cast<uint16_t*>(p.lo) + at, p.ldc, rows, (int)p.ldc - n0 - c);
          __syncwarp();
        }
      }
      tc_fence_before();
      mbar_arrive_remote(mapa_u32(&acc_empty[acc], 0));
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

// ------------------------------------------------------------------ norms and the f16 copy
// Two passes over the matrix, 16 bytes a load; the second finds what the first left in L2 (the launcher takes matrices in groups
// that fit).  Squares in 64 bits: no scale of the input overflows or vanishes, and the order of the sum is fixed.
constexpr int NORM_BLOCKS = 512;            // partial sums per matrix at most
constexpr int CAST_THREADS = 256;

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) s += part[i];
  return s;
}

// partial[b][j]: the squares of one of gridDim.x interleaved pieces of matrix b
template <class T>
__global__ void __launch_bounds__(CAST_THREADS) ns_squares_kernel(const T* __restrict__ g, long long n, double* __restrict__ partial) {
  constexpr int VEC = 16 / (int)sizeof(T), UNROLL = 4;
  const T* x = g + (long long)blockIdx.y * n;
  const long long tid = (long long)blockIdx.x * CAST_THREADS + threadIdx.x, step = (long long)gridDim.x * CAST_THREADS;
  const long long nv = (reinterpret_cast<uintptr_t>(x) & 15) == 0 ? n / VEC : 0;
  double s[UNROLL] = {0, 0, 0, 0};
  for (long long v = tid; v < nv; v += step * UNROLL) {
    uint4 raw[UNROLL];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) raw[k] = v + k * step < nv ? __ldg(reinterpret_cast<const uint4*>(x) + v + k * step) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < UNROLL; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) { const double e = (double)to_f32(reinterpret_cast<const T*>(&raw[k])[j]); s[k] = fma(e, e, s[k]); }
  }
  for (long long i = nv * VEC + tid; i < n; i += step) { const double e = (double)to_f32(x[i]); s[0] = fma(e, e, s[0]); }
  const double sum = block_sum((s[0] + s[1]) + (s[2] + s[3]));
  if (threadIdx.x == 0) partial[(long long)blockIdx.y * NORM_BLOCKS + blockIdx.x] = sum;
}

// x [rows, ld] = f16(scale g / |g|), norm[b] = |g|; lo (or null): what the rounding leaves
template <class T>
__global__ void __launch_bounds__(CAST_THREADS) ns_cast_kernel(const T* __restrict__ g, int rows, int cols, const double* __restrict__ partial,
                                                              int parts, float scale, __half* __restrict__ x, __half* __restrict__ lo, int ld,
                                                              double* __restrict__ norm) {
  const int b = blockIdx.y;
  double v = 0;
  for (int i = threadIdx.x; i < parts; i += CAST_THREADS) v += partial[(long long)b * NORM_BLOCKS + i];
  const double whole = sqrt(block_sum(v));
  if (blockIdx.x == 0 && threadIdx.x == 0) norm[b] = whole;
  // the factor as a product of two floats, so that no finite norm takes it out of their range: 2^e times something near `scale`
  const double f = whole == 0.0 ? 0.0 : (double)scale / whole;
  int e = 0;
  const double mant = frexp(f, &e);
  const float f0 = (float)ldexp(mant, e / 2), f1 = (float)ldexp(1.0, e - e / 2);
  const T* src = g + (long long)b * rows * cols;
  __half* dst = x + (long long)b * rows * ld;
  __half* rest = lo ? lo + (long long)b * rows * ld : nullptr;
  const long long n = (long long)rows * cols, step = (long long)gridDim.x * CAST_THREADS;
  if (ld == cols && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {      // no padding: eight elements at a time
    constexpr int LOADS = 8 * (int)sizeof(T) / 16, UNROLL = sizeof(T) == 4 ? 2 : 4;
    const long long nv = n / 8;
    for (long long i = (long long)blockIdx.x * CAST_THREADS + threadIdx.x; i < nv; i += step * UNROLL) {
      uint4 raw[UNROLL][LOADS];
#pragma unroll
      for (int k = 0; k < UNROLL; ++k)
#pragma unroll
        for (int l = 0; l < LOADS; ++l)
          if (i + k * step < nv) raw[k][l] = __ldcs(reinterpret_cast<const uint4*>(src) + (i + k * step) * LOADS + l);
#pragma unroll
      for (int k = 0; k < UNROLL; ++k) {
        if (i + k * step < nv) {
          const T* t = reinterpret_cast<const T*>(&raw[k][0]);
          uint4 o, q;
          __half2 *h = reinterpret_cast<__half2*>(&o), *l = reinterpret_cast<__half2*>(&q);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float a = to_f32(t[2 * j]) * f0 * f1, c = to_f32(t[2 * j + 1]) * f0 * f1;
            h[j] = __floats2half2_rn(a, c);
            l[j] = left_over(h[j], a, c);
          }
          reinterpret_cast<uint4*>(dst)[i + k * step] = o;
          if (rest) reinterpret_cast<uint4*>(rest)[i + k * step] = q;
        }
      }
    }
    return;
  }
  for (int r = blockIdx.x; r < rows; r += gridDim.x)
    for (int c = threadIdx.x; c < cols; c += CAST_THREADS) {
      const float v = to_f32(src[(long long)r * cols + c]) * f0 * f1;
      const __half h = __float2half_rn(v);
      dst[(long long)r * ld + c] = h;
      if (rest) rest[(long long)r * ld + c] = __float2half_rn(v - __half2float(h));
    }
}

// ------------------------------------------------------------------ few rows or columns: everything on chip
// d <= 128 and L <= 4096 (not all of them: `is_small`): one CTA, or a cluster of up to eight with 512 columns each, holds x [128, L]
// (transposed when rows > cols), G and P in shared memory and runs all iterations in one launch; what such sizes cost otherwise is
// launches.  The lower half of x goes through L2: on chip, up to 256 columns a CTA, it was no faster.  x lies as blocks of 128
// rows x 64 columns with 128-byte swizzle, which is the K-major operand of G = x x^T and, read with its columns as N, the MN-major
// one of P x.  Rows and columns beyond the matrix are zero and stay so.  In a cluster each CTA adds up a share of the partial G of
// all, rounds it and hands it round; P is then formed by everyone.  Also the derivative (`apply`): the kept P of every iteration is
// read back.  A wait that runs out sets the status word and the kernel goes on to its end, so that no CTA waits for one that left.
// Five steps with keep and their derivative, here / as products of their own, in us (* : where `is_small` sends them to the products):
//   one matrix                                                                     300 of them
//   16 x 64      23 + 14 / 65 + 23      64 x 256    35 + 22 / 76 + 27               16 x 64     66 + 39 / 330 + 78
//   128 x 256    42 + 25 / 81 + 28      128 x 512   65 + 42 / 86 + 29               128 x 512   209 + 135 / 735 + 306
//   512 x 128    70 + 52 / 86 + 29      64 x 1024   72 + 35 / 91 + 28               64 x 1024   373 + 176 / 1020 + 526
//   128 x 1024   88 + 44 / 97 + 30      128 x 4096  109 + 44 / 149 + 31             128 x 4096  2374 + 953 / 3554 + 1857
//   1024 x 64    78 + 44 / 90 + 28      2048 x 128  103 + 53 / 115 + 30             1024 x 64   400 + 221 / 701 + 282
//   4096 x 16    79 + 40 / 142 + 29     4095 x 127  113 + 53 / 155 + 35             4096 x 128  2425 + 1130 / 2493 + 1246
//   16 x 601     58 + 31 / 83 + 28      30 x 2049   71 + 36 / 112 + 32              30 x 2049   1463 + 719 / 1871 + 1160
//   84 x 915   * 124 + 82 / 102 + 34    100 x 701 * 115 + 73 / 95 + 33              84 x 915    648 + 436 / 1286 + 680
//   127 x 2049 * 136 + 74 / 130 + 35    (16 of 84 x 915 * 126 + 84 / 133 + 58, 32 of them 126 + 85 / 185 + 95)
//                                                                                  127 x 2049 * 2965 + 1645 / 2637 + 1476
// Bound by the latency of its three dependent products a step and, with many matrices, by loading x and by the epilogues.
constexpr int SMALL_D = 128, SMALL_L = 512, SMALL_RANKS = 8, SMALL_THREADS = 512;
constexpr int BLOCK_BYTES = SMALL_D * 128;                     // 128 rows x 64 f16

struct SmallParams {
  const void* in;
  int rows, cols, steps, apply, keep, out, ldd, ranks, slice;      // `slice`: columns of x per CTA, a multiple of 64
  float scale;                 // of the f16 copy
  __half* lo;                  // what the f16 roundings of x leave, pieces of 8 columns with neighbouring rows side by side (null: not kept)
  __half* maps;                // [steps or 1, batch, d, ldd]
  long long map_stride;
  double* norms;               // written by the forward, read by the derivative (null: 1)
  void* y;
  int* status;
  float alpha[MAX_STEPS];      // x' = alpha x + M x with M = P + (a - alpha) I
};

// elements of `lo` per CTA
__host__ __device__ inline long long small_lo(int d, int slice) { return (long long)((d + 31) / 32 * 32) * slice; }
__device__ __forceinline__ int small_offset(int row, int col) {      // bytes; of the 16-byte piece that starts at col
  return (col >> 6) * BLOCK_BYTES + row * 128 + ((((col >> 3) & 7) ^ (row & 7)) * 16);
}
__device__ __forceinline__ void store_small(uint8_t* at, int row, int col, const float (&v)[32]) {      // 32 columns from a multiple of 32
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint4 o;
    __half2* h = reinterpret_cast<__half2*>(&o);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = __floats2half2_rn(v[8 * q + 2 * e], v[8 * q + 2 * e + 1]);
    *reinterpret_cast<uint4*>(at + small_offset(row, col + 8 * q)) = o;
  }
}

// piece of four floats `q` of row `row` of a 128 x 128 f32 matrix, swizzled so that neighbouring rows fall into different banks
__device__ __forceinline__ int part_offset(int row, int q) { return row * 512 + ((q ^ (row & 31)) * 16); }
__device__ __forceinline__ float4 ld_cluster_f32x4(const void* p, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(mapa_u32(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ double ld_cluster_f64(const double* p, int rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(mapa_u32(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster_b128(void* p, int rank, const uint4& v) {
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mapa_u32(p, rank)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

template <class T>
__global__ void __launch_bounds__(SMALL_THREADS, 1) ns_small_kernel(const SmallParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sx = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const bool wide = p.rows <= p.cols;
  const int me = p.ranks > 1 ? (int)cluster_ctarank() : 0, b = blockIdx.x / p.ranks;
  const int d = wide ? p.rows : p.cols, c0 = me * p.slice, L = max(0, min(p.slice, (wide ? p.cols : p.rows) - c0));
  const int Lp = max(64, (L + 63) / 64 * 64);                  // a CTA without columns keeps a block of zeros
  uint8_t* sg = sx + (p.slice / 64) * BLOCK_BYTES;
  uint8_t* sp = sg + 2 * BLOCK_BYTES;                          // P; in a cluster first this CTA's part of G, 128 x 128 f32
  uint64_t* bar = reinterpret_cast<uint64_t*>(sp + (p.ranks > 1 ? 4 : 2) * BLOCK_BYTES);
  double* squares = reinterpret_cast<double*>(bar + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(squares + 1);
  volatile int* abort_word = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t tmem_cols = Lp > 256 ? 512 : Lp > 128 ? 256 : 128;
  if (tid == 0) {
    mbar_init(bar, 1);
    *abort_word = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, tmem_cols);
    tmem_relinquish();
  }
  // the norm, then the scaled f16 copy
  const T* __restrict__ g = reinterpret_cast<const T*>(p.in) + (long long)b * p.rows * p.cols;
  constexpr int VEC = 16 / (int)sizeof(T);
  const bool aligned = (reinterpret_cast<uintptr_t>(g) & 15) == 0;
  const int n = p.rows * p.cols, nv = aligned ? n / VEC : 0;
  double s = 0;
  for (int i = tid + me * 8 * SMALL_THREADS; i < nv; i += 8 * SMALL_THREADS * p.ranks) {
    uint4 raw[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      raw[k] = i + k * SMALL_THREADS < nv ? __ldg(reinterpret_cast<const uint4*>(g) + i + k * SMALL_THREADS) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) { const double e = (double)to_f32(reinterpret_cast<const T*>(&raw[k])[j]); s = fma(e, e, s); }
  }
  for (int i = nv * VEC + tid + me * 8 * SMALL_THREADS; i < n; i += 8 * SMALL_THREADS * p.ranks) {
    float e[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = i + k * SMALL_THREADS < n ? to_f32(g[i + k * SMALL_THREADS]) : 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s = fma((double)e[k], (double)e[k], s);
  }
  s = block_sum(s);
  if (p.ranks > 1) {
    if (tid == 0) *squares = s;
    cluster_sync_all();
    s = 0;
    for (int r = 0; r < p.ranks; ++r) s += ld_cluster_f64(squares, r);      // the same order for all
  }
  const double whole = sqrt(s);
  if (!p.apply && tid == 0 && me == 0) p.norms[b] = whole;
  const double f = whole == 0.0 ? 0.0 : (double)p.scale / whole;
  int ex = 0;
  const double mant = frexp(f, &ex);
  const float f0 = (float)ldexp(mant, ex / 2), f1 = (float)ldexp(1.0, ex - ex / 2);      // two factors: no finite norm leaves their range
  uint4* lo = p.lo ? reinterpret_cast<uint4*>(p.lo + blockIdx.x * small_lo(d, p.slice)) : nullptr;
  const int lo_rows = (d + 31) / 32 * 32;
  // pieces of 8 columns of x, neighbouring threads on neighbouring memory; four of them in flight
  const int pieces = Lp / 8, all = d * pieces;
  for (int i = all + tid; i < SMALL_D * pieces; i += SMALL_THREADS)      // rows beyond the matrix
    *reinterpret_cast<uint4*>(sx + small_offset(i / pieces, i % pieces * 8)) = make_uint4(0, 0, 0, 0);
  for (int i = tid; i < 4 * BLOCK_BYTES / 16; i += SMALL_THREADS) reinterpret_cast<uint4*>(sg)[i] = make_uint4(0, 0, 0, 0);      // of G and P
  const bool vec = wide && aligned && p.cols % 8 == 0;
  for (int i0 = tid; i0 < all; i0 += 4 * SMALL_THREADS) {
    float x[4][8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + k * SMALL_THREADS;
      const int row = wide ? i / pieces : i % d, col = (wide ? i % pieces : i / d) * 8;
      const bool rows_in = i < all;
      if (vec) {
        uint4 raw[8 / VEC];
#pragma unroll
        for (int l = 0; l < 8 / VEC; ++l)
          raw[l] = rows_in && col < L ? __ldg(reinterpret_cast<const uint4*>(g + row * p.cols + c0 + col) + l) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[k][e] = to_f32(reinterpret_cast<const T*>(raw)[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[k][e] = rows_in && col + e < L ? to_f32(g[wide ? row * p.cols + c0 + col + e : (c0 + col + e) * p.cols + row]) : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int i = i0 + k * SMALL_THREADS;
      const int row = wide ? i / pieces : i % d, col = (wide ? i % pieces : i / d) * 8;
      uint4 o, w;
      __half2 *h = reinterpret_cast<__half2*>(&o), *l = reinterpret_cast<__half2*>(&w);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = x[k][2 * e] * f0 * f1, c = x[k][2 * e + 1] * f0 * f1;
        h[e] = __floats2half2_rn(a, c);
        l[e] = left_over(h[e], a, c);
      }
      if (i < all) {
        *reinterpret_cast<uint4*>(sx + small_offset(row, col)) = o;
        if (lo) lo[(col >> 3) * lo_rows + row] = w;
      }
    }
  }
  float last = 1.f / p.scale;                                  // brings the last product to the result's scale
  bool none = false;                                           // a zero matrix has a zero derivative, whatever the cotangent
  if (p.apply) { const double n = p.norms ? p.norms[b] : 1.0; none = n == 0.0; last = (float)(whole / n / (double)p.scale); }
  tc_fence_before();
  fence_async_proxy();                                         // the tensor core reads what these threads wrote
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int quarter = warp & 3, part = warp >> 2, row = quarter * 32 + lane;
  const bool rows_here = quarter * 32 < d;                      // the others stay zero
  const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
  uint32_t phase = 0;
  // one product: issued by thread 0, waited for by all
  auto wait = [&]() {
    mbar_wait_bounded(bar, phase, abort_word, p.status, ERR_WAIT_TMEM_FULL);
    phase ^= 1;
    __syncthreads();
    tc_fence_after();
  };
  auto hand_over = [&]() {                                     // accumulators read, operands written: the next product may start
    tc_fence_before();
    fence_async_proxy();
    __syncthreads();
    tc_fence_after();
  };
  // the kept P, [d, ldd], as rows of 16-byte pieces; the derivative takes them from the last to the first, each read a step ahead
  constexpr int KEPT = SMALL_D * SMALL_D / 8 / SMALL_THREADS;
  const int kept_pieces = p.ldd / 8;
  auto map_of = [&](int k) { return p.maps + k * p.map_stride + (long long)b * d * p.ldd; };
  uint4 next[KEPT];                                            // (or, in the forward, what the rounding of x left)
  auto fetch = [&](int k) {
    const __half* map = map_of(p.steps - 1 - k);
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
      const int at = tid + i * SMALL_THREADS, r = at / (SMALL_D / 8), q = at % (SMALL_D / 8);
      next[i] = r < d && q < kept_pieces ? reinterpret_cast<const uint4*>(map + r * p.ldd)[q] : make_uint4(0, 0, 0, 0);
    }
  };
  if (p.apply) fetch(0);
  for (int k = 0; k < p.steps; ++k) {
    const float alpha = p.alpha[p.apply ? p.steps - 1 - k : k];
    if (!p.apply) {
      if (tid == 0) {
        const uint32_t a = smem_u32(sx), idesc = make_idesc_f16(128, 128, 0, 0);
        for (int i = 0; i < Lp / 16; ++i) {
          const uint64_t desc = make_smem_desc(a + (i >> 2) * BLOCK_BYTES + (i & 3) * 32, 16, 1024);
          umma_f16(tmem, desc, desc, idesc, i > 0);
        }
        umma_commit(bar);
      }
      wait();
      float gr[32];                                            // this thread's entries of G
      if (rows_here) {
        uint32_t r[32];
        tmem_ld_32x32(lanes + part * 32, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float v = __uint_as_float(r[j]) * (1.f / X_SCALE);
          gr[j] = p.ranks == 1 ? __half2float(__float2half_rn(v)) : v;      // one G, rounded, for both terms
        }
        if (p.ranks == 1) {
          store_small(sg, row, part * 32, gr);
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            *reinterpret_cast<float4*>(sp + part_offset(row, part * 8 + q)) = make_float4(gr[4 * q], gr[4 * q + 1], gr[4 * q + 2], gr[4 * q + 3]);
        }
      }
      if (p.ranks > 1) {
        tc_fence_before();
        cluster_sync_all();
        // this CTA's share of the rows: summed over the parts in order, to everyone's G
        const int share = SMALL_D / p.ranks, live = (d + 31) / 32 * 32;
        for (int i = tid; i < share * 16; i += SMALL_THREADS) {
          const int r = me * share + i / 16, q = i % 16;
          if (r >= live) continue;
          float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 1
          for (int k0 = 0; k0 < p.ranks; k0 += 2) {            // two or more; four loads in flight
            const float4 a0 = ld_cluster_f32x4(sp + part_offset(r, 2 * q), k0), a1 = ld_cluster_f32x4(sp + part_offset(r, 2 * q + 1), k0);
            const float4 b0 = ld_cluster_f32x4(sp + part_offset(r, 2 * q), k0 + 1), b1 = ld_cluster_f32x4(sp + part_offset(r, 2 * q + 1), k0 + 1);
            v[0] += a0.x + b0.x; v[1] += a0.y + b0.y; v[2] += a0.z + b0.z; v[3] += a0.w + b0.w;
            v[4] += a1.x + b1.x; v[5] += a1.y + b1.y; v[6] += a1.z + b1.z; v[7] += a1.w + b1.w;
          }
          uint4 o;
          __half2* h = reinterpret_cast<__half2*>(&o);
#pragma unroll
          for (int e = 0; e < 4; ++e) h[e] = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
          for (int k2 = 0; k2 < p.ranks; ++k2) st_cluster_b128(sg + small_offset(r, q * 8), k2, o);
        }
        asm volatile("fence.proxy.async;" ::: "memory");       // the tensor cores of all read what these threads wrote
        cluster_sync_all();
        tc_fence_after();
        if (rows_here) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint4 o = *reinterpret_cast<const uint4*>(sg + small_offset(row, part * 32 + q * 8));
            const __half* h = reinterpret_cast<const __half*>(&o);
#pragma unroll
            for (int e = 0; e < 8; ++e) gr[8 * q + e] = __half2float(h[e]);
          }
        }
      }
      hand_over();
      if (tid == 0) {
        const uint32_t a = smem_u32(sg), idesc = make_idesc_f16(128, 128, 0, 0);
        for (int i = 0; i < 8; ++i) {
          const uint64_t desc = make_smem_desc(a + (i >> 2) * BLOCK_BYTES + (i & 3) * 32, 16, 1024);
          umma_f16(tmem, desc, desc, idesc, i > 0);
        }
        umma_commit(bar);
      }
      wait();
      if (rows_here) {
        uint32_t r[32];
        tmem_ld_32x32(lanes + part * 32, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 32; ++j)
          gr[j] = fmaf(NS_B, gr[j], NS_C / X_SCALE * __uint_as_float(r[j])) + (row == part * 32 + j ? (NS_A - alpha) * X_SCALE : 0.f);
        store_small(sp, row, part * 32, gr);
      }
    } else {
#pragma unroll
      for (int i = 0; i < KEPT; ++i) {
        const int at = tid + i * SMALL_THREADS;
        *reinterpret_cast<uint4*>(sp + small_offset(at / (SMALL_D / 8), at % (SMALL_D / 8) * 8)) = next[i];
      }
      if (k + 1 < p.steps) fetch(k + 1);
    }
    hand_over();
    if (tid == 0) {
      const uint32_t a = smem_u32(sp), x = smem_u32(sx);
      for (int n0 = 0; n0 < Lp; n0 += 256) {
        const int n = min(256, Lp - n0);
        const uint32_t idesc = make_idesc_f16(128, n, 0, 1);
        for (int i = 0; i < 8; ++i)
          umma_f16(tmem + n0, make_smem_desc(a + (i >> 2) * BLOCK_BYTES + (i & 3) * 32, 16, 1024),
                   make_smem_desc(x + (n0 >> 6) * BLOCK_BYTES + i * (UMMA_K * 128), BLOCK_BYTES, 1024), idesc, i > 0);
      }
      umma_commit(bar);
    }
    if (!p.apply && p.keep)                                    // while the product runs; the padding of P is zero
      for (int i = tid + me * SMALL_THREADS; i < d * kept_pieces; i += SMALL_THREADS * p.ranks) {
        const int r = i / kept_pieces, q = i % kept_pieces;
        reinterpret_cast<uint4*>(map_of(k) + r * p.ldd)[q] = *reinterpret_cast<const uint4*>(sp + small_offset(r, q * 8));
      }
    // what the rounding of x left, of the columns that come first: this thread's own stores, or those before the first product
    const bool end = k == p.steps - 1, has_lo = lo && row < d && !end;
    static_assert(KEPT == 4, "32 columns of the low half");
    auto fetch_lo = [&](int col) {
#pragma unroll
      for (int q = 0; q < 4; ++q) next[q] = has_lo ? lo[((col >> 3) + q) * lo_rows + row] : make_uint4(0, 0, 0, 0);
    };
    if (!p.apply && part * 32 < Lp) fetch_lo(part * 32);
    wait();
    const float fx = (end ? last : 1.f) * alpha, fr = (end ? last : 1.f) / X_SCALE;
    for (int col = rows_here ? part * 32 : Lp; col < Lp; col += 128) {
      uint32_t r[32];
      tmem_ld_32x32(lanes + col, r);
      tmem_ld_wait();
      float v[32];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint4 o = *reinterpret_cast<const uint4*>(sx + small_offset(row, col + 8 * q));
        const __half *h = reinterpret_cast<const __half*>(&o), *l = reinterpret_cast<const __half*>(&next[q]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[8 * q + e] = fmaf(fx, __half2float(h[e]), __uint_as_float(r[8 * q + e]) * fr);
          if (!p.apply) v[8 * q + e] = fmaf(NS_A, __half2float(l[e]), v[8 * q + e]);
        }
      }
      if (!p.apply && col + 128 < Lp) fetch_lo(col + 128);
      if (none && end) {
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = 0.f;
      }
      if (!end && has_lo && k < p.steps - 2) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint4 o, w;
          __half2 *h = reinterpret_cast<__half2*>(&o), *l = reinterpret_cast<__half2*>(&w);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float a = v[8 * q + 2 * e], c = v[8 * q + 2 * e + 1];
            h[e] = __floats2half2_rn(a, c);
            l[e] = left_over(h[e], a, c);
          }
          *reinterpret_cast<uint4*>(sx + small_offset(row, col + 8 * q)) = o;
          lo[((col >> 3) + q) * lo_rows + row] = w;
        }
      } else if (!end) {
        store_small(sx, row, col, v);
      } else if (row < d && wide && p.out == OUT_BF16 && p.cols % 8 == 0) {
        uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.y) + (long long)b * n + row * p.cols + c0 + col);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint4 w;
          __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
          for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(v[8 * q + 2 * e], v[8 * q + 2 * e + 1]);
          if (col + 8 * q < L) o[q] = w;
        }
      } else if (row < d) {
        const long long base = (long long)b * n;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (col + j < L) {
            const long long o = base + (wide ? (long long)row * p.cols + c0 + col + j : (long long)(c0 + col + j) * p.cols + row);
            if (p.out == OUT_F32) reinterpret_cast<float*>(p.y)[o] = v[j];
            else reinterpret_cast<__nv_bfloat16*>(p.y)[o] = __float2bfloat16(v[j]);
          }
      }
    }
    hand_over();
  }
  tc_fence_before();
  if (p.ranks > 1) cluster_sync_all();                         // nobody leaves while a peer may still reach in
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

// Which matrices take one launch: all up to 128 x 512 or 512 x 128, all tall ones up to 4096 x 128, and wide ones up to 128 x 4096 whose
// rows start at 16 bytes.  The rows of other wide ones beyond 512 columns come element by element into every CTA of a cluster, which is
// made up for where there are few of them (d <= 64) or where many matrices of at most two CTAs each share the device; so the same
// matrix may take either way, and round differently, by the size of its batch.
static bool is_small(int batch, int rows, int cols) {
  const int d = rows < cols ? rows : cols, L = rows < cols ? cols : rows;
  if (d > SMALL_D || L > SMALL_L * SMALL_RANKS) return false;
  return L <= SMALL_L || rows > cols || cols % 8 == 0 || d <= 64 || (batch >= 24 && L <= 2 * SMALL_L);
}
static constexpr int small_smem(int slice, int ranks) { return (slice / 64 + (ranks > 1 ? 6 : 4)) * BLOCK_BYTES + 2048; }
static_assert(small_smem(SMALL_L, SMALL_RANKS) + 256 <= 227 * 1024, "shared memory of an SM");

static void small_split(int rows, int cols, int* ranks, int* slice) {
  const int L = rows < cols ? cols : rows;
  *ranks = 1;
  while (*ranks * SMALL_L < L) *ranks *= 2;
  *slice = ((L + *ranks - 1) / *ranks + 63) / 64 * 64;
}

static int launch_small(SmallParams p, int f32, int batch, cudaStream_t stream) {
  small_split(p.rows, p.cols, &p.ranks, &p.slice);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(batch * p.ranks);
  cfg.blockDim = dim3(SMALL_THREADS);
  cfg.dynamicSmemBytes = small_smem(p.slice, p.ranks);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = f32 ? cudaLaunchKernelEx(&cfg, ns_small_kernel<float>, p) : cudaLaunchKernelEx(&cfg, ns_small_kernel<__nv_bfloat16>, p);
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  });
  return fn;
}

// A stored f16 matrix [rows, cols] per batch entry, rows `ld` apart.
struct Mat {
  const void* ptr;
  int rows, cols;
  long long ld;
};

// `mn`: the operand's rows run along the contraction (its M or N index is contiguous); the box is then 64 x BK, else BK x box_rows.
static int encode_map(CUtensorMap* map, const Mat& m, int batch, bool mn, int box_rows) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return 101;
  cuuint64_t dims[3] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows, (cuuint64_t)batch};
  cuuint64_t strides[2] = {(cuuint64_t)m.ld * 2, (cuuint64_t)m.ld * m.rows * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)(mn ? BK : box_rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  if (int c = check_map(m.ptr, 3, dims, strides, 2)) return c;
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(m.ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 200 + (int)r;
}

// One call's tensor maps: its products use the same few buffers again and again, and encoding a map takes the host a microsecond.
struct Maps {
  struct Entry { Mat m; bool mn; int box_rows; CUtensorMap map; } e[24];
  int n = 0;
  int get(const CUtensorMap** out, const Mat& m, int batch, bool mn, int box_rows) {
    for (int i = 0; i < n; ++i)
      if (e[i].m.ptr == m.ptr && e[i].m.rows == m.rows && e[i].m.cols == m.cols && e[i].m.ld == m.ld && e[i].mn == mn &&
          (mn || e[i].box_rows == box_rows)) { *out = &e[i].map; return 0; }
    const int at = n < 24 ? n++ : 23;                        // more than there is room for (kept maps of many steps): the last is replaced
    if (int r = encode_map(&e[at].map, m, batch, mn, box_rows)) return r;
    e[at].m = m; e[at].mn = mn; e[at].box_rows = box_rows;
    *out = &e[at].map;
    return 0;
  }
};

struct ProductKernel {
  void (*kernel)(const CUtensorMap, const CUtensorMap, const Params);
  int smem;
};
template <int BN, int MODE> constexpr ProductKernel product_kernel() { return {ns_product_kernel<BN, MODE>, Tile<BN, MODE>::SMEM}; }
static const ProductKernel wide_kernels[4] = {product_kernel<256, 0>(), product_kernel<256, 1>(), product_kernel<256, 2>(), product_kernel<256, 3>()};
static const ProductKernel narrow_kernels[4] = {product_kernel<128, 0>(), product_kernel<128, 1>(), product_kernel<128, 2>(), product_kernel<128, 3>()};

static int prepare_device(int* n_sm) {
  static std::mutex mu;
  static unsigned long long attr_mask = 0;
  static int sms[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 301;
  static thread_local int bound_dev = -1;
  // The encoder needs a current context, which cudaSetDevice makes.  (cudaFree(0) would too, but a thread's first call may lie inside a
  // capture, autograd's for a captured backward say, and ends that.)
  if (bound_dev != dev) { if (cudaSetDevice(dev) != cudaSuccess) return 301; bound_dev = dev; }
  std::lock_guard<std::mutex> lock(mu);
  if (!(attr_mask >> dev & 1ull)) {
    for (int k = 0; k < 4; ++k)
      if (cudaFuncSetAttribute(wide_kernels[k].kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, wide_kernels[k].smem) != cudaSuccess ||
          cudaFuncSetAttribute(narrow_kernels[k].kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, narrow_kernels[k].smem) != cudaSuccess) return 302;
    if (cudaFuncSetAttribute(ns_small_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, small_smem(SMALL_L, SMALL_RANKS)) != cudaSuccess ||
        cudaFuncSetAttribute(ns_small_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, small_smem(SMALL_L, SMALL_RANKS)) != cudaSuccess) return 302;
    cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
    attr_mask |= 1ull << dev;
  }
  *n_sm = sms[dev] > 1 ? sms[dev] : 148;
  return 0;
}

struct Out {
  void* C;
  int kind;
  long long ld;
  const double *num, *den;
  void* lo = nullptr;          // with D2: takes what the rounding of C leaves
};

// C [M, N] = alpha op(A) op(B) + beta D (+ beta2 D2, with the layout of D) + diag I over the batch (symmetric: C and D are, and only f16)
static int product(Maps& maps, int batch, int M, int N, int K, const Mat& A, bool a_mn, const Mat& B, bool b_mn, float alpha, float beta, const Mat* D,
                   const Out& o, bool symmetric, int* status, int n_sm, cudaStream_t stream, const Mat* D2 = nullptr, float beta2 = 0.f,
                   float diag = 0.f) {
  Params p;
  memset(&p, 0, sizeof(p));
  p.M = M; p.N = N; p.K = K; p.batch = batch; p.a_mn_major = a_mn; p.b_mn_major = b_mn; p.alpha = alpha; p.beta = beta;
  if (D) { p.D = (const __half*)D->ptr; p.ldd = D->ld; p.d_batch = D->ld * D->rows; }
  if (D2) { p.D2 = (const __half*)D2->ptr; p.beta2 = beta2; }
  p.diag = diag;
  p.lo = (__half*)o.lo;
  p.C = o.C; p.out = o.kind; p.ldc = o.ld; p.c_batch = o.ld * M; p.num = o.num; p.den = o.den; p.status = status;
  p.symmetric = symmetric;
  p.tiles_m = (M + 2 * BM - 1) / (2 * BM);
  // Tiles of 256 or of 128 columns: whichever needs less time for its rounds over the pairs of SMs.  A narrow tile's k-block takes
  // 0.62 of a wide one's (it moves 3/4 of the bytes for half the products), its share outside the main loop about half.
  const int pairs = n_sm / 2, kb = (K + BK - 1) / BK;
  long long tiles[2];
  double cost[2];
  for (int i = 0; i < 2; ++i) {
    p.tiles_n = (N + (256 >> i) - 1) / (256 >> i);
    tiles[i] = (long long)batch * tiles_per_matrix(p, 1 << i);
    cost[i] = (double)((tiles[i] + pairs - 1) / pairs) * (kb * (i ? 0.62 : 1.0)) + (i ? 15 : 30);
  }
  const int narrow = cost[1] < cost[0];
  p.tiles_n = (N + (256 >> narrow) - 1) / (256 >> narrow);
  if (tiles[narrow] > 0x3fffffff) return 303;
  const CUtensorMap *mapA, *mapB;
  CUtensorMap copyA;                                           // a later lookup may replace an entry
  if (int r = maps.get(&mapA, A, batch, a_mn, BM)) return r;
  copyA = *mapA;
  if (int r = maps.get(&mapB, B, batch, b_mn, narrow ? 64 : 128)) return r;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (int)(tiles[narrow] < pairs ? tiles[narrow] : pairs));
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;      // the prologue overlaps the product before
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int mode = o.lo ? MODE_SPLIT : D2 ? MODE_SUM : diag != 0.f ? MODE_DIAG : MODE_PLAIN;
  const ProductKernel& k = (narrow ? narrow_kernels : wide_kernels)[mode];
  cfg.dynamicSmemBytes = k.smem;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k.kernel, copyA, *mapB, p);
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}

// r (f16) -> beta r + alpha M r (r M^T of a tall one), or with the transpose of M, + beta2 D2: into f16 or, at the end, into the caller's
// tensor
static int apply(Maps& maps, int batch, int rows, int cols, const Mat& r, const Mat& M, bool transposed, float alpha, float beta, const Out& o, int* status,
                 int n_sm, cudaStream_t stream, const Mat* D2 = nullptr, float beta2 = 0.f) {
  if (rows <= cols) return product(maps, batch, rows, cols, rows, M, transposed, r, true, alpha, beta, &r, o, false, status, n_sm, stream, D2, beta2);
  return product(maps, batch, rows, cols, cols, r, false, M, transposed, alpha, beta, &r, o, false, status, n_sm, stream, D2, beta2);
}

// Matrices of `bytes` each whose two passes run together: about 48 MB, so that the second reads them from L2 (126 MB) while the f16
// copies are written.
static int cast_group(long long bytes) { return (int)(bytes > (48ll << 20) ? 1 : (48ll << 20) / bytes); }

template <class T>
static int cast(const T* g, int batch, int rows, int cols, double* partial, float scale, __half* x, __half* lo, int ld, double* norm, int n_sm,
                cudaStream_t stream) {
  const long long n = (long long)rows * cols, bytes = n * (long long)sizeof(T);
  auto blocks = [](long long work, long long each, int most) { const long long w = (work + each - 1) / each; return (int)(w < most ? w : most); };
  const int parts = blocks(n, 8192, NORM_BLOCKS);
  const int casts = ld == cols ? blocks(n, 4096, 8 * n_sm) : blocks(rows, 1, 8 * n_sm);
  const int group = cast_group(bytes);
  for (int b = 0; b < batch; b += group) {
    const int k = batch - b < group ? batch - b : group;
    double* part = partial + (long long)b * NORM_BLOCKS;
    ns_squares_kernel<T><<<dim3(parts, k), CAST_THREADS, 0, stream>>>(g + b * n, n, part);
    ns_cast_kernel<T><<<dim3(casts, k), CAST_THREADS, 0, stream>>>(g + b * n, rows, cols, part, parts, scale, x + (long long)b * rows * ld,
                                                                  lo ? lo + (long long)b * rows * ld : nullptr, ld, norm + b);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}

static int cast(const void* g, int f32, int batch, int rows, int cols, double* partial, float scale, void* x, void* lo, int ld, double* norm, int n_sm,
                cudaStream_t stream) {
  if (f32) return cast<float>((const float*)g, batch, rows, cols, partial, scale, (__half*)x, (__half*)lo, ld, norm, n_sm, stream);
  return cast<__nv_bfloat16>((const __nv_bfloat16*)g, batch, rows, cols, partial, scale, (__half*)x, (__half*)lo, ld, norm, n_sm, stream);
}

}  // namespace ns
}  // namespace dttt

namespace dttt {
namespace ns {

// How the iterations are grouped.  Two of them in one,
//   x'' = (a I + P')(a I + P) x = (a^2 - s) x + N x,   N = P' P + a (P + P') + s I,
// need G' of the second from G alone: with H = (a I + P) G = a G + P G, G' = a H + H P.  That replaces one product with x on each side
// of the group (d^2 L and 2 d^2 L of the longer side L) by three d x d ones, which pays from about L = 2 d on where the products are
// large enough to be bound by the tensor cores: 4 x 2048 x 8192, five steps, 2.36 -> 1.77 ms.  `s` shifts N by its value at the singular
// value of a matrix with equal ones, so that what rounds is the spread and not the bulk of it.  Single ones are shifted likewise:
// unshifted, 2.7 I next to a result of 0.7 rounds (101 x 346, five steps: 1.5e-3 off before the rounding to bf16 instead of 1.1e-3).
// With s = b^2 / 4c, P + s I would be the one product c (G + b / 2c I)^2: 170 instead of 173 us for 1000 x 1024, but 2.34e-3 off
// instead of 2.06e-3.  P, P' and G commute only up to their roundings: G' is formed as H P, which is symmetric even so (P H, or N mirrored across its diagonal, is not, and the
// difference is amplified: 5.2e-3 and 2.5e-3 off instead of 2.2e-3).  The first two and, from five on, the last two are grouped; a
// pair in the middle, or three in one, loses to the cancellation in N what single steps keep.
struct Group {
  int steps;
  float alpha, shift;          // x' = alpha x + M x
};

static int make_plan(int rows, int cols, int steps, Group* g) {
  const double d = rows < cols ? rows : cols, len = rows < cols ? cols : rows;
  const bool pairs = d >= 512 && len >= 2 * d;
  auto q = [](double l) { return (double)NS_A + NS_B * l + NS_C * l * l; };
  double l = 1.0 / d;
  int n = 0;
  for (int k = 0; k < steps; ++n) {
    const bool two = pairs && ((k == 0 && steps >= 2) || (k == steps - 2 && k >= 3));
    const double next = l * q(l) * q(l);
    if (two) {
      g[n] = {2, (float)(q(l) * q(next)), (float)((double)NS_A * NS_A - q(l) * q(next))};
      l = next * q(next) * q(next);
      k += 2;
    } else {
      g[n] = {1, (float)q(l), (float)(NS_A - q(l))};
      l = next;
      k += 1;
    }
  }
  return n;
}

struct Scratch {
  void *x[2], *lo, *gram, *h, *p;
  double *partial, *norm;
  long long bytes;
  int ld, d, ldd;
  Scratch(void* base, int batch, int rows, int cols) {
    auto up = [](long long v) { return (v + 255) / 256 * 256; };
    ld = (cols + 7) / 8 * 8; d = rows < cols ? rows : cols; ldd = (d + 7) / 8 * 8;
    const long long xb = up((long long)batch * rows * ld * 2), gb = up((long long)batch * d * ldd * 2);
    uint8_t* s = (uint8_t*)base;
    auto take = [&](long long n) { uint8_t* r = s; s += n; return r; };
    x[0] = take(xb); x[1] = take(xb); lo = take(xb);
    gram = take(gb); h = take(gb); p = take(gb);
    partial = (double*)take(up((long long)batch * NORM_BLOCKS * 8));
    norm = (double*)take(up((long long)batch * 8));
    bytes = s - (uint8_t*)base;
  }
};

}  // namespace ns
}  // namespace dttt

// Bytes of the scratch area for `batch` matrices [rows, cols] (256-byte aligned base).
extern "C" long long dttt_newton_schulz_scratch(int batch, int rows, int cols) {
  using namespace dttt::ns;
  if (!is_small(batch, rows, cols)) return Scratch(nullptr, batch, rows, cols).bytes;
  int ranks, slice;
  small_split(rows, cols, &ranks, &slice);
  return batch * (long long)ranks * small_lo(rows < cols ? rows : cols, slice) * 2;      // (of the forward)
}

// Kernels that a forward (`parts` 0) or a part of `parts` groups of the derivative launches.
extern "C" int dttt_newton_schulz_launches(int f32, int batch, int rows, int cols, int steps, int parts) {
  using namespace dttt::ns;
  if (batch <= 0 || rows <= 0 || cols <= 0 || steps <= 0 || steps > MAX_STEPS) return 0;
  if (is_small(batch, rows, cols)) return 1;
  const int group = cast_group((long long)rows * cols * (f32 ? 4 : 2)), casts = 2 * ((batch + group - 1) / group);
  if (parts) return casts + parts;
  Group plan[MAX_STEPS];
  int n = casts;
  for (int k = make_plan(rows, cols, steps, plan) - 1; k >= 0; --k) n += plan[k].steps == 1 ? 3 : 7;
  return n;
}

// Groups of iterations, each with one d x d matrix of the linear map.
extern "C" int dttt_newton_schulz_groups(int rows, int cols, int steps) {
  dttt::ns::Group g[dttt::ns::MAX_STEPS];
  return steps <= 0 || steps > dttt::ns::MAX_STEPS ? 0 : dttt::ns::make_plan(rows, cols, steps, g);
}

// g [batch, rows, cols] (f32 or bf16, contiguous) -> y bf16.  kept: f16 [groups or 1, batch, d, ceil8(d)]; with keep every group's
// matrix stays there for the backward, else one slot is used again and again.  norms: f64 [batch].
extern "C" int dttt_newton_schulz(const void* g, int f32, int batch, int rows, int cols, int steps, void* scratch, void* kept, int keep,
                                  double* norms, void* y, int* status, cudaStream_t stream) {
  using namespace dttt::ns;
  if (batch <= 0 || rows <= 0 || cols <= 0 || steps <= 0 || steps > MAX_STEPS || batch > 65535) return -2;
  int n_sm;
  if (int r = prepare_device(&n_sm)) return r;
  Group plan[MAX_STEPS];
  const int groups = make_plan(rows, cols, steps, plan);
  if (is_small(batch, rows, cols)) {
    const int small = rows < cols ? rows : cols, ld = (small + 7) / 8 * 8;
    SmallParams p = {g, rows, cols, steps, 0, keep, OUT_BF16, ld, 1, 0, X_SCALE, steps > 1 ? (__half*)scratch : nullptr, (__half*)kept,
                     (long long)batch * small * ld, norms, y, status};
    for (int k = 0; k < steps; ++k) p.alpha[k] = plan[k].alpha;
    return launch_small(p, f32, batch, stream);
  }
  const Scratch s(scratch, batch, rows, cols);
  const int d = s.d, ldd = s.ldd;
  if (int r = cast(g, f32, batch, rows, cols, s.partial, X_SCALE, s.x[0], groups > 1 ? s.lo : nullptr, s.ld, norms, n_sm, stream)) return r;
  const bool wide = rows <= cols;
  Maps maps;
  const Mat G = {s.gram, d, d, ldd}, H = {s.h, d, d, ldd}, P1 = {s.p, d, d, ldd}, Lo = {s.lo, rows, cols, s.ld};
  auto square = [&](const Mat& A, const Mat& B, float alpha, float beta, const Mat& D, const Mat& C, const Mat* D2 = nullptr, float beta2 = 0.f,
                    float diag = 0.f) {
    const Out o = {const_cast<void*>(C.ptr), OUT_F16, ldd, nullptr, nullptr};
    return product(maps, batch, d, d, d, A, false, B, false, alpha / X_SCALE, beta, &D, o, D2 == nullptr, status, n_sm, stream, D2, beta2, diag);
  };
  for (int k = 0; k < groups; ++k) {
    const Mat X = {s.x[k & 1], rows, cols, s.ld};
    const Mat M = {(uint8_t*)kept + (keep ? (long long)k * batch * d * ldd * 2 : 0), d, d, ldd};
    const Out og = {s.gram, OUT_F16, ldd, nullptr, nullptr};
    if (int r = product(maps, batch, d, d, wide ? cols : rows, X, !wide, X, !wide, 1.f / X_SCALE, 0.f, nullptr, og, true, status, n_sm, stream)) return r;
    if (plan[k].steps == 1) {
      if (int r = square(G, G, NS_C, NS_B, G, M, nullptr, 0.f, plan[k].shift * X_SCALE)) return r;      // M = b G + c G G + s I
    } else {
      if (int r = square(G, G, NS_C, NS_B, G, P1)) return r;
      if (int r = square(P1, G, 1.f, NS_A, G, H)) return r;                                  // H = a G + P G
      if (int r = square(H, P1, 1.f, NS_A, H, G)) return r;                                  // G' = a H + H P
      if (int r = square(G, G, NS_C, NS_B, G, H)) return r;                                  // P'
      if (int r = square(H, P1, 1.f, NS_A, P1, M, &H, NS_A, plan[k].shift * X_SCALE)) return r;      // N = P' P + a P + a P' + s I
    }
    const bool last = k == groups - 1;
    const float f = last ? 1.f / X_SCALE : 1.f;
    // The last group goes without the low half: what x_k lost grows only by this group's factor there (3.4445, or 11.9 of a pair, times
    // 2.8e-4), and a third of the traffic is saved.
    const Out ox = {last ? y : s.x[(k + 1) & 1], last ? OUT_BF16 : OUT_F16, last ? cols : s.ld, nullptr, nullptr, k < groups - 2 ? s.lo : nullptr};
    const float beta2 = plan[k].alpha + plan[k].shift;
    if (int r = apply(maps, batch, rows, cols, X, M, false, f / X_SCALE, f * plan[k].alpha, ox, status, n_sm, stream, last ? nullptr : &Lo, beta2)) return r;
  }
  return 0;
}

// The derivative is applied in parts of at most PART_STEPS iterations, the last groups first, each a call with the result of the one
// before (f32): the first group of the part that ends before group `upto`.
extern "C" int dttt_newton_schulz_part(int rows, int cols, int steps, int upto) {
  using namespace dttt::ns;
  if (steps <= PART_STEPS || steps > MAX_STEPS) return 0;
  Group plan[MAX_STEPS];
  const int groups = make_plan(rows, cols, steps, plan);
  int k = upto < groups ? upto : groups, sum = 0;
  while (k > 0 && sum + plan[k - 1].steps <= PART_STEPS) sum += plan[--k].steps;
  return k;
}

// r [batch, rows, cols] (f32 or bf16) -> out (f32 or bf16) = prod_{k in first .. upto - 1} (alpha_k I + M_k)^T r / norms (null: 1), the
// maps of a forward with keep.
extern "C" int dttt_newton_schulz_apply(const void* r_in, int f32, int batch, int rows, int cols, int steps, int first, int upto, void* scratch,
                                        const void* kept, const double* norms, void* out, int out_f32, int* status, cudaStream_t stream) {
  using namespace dttt::ns;
  if (batch <= 0 || rows <= 0 || cols <= 0 || steps <= 0 || steps > MAX_STEPS || batch > 65535) return -2;
  int n_sm;
  if (int r = prepare_device(&n_sm)) return r;
  Group plan[MAX_STEPS];
  const int groups = make_plan(rows, cols, steps, plan), count = upto - first;
  if (first < 0 || count <= 0 || upto > groups) return -2;
  if (is_small(batch, rows, cols)) {
    const int small = rows < cols ? rows : cols, ld = (small + 7) / 8 * 8;
    const long long stride = (long long)batch * small * ld;
    SmallParams p = {r_in, rows, cols, count, 1, 1, out_f32 ? OUT_F32 : OUT_BF16, ld, 1, 0, R_SCALE, nullptr,
                     (__half*)const_cast<void*>(kept) + first * stride, stride, const_cast<double*>(norms), out, status};
    for (int k = 0; k < count; ++k) p.alpha[k] = plan[first + k].alpha;
    return launch_small(p, f32, batch, stream);
  }
  const Scratch s(scratch, batch, rows, cols);
  if (int r = cast(r_in, f32, batch, rows, cols, s.partial, R_SCALE, s.x[0], nullptr, s.ld, s.norm, n_sm, stream)) return r;
  Maps maps;
  for (int i = 0; i < count; ++i) {
    const int k = upto - 1 - i;
    const Mat X = {s.x[i & 1], rows, cols, s.ld};
    const Mat M = {(const uint8_t*)kept + (long long)k * batch * s.d * s.ldd * 2, s.d, s.d, s.ldd};
    const bool last = k == first;
    const float f = last ? 1.f / R_SCALE : 1.f;
    const Out o = {last ? out : s.x[(i + 1) & 1], last ? (out_f32 ? OUT_F32 : OUT_BF16) : OUT_F16, last ? cols : s.ld, last ? s.norm : nullptr,
                   last ? norms : nullptr};
    if (int r = apply(maps, batch, rows, cols, X, M, true, f / X_SCALE, f * plan[k].alpha, o, status, n_sm, stream)) return r;
  }
  return 0;
}
