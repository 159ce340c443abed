// Decoding a block: one token for every slot from its logits, and the commit of the surest slots.
//
//   sample   per row of logits x [V] (x = fl32(logit + bias), bias per sequence), with m = max x:
//              logp     = x_tok - m - log sum_i exp(x_i - m)                       (untempered, the whole vocabulary)
//              priority = logp | p_(1) - p_(2) | sum_i p_i log p_i
//              w_i      = exp((x_i - m) / T), order: x descending, index ascending
//              kept     = the first top_k; of those the shortest prefix of mass >= top_p * mass(first top_k);
//                         of those w_i >= min_p
//              token    = first kept i in index order with w_0 + .. + w_i > u * (mass of the kept)
//            T <= 0: the lowest index of the maximum (T > 0 is clamped to [1e-6, 1e6]).  A row that holds NaN or +inf, or nothing above -inf, has no
//            distribution: token -1, logp and priority NaN.
//   unmask   per row of C slots: where = (rank by (priority descending, NaN last, slot ascending; closed slots as -inf) < quota
//            and open) or (logp >= sure and not known); ids / known / committed logp updated there.
//
// Masses are integers: w in [0, 1] is rounded to a multiple of 2^-S with V 2^S <= 2^63, so sums are exact, independent of their
// order, and every pass over the row that adds up a part of it sees the same numbers.  w itself is evaluated in 64 bits: the
// draw and the top-p cut are comparisons of sums over up to V terms, and a 32-bit sum over 128k terms is off by more than the
// gap between neighbouring borders of a flat row.
//
// A row is spread over a cluster of 1 .. 8 CTAs, each of which keeps its slice (f32, after the bias) in shared memory, so the
// logits are read from global memory once whatever the number of passes; the CTAs exchange maxima, histograms and masses
// through distributed shared memory.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace cg = cooperative_groups;

namespace {

typedef unsigned long long u64;

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int BINS = 256;
constexpr int SLICE_MAX = 49152;            // elements of a slice at most (192 KB)
constexpr int SLICE_GOOD = 16384;           // a slice up to which three CTAs fit an SM

enum { PRI_LOGP = 0, PRI_MARGIN = 1, PRI_ENTROPY = 2 };

struct SampleParams {
  const void* logits;
  long long s_outer, s_inner;               // element strides of a row's two indices
  int inner;                                // rows per outer index
  int V, slice, scale_bits, priority;
  const float* u;
  const float* bias;                        // [outer, V] or null
  const float* t_row;                       // per-row parameters, or null and the scalar
  const int* k_row;
  const float* p_row;
  const float* m_row;
  double temperature, top_p, min_p;
  int top_k;
  long long* tokens;
  float* logp;
  float* prio;
};

// a total order of f32 values as unsigned integers (-0 is folded into +0 before)
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {      // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

struct Shared {
  // what this CTA tells the others; every exchange has fields of its own, so nothing is overwritten while a peer reads it
  float m;
  int bad;
  double z, ent;
  float second;
  int at_max, first_max;
  u64 mass;
  unsigned int count[2][BINS];              // histograms of the threshold search, alternating between rounds
  u64 hmass[2][BINS];
  // this CTA alone
  float fred[WARPS];
  double dred[2][WARPS];
  u64 ured[WARPS];
  int ired[WARPS];
  u64 tot_mass[BINS];
  unsigned int tot_count[BINS];
  unsigned int below_count[BINS];           // of the CTAs with a lower rank
  int pick_bin, idx_star;
  u64 pick_above_count, pick_above_mass;
};

// (x - m) / T as a mass of `scale` = 2^S units
struct Weigher {
  double m, inv_t, scale;
  __device__ __forceinline__ u64 operator()(float x) const { return (u64)__double2ll_rn(exp(((double)x - m) * inv_t) * scale); }
};

struct Cut {
  uint32_t k0, k1;                          // keys above k1 are kept; of those in [k0, k1] the first `ties` by index
  u64 ties, mass;                           // mass: of everything kept
  u64 before;                               // elements of [k0, k1] in CTAs with a lower rank
  u64 here;                                 // ... and in this one
};

struct Segment { int a, b; };
__device__ __forceinline__ Segment split(int a, int b, int parts, int i) {      // part i of [a, b), starts 32 apart
  const int len = ((b - a + parts * 32 - 1) / (parts * 32)) * 32;
  const int s = min(b, a + i * len);
  return {s, min(b, s + len)};
}

// The shortest prefix of the row (value descending, index ascending) whose count (MASS false) or mass (MASS true) reaches
// `target`: 256-way search over the order keys, one pass over the slice and one cluster barrier per round.
template <bool MASS>
__device__ Cut find_cut(Shared& sh, const float* xs, int n, const Weigher& w, u64 target, bool want_mass, int& round) {
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Segment seg = split(0, n, WARPS, warp);
  uint32_t k0 = 0, k1 = 0xffffffffu;
  u64 above_c = 0, above_m = 0;
  for (;;) {
    const int buf = round & 1;
    ++round;
    int shift = 0;
    while ((k1 - k0) >> shift >= BINS) ++shift;
    for (int i = tid; i < BINS; i += THREADS) { sh.count[buf][i] = 0; sh.hmass[buf][i] = 0; }
    __syncthreads();
    for (int i = seg.a + lane; i < seg.b; i += 32) {
      const uint32_t k = order_key(xs[i]);
      if (k >= k0 && k <= k1) {
        const uint32_t bin = (k - k0) >> shift;
        atomicAdd(&sh.count[buf][bin], 1u);
        if (MASS || want_mass) atomicAdd(&sh.hmass[buf][bin], w(xs[i]));
      }
    }
    cluster.sync();
    const int ranks = (int)cluster.num_blocks(), me = (int)cluster.block_rank();
    for (int i = tid; i < BINS; i += THREADS) {
      unsigned int c = 0, below = 0;
      u64 m = 0;
      for (int r = 0; r < ranks; ++r) {
        const Shared* p = cluster.map_shared_rank(&sh, r);
        if (r == me) below = c;
        c += p->count[buf][i];
        m += p->hmass[buf][i];
      }
      sh.tot_count[i] = c; sh.tot_mass[i] = m; sh.below_count[i] = below;
    }
    __syncthreads();
    if (warp == 0) {
      // lane 0 holds the highest bins: running totals from the top
      u64 c = 0, m = 0;
      for (int j = 0; j < BINS / 32; ++j) { const int b = BINS - 1 - (lane * (BINS / 32) + j); c += sh.tot_count[b]; m += sh.tot_mass[b]; }
      u64 pc = above_c + warp_scan(c, lane) - c, pm = above_m + warp_scan(m, lane) - m;      // before this lane's bins
      int found = -1;
      u64 fc = 0, fm = 0;
      for (int j = 0; j < BINS / 32; ++j) {
        const int b = BINS - 1 - (lane * (BINS / 32) + j);
        const u64 reach = MASS ? pm + sh.tot_mass[b] : pc + sh.tot_count[b];
        if (found < 0 && reach >= target) { found = b; fc = pc; fm = pm; }
        pc += sh.tot_count[b]; pm += sh.tot_mass[b];
      }
      const unsigned int any = __ballot_sync(0xffffffffu, found >= 0);
      if (any && lane == __ffs(any) - 1) { sh.pick_bin = found; sh.pick_above_count = fc; sh.pick_above_mass = fm; }
    }
    __syncthreads();
    const uint32_t bin = sh.pick_bin;
    above_c = sh.pick_above_count; above_m = sh.pick_above_mass;
    const u64 cnt = sh.tot_count[bin], mass = sh.tot_mass[bin];
    const uint32_t lo = k0 + (bin << shift), hi = lo + ((1u << shift) - 1u);
    const uint32_t top = k1;
    k0 = lo; k1 = min(hi, top);
    if (shift == 0 || cnt == 1) {
      Cut c;
      c.k0 = k0; c.k1 = k1;
      c.before = sh.below_count[bin]; c.here = sh.count[buf][bin];
      if (MASS) {
        const u64 each = mass / cnt;                              // equal keys: equal masses
        c.ties = (target - above_m + each - 1) / each;
        c.mass = above_m + c.ties * each;
      } else {
        c.ties = target - above_c;
        c.mass = above_m + c.ties * (mass / cnt);
      }
      __syncthreads();
      return c;
    }
    __syncthreads();                                              // pick_* and tot_* are written again in the next round
  }
}

template <class T>
__global__ void __launch_bounds__(THREADS) sample_kernel(const SampleParams p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared& sh = *reinterpret_cast<Shared*>(smem_raw);
  float* xs = reinterpret_cast<float*>(smem_raw + ((sizeof(Shared) + 15) / 16) * 16);
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), me = (int)cluster.block_rank();
  const long long row = blockIdx.x / ranks;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long outer = row / p.inner;
  const int first = me * p.slice;
  const int n = max(0, min(p.slice, p.V - first));

  // ---- the slice into shared memory, its maximum
  const T* src = reinterpret_cast<const T*>(p.logits) + outer * p.s_outer + (row - outer * p.inner) * p.s_inner + first;
  const float* bias = p.bias ? p.bias + outer * p.V + first : nullptr;
  constexpr int VEC = 16 / (int)sizeof(T);
  const int mis = (int)((reinterpret_cast<uintptr_t>(src) / sizeof(T)) % VEC);      // keeps 16-byte pieces aligned on both sides
  float mx = -INFINITY;
  int bad = 0;
  for (int v = tid; v * VEC < mis + n; v += THREADS) {
    const int i0 = v * VEC - mis;
    T e[VEC];
    if (i0 >= 0 && i0 + VEC <= n) {
      *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(src + i0);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (i0 + j >= 0 && i0 + j < n) e[j] = src[i0 + j];
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const int i = i0 + j;
      if (i >= 0 && i < n) {
        const float x = bias ? to_f32(e[j]) + bias[i] + 0.f : to_f32(e[j]) + 0.f;      // + 0: no negative zero
        bad |= !(x < INFINITY);                                    // NaN or +inf
        mx = fmaxf(mx, x);
        xs[mis + i] = x;
      }
    }
  }
  xs += mis;
  mx = warp_max(mx);
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) { sh.fred[warp] = mx; sh.ired[warp] = bad; }
  __syncthreads();
  if (tid == 0) {
    float m = -INFINITY;
    int b = 0;
    for (int i = 0; i < WARPS; ++i) { m = fmaxf(m, sh.fred[i]); b |= sh.ired[i]; }
    sh.m = m; sh.bad = b;
  }
  cluster.sync();
  float m = -INFINITY;
  bad = 0;
  for (int r = 0; r < ranks; ++r) { const Shared* q = cluster.map_shared_rank(&sh, r); m = fmaxf(m, q->m); bad |= q->bad; }
  if (bad || m == -INFINITY) {                                     // the same in every CTA of the cluster
    if (me == 0 && tid == 0) { p.tokens[row] = -1; p.logp[row] = NAN; if (p.priority != PRI_LOGP) p.prio[row] = NAN; }
    cluster.sync();
    return;
  }

  // ---- untempered sums
  const Segment seg = split(0, n, WARPS, warp);
  {
    double z = 0, ent = 0;
    float second = -INFINITY;
    int at_max = 0, first_max = 0x7fffffff;
    for (int i = seg.a + lane; i < seg.b; i += 32) {
      const float x = xs[i], d = fmaxf(x - m, -1e4f), e = __expf(d);
      z += e;
      ent += (double)(e * d);
      if (x == m) { ++at_max; first_max = min(first_max, first + i); }
      else second = fmaxf(second, x);
    }
    z = warp_sum(z); ent = warp_sum(ent); second = warp_max(second);
    at_max = __reduce_add_sync(0xffffffffu, at_max);
    first_max = __reduce_min_sync(0xffffffffu, first_max);
    if (tid == 0) { sh.at_max = 0; sh.first_max = 0x7fffffff; }
    __syncthreads();
    if (lane == 0) {
      sh.dred[0][warp] = z; sh.dred[1][warp] = ent; sh.fred[warp] = second;
      atomicAdd(&sh.at_max, at_max); atomicMin(&sh.first_max, first_max);
    }
    __syncthreads();
    if (tid == 0) {
      double a = 0, b = 0;
      float s = -INFINITY;
      for (int i = 0; i < WARPS; ++i) { a += sh.dred[0][i]; b += sh.dred[1][i]; s = fmaxf(s, sh.fred[i]); }
      sh.z = a; sh.ent = b; sh.second = s;
    }
  }

  // ---- tempered: the kept set, its mass
  const float t_f = p.t_row ? p.t_row[row] : 1.f;
  const double t_raw = p.t_row ? (double)t_f : p.temperature;
  const bool greedy = !(t_raw > 0);
  const double temp = fmin(fmax(t_raw, 1e-6), 1e6);
  Weigher w;
  w.m = (double)m; w.inv_t = 1.0 / temp; w.scale = (double)(1ull << p.scale_bits);
  Cut cut;
  cut.k0 = cut.k1 = 0; cut.ties = 1; cut.before = 0; cut.here = 0; cut.mass = 0;
  uint32_t k_min = 0;
  bool chosen_cut = false;
  u64 my_mass = 0;
  const double min_p = p.m_row ? (double)p.m_row[row] : p.min_p;
  int round = 0;
  auto kept = [&](float x, int i, int last_tie) {
    const uint32_t k = order_key(x);
    return (k > cut.k1 || (k >= cut.k0 && i <= last_tie)) && k >= k_min;
  };
  int last_tie = 0x7fffffff;
  if (!greedy) {
    if (min_p > 0) k_min = order_key(__double2float_ru((double)m + temp * log(fmin(min_p, 1.0))));
    const double top_p = p.p_row ? (double)p.p_row[row] : p.top_p;
    const int top_k = p.k_row ? p.k_row[row] : p.top_k;
    u64 whole = 0;
    if (top_k > 0 && top_k < p.V) {
      cut = find_cut<false>(sh, xs, n, w, (u64)top_k, top_p < 1.0, round);
      whole = cut.mass;
      chosen_cut = true;
    } else if (top_p < 1.0) {
      u64 s = 0;
      for (int i = seg.a + lane; i < seg.b; i += 32) s += w(xs[i]);
      s = warp_sum(s);
      if (lane == 0) sh.ured[warp] = s;
      __syncthreads();
      if (tid == 0) { u64 a = 0; for (int i = 0; i < WARPS; ++i) a += sh.ured[i]; sh.mass = a; }
      cluster.sync();
      for (int r = 0; r < ranks; ++r) whole += cluster.map_shared_rank(&sh, r)->mass;
      cluster.sync();                                              // sh.mass is written once more below
    }
    if (top_p < 1.0) {
      const double goal = ceil(fmax(top_p, 0.0) * (double)whole);
      const u64 target = max((u64)1, min(whole, (u64)goal));
      cut = find_cut<true>(sh, xs, n, w, target, true, round);
      chosen_cut = true;
    }
    if (chosen_cut && cut.before + cut.here > cut.ties) {          // this CTA holds ties that are not kept
      if (cut.before >= cut.ties) {
        last_tie = -1;
      } else {
        // the (ties - before)-th element of [k0, k1] in this slice
        const u64 want = cut.ties - cut.before;
        int c = 0;
        for (int i = seg.a + lane; i < seg.b; i += 32) { const uint32_t k = order_key(xs[i]); c += k >= cut.k0 && k <= cut.k1; }
        c = __reduce_add_sync(0xffffffffu, c);
        if (lane == 0) sh.ired[warp] = c;
        __syncthreads();
        u64 run = 0;
        for (int i = 0; i < warp; ++i) run += sh.ired[i];
        if (run < want && run + sh.ired[warp] >= want) {
          for (int i0 = seg.a; i0 < seg.b; i0 += 32) {
            const int i = i0 + lane;
            const uint32_t k = i < seg.b ? order_key(xs[i]) : 0;
            const unsigned int hit = __ballot_sync(0xffffffffu, i < seg.b && k >= cut.k0 && k <= cut.k1);
            const int cnt = __popc(hit);
            if (run + cnt >= want) {
              if ((hit >> lane & 1) && run + __popc(hit & ((2u << lane) - 1)) == want) sh.idx_star = i;
              break;
            }
            run += cnt;
          }
        }
        __syncthreads();
        last_tie = sh.idx_star;
      }
    }
    u64 s = 0;
    for (int i = seg.a + lane; i < seg.b; i += 32)
      if (kept(xs[i], i, last_tie)) s += w(xs[i]);
    s = warp_sum(s);
    if (lane == 0) sh.ured[warp] = s;
    __syncthreads();
    if (tid == 0) { u64 a = 0; for (int i = 0; i < WARPS; ++i) a += sh.ured[i]; sh.mass = a; }
  }
  cluster.sync();

  // ---- totals of the cluster, the draw
  double z = 0, ent = 0;
  u64 total = 0, base = 0;
  float second = -INFINITY;
  int at_max = 0, first_max = 0x7fffffff;
  for (int r = 0; r < ranks; ++r) {
    const Shared* q = cluster.map_shared_rank(&sh, r);
    z += q->z; ent += q->ent;
    second = fmaxf(second, q->second);
    at_max += q->at_max; first_max = min(first_max, q->first_max);
    if (!greedy) {
      if (r == me) { base = total; my_mass = q->mass; }
      total += q->mass;
    }
  }
  const float logz = logf((float)z);
  auto answer = [&](long long tok, float x) {
    const float lp = (x - m) - logz;
    p.tokens[row] = tok;
    p.logp[row] = lp;
    if (p.priority == PRI_LOGP) return;
    float pr;
    if (p.priority == PRI_MARGIN) pr = at_max > 1 ? 0.f : (float)((1.0 - (double)__expf(second - m)) / z);
    else pr = (float)(ent / z - (double)logz);
    p.prio[row] = pr;
  };
  if (greedy) {
    if (me == 0 && tid == 0) answer(first_max, m);
  } else {
    const double u = (double)p.u[row];
    u64 goal = u > 0 ? (u64)(fmin(u, 1.0) * (double)total) : 0;
    if (goal >= total) goal = total - 1;
    if (goal >= base && goal < base + my_mass) {                   // the draw falls into this slice
      u64 run = base;
      int own = 0;
      while (own < WARPS - 1 && run + sh.ured[own] <= goal) run += sh.ured[own++];
      const Segment big = split(0, n, WARPS, own);
      const Segment part = split(big.a, big.b, WARPS, warp);
      u64 s = 0;
      for (int i = part.a + lane; i < part.b; i += 32)
        if (kept(xs[i], i, last_tie)) s += w(xs[i]);
      s = warp_sum(s);
      __syncthreads();
      if (lane == 0) sh.ured[warp] = s;
      __syncthreads();
      for (int i = 0; i < warp; ++i) run += sh.ured[i];
      if (goal >= run && goal < run + s) {
        for (int i0 = part.a; i0 < part.b; i0 += 32) {
          const int i = i0 + lane;
          const u64 wi = i < part.b && kept(xs[i], i, last_tie) ? w(xs[i]) : 0;
          const u64 inc = run + warp_scan(wi, lane);
          const unsigned int hit = __ballot_sync(0xffffffffu, inc > goal);
          if (hit) {
            if (lane == __ffs(hit) - 1) answer(first + i, xs[i]);
            break;
          }
          run = __shfl_sync(0xffffffffu, inc, 31);
        }
      }
    }
  }
  cluster.sync();                                                  // nobody leaves while a peer may still read its memory
}

template <class T>
int launch_sample(const SampleParams& p, long long rows, int ranks, cudaStream_t s) {
  const size_t smem = ((sizeof(Shared) + 15) / 16) * 16 + ((size_t)p.slice + 16) * sizeof(float);
  cudaError_t e = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return 1000 + (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned int)(rows * ranks));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned int)ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, sample_kernel<T>, p);
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}

// ------------------------------------------------------------------------------------------------------ unmask
// One block per row.  The quota-th slot in rank order is found by a radix search over the order keys in shared memory.
constexpr int UM_THREADS = 256;
constexpr int UM_SLOTS_MAX = 32768;

__global__ void __launch_bounds__(UM_THREADS) unmask_kernel(const long long* __restrict__ ids, const uint8_t* __restrict__ known,
                                                           const float* __restrict__ held, const long long* __restrict__ tokens,
                                                           const float* __restrict__ logp, const float* __restrict__ priority,
                                                           const long long* __restrict__ quota, const uint8_t* __restrict__ allowed,
                                                           float sure, int use_sure, long long* __restrict__ ids_out,
                                                           uint8_t* __restrict__ known_out, float* __restrict__ held_out,
                                                           uint8_t* __restrict__ where_out, int C) {
  extern __shared__ uint32_t keys[];
  __shared__ unsigned int hist[256];
  __shared__ int warp_count[UM_THREADS / 32];
  __shared__ unsigned int s_bin, s_above;
  const long long row = blockIdx.x, at = row * C;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int i = tid; i < C; i += UM_THREADS) {
    const bool shut = known[at + i] || (allowed && !allowed[at + i]);
    const float v = shut ? -INFINITY : priority[at + i] + 0.f;
    keys[i] = v != v ? 0u : order_key(v);
  }
  const long long q = quota[row];
  uint32_t key = 0;                                                // slots above `key` are picked, of those equal the first `ties`
  long long ties = 0;
  if (q >= C) {
    ties = C;                                                      // key 0: NaN slots last, all of them picked
  } else if (q <= 0) {
    key = 0xffffffffu;
  } else {
    unsigned int left = (unsigned int)q;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += UM_THREADS) hist[i] = 0;
      __syncthreads();
      const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
      for (int i = tid; i < C; i += UM_THREADS)
        if ((keys[i] & mask) == key) atomicAdd(&hist[keys[i] >> shift & 255u], 1u);
      __syncthreads();
      if (warp == 0) {
        unsigned int c = 0;
        for (int j = 0; j < 8; ++j) c += hist[255 - (lane * 8 + j)];
        unsigned int run = (unsigned int)warp_scan((u64)c, lane) - c;
        for (int j = 0; j < 8; ++j) {
          const int b = 255 - (lane * 8 + j);
          if (run < left && run + hist[b] >= left) { s_bin = b; s_above = run; }
          run += hist[b];
        }
      }
      __syncthreads();
      key |= s_bin << shift;
      left -= s_above;
      __syncthreads();
    }
    ties = left;
  }
  // ties by slot: warps own contiguous pieces
  __syncthreads();
  const Segment seg = split(0, C, UM_THREADS / 32, warp);
  int c = 0;
  for (int i = seg.a + lane; i < seg.b; i += 32) c += keys[i] == key;
  c = __reduce_add_sync(0xffffffffu, c);
  if (lane == 0) warp_count[warp] = c;
  __syncthreads();
  long long run = 0;
  for (int i = 0; i < warp; ++i) run += warp_count[i];
  for (int i0 = seg.a; i0 < seg.b; i0 += 32) {
    const int i = i0 + lane;
    const bool in = i < seg.b;
    const uint32_t k = in ? keys[i] : 0u;
    const unsigned int eq = __ballot_sync(0xffffffffu, in && k == key);
    if (in) {
      const bool is_known = known[at + i];
      const bool shut = is_known || (allowed && !allowed[at + i]);
      const float lp = logp[at + i];
      bool take = (k > key || (k == key && run + __popc(eq & ((1u << lane) - 1)) < ties)) && !shut;
      if (use_sure && lp >= sure && !is_known) take = true;
      ids_out[at + i] = take ? tokens[at + i] : ids[at + i];
      known_out[at + i] = is_known || take;
      held_out[at + i] = take ? lp : held[at + i];
      where_out[at + i] = take;
    }
    run += __popc(eq);
  }
}

}  // namespace

// CTAs per row for a vocabulary of V (0: not supported).
extern "C" int dttt_sample_ranks(int V) {
  if (V <= 0) return 0;
  for (int r = 1; r <= 8; r *= 2)
    if (V <= r * SLICE_GOOD) return r;
  return V <= 8 * SLICE_MAX ? 8 : 0;
}

// logits: rows [outer, inner] of V elements (dtype 0 f32, 1 bf16, 2 f16), element strides s_outer / s_inner, contiguous along V.
// *_row: per-row parameter arrays or null (then the scalar).  Outputs contiguous [rows].
extern "C" int dttt_sample(const void* logits, int dtype, long long rows, int inner, long long s_outer, long long s_inner, int V,
                           const float* u, const float* bias, double temperature, const float* t_row, int top_k, const int* k_row,
                           double top_p, const float* p_row, double min_p, const float* m_row, int priority, long long* tokens,
                           float* logp, float* prio, cudaStream_t stream) {
  if (rows <= 0) return 0;
  const int ranks = dttt_sample_ranks(V);
  if (ranks == 0 || inner <= 0 || rows * ranks > 0x7fffffffll) return -2;
  SampleParams p;
  p.logits = logits; p.s_outer = s_outer; p.s_inner = s_inner; p.inner = inner;
  p.V = V; p.slice = ((V + ranks - 1) / ranks + 7) / 8 * 8; p.priority = priority;
  int lg = 0;
  while ((1ll << lg) < V) ++lg;
  p.scale_bits = min(50, 62 - lg);
  p.u = u; p.bias = bias; p.t_row = t_row; p.k_row = k_row; p.p_row = p_row; p.m_row = m_row;
  p.temperature = temperature; p.top_p = top_p; p.min_p = min_p; p.top_k = top_k;
  p.tokens = tokens; p.logp = logp; p.prio = prio;
  switch (dtype) {
    case 0: return launch_sample<float>(p, rows, ranks, stream);
    case 1: return launch_sample<__nv_bfloat16>(p, rows, ranks, stream);
    case 2: return launch_sample<__half>(p, rows, ranks, stream);
  }
  return -2;
}

extern "C" int dttt_unmask(const long long* ids, const void* known, const float* held, const long long* tokens, const float* logp,
                           const float* priority, const long long* quota, const void* allowed, float sure, int use_sure,
                           long long* ids_out, void* known_out, float* held_out, void* where_out, int B, int C, cudaStream_t stream) {
  if (B <= 0 || C <= 0) return 0;
  if (C > UM_SLOTS_MAX) return -2;
  const size_t smem = (size_t)C * sizeof(uint32_t);
  cudaError_t e = cudaFuncSetAttribute(unmask_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, UM_SLOTS_MAX * (int)sizeof(uint32_t));
  if (e != cudaSuccess) return 1000 + (int)e;
  unmask_kernel<<<B, UM_THREADS, smem, stream>>>(ids, (const uint8_t*)known, held, tokens, logp, priority, quota, (const uint8_t*)allowed,
                                                 sure, use_sure, ids_out, (uint8_t*)known_out, held_out, (uint8_t*)where_out, C);
  e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}
