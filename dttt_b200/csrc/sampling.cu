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
// gap between neighbouring borders of a flat row.  A draw of fewer units than there are elements (u = 0; else u < 2^-24) may end
// among tokens that have less than a unit: it is made again with masses in 64-bit floating point (`tiny_draw`).
//
// A row is spread over a cluster of 1 .. 8 CTAs, each of which keeps its slice (f32, after the bias) in shared memory, so the
// logits are read from global memory once whatever the number of passes; the CTAs exchange maxima, histograms and masses
// through distributed shared memory.  A pass counts every element into octaves of its mass, 1/8 octave wide, which bounds where the
// truncation can end; if no more than 256 elements lie in the octaves that are kept, one CTA finishes the row from a list of them
// (top-p, 512 x 128256: 383 us without that, 212 with), else a 128-way search goes on among the elements of the last
// octaves.  Without truncation nothing has to wait for the maximum, and many rows take two streaming launches instead.
//
// What bounds it, at V = 128256 (f32, 525 MB for 1024 rows, 81 us at the copy rate):
//   one row, top-p: 16 us.  Latency: load 1.5 us, three exchanges over the cluster, ranking the list 3.4 us.
//   1024 rows, top-p 0.9: 465 us = 1.1 TB/s.  A CTA takes 17 us, of which loading 4.5, its pass 4, looking for candidates 1.4 and the
//     exchanges 6.5; three to an SM hide each other's waits only in part (issue slots 42 % busy).
//   1024 rows, untruncated: 203 + 12 us = 2.5 TB/s, bound by issue: 38 instructions an element, of which the 64-bit exponential
//     (FP64 pipe 36 % busy, issue slots 68 %) is most.
//   252 rows bf16 with bias, top-k 50 and min-p: 115 us for 67 MB: 4.5 rounds of CTAs as above, whose slices are f32.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace cg = cooperative_groups;

namespace {

typedef unsigned long long u64;

constexpr int MAX_WARPS = 16;
constexpr int OCTAVES = 256;                 // bins of the octave counts
constexpr int BINS = 128;                    // of a round of the search
constexpr int TAB = 64, COPIES = 8;
constexpr int FEW = 256;                     // candidates up to which one CTA finishes a row
constexpr int LIST = 256;                    // entries of all warps
constexpr int SLICE_MAX = 49152;            // elements of a slice at most (192 KB)
constexpr int SLICE_GOOD = 16384;           // a slice up to which three CTAs fit an SM

constexpr int SLICE_SMALL = 4096;

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
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// the maximum, NaN if there is one
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
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

// 2^(j / 64)
__constant__ double ROOTS[TAB] = {
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284, 1.0442737824274138, 1.0556451783605572,
    1.0671404006768237, 1.0787607977571199, 1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812, 1.189207115002721, 1.202156731452703,
    1.215247359980469, 1.22848053610687, 1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303, 1.3542555469368927, 1.3690024229745905,
    1.383909881963832, 1.3989796725383112, 1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384, 1.5422108254079407, 1.559004400237837,
    1.5759808451078865, 1.593142151342267, 1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062, 1.7562521603732995, 1.7753764925265212,
    1.7947090750031072, 1.8142521755003989, 1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951};

struct Shared {
  // what the other CTAs read; nothing of it is overwritten before a cluster barrier that follows their reads
  float m;
  float z[MAX_WARPS], ent[MAX_WARPS];       // a value per warp (`ent`: of either priority)
  int at_max[MAX_WARPS], first_max[MAX_WARPS];
  u64 mass[MAX_WARPS];                      // of every element, or of the kept ones
  unsigned int octaves_here[OCTAVES];
  u64 all_mass;                             // of every element, where the search adds it up
  float zt[MAX_WARPS];                      // tempered sums in 32 bits, of every element
  int pushed;                               // entries of the candidate list, which in CTA 0 takes the place of the histograms
  alignas(16) u64 hmass[2][BINS];           // histograms of the threshold search, alternating between rounds
  unsigned int count[2][BINS];
  unsigned int above_count[2];
  u64 above_mass[2];
  // this CTA alone
  float fred[MAX_WARPS];
  u64 above[MAX_WARPS], sub[MAX_WARPS];
  int ties[MAX_WARPS], listed[MAX_WARPS];
  unsigned short list[LIST];                // indices of each warp's elements in the search's first range, if they fit its share
  union {
    struct {
      u64 tot_mass[BINS];
      unsigned int tot_count[BINS];
      unsigned int octaves[OCTAVES];        // of all CTAs
    };
    u64 few_mass[FEW];                      // of the candidates, where CTA 0 finishes the row
  };
  uint32_t range[2];
  int last_bin, candidates;                 // the octaves down to last_bin hold the prefix; so many elements
  u64 tot_above_count, tot_above_mass;
  int pick_bin, idx_star;
  u64 pick_above_count, pick_above_mass;
  double tab[TAB * COPIES];
  // this row's parameters, and at the end its answer but for the token
  double temp, min_p, top_p, log2e_t, cut;
  double rough;                             // 32-bit sum of the tempered masses, in units of the maximum's
  float scale, u, logz, pr;
  int top_k, greedy;
  u64 whole, goal, base, mine;
  int tiny;                                 // the draw is made again by tiny_draw
  double part[MAX_WARPS];                   // its masses, per warp
};

// exp((x - m) / T) as a mass of 2^S units, rounded to nearest.  Table-driven (Tang's scheme, from the mathematics): with
// z = 64 log2(e) (x - m) / T = n + r, |r| <= 1/2, it is 2^(n >> 6) 2^((n & 63) / 64) 2^(r / 64); the last factor by its Taylor series to
// the third order (|r| ln2 / 64 <= 0.0054: truncated by 3.6e-11, which is the same for equal values, smooth in r and shifts a
// border of the draw by about 1e-11 of the whole).  The table holds copies of its values in banks of their own, so that a half
// warp's lookups collide two by two at most.  Half the FP64 instructions of the library's exp, and no conversion back: adding
// 1.5 2^(52 - S) leaves the rounded mass in the low bits.
// `coarse`: T is so small that the floats next to m are 400 octaves away: whatever is below m has no mass.
struct Weigher {
  double c, mc, magic;                      // z = x c + mc
  float m, least;                           // the mass of `least` rounds to 0, as that of everything below
  bool coarse;
  const double* tab;                        // this thread's copy
  __device__ __forceinline__ Weigher(double log2e_t, float m_, double cut, int bits, const double* tab_) : m(m_), tab(tab_) {
    c = TAB * log2e_t;
    mc = -(double)m * c;
    magic = __hiloint2double(0x3ff80000 + ((52 - bits) << 20), 0);         // 1.5 2^(52 - S)
    least = fminf(__double2float_rd((double)m - cut), nextafterf(m, -INFINITY));      // below m, even where m - cut is m
    coarse = !(((double)m - (double)least) * c < 400.0 * TAB);
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    if (coarse) return x >= m ? (u64)(__double_as_longlong(magic + 1.0) - __double_as_longlong(magic)) : 0;
    return fine(x) - (u64)__double_as_longlong(magic);
  }
  // not coarse; with the bits of `magic` still in it: for sums of many, from which they are taken once
  __device__ __forceinline__ u64 fine(float x) const {
    constexpr double SHIFT = 6755399441055744.0;                   // 1.5 2^52: the sum's low word is the rounded integer
    constexpr double L = 0.010830424696249145;                     // ln2 / 64
    const double z = fma((double)fmaxf(x, least), c, mc);
    const double t = z + SHIFT;
    const int n = __double2loint(t);
    const double r = z - (t - SHIFT);
    double q = L * L * L / 6;
    q = fma(q, r, L * L / 2);
    q = fma(q, r, L);
    q = fma(q, r, 1.0);
    const double v = q * tab[(n & (TAB - 1)) * COPIES];
    return (u64)__double_as_longlong(__hiloint2double(__double2hiint(v) + (n & ~(TAB - 1)) * (1 << 14), __double2loint(v)) + magic);
  }
};

__device__ __forceinline__ float key_value(uint32_t k) {
  if (k <= 0x007fffffu) return -INFINITY;                          // -inf and what has no value
  if (k >= 0xff800000u) return INFINITY;
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct Cut {
  float lo, hi;                             // values above hi are kept; of those in [lo, hi] the first `ties` by index
  u64 ties, mass;                           // mass: of everything kept
  float first_hi;                           // the first round's upper end: each warp's mass above it is in Shared::above
  u64 before;                               // elements of [lo, hi] in CTAs with a lower rank
  u64 here;                                 // ... and in this one
};

struct Segment { int a, b; };
__device__ __forceinline__ Segment split(int a, int b, int parts, int i) {      // part i of [a, b), starts 32 apart
  const int len = ((b - a + parts * 32 - 1) / (parts * 32)) * 32;
  const int s = min(b, a + i * len);
  return {s, min(b, s + len)};
}

// Octaves of the tempered mass: bin j of the counts holds the elements whose (m - x) / T log2(e) rounds to j / 8; the last one is
// not counted.  The rounding is monotone in x, so bins are ranges of the order, and an element's mass is known within 9 %.
constexpr float PER_OCTAVE = 8.f;
__device__ __forceinline__ int octave_bin(float x, float m, float scale) {
  return __float_as_int(fminf((m - x) * scale, (float)(OCTAVES - 1)) + 8388608.f) - 0x4b000000;
}

constexpr int MAX_RANKS = 8;
// The sum over the cluster's CTAs of what `get` takes from one's shared memory; all loads in flight at once.
template <class V, class F>
__device__ __forceinline__ V over_ranks(Shared& sh, F get) {
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks();
  V v[MAX_RANKS], sum = 0;
#pragma unroll
  for (int r = 0; r < MAX_RANKS; ++r) v[r] = r < ranks ? get(*cluster.map_shared_rank(&sh, r)) : V(0);
#pragma unroll
  for (int r = 0; r < MAX_RANKS; ++r) sum += v[r];
  return sum;
}

// The per-warp values of all CTAs, in order of the slices, over the lanes of a warp: `per` of them to a lane (a CTA's warps are a
// whole number of lanes).
template <int WARPS, class V, class F>
__device__ __forceinline__ V warp_values(Shared& sh, int lane, V none, F get) {
  cg::cluster_group cluster = cg::this_cluster();
  const int all = (int)cluster.num_blocks() * WARPS, per = max(1, all / 32);
  V v = none;
  for (int j = 0; j < per; ++j) {
    const int e = lane * per + j;
    if (e < all) v = get(v, *cluster.map_shared_rank(&sh, e / WARPS), e % WARPS);
  }
  return v;
}

// From the octave counts, the range of values that has to hold the last element of the prefix whose count or mass reaches
// `goal` (a mass as a part of exp(0), known to 2e-4 of itself, give or take `slack`).  Warp 0 computes it, from the top bin down, with
// every element's mass between those of its bin's borders (1e-4 is far more than the rounding of the bins can shift them); the
// borders are widened by more than the rounding of m - x.
template <bool MASS>
__device__ __forceinline__ void first_range(Shared& sh, float m, float scale, float goal, float slack) {
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    constexpr int EACH = OCTAVES / 32;
    constexpr float STEP = 0.917004043f;                           // 2^(-1/8); its powers here are off by less than 1e-6
    const float w_lo = exp2f(-(lane * EACH + 0.5f) / PER_OCTAVE), w_hi = exp2f(-(lane * EACH - 0.5f) / PER_OCTAVE);
    float lo[EACH], hi[EACH], wl = w_lo, wh = w_hi;
    float slo = 0, shi = 0;
    unsigned int n[EACH], sn = 0;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      sn += sh.octaves[lane * EACH + j];
      n[j] = sn;
      const float c = (float)sh.octaves[lane * EACH + j];
      slo += MASS ? c * wl : c;
      shi += MASS ? c * fminf(wh, 1.f) : c;
      lo[j] = slo; hi[j] = shi;
      wl *= STEP; wh *= STEP;
    }
    float blo = slo, bhi = shi;
    unsigned int bn = sn;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float a = __shfl_up_sync(0xffffffffu, blo, o), b = __shfl_up_sync(0xffffffffu, bhi, o);
      const unsigned int c = __shfl_up_sync(0xffffffffu, bn, o);
      if (lane >= o) { blo += a; bhi += b; bn += c; }
    }
    blo -= slo; bhi -= shi; bn -= sn;
    // counts are whole numbers below 2^24: their float sums are exact
    int first = OCTAVES - 1, last = OCTAVES - 1;
#pragma unroll
    for (int j = EACH - 1; j >= 0; --j) {
      if ((MASS ? (bhi + hi[j]) * 1.0003f + slack : bhi + hi[j]) >= goal) first = min(first, lane * EACH + j);
      if ((MASS ? (blo + lo[j]) * 0.9997f - slack : blo + lo[j]) >= goal) last = min(last, lane * EACH + j);
    }
    first = __reduce_min_sync(0xffffffffu, first);
    last = __reduce_min_sync(0xffffffffu, last);
#pragma unroll
    for (int j = 0; j < EACH; ++j)
      if (lane * EACH + j == last) { sh.last_bin = last; sh.candidates = last == OCTAVES - 1 ? 0x7fffffff : (int)(bn + n[j]); }
    if (lane < 2) {
      const float edge = lane ? fmaxf(first - 0.5f, 0.f) * (1.f - 1e-5f) : (last + 0.5f) * (1.f + 1e-5f);
      const double at = (double)m - (double)edge / (double)scale, eps = fabs((double)m) * 1e-6;
      sh.range[lane] = lane ? (first == 0 ? 0xffffffffu : order_key(__double2float_ru(at + eps) + 0.f))
                            : (last == OCTAVES - 1 ? 0u : order_key(__double2float_rd(at - eps) + 0.f));
    }
  }
  __syncthreads();
}

// f(x, index, whether there is one) over a warp's elements of the search's first range, or over all of its elements where their
// list overflowed; all lanes together.
template <int WARPS, class F>
__device__ __forceinline__ void for_range(const Shared& sh, const float* xs, Segment seg, int warp, int lane, F f) {
  const int listed = sh.listed[warp];
  constexpr int ROOM = LIST / WARPS;
  if (listed <= ROOM) {
    for (int j = lane; j - lane < listed; j += 32) { const int i = j < listed ? sh.list[warp * ROOM + j] : 0; f(xs[i], i, j < listed); }
  } else {
    for (int i = seg.a + lane; i - lane < seg.b; i += 32) f(i < seg.b ? xs[i] : -INFINITY, i, i < seg.b);
  }
}

// The shortest prefix of the row (value descending, index ascending) whose count (MASS false) or mass (MASS true) reaches
// `target`: 128-way search over the order keys from the range above; a pass over the slice and a cluster barrier per round.  Only
// elements of the range and, in the first round, those above it cost more than a comparison.
//
// ALL: the target is a part, `target_of`, of the mass of all elements, which the first round adds up on its way: every element is
// weighed once, and the range comes from a 32-bit sum.
template <int WARPS, bool MASS, bool ALL, class F>
__device__ Cut find_cut(Shared& sh, const float* xs, int n, const Weigher& w, u64 target, F target_of, int& round) {
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Segment seg = split(0, n, WARPS, warp);
  uint32_t k0 = sh.range[0], k1 = sh.range[1];
  const float first_hi = key_value(k1);
  u64 above_c = 0, above_m = 0;
  bool fresh = true;                                               // what lies above the range is not known yet
  for (;;) {
    const int buf = round & 1;
    ++round;
    int shift = 0;
    while ((k1 - k0) >> shift >= BINS) ++shift;
    const float lo = key_value(k0), hi = key_value(k1);
    // `any`: the lanes that have one.  With many of them equal values meet in one addition: 16-bit logits and flat rows would put
    // thousands of elements on one counter.
    auto count = [&](float x, u64 wx, unsigned int any) {
      if (any >> lane & 1) {
        int k = 1;
        bool adds = true;
        if (__popc(any) >= 8) {
          const unsigned int peers = __match_any_sync(any, __float_as_uint(x));
          k = __popc(peers);
          adds = lane == __ffs(peers) - 1;
        }
        if (adds) {
          const uint32_t bin = (order_key(x) - k0) >> shift;
          atomicAdd(&sh.count[buf][bin], (unsigned int)k);
          atomicAdd(&sh.hmass[buf][bin], (u64)k * wx);
        }
      }
      __syncwarp();
    };
    if (fresh) {
      unsigned int ac = 0;
      u64 am = 0, all = 0;
      int listed = 0;
      for (int i0 = seg.a; i0 < seg.b; i0 += 128) {
        float xk[4];
        bool some = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          xk[k] = i0 + k * 32 + lane < seg.b ? xs[i0 + k * 32 + lane] : NAN;
          some |= xk[k] >= lo;
        }
        if (!ALL && !__any_sync(0xffffffffu, some)) continue;
        u64 wk[4];
        if (ALL) {
#pragma unroll
          for (int k = 0; k < 4; ++k) { wk[k] = w(xk[k]); all += wk[k]; }      // NaN, where there is none: 0
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float x = xk[k];
          const unsigned int cand = __ballot_sync(0xffffffffu, x >= lo);
          if (!cand) continue;
          const u64 wx = ALL ? wk[k] : w(x);
          const unsigned int over = __ballot_sync(0xffffffffu, x > hi), any = cand & ~over;
          if (over >> lane & 1) { ++ac; am += wx; }
          if (any) {
            const int at = listed + __popc(any & ((1u << lane) - 1));
            if ((any >> lane & 1) && at < LIST / WARPS) sh.list[warp * (LIST / WARPS) + at] = (unsigned short)(i0 + k * 32 + lane);
            listed += __popc(any);
            count(x, wx, any);
          }
        }
      }
      ac = __reduce_add_sync(0xffffffffu, ac);
      am = warp_sum(am);
      if (ALL) all = warp_sum(all);
      if (lane == 0) {
        if (ALL) atomicAdd(&sh.all_mass, all);
        sh.above[warp] = am;
        sh.listed[warp] = listed;
        if (ac) { atomicAdd(&sh.above_count[buf], ac); atomicAdd(&sh.above_mass[buf], am); }
      }
    } else {
      for_range<WARPS>(sh, xs, seg, warp, lane, [&](float x, int, bool in) {
        const unsigned int any = __ballot_sync(0xffffffffu, in && x >= lo && x <= hi);
        if (any) count(x, w(x), any);
      });
    }
    cluster.sync();
    for (int i = tid; i < BINS; i += WARPS * 32) {
      sh.tot_count[i] = over_ranks<unsigned int>(sh, [&](const Shared& q) { return q.count[buf][i]; });
      sh.tot_mass[i] = over_ranks<u64>(sh, [&](const Shared& q) { return q.hmass[buf][i]; });
      sh.count[buf ^ 1][i] = 0; sh.hmass[buf ^ 1][i] = 0;             // the next round's; the last round's readers are past the barrier
    }
    if (warp == WARPS - 1) {
      if (lane == 0) sh.tot_above_count = over_ranks<unsigned int>(sh, [&](const Shared& q) { return q.above_count[buf]; });
      if (lane == 1) sh.tot_above_mass = over_ranks<u64>(sh, [&](const Shared& q) { return q.above_mass[buf]; });
      if (lane == 2) { sh.above_count[buf ^ 1] = 0; sh.above_mass[buf ^ 1] = 0; }
      if (ALL && fresh && lane == 3) sh.whole = over_ranks<u64>(sh, [&](const Shared& q) { return q.all_mass; });
    }
    __syncthreads();
    if (ALL && fresh) target = target_of(sh.whole);
    if (fresh) { above_c = sh.tot_above_count; above_m = sh.tot_above_mass; fresh = false; }
    if (warp == 0) {
      // lane 0 holds the highest bins: running totals from the top
      constexpr int EACH = BINS / 32;
      u64 part[EACH], sum = 0;
#pragma unroll
      for (int j = 0; j < EACH; ++j) { const int b = BINS - 1 - (lane * EACH + j); part[j] = MASS ? sh.tot_mass[b] : sh.tot_count[b]; sum += part[j]; }
      u64 run = (MASS ? above_m : above_c) + warp_scan(sum, lane) - sum, at = 0;      // before this lane's bins
      int found = -1;
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        if (found < 0 && run + part[j] >= target) { found = BINS - 1 - (lane * EACH + j); at = run; }
        run += part[j];
      }
      const unsigned int any = __ballot_sync(0xffffffffu, found >= 0);
      const int from = any ? __ffs(any) - 1 : 0, bin = max(__shfl_sync(0xffffffffu, found, from), 0);
      u64 over = 0;                                                  // the other measure of the bins above
#pragma unroll
      for (int j = 0; j < EACH; ++j) { const int b = BINS - 1 - (lane * EACH + j); if (!MASS && b > bin) over += sh.tot_mass[b]; }
      if (!MASS) over = warp_sum(over);
      if (lane == from) { sh.pick_bin = bin; sh.pick_above_count = at; sh.pick_above_mass = MASS ? at : above_m + over; }
    }
    __syncthreads();
    const uint32_t bin = (uint32_t)sh.pick_bin;
    above_c = MASS ? 0 : sh.pick_above_count; above_m = sh.pick_above_mass;
    const u64 cnt = sh.tot_count[bin], mass = sh.tot_mass[bin];
    const uint32_t low = k0 + (bin << shift);
    k1 = min(low + ((1u << shift) - 1u), k1);
    k0 = low;
    if (shift == 0 || cnt == 1) {
      Cut c;
      c.lo = key_value(k0); c.hi = key_value(k1); c.first_hi = first_hi;
      c.before = __reduce_add_sync(0xffffffffu, lane < (int)cluster.block_rank() ? cluster.map_shared_rank(&sh, lane)->count[buf][bin] : 0u);
      c.here = sh.count[buf][bin];
      if (MASS) {
        const u64 each = mass / cnt;                              // equal values: equal masses
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

// One pass over the slice for everything that needs every element: the untempered sum of exponentials, what the priority needs,
// the tempered masses (per warp, MASS) or their 32-bit sum (ROUGH) and the octave counts (HIST).
// The 32-bit sum is off by less than 1e-5 of itself: three roundings of the argument shift a term by 3 2^-24 ln2 |y| of itself, 4e-6
// at |y| = 32 octaves (below which all terms together make up less than V 2^-32), the exponential is off by 2^-22, and at most
// 51 terms to an accumulator (a slice of 49152 elements, 256 threads) and the tree after it add (51 + 8) 2^-24 = 3.5e-6.
template <int WARPS, bool MASS, bool HIST, bool ROUGH, int PRI>
__device__ __forceinline__ void whole_pass(Shared& sh, const float* xs, Segment seg, float m, float scale, const Weigher& w) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float z = 0, zt[4] = {0, 0, 0, 0}, ent = 0, second = -INFINITY;
  int at_max = 0;
  u64 mass = 0;
  auto one = [&](float x, int k) {
    const float y = (x - m) * 1.44269504f, e = ex2(y);
    z += e;
    if (PRI == PRI_ENTROPY) ent = fmaf(e, fmaxf(y, -1e4f), ent);
    if (PRI == PRI_MARGIN) { at_max += x == m; second = x < m ? fmaxf(second, x) : second; }
    if (ROUGH) zt[k] += ex2((x - m) * (scale * (1.f / PER_OCTAVE)));
    if (MASS) mass += w.fine(x);
    if (HIST) {
      const int b = octave_bin(x, m, scale);
      if (b < OCTAVES - 1) atomicAdd(&sh.octaves_here[b], 1u);
    }
  };
  int i = seg.a + lane;
  for (; i + 96 < seg.b; i += 128) {
    const float x0 = xs[i], x1 = xs[i + 32], x2 = xs[i + 64], x3 = xs[i + 96];
    one(x0, 0); one(x1, 1); one(x2, 2); one(x3, 3);
  }
  for (; i < seg.b; i += 32) one(xs[i], 0);
  const int count = max(0, (seg.b - seg.a - lane + 31) >> 5);
  z = warp_sum(z);
  if (lane == 0) sh.z[warp] = z;
  if (ROUGH) { const float t = warp_sum((zt[0] + zt[1]) + (zt[2] + zt[3])); if (lane == 0) sh.zt[warp] = t; }
  if (PRI == PRI_ENTROPY) { ent = warp_sum(ent); if (lane == 0) sh.ent[warp] = ent; }
  if (PRI == PRI_MARGIN) {
    second = warp_max(second);
    at_max = __reduce_add_sync(0xffffffffu, at_max);
    if (lane == 0) { sh.ent[warp] = second; sh.at_max[warp] = at_max; }
  }
  if (MASS) {
    mass -= (u64)count * (u64)__double_as_longlong(w.magic);
    if (w.coarse) {                                                // the same for the whole row
      mass = 0;
      for (int k = seg.a + lane; k < seg.b; k += 32) mass += w(xs[k]);
    }
    mass = warp_sum(mass);
    if (lane == 0) sh.mass[warp] = mass;
  }
}

template <int WARPS, bool MASS, bool HIST, bool ROUGH>
__device__ __forceinline__ void whole_pass(int pri, Shared& sh, const float* xs, Segment seg, float m, float scale, const Weigher& w) {
  if (pri == PRI_LOGP) whole_pass<WARPS, MASS, HIST, ROUGH, PRI_LOGP>(sh, xs, seg, m, scale, w);
  else if (pri == PRI_MARGIN) whole_pass<WARPS, MASS, HIST, ROUGH, PRI_MARGIN>(sh, xs, seg, m, scale, w);
  else whole_pass<WARPS, MASS, HIST, ROUGH, PRI_ENTROPY>(sh, xs, seg, m, scale, w);
}

__device__ __forceinline__ unsigned int cluster_id() {
  unsigned int r;
  asm("mov.u32 %0, %%clusterid.x;" : "=r"(r));
  return r;
}

// By one warp: log of the untempered sum, and the priority where it is not the log-probability.
template <int WARPS>
__device__ __forceinline__ float2 untempered(const SampleParams& p, Shared& sh, int lane, float m) {
  const double z = warp_sum(warp_values<WARPS>(sh, lane, 0.0, [](double v, const Shared& q, int k) { return v + (double)q.z[k]; }));
  const float logz = logf((float)z);
  float pr = 0.f;
  if (p.priority == PRI_MARGIN) {
    const float second = warp_max(warp_values<WARPS>(sh, lane, -INFINITY, [](float v, const Shared& q, int k) { return fmaxf(v, q.ent[k]); }));
    const int at_max = __reduce_add_sync(0xffffffffu, warp_values<WARPS>(sh, lane, 0, [](int v, const Shared& q, int k) { return v + q.at_max[k]; }));
    pr = at_max > 1 ? 0.f : (float)((1.0 - (double)__expf(second - m)) / z);
  } else if (p.priority == PRI_ENTROPY) {
    const double ent = warp_sum(warp_values<WARPS>(sh, lane, 0.0, [](double v, const Shared& q, int k) { return v + (double)q.ent[k]; }));
    pr = (float)(ent * 0.6931471805599453 / z - (double)logz);
  }
  return make_float2(logz, pr);
}

// A row of global memory as chunks of 1024 elements that start at 16-byte boundaries; the first may be short.
constexpr int CHUNK = 1024;
template <class T>
struct RowView {
  const T* src;
  const float* bias;
  int mis, chunks;
  __device__ __forceinline__ RowView(const SampleParams& p, unsigned int row) {
    const unsigned int outer = row / (unsigned int)p.inner;
    src = reinterpret_cast<const T*>(p.logits) + outer * p.s_outer + (row - outer * (unsigned int)p.inner) * p.s_inner;
    bias = p.bias ? p.bias + (long long)outer * p.V : nullptr;
    constexpr int VEC = 16 / (int)sizeof(T);
    mis = (int)((reinterpret_cast<uintptr_t>(src) / sizeof(T)) % VEC);
    chunks = (mis + p.V + CHUNK - 1) / CHUNK;
  }
  // the lane's elements of chunk c: pieces of 16 bytes, 32 lanes side by side; -inf where the row has none.  Element k of them has index
  // c CHUNK - mis + ((k / VEC) 32 + lane) VEC + k % VEC.
  __device__ __forceinline__ void load(int V, int c, int lane, float (&x)[32]) const {
    constexpr int VEC = 16 / (int)sizeof(T), PIECES = 32 / VEC;
    const int at0 = c * CHUNK - mis + lane * VEC;
    uint4 raw[PIECES];
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int at = at0 + j * 32 * VEC;
      if (at >= 0 && at + VEC <= V) {
        raw[j] = __ldcs(reinterpret_cast<const uint4*>(src + at));
      } else {
        T e[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) e[k] = at + k >= 0 && at + k < V ? src[at + k] : T(-INFINITY);
        raw[j] = *reinterpret_cast<const uint4*>(e);
      }
    }
#pragma unroll
    for (int j = 0; j < PIECES; ++j)
#pragma unroll
      for (int k = 0; k < VEC; ++k) x[j * VEC + k] = to_f32(reinterpret_cast<const T*>(&raw[j])[k]);
    if (bias) {
#pragma unroll
      for (int j = 0; j < PIECES; ++j)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const int i = at0 + j * 32 * VEC + k;
          if (i >= 0 && i < V) x[j * VEC + k] += __ldg(bias + i);
        }
    }
  }
};

// The row's end where no more than FEW elements lie in the octaves that hold the kept ones: all CTAs push theirs into the list of CTA
// 0 and leave; it ranks them against one another (by value, then index), which gives every cut at once, and draws.  The pushes come
// in any order and nothing depends on it.
struct Candidate { float x; int i; };
static_assert(sizeof(Shared::hmass) + sizeof(Shared::count) >= FEW * sizeof(Candidate), "the candidate list takes the histograms' place");
//
// The goal of top-p is a part of the mass of all elements, of which the caller has a 32-bit sum.  What the kept set is follows from
// it, except where a border lies in the few 1e-5 that it leaves open: then CTA 0 reads the row once more and adds up the masses.
constexpr double ROUGH_ERROR = 1e-5;
template <class T, int WARPS>
__device__ __noinline__ void few_candidates(const SampleParams& p, Shared& sh, const float* xs, Segment seg, int first, unsigned int row, float m,
                                            float scale, const Weigher& w_in, int top_k, double top_p, float least) {
  const Weigher w = w_in;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, me = (int)cluster.block_rank();
  Shared* home = cluster.map_shared_rank(&sh, 0);
  Candidate* list = reinterpret_cast<Candidate*>(&home->hmass[0][0]);
  const int last = sh.last_bin, n = sh.candidates;
  const bool all = top_k >= p.V;                                   // the goal is a part of every element's mass
  const float lo = key_value(sh.range[0]);                         // not above any element of the octaves
  for (int i0 = seg.a; i0 < seg.b; i0 += 256) {
    float x[8];
    float most = -INFINITY;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = i0 + k * 32 + lane;
      x[k] = i < seg.b ? xs[i] : -INFINITY;
      most = fmaxf(most, x[k]);
    }
    if (!__any_sync(0xffffffffu, most >= lo)) continue;
    unsigned int in = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (octave_bin(x[k], m, scale) <= last) in |= 1u << k;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const unsigned int any = __ballot_sync(0xffffffffu, in >> k & 1);
      if (!any) continue;
      int at = 0;
      if (lane == 0) at = atomicAdd(&home->pushed, __popc(any));
      at = __shfl_sync(0xffffffffu, at, 0) + __popc(any & ((1u << lane) - 1));
      if ((in >> k & 1) && at < FEW) list[at] = {x[k], first + i0 + k * 32 + lane};
    }
  }
  if (me == 0 && warp == 1) {                                      // the others' sums, before they leave
    const float2 t = untempered<WARPS>(p, sh, lane, m);
    if (lane == 0) { sh.logz = t.x; sh.pr = t.y; }
  }
  cluster.sync();
  if (me != 0) return;
  // a candidate per thread (or two): its place in the order and the mass before it
  constexpr int THREADS = WARPS * 32, EACH = (FEW + THREADS - 1) / THREADS;
  u64* mass = sh.few_mass;
  u64 before[EACH], upto[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e)
    if (tid + e * THREADS < n) mass[tid + e * THREADS] = w(list[tid + e * THREADS].x);
  __syncthreads();
  int rank[EACH];
  u64 topped = 0;                                                  // the mass of the first top_k
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int j = tid + e * THREADS;
    before[e] = 0; rank[e] = 0;
    if (j < n) {
      const Candidate c = list[j];
#pragma unroll 4
      for (int o = 0; o < n; ++o) {
        const Candidate q = list[o];
        const bool ahead = q.x > c.x || (q.x == c.x && q.i < c.i);
        rank[e] += ahead;
        before[e] += ahead ? mass[o] : 0;
      }
      if (rank[e] < top_k) topped += mass[j];
    }
  }
  topped = warp_sum(topped);
  if (lane == 0) sh.sub[warp] = topped;
  __syncthreads();
  auto target_of = [&](u64 whole) { return max((u64)1, min(whole, (u64)ceil(fmax(top_p, 0.0) * (double)whole))); };
  u64 whole = 0, goal = 0;
  if (!all) {
    for (int k = 0; k < WARPS; ++k) whole += sh.sub[k];
    goal = target_of(whole);
    __syncthreads();
  } else {
    const double rough = sh.rough * (double)(1ull << p.scale_bits), off = rough * ROUGH_ERROR + p.V;
    goal = target_of((u64)fmax(rough - off, 0.0));
    const u64 goal_hi = target_of((u64)(rough + off));
    bool open = false;
#pragma unroll
    for (int e = 0; e < EACH; ++e) open |= tid + e * THREADS < n && before[e] >= goal && before[e] < goal_hi;
    if (__syncthreads_or(open)) {
      const RowView<T> view(p, row);
      for (int c = warp; c < view.chunks; c += WARPS) {
        float x[32];
        view.load(p.V, c, lane, x);
#pragma unroll 8
        for (int k = 0; k < 32; ++k) whole += w(x[k]);
      }
      whole = warp_sum(whole);
      if (lane == 0) sh.sub[warp] = whole;
      __syncthreads();
      whole = 0;
      for (int k = 0; k < WARPS; ++k) whole += sh.sub[k];
      goal = target_of(whole);
      __syncthreads();
    }
  }
  u64 kept = 0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int j = tid + e * THREADS;
    if (j < n) {
      if (!(rank[e] < top_k && (top_p >= 1.0 || before[e] < goal) && list[j].x >= least)) mass[j] = 0;
      kept += mass[j];
    }
  }
  kept = warp_sum(kept);
  if (lane == 0) sh.sub[warp] = kept;
  __syncthreads();
  u64 total = 0;
  for (int k = 0; k < WARPS; ++k) total += sh.sub[k];
  const double u = (double)sh.u;
  const u64 want = min(u > 0 ? (u64)(fmin(u, 1.0) * (double)total) : 0, total - 1);
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    const int j = tid + e * THREADS;
    if (j < n && mass[j]) {
      const Candidate c = list[j];
      upto[e] = 0;                                                 // in order of the indices
#pragma unroll 4
      for (int o = 0; o < n; ++o) upto[e] += list[o].i <= c.i ? mass[o] : 0;
      if (upto[e] > want && upto[e] - mass[j] <= want) {
        p.tokens[row] = c.i;
        p.logp[row] = (c.x - m) - sh.logz;
        if (p.priority != PRI_LOGP) p.prio[row] = sh.pr;
      }
    }
  }
}

// The draw of a row whose goal is less than a unit of mass for every element: with masses as doubles, in order of the indices, over
// all CTAs of the row.  `kept` as the caller has it.
template <int WARPS>
__device__ __noinline__ void tiny_draw(const SampleParams& p, Shared& sh, const float* xs, Segment seg, int first, unsigned int row, float m,
                                       float least, float lo, float hi, int last_tie) {
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), me = (int)cluster.block_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto mass = [&](int i) {
    const float x = i < seg.b ? xs[i] : -INFINITY;
    return i < seg.b && x >= least && (x > hi || (x >= lo && i <= last_tie)) ? exp(((double)x - (double)m) / sh.temp) : 0.0;
  };
  double s = 0;
  for (int i = seg.a + lane; i < seg.b; i += 32) s += mass(i);
  s = warp_sum(s);
  if (lane == 0) sh.part[warp] = s;
  cluster.sync();
  double run = 0, total = 0;
  for (int e = 0; e < ranks * WARPS; ++e) {
    const double v = cluster.map_shared_rank(&sh, e / WARPS)->part[e % WARPS];
    if (e < me * WARPS + warp) run += v;
    total += v;
  }
  const double u = (double)sh.u, goal = u > 0 ? u * total : 0.0;
  if (!(run <= goal && run + s > goal)) return;                    // one warp's, as the sums before it are the same for all
  auto answer = [&](int i) {
    p.tokens[row] = first + i;
    p.logp[row] = (xs[i] - m) - sh.logz;
    if (p.priority != PRI_LOGP) p.prio[row] = sh.pr;
  };
  int last = -1;                                                   // with a mass: the answer where only a rounding is missing
  for (int i0 = seg.a; i0 < seg.b; i0 += 32) {
    double inc = mass(i0 + lane);
    if (inc > 0) last = i0 + lane;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    const unsigned int hit = __ballot_sync(0xffffffffu, run + inc > goal);
    if (hit) {
      if (lane == __ffs(hit) - 1) answer(i0 + lane);
      return;
    }
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
  last = __reduce_max_sync(0xffffffffu, last);
  if (lane == 0) answer(last);
}

static_assert(sizeof(Shared) <= 12600, "three CTAs with slices of 16032 elements (V = 128256) on an SM");

template <class T, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, WARPS == 4 ? 9 : WARPS == 8 ? 3 : 1) sample_kernel(const SampleParams p) {
  constexpr int THREADS = WARPS * 32;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  Shared& sh = *reinterpret_cast<Shared*>(smem_raw);
  float* xs = reinterpret_cast<float*>(smem_raw + ((sizeof(Shared) + 15) / 16) * 16);
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), me = (int)cluster.block_rank();
  const unsigned int row = cluster_id();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long outer = row / (unsigned int)p.inner;
  const int first = me * p.slice;
  const int n = max(0, min(p.slice, p.V - first));

  // ---- the slice into shared memory, its maximum
  const T* src = reinterpret_cast<const T*>(p.logits) + outer * p.s_outer + (row - outer * p.inner) * p.s_inner + first;
  const float* bias = p.bias ? p.bias + outer * p.V + first : nullptr;
  constexpr int VEC = 16 / (int)sizeof(T), UNROLL = sizeof(T) == 4 ? 4 : 2;
  const int mis = (int)((reinterpret_cast<uintptr_t>(src) / sizeof(T)) % VEC);      // keeps 16-byte pieces aligned on both sides
  const int v0 = mis ? 1 : 0, v1 = (mis + n) / VEC;                                 // the whole pieces
  const bool bias_vec = bias && ((reinterpret_cast<uintptr_t>(bias) / sizeof(float) + VEC - mis) & 3) == 0;
  if (tid == 0) {
    const double t = p.t_row ? (double)p.t_row[row] : p.temperature;
    sh.greedy = !(t > 0);
    sh.temp = fmin(fmax(t, 1e-6), 1e6);
    sh.min_p = p.m_row ? (double)p.m_row[row] : p.min_p;
    sh.top_p = p.p_row ? (double)p.p_row[row] : p.top_p;
    sh.top_k = p.k_row ? p.k_row[row] : p.top_k;
    sh.log2e_t = 1.4426950408889634 / sh.temp;
    sh.cut = (p.scale_bits + 1.5) / sh.log2e_t;
    sh.scale = (float)(PER_OCTAVE * sh.log2e_t);
    sh.u = p.u[row];
    for (int b = 0; b < 2; ++b) { sh.above_count[b] = 0; sh.above_mass[b] = 0; }
    sh.pushed = 0;
    sh.all_mass = 0;
  }
  float mx = -INFINITY;
  for (int v = v0 + tid; v < v1; v += THREADS * UNROLL) {
    uint4 raw[UNROLL];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k)
      if (v + k * THREADS < v1) raw[k] = __ldcs(reinterpret_cast<const uint4*>(src - mis) + v + k * THREADS);
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) {
      const int at = (v + k * THREADS) * VEC;
      if (v + k * THREADS < v1) {
        const T* e = reinterpret_cast<const T*>(&raw[k]);
        float x[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[j] = to_f32(e[j]);
        if (bias_vec) {
#pragma unroll
          for (int j = 0; j < VEC; j += 4) {
            const float4 t = __ldg(reinterpret_cast<const float4*>(bias + at - mis + j));
            x[j] += t.x; x[j + 1] += t.y; x[j + 2] += t.z; x[j + 3] += t.w;
          }
        } else if (bias) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) x[j] += __ldg(bias + at - mis + j);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) { x[j] += 0.f; mx = max_nan(mx, x[j]); }       // + 0: no negative zero
#pragma unroll
        for (int j = 0; j < VEC; j += 4) *reinterpret_cast<float4*>(xs + at + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
      }
    }
  }
  if (tid < 2 * VEC) {                                             // the ragged ends, an element each
    const int head = v0 ? min(n, VEC - mis) : 0, tail = max(head, v1 * VEC - mis);
    const int i = tid < VEC ? tid : tail + tid - VEC;
    if (tid < VEC ? i < head : i < n) {
      float x = to_f32(src[i]);
      if (bias) x += bias[i];
      x += 0.f;
      mx = max_nan(mx, x);
      xs[mis + i] = x;
    }
  }
  xs += mis;
  for (int i = tid; i < OCTAVES; i += WARPS * 32) sh.octaves_here[i] = 0;
  for (int i = tid; i < BINS; i += WARPS * 32) { sh.count[0][i] = 0; sh.hmass[0][i] = 0; }
  for (int i = tid; i < TAB * COPIES; i += WARPS * 32) sh.tab[i] = ROOTS[i / COPIES];
  mx = warp_max_nan(mx);
  if (lane == 0) sh.fred[warp] = mx;
  __syncthreads();
  if (warp == 0) { mx = warp_max_nan(lane < WARPS ? sh.fred[lane] : -INFINITY); if (lane == 0) sh.m = mx; }
  cluster.sync();
  const float m = warp_max_nan(lane < ranks ? cluster.map_shared_rank(&sh, lane)->m : -INFINITY);
  if (!(m > -INFINITY && m < INFINITY)) {                          // NaN, +inf or nothing above -inf: the same in every CTA of the cluster
    if (me == 0 && tid == 0) { p.tokens[row] = -1; p.logp[row] = NAN; if (p.priority != PRI_LOGP) p.prio[row] = NAN; }
    cluster.sync();
    return;
  }

  // ---- this row's parameters
  const bool greedy = sh.greedy;
  const double min_p = sh.min_p, top_p = sh.top_p;
  const int top_k = sh.top_k;
  const bool by_count = !greedy && top_k > 0 && top_k < p.V, by_mass = !greedy && top_p < 1.0, by_ratio = !greedy && min_p > 0;
  const float scale = sh.scale;
  const Weigher w(sh.log2e_t, m, sh.cut, p.scale_bits, sh.tab + (lane & (COPIES - 1)));

  // ---- the pass over every element
  const Segment seg = split(0, n, WARPS, warp);
  if (greedy) whole_pass<WARPS, false, false, false>(p.priority, sh, xs, seg, m, scale, w);
  else if (by_count) whole_pass<WARPS, false, true, false>(p.priority, sh, xs, seg, m, scale, w);
  else if (by_mass) whole_pass<WARPS, false, true, true>(p.priority, sh, xs, seg, m, scale, w);
  else if (by_ratio) whole_pass<WARPS, false, false, false>(p.priority, sh, xs, seg, m, scale, w);
  else whole_pass<WARPS, true, false, false>(p.priority, sh, xs, seg, m, scale, w);

  // ---- the kept set and its mass
  Cut cut;
  cut.lo = cut.hi = cut.first_hi = -INFINITY; cut.ties = 1; cut.before = 0; cut.here = 0; cut.mass = 0;
  float least = -INFINITY;
  int last_tie = 0x7fffffff, round = 0;
  auto kept = [&](float x, int i) { return x >= least && (x > cut.hi || (x >= cut.lo && i <= last_tie)); };
  if (greedy) {
    int at = 0x7fffffff;
    for (int i = seg.a + lane; i < seg.b; i += 32)
      if (xs[i] == m) { at = first + i; break; }
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) sh.first_max[warp] = at;
  } else if (by_count || by_mass || by_ratio) {
    if (by_ratio) least = __double2float_ru((double)m + sh.temp * log(fmin(min_p, 1.0)));
    if (by_count || by_mass) {
      cluster.sync();
      for (int i = tid; i < OCTAVES; i += WARPS * 32)
        sh.octaves[i] = over_ranks<unsigned int>(sh, [&](const Shared& q) { return q.octaves_here[i]; });
      if (warp == WARPS - 1 && !by_count) {
        const double t = warp_sum(warp_values<WARPS>(sh, lane, 0.0, [](double v, const Shared& q, int k) { return v + (double)q.zt[k]; }));
        if (lane == 0) sh.rough = t;
      }
      __syncthreads();
      const double unit = 1.0 / (double)(1ull << p.scale_bits);
      const float slack = (float)((double)(p.V + 1) * unit);       // masses are rounded to units
      if (by_count) first_range<false>(sh, m, scale, (float)top_k, 0.f);
      else first_range<true>(sh, m, scale, (float)(fmin(fmax(top_p, 0.0), 1.0) * sh.rough), slack);
      if (sh.candidates <= FEW) {
        few_candidates<T, WARPS>(p, sh, xs, seg, first, row, m, scale, w, by_count ? top_k : p.V, by_mass ? top_p : 2.0, least);
        return;
      }
      auto target_of = [&](u64 whole) { return max((u64)1, min(whole, (u64)ceil(fmax(top_p, 0.0) * (double)whole))); };
      if (by_count) {
        cut = find_cut<WARPS, false, false>(sh, xs, n, w, (u64)top_k, target_of, round);
        if (by_mass) {
          const u64 target = target_of(cut.mass);
          first_range<true>(sh, m, scale, (float)((double)target * unit), slack);
          cut = find_cut<WARPS, true, false>(sh, xs, n, w, target, target_of, round);
        }
      } else {
        cut = find_cut<WARPS, true, true>(sh, xs, n, w, 0, target_of, round);
      }
    }
    if (cut.before + cut.here > cut.ties) {                        // this CTA holds ties that are not kept
      if (cut.before >= cut.ties) {
        last_tie = -1;
      } else {
        // the (ties - before)-th element of [lo, hi] in this slice
        const u64 want = cut.ties - cut.before;
        int c = 0;
        for (int i = seg.a + lane; i < seg.b; i += 32) c += xs[i] >= cut.lo && xs[i] <= cut.hi;
        c = __reduce_add_sync(0xffffffffu, c);
        if (lane == 0) sh.ties[warp] = c;
        __syncthreads();
        u64 run = 0;
        for (int i = 0; i < warp; ++i) run += sh.ties[i];
        if (run < want && run + sh.ties[warp] >= want) {
          for (int i0 = seg.a; i0 < seg.b; i0 += 32) {
            const int i = i0 + lane;
            const unsigned int hit = __ballot_sync(0xffffffffu, i < seg.b && xs[i] >= cut.lo && xs[i] <= cut.hi);
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
    // what lies above the search's first range is summed already, unless min_p cuts into it
    const bool summed = (by_count || by_mass) && least <= cut.first_hi;
    u64 s = 0;
    if (summed) {
      for_range<WARPS>(sh, xs, seg, warp, lane, [&](float x, int i, bool in) { if (in && x <= cut.first_hi && kept(x, i)) s += w(x); });
      s = warp_sum(s) + sh.above[warp];
    } else {
      for (int i = seg.a + lane; i < seg.b; i += 32)
        if (kept(xs[i], i)) s += w(xs[i]);
      s = warp_sum(s);
    }
    if (lane == 0) sh.mass[warp] = s;
  }
  cluster.sync();

  // ---- totals of the cluster, the draw
  if (warp == 0) {
    if (greedy) {
      const int at = __reduce_min_sync(0xffffffffu, warp_values<WARPS>(sh, lane, 0x7fffffff, [](int v, const Shared& q, int k) { return min(v, q.first_max[k]); }));
      if (me == 0 && lane == 0) p.tokens[row] = at;
    } else {
      const u64 part = warp_values<WARPS>(sh, lane, (u64)0, [](u64 v, const Shared& q, int k) { return v + q.mass[k]; });
      const u64 upto = warp_scan(part, lane), total = __shfl_sync(0xffffffffu, upto, 31);
      const int each = WARPS / max(1, ranks * WARPS / 32);           // lanes to a CTA
      const u64 base = __shfl_sync(0xffffffffu, upto - part, me * each);
      const u64 end = __shfl_sync(0xffffffffu, upto, (me + 1) * each - 1);
      if (lane == 0) {
        const double u = (double)sh.u;
        const u64 goal = u > 0 ? (u64)(fmin(u, 1.0) * (double)total) : 0;
        sh.goal = min(goal, total - 1);
        sh.tiny = goal < (u64)p.V;
        sh.base = base; sh.mine = end - base;
      }
    }
  } else if (warp == 1) {
    const float2 t = untempered<WARPS>(p, sh, lane, m);
    const float logz = t.x, pr = t.y;
    if (lane == 0) {
      sh.logz = logz; sh.pr = pr;
      if (greedy && me == 0) {
        p.logp[row] = -logz;
        if (p.priority != PRI_LOGP) p.prio[row] = pr;
      }
    }
  }
  __syncthreads();
  const bool tiny = !greedy && sh.tiny;                            // the same in every CTA of the row
  if (tiny) tiny_draw<WARPS>(p, sh, xs, seg, first, row, m, least, cut.lo, cut.hi, last_tie);
  __syncwarp();
  cluster.barrier_arrive();                                        // nothing of a peer's memory is read any more
  if (!greedy && !tiny) {
    const u64 goal = sh.goal, base = sh.base;
    auto answer = [&](int tok, float x) {
      p.tokens[row] = tok;
      p.logp[row] = (x - m) - sh.logz;
      if (p.priority != PRI_LOGP) p.prio[row] = sh.pr;
    };
    if (goal >= base && goal < base + sh.mine) {                   // the draw falls into this slice
      u64 run = base;
      int own = 0;
      while (own < WARPS - 1 && run + sh.mass[own] <= goal) run += sh.mass[own++];
      const Segment big = split(0, n, WARPS, own);
      const Segment part = split(big.a, big.b, WARPS, warp);
      u64 s = 0;
      for (int i = part.a + lane; i < part.b; i += 32)
        if (kept(xs[i], i)) s += w(xs[i]);
      s = warp_sum(s);
      if (lane == 0) sh.sub[warp] = s;
      __syncthreads();
      for (int i = 0; i < warp; ++i) run += sh.sub[i];
      if (goal >= run && goal < run + s) {
        for (int i0 = part.a; i0 < part.b; i0 += 32) {
          const int i = i0 + lane;
          const u64 wi = i < part.b && kept(xs[i], i) ? w(xs[i]) : 0;
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
  __syncwarp();
  cluster.barrier_wait();                                          // nobody leaves while a peer may still read its memory
}

// ------------------------------------------------------------------------------------------------ the untruncated draw
// Without top-k, top-p and min-p nothing has to wait for the row's maximum: a warp reads a chunk of 1024 elements into registers,
// takes the chunk's own maximum, and leaves the chunk's sums relative to it (the masses as integers, as above).  A second launch, a
// warp per row, brings them to the row's maximum in 64 bits, finds the chunk that holds the draw and reads it once more.
constexpr int CHUNK_BITS = 50;                    // 1024 2^50 <= 2^62
// A draw takes two launches from 6.2 million elements on, for vocabularies above 4096.  One / two, us (f32; bf16 within
// 10 %; of 30 sizes in both types the form chosen here is at most 2 us slower than the other one):
//   V = 128256: 8 rows 12.3 / 20.0, 32 rows 21.8 / 25.2, 48 rows (6.16 million) 26.4 / 28.7, 64 rows 37.1 / 30.8, 96 rows 45.4 / 35.7
//   V = 390001: 8 rows 23.9 / 28.0, 16 rows (6.24 million) 55.3 / 32.8    V = 50257: 64 rows 19.2 / 22.0, 128 rows (6.43) 32.8 / 27.7
//   V = 32000: 192 rows 26.4 / 26.7, 256 rows 36.5 / 28.7    V = 16384: 256 rows 20.5 / 23.3, 512 rows 37.1 / 28.7
//   V = 8192: 512 rows 26.1 / 24.6, 1024 rows 39.0 / 30.8    V = 4096: 1024 rows 22.6 / 24.3, 2048 rows 39.0 / 39.2
//   V = 2048: 4096 rows 49.2 / 58.9    V = 1000: 16384 rows 145.5 / 175.5 (a chunk of 1024 is mostly empty, and a row has its own second warp)
constexpr long long STREAM_LEAST = 6200000;
constexpr int STREAM_VOCAB = 4096;

struct __align__(16) Chunk {
  float m, z, e;               // maximum (NaN or +inf if there is one), sum of exp(x - m), the priority's own value
  int at_max;                  // elements at the maximum (margin)
  u64 mass;
  int first, pad;              // index of the first element at the maximum
};

__device__ __forceinline__ double row_temperature(const SampleParams& p, unsigned int row) {
  const double t = p.t_row ? (double)p.t_row[row] : p.temperature;
  return t > 0 ? fmin(fmax(t, 1e-6), 1e6) : 0.0;                   // 0: greedy
}

// the masses of one chunk, relative to its maximum
__device__ __forceinline__ Weigher chunk_weigher(double temp, float m, const double* tab) {
  const double log2e_t = 1.4426950408889634 / temp;
  return Weigher(log2e_t, m, (CHUNK_BITS + 1.5) / log2e_t, CHUNK_BITS, tab);
}

constexpr int STREAM_THREADS = 256;

template <class T, int PRI>
__global__ void __launch_bounds__(STREAM_THREADS, 3) chunk_kernel(const SampleParams p, unsigned int rows, unsigned int most, Chunk* __restrict__ out) {
  __shared__ double tab[TAB * COPIES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < TAB * COPIES; i += STREAM_THREADS) tab[i] = ROOTS[i / COPIES];
  __syncthreads();
  const unsigned int all = rows * most, step = gridDim.x * (STREAM_THREADS / 32);      // below 2^31 (the launcher)
  for (unsigned int t = blockIdx.x * (STREAM_THREADS / 32) + warp; t < all; t += step) {
    const unsigned int row = t / most;
    const int c = (int)(t - row * most);
    const RowView<T> view(p, row);
    if (c >= view.chunks) continue;
    const double temp = row_temperature(p, row);
    float x[32];
    view.load(p.V, c, lane, x);
    float m = x[0];
#pragma unroll
    for (int k = 1; k < 32; ++k) m = max_nan(m, x[k]);
    m = warp_max_nan(m);
    Chunk r = {m, 0.f, PRI == PRI_MARGIN ? -INFINITY : 0.f, 0, 0, 0x7fffffff, 0};
    if (m > -INFINITY && m < INFINITY) {
      float z = 0, e = r.e;
      int n = 0;
      if (PRI == PRI_ENTROPY || temp != 1.0) {                     // at T = 1 the masses are these exponentials
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const float y = (x[k] - m) * 1.44269504f, v = ex2(y);
          z += v;
          if (PRI == PRI_ENTROPY) e = fmaf(v, fmaxf(y, -1e4f), e);
        }
        r.z = warp_sum(z);
      }
      if (PRI == PRI_MARGIN) {
#pragma unroll
        for (int k = 0; k < 32; ++k) { n += x[k] == m; e = x[k] < m ? fmaxf(e, x[k]) : e; }
      }
      if (PRI == PRI_ENTROPY) r.e = warp_sum(e);
      if (PRI == PRI_MARGIN) { r.e = warp_max(e); r.at_max = __reduce_add_sync(0xffffffffu, n); }
      if (temp > 0) {
        const Weigher w = chunk_weigher(temp, m, tab + (lane & (COPIES - 1)));
        u64 mass = 0;
        if (w.coarse) {
#pragma unroll
          for (int k = 0; k < 32; ++k) mass += w(x[k]);
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) mass += w.fine(x[k]);
          mass -= 32 * (u64)__double_as_longlong(w.magic);
        }
        r.mass = warp_sum(mass);
        if (PRI != PRI_ENTROPY && temp == 1.0) r.z = (float)((double)r.mass * (1.0 / (double)(1ull << CHUNK_BITS)));
      } else {
        constexpr int VEC = 16 / (int)sizeof(T);
        int at = 0x7fffffff;
#pragma unroll
        for (int k = 31; k >= 0; --k)
          if (x[k] == m) at = c * CHUNK - view.mis + ((k / VEC) * 32 + lane) * VEC + k % VEC;
        r.first = __reduce_min_sync(0xffffffffu, at);
      }
    }
    if (lane == 0) out[t] = r;
  }
}

// The draw inside a chunk where less than a unit of mass for every element is left: masses as doubles, relative to the row's maximum,
// in order of the indices.  By one warp.
template <class T>
__device__ __noinline__ void tiny_chunk_draw(const SampleParams& p, unsigned int row, int chunk, float m, double temp, double left, float logz,
                                             float pr) {
  const RowView<T> view(p, row);
  const int lane = threadIdx.x & 31, start = max(0, chunk * CHUNK - view.mis), end = min(p.V, (chunk + 1) * CHUNK - view.mis);
  auto value = [&](int i) {
    if (i >= end) return -INFINITY;
    const float x = to_f32(view.src[i]);
    return view.bias ? x + view.bias[i] : x;
  };
  auto answer = [&](int i) {
    p.tokens[row] = i;
    p.logp[row] = (value(i) - m) - logz;
    if (p.priority != PRI_LOGP) p.prio[row] = pr;
  };
  double run = 0;
  int last = -1;                                                   // with a mass: the answer where only a rounding is missing
  for (int i0 = start; i0 < end; i0 += 32) {
    double inc = exp(((double)value(i0 + lane) - (double)m) / temp);
    if (inc > 0) last = i0 + lane;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double t = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += t;
    }
    const unsigned int hit = __ballot_sync(0xffffffffu, run + inc > left);
    if (hit) {
      if (lane == __ffs(hit) - 1) answer(i0 + lane);
      return;
    }
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
  last = __reduce_max_sync(0xffffffffu, last);
  if (lane == 0) answer(last);
}

// A warp per row.
template <class T>
__global__ void __launch_bounds__(32) chunk_draw_kernel(const __grid_constant__ SampleParams p, int most, const Chunk* __restrict__ in) {
  __shared__ double tab[TAB * COPIES];
  const int lane = threadIdx.x;
  const unsigned int row = blockIdx.x;
  const RowView<T> view(p, row);
  const Chunk* r = in + (long long)row * most;
  const double temp = row_temperature(p, row), u = (double)p.u[row];
  for (int i = lane; i < TAB * COPIES; i += 32) tab[i] = ROOTS[i / COPIES];
  __syncwarp();
  const int per = (view.chunks + 31) / 32, c0 = min(view.chunks, lane * per), c1 = min(view.chunks, c0 + per);      // in order over the lanes
  float m = -INFINITY;
  for (int c = c0; c < c1; ++c) m = max_nan(m, r[c].m);
  m = warp_max_nan(m);
  if (!(m > -INFINITY && m < INFINITY)) {
    if (lane == 0) { p.tokens[row] = -1; p.logp[row] = NAN; if (p.priority != PRI_LOGP) p.prio[row] = NAN; }
    return;
  }
  // everything relative to the row's maximum, in 64 bits
  double z = 0, ent = 0, mass = 0;
  float second = -INFINITY;
  int at_max = 0, first = 0x7fffffff;
  for (int c = c0; c < c1; ++c) {
    const Chunk q = r[c];
    if (q.m == -INFINITY) continue;
    const double d = (double)q.m - (double)m, f = exp(d);
    z += (double)q.z * f;
    if (p.priority == PRI_ENTROPY) ent += ((double)q.e * 0.6931471805599453 + (double)q.z * d) * f;      // sum e^(x - m) (x - m)
    if (p.priority == PRI_MARGIN) {
      second = fmaxf(second, q.m == m ? q.e : q.m);
      if (q.m == m) at_max += q.at_max;
    }
    if (temp > 0) mass += (double)q.mass * exp(d / temp);
    else if (q.m == m) first = min(first, q.first);
  }
  z = warp_sum(z);
  const float logz = logf((float)z);
  float pr = 0.f;
  if (p.priority == PRI_MARGIN) {
    second = warp_max(second);
    at_max = __reduce_add_sync(0xffffffffu, at_max);
    pr = at_max > 1 ? 0.f : (float)((1.0 - (double)__expf(second - m)) / z);
  } else if (p.priority == PRI_ENTROPY) {
    pr = (float)(warp_sum(ent) / z - (double)logz);
  }
  auto answer = [&](int tok, float x) {
    p.tokens[row] = tok;
    p.logp[row] = (x - m) - logz;
    if (p.priority != PRI_LOGP) p.prio[row] = pr;
  };
  if (!(temp > 0)) {
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) answer(first, m);
    return;
  }
  double upto = mass;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double t = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += t;
  }
  // the sum before a lane comes from the lane before it: upto - mass would lose what is small beside the lane's own mass
  const double up = __shfl_up_sync(0xffffffffu, upto, 1), before = lane ? up : 0.0;
  const double total = __shfl_sync(0xffffffffu, upto, 31), goal = u > 0 ? fmin(u, 1.0) * total : 0.0;
  // the first lane, and its first chunk, whose running mass exceeds the goal; rounding at the very end: the last chunk with a mass
  const unsigned int past = __ballot_sync(0xffffffffu, upto > goal), some = __ballot_sync(0xffffffffu, mass > 0);
  const int own = past & some ? __ffs(past & some) - 1 : 31 - __clz(some);
  int chunk = -1;
  double rest = 0, left = 0;
  if (lane == own) {
    double run = before;
    for (int c = c0; c < c1; ++c) {
      const Chunk q = r[c];
      if (q.m == -INFINITY || q.mass == 0) continue;
      const double f = exp(((double)q.m - (double)m) / temp), v = (double)q.mass * f;
      if (!(v > 0)) continue;
      chunk = c;
      left = goal - run;
      rest = left / f;
      if (run + v > goal) break;
      run += v;
    }
  }
  chunk = __shfl_sync(0xffffffffu, chunk, own);
  rest = __shfl_sync(0xffffffffu, rest, own);
  if (rest < CHUNK) {
    left = __shfl_sync(0xffffffffu, left, own) * (1.0 / (double)(1ull << CHUNK_BITS));
    tiny_chunk_draw<T>(p, row, chunk, m, temp, left, logz, pr);
    return;
  }
  const u64 held = r[chunk].mass;
  const u64 want = min(rest > 0 ? (u64)rest : 0, held - 1);
  const float mc = r[chunk].m;
  const Weigher w = chunk_weigher(temp, mc, tab + (lane & (COPIES - 1)));
  float x[32];
  view.load(p.V, chunk, lane, x);
  constexpr int VEC = 16 / (int)sizeof(T), PIECES = 32 / VEC;
  u64 run = 0;
  for (int j = 0; j < PIECES; ++j) {
    u64 s = 0;
#pragma unroll
    for (int jj = 0; jj < PIECES; ++jj)
      if (jj == j)
#pragma unroll
        for (int k = 0; k < VEC; ++k) s += w(x[jj * VEC + k]);
    const u64 inc = run + warp_scan(s, lane);
    const unsigned int hit = __ballot_sync(0xffffffffu, inc > want);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        u64 before = inc - s;
        bool done = false;
#pragma unroll
        for (int jj = 0; jj < PIECES; ++jj)
          if (jj == j)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
              before += w(x[jj * VEC + k]);
              if (!done && before > want) { done = true; answer(chunk * CHUNK - view.mis + (j * 32 + lane) * VEC + k, x[jj * VEC + k]); }
            }
      }
      break;
    }
    run = __shfl_sync(0xffffffffu, inc, 31);
  }
}

template <class T>
int launch_stream(const SampleParams& p, long long rows, Chunk* scratch, cudaStream_t s) {
  const int most = (p.V + 7 + CHUNK - 1) / CHUNK;
  const long long warps = rows * most, blocks = (warps + STREAM_THREADS / 32 - 1) / (STREAM_THREADS / 32);
  const int grid = (int)(blocks < 148 * 3 ? blocks : 148 * 3);
  if (p.priority == PRI_LOGP) chunk_kernel<T, PRI_LOGP><<<grid, STREAM_THREADS, 0, s>>>(p, (unsigned int)rows, most, scratch);
  else if (p.priority == PRI_MARGIN) chunk_kernel<T, PRI_MARGIN><<<grid, STREAM_THREADS, 0, s>>>(p, (unsigned int)rows, most, scratch);
  else chunk_kernel<T, PRI_ENTROPY><<<grid, STREAM_THREADS, 0, s>>>(p, (unsigned int)rows, most, scratch);
  chunk_draw_kernel<T><<<(unsigned int)rows, 32, 0, s>>>(p, most, scratch);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}

// Raises a kernel's shared memory limit once per device (`ready`: a bit per device).
template <class K>
cudaError_t allow_shared(K kernel, int bytes, std::atomic<u64>& ready) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && (ready.load() >> dev & 1))) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) ready.fetch_or(1ull << dev);
  return e;
}

template <class T, int WARPS>
int launch_sample(const SampleParams& p, long long rows, int ranks, cudaStream_t s) {
  const size_t smem = ((sizeof(Shared) + 15) / 16) * 16 + ((size_t)p.slice + 16) * sizeof(float);
  constexpr size_t most = ((sizeof(Shared) + 15) / 16) * 16 + ((size_t)SLICE_MAX + 16) * sizeof(float);
  static_assert(most <= 227 * 1024, "a slice has to fit the shared memory of an SM");
  static std::atomic<u64> ready{0};
  cudaError_t e = allow_shared(sample_kernel<T, WARPS>, (int)most, ready);
  if (e != cudaSuccess) return 1000 + (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned int)(rows * ranks));
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned int)ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, sample_kernel<T, WARPS>, p);
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}

// Warps to a CTA.  Sixteen while every CTA finds an SM of its own (clusters of eight: fourteen of them are resident at once),
// else eight, three CTAs to an SM; small slices, of which there are more than that, take four, so that fewer warps pay what a
// row costs apart from its elements.  Top-p, us with 16 / 8 / 4 warps:
//   V = 128256: 14 rows 14.5 / 18.6, 16 rows 24.7 / 18.6, 64 rows 57 / 38      V = 4000: 148 rows 12.4 / 12.4 / 16.5, 296 rows
//   22.6 / 14.5 / 16.7, 600 rows 47 / 26.8 / 23.0                               V = 1000: 600 rows 48 / 27 / 18.6
template <class T>
int launch_sample(const SampleParams& p, long long rows, int ranks, cudaStream_t s) {
  const long long ctas = rows * ranks;
  if (ctas <= (ranks == 8 ? 112 : 148)) return launch_sample<T, 16>(p, rows, ranks, s);
  if (p.slice <= SLICE_SMALL && ctas > 444) return launch_sample<T, 4>(p, rows, ranks, s);
  return launch_sample<T, 8>(p, rows, ranks, s);
}

// ------------------------------------------------------------------------------------------------------ unmask
// One block per row.  Rows of up to 1024 slots: a thread per slot, everything it needs loaded at once, and the key of the quota-th slot
// in rank order built bit by bit from counts over the block (32 barriers, about 1.5 us; latency is all there is to it).  Longer
// rows: a radix search over the order keys in shared memory.  Thread per slot / radix: 1 x 16 4.3 / 6.3 us, 1 x 1024 and 64 x 1024
// 6.3 / 10.4, 256 x 1024 10.4 / 10.3.
constexpr int UM_ROW = 1024;

__global__ void __launch_bounds__(UM_ROW) unmask_row_kernel(const long long* __restrict__ ids, const uint8_t* __restrict__ known,
                                                           const float* __restrict__ held, const long long* __restrict__ tokens,
                                                           const float* __restrict__ logp, const float* __restrict__ priority,
                                                           const long long* __restrict__ quota, const uint8_t* __restrict__ allowed,
                                                           float sure, int use_sure, long long* __restrict__ ids_out,
                                                           uint8_t* __restrict__ known_out, float* __restrict__ held_out,
                                                           uint8_t* __restrict__ where_out, int C) {
  __shared__ int warp_count[UM_ROW / 32];
  const int i = threadIdx.x, warp = i >> 5, lane = i & 31;
  const long long at = (long long)blockIdx.x * C + i;
  const bool in = i < C;
  const long long q = quota[blockIdx.x];
  bool is_known = true, ok = false;
  float pri = 0.f, lp = 0.f, was = 0.f;
  long long id = 0, token = 0;
  if (in) {
    is_known = known[at]; ok = allowed ? allowed[at] : true;
    pri = priority[at]; lp = logp[at]; was = held[at]; id = ids[at]; token = tokens[at];
  }
  const bool shut = is_known || !ok;
  const float v = shut ? -INFINITY : pri + 0.f;
  const uint32_t key = !in || v != v ? 0u : order_key(v);         // 0: NaN, and threads without a slot, which come after the slots
  bool take = q >= C;
  if (q > 0 && q < C) {
    const int want = (int)q;
    uint32_t least = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t cand = least | 1u << bit;
      if (__syncthreads_count(key >= cand) >= want) least = cand;
    }
    const int ties = want - __syncthreads_count(key > least);
    const unsigned int eq = __ballot_sync(0xffffffffu, in && key == least);
    if (lane == 0) warp_count[warp] = __popc(eq);
    __syncthreads();
    int run = __popc(eq & ((1u << lane) - 1));
    for (int k = 0; k < warp; ++k) run += warp_count[k];
    take = key > least || (key == least && run < ties);
  }
  if (in) {
    take = (take && !shut) || (use_sure && lp >= sure && !is_known);
    ids_out[at] = take ? token : id;
    known_out[at] = is_known || take;
    held_out[at] = take ? lp : was;
    where_out[at] = take;
  }
}

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

// Bytes of scratch that dttt_sample wants for `rows` rows whose draw no parameter truncates (0: none).
extern "C" long long dttt_sample_scratch(long long rows, int V) {
  const long long most = (V + 7ll + CHUNK - 1) / CHUNK;
  return V > STREAM_VOCAB && rows * V >= STREAM_LEAST && rows * most <= 0x7fffffffll ? rows * most * (long long)sizeof(Chunk) : 0;
}

// logits: rows [outer, inner] of V elements (dtype 0 f32, 1 bf16, 2 f16), element strides s_outer / s_inner, contiguous along V.
// *_row: per-row parameter arrays or null (then the scalar).  Outputs contiguous [rows].  `scratch` (16-byte aligned): of
// dttt_sample_scratch, only for rows that no parameter truncates; null takes the kernel on clusters.
extern "C" int dttt_sample(const void* logits, int dtype, long long rows, int inner, long long s_outer, long long s_inner, int V,
                           const float* u, const float* bias, double temperature, const float* t_row, int top_k, const int* k_row,
                           double top_p, const float* p_row, double min_p, const float* m_row, int priority, long long* tokens,
                           float* logp, float* prio, void* scratch, cudaStream_t stream) {
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
  if (scratch) {
    switch (dtype) {
      case 0: return launch_stream<float>(p, rows, (Chunk*)scratch, stream);
      case 1: return launch_stream<__nv_bfloat16>(p, rows, (Chunk*)scratch, stream);
      case 2: return launch_stream<__half>(p, rows, (Chunk*)scratch, stream);
    }
    return -2;
  }
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
  if (C <= UM_ROW) {
    unmask_row_kernel<<<B, (C + 31) / 32 * 32, 0, stream>>>(ids, (const uint8_t*)known, held, tokens, logp, priority, quota, (const uint8_t*)allowed,
                                                            sure, use_sure, ids_out, (uint8_t*)known_out, held_out, (uint8_t*)where_out, C);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : 1000 + (int)e;
  }
  const size_t smem = (size_t)C * sizeof(uint32_t);
  static std::atomic<u64> ready{0};
  cudaError_t e = allow_shared(unmask_kernel, UM_SLOTS_MAX * (int)sizeof(uint32_t), ready);
  if (e != cudaSuccess) return 1000 + (int)e;
  unmask_kernel<<<B, UM_THREADS, smem, stream>>>(ids, (const uint8_t*)known, held, tokens, logp, priority, quota, (const uint8_t*)allowed,
                                                 sure, use_sure, ids_out, (uint8_t*)known_out, held_out, (uint8_t*)where_out, C);
  e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 1000 + (int)e;
}
