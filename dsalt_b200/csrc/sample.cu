// Token sampling with temperature, top-k, top-p and min-p from given uniform numbers
// (dsalt_sample).
//
// Of a row of logits l, with m = max l and weights w = exp((l - m) / T):
//   top-k: the k first in the order (logit descending, index ascending)
//   top-p: of those the shortest prefix whose mass reaches p times theirs
//   min-p: of those the weights of at least min_p (the largest weight is 1), or the first alone
//   token: the first index whose running sum of kept weights, in index order, exceeds u
//          times their total.
// T <= 0 takes the first index of the largest logit. A NaN counts as -inf, +inf logits share
// the draw among themselves, a row of nothing but -inf gives token 0 with log-probability -inf.
//
// No sort of the row: all three filters keep a prefix of one order, so there is one element
// (key, index) at which the row is cut. Where at most LIST_CAP elements can matter they are
// gathered and sorted in one block's shared memory, and the row is settled there:
//   top-k: the k-th largest of the maxima of any threads is at most the k-th largest logit, so
//          the elements from there on up hold the k first and few more (groups of 8 or 16 threads
//          for a small k, every thread for a larger one);
//   top-p: masses and counts of 16 bins of (m - l) / T. Each thread has bins of its own (no
//          atomics: a word per thread and bin).
// Otherwise each warp puts its elements of the bin where p is reached into a queue: only they
// are looked at again, by a histogram of 1024 parts of the bin and, where a part still holds
// more than the list, by histograms over (key, index). The mass of what stays is then known
// per warp, and the draw goes down from block to warp to 256 elements to the token.
//
// Masses are whole numbers, w * 2^43 rounded from 64-bit arithmetic: their sums do not depend
// on the order in which threads arrive, so a row gives the same token in every batch and in
// every run, and a border lies within 2^20 roundings of 2^-44 (6e-8 of the largest weight at
// the very worst, about 1e-11 in practice) of where sums in 64-bit floating point put it. The
// log-probability is formed from the drawn logit and the sum, not from the token's own mass.
//
// One cluster of C blocks owns a row, each a share of it. The row comes from HBM once; later
// passes find it in L1 or L2, which hold it for all rows under way.
//
// Measured on a B200 (device time, 64 rows of 151936 in bf16, 19 MB): the largest logit 9.9 us,
// temperature alone 27.1, top-k 50 19.8, top-p 0.9 88.5, every row its own settings 94.4. Bytes are
// 3 us of each. Temperature alone is bound by the 64-bit instructions of the weights (10 per
// element), the draws of a wide nucleus by latency: some ten steps of one cluster one after
// another, of which the pass over the bins takes 15 us, the queue 11, the histogram and its
// joining 14, list and sort 14. Measured and not kept: a rough pass in 32 bits before one exact
// pass that also queues (107 us for top-p 0.9: the queue's places cost more beside the
// weights than in a pass of their own), queues per lane (112), queues by votes (93), queues
// that hold the logits too (91).
#include <cooperative_groups.h>

#include <type_traits>

#include "common.cuh"

namespace dsalt {

namespace cg = cooperative_groups;

constexpr int SAMPLE_THREADS = 512;
constexpr int SAMPLE_WARPS = SAMPLE_THREADS / 32;
constexpr int PBINS = SAMPLE_WARPS;           // private bins, one per warp where they are summed
constexpr int NBINS = 2 * SAMPLE_THREADS;     // of a joint histogram, two per thread where they are summed
constexpr int LIST_CAP = 2 * SAMPLE_THREADS;
constexpr int IDX_BITS = 20;                  // vocabulary of at most 2^20
constexpr int BLOCK_ELEMS = 256;              // a warp's step: eight consecutive elements per lane
constexpr int MAX_SHARE = 131328;             // 2^20 / 8 and a skew, in whole steps: 513 of them
constexpr int MAX_STEPS = (MAX_SHARE / BLOCK_ELEMS + SAMPLE_WARPS - 1) / SAMPLE_WARPS;  // of one warp
constexpr int QUEUE = 992;                    // elements of the decisive bin that a warp keeps
constexpr int MAX_GROUPS = 256;
constexpr int MASS_BITS = 43;
constexpr double MASS_ONE = 8796093022208.0;  // 2^43: 2^20 of them are 2^63, within 64 bits without a sign
// A mass (at most 2^43) in the joint histogram's 32-bit words: limbs of 14 bits, so that no word overflows
// where a whole share falls into one bin (131328 limbs of 15 bits would reach past 2^32).
constexpr int LIMBS = 4, LIMB_BITS = 14;
constexpr uint32_t LIMB_MAX = (1u << LIMB_BITS) - 1;
static_assert((uint64_t)MAX_SHARE * LIMB_MAX <= 0xffffffffull, "a limb's sum over a share");
static_assert(MASS_BITS < LIMBS * LIMB_BITS, "the limbs hold a mass");
constexpr float BIN_SPAN = 32.f;              // (m - l) / T that the joint histogram covers
constexpr float MIN_LOG2 = -45.f;             // weights below 2^-45 round to no mass

typedef unsigned long long u64;

struct SampleArgs {
  const void* logits;
  int64_t row_stride;
  int V, share;  // share: elements of one block, a multiple of BLOCK_ELEMS
  const float* u;
  const float *temperature, *top_p, *min_p;  // per row, or null and the value below
  const int32_t* top_k;
  float temperature_v, top_p_v, min_p_v;
  int top_k_v;
  int64_t* token;
  float* logprob;
};

// What one block holds. The arrays of a group share their memory: none outlives the next use.
struct SampleShared {
  union {
    u64 priv[PBINS][SAMPLE_THREADS];  // count (12 bits) and mass (52) of each thread's elements per bin
    struct {
      uint32_t count[NBINS], limb[LIMBS][NBINS];  // this block's joint histogram; masses in limbs
    };
    struct {
      u64 sorted[LIST_CAP], weight[LIST_CAP];  // the leader's candidates in order, and their masses
      uint32_t by_index[LIST_CAP];
    };
  };
  uint16_t queue[SAMPLE_WARPS][QUEUE];  // places within the warp's stretch (below 2^16)
  union {
    u64 mass[NBINS];     // joined over the cluster, in the leader's copy
    u64 item[LIST_CAP];  // candidates as they arrive, in the leader's copy
  };
  uint32_t total[NBINS];  // joined counts, in the leader's copy
  u64 warp_bin[PBINS][SAMPLE_WARPS];  // first level's masses, per warp
  u64 bin_mass[PBINS];
  uint32_t bin_count[PBINS];
  u64 steps[MAX_STEPS];  // masses of the steps of the warp that holds the draw
  u64 kept[SAMPLE_WARPS];
  uint32_t n_items, first_index;
  float best, bound;
  float group_max[64], all_max[MAX_GROUPS];  // of 8 or 16 threads: this block's, the cluster's
  u64 share_mass, range[2], result[4];  // result: written by the leader only
  u64 warp_red[SAMPLE_WARPS];
  double exp2_128[128];  // 2^(j / 128)
};

// the block's own, by its shared-memory address (a pointer handed to a function would be generic)
__device__ __forceinline__ SampleShared& block_shared() {
  extern __shared__ __align__(16) unsigned char sample_smem[];
  return *reinterpret_cast<SampleShared*>(sample_smem);
}

// (key, index) as one number: larger comes first in the order of the filters
__device__ __forceinline__ u64 compose(float l, int idx) {
  return ((u64)order_f32(l + 0.0f) << IDX_BITS) | (u64)((1 << IDX_BITS) - 1 - idx);  // -0 as 0
}
__device__ __forceinline__ int index_of(u64 c) { return (1 << IDX_BITS) - 1 - (int)(c & ((1u << IDX_BITS) - 1)); }
__device__ __forceinline__ float logit_of(u64 c) {
  const uint32_t k = (uint32_t)(c >> IDX_BITS);
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}

// Weights of one row. 2^t, t = (l - m) log2(e) / T: t = k / 128 + g with |g| <= 1/256,
// then 2^(k/128) from a table of 128 and the exponent, 2^g by its Taylor series to the fourth power
// (the fifth term is below (ln 2 / 256)^5 / 5! = 1.3e-15). The passes are bound by instructions, and
// one in 64 bits takes two turns: ten of them here, no branch and no selection (a table of 32 and
// the fifth power: 27.7 us at temperature alone, 26.9 so).
struct Weights {
  float top;    // the largest logit
  float floor;  // logits below it (and NaN) are taken as it
  double c;
  bool only_top;   // +inf: equal ones have weight 1, all others none
  bool vanishing;  // the floor's weight rounds to no mass (else -inf and NaN have to be left out)
  __device__ __forceinline__ double finite(float l) const {  // where !only_top
    constexpr double MAGIC = 52776558133248.0;  // 1.5 * 2^45: adding it leaves steps of 1/128
    constexpr double C1 = 0.6931471805599453094, C2 = C1 * C1 / 2, C3 = C2 * C1 / 3, C4 = C3 * C1 / 4;
    const double d = (double)fmaxf(l, floor) - (double)top, r = fma(d, c, MAGIC);
    const int k = __double2loint(r);
    const double g = fma(d, c, MAGIC - r);
    double p = fma(g, C4, C3);
    p = fma(p, g, C2);
    p = fma(p, g, C1);
    p = fma(p, g, 1.0) * block_shared().exp2_128[k & 127];
    return __hiloint2double(__double2hiint(p) + ((k >> 7) << 20), __double2loint(p));
  }
  __device__ __forceinline__ double operator()(float l) const {
    return only_top ? (l == top ? 1.0 : 0.0) : finite(l);
  }
  // w * 2^43 to the nearest whole number
  static __device__ __forceinline__ u64 mass(double w) {
    return (u64)__double_as_longlong(fma(w, MASS_ONE, 4503599627370496.0)) & 0xfffffffffffffull;  // + 2^52
  }
  __device__ __forceinline__ u64 mass(float l) const { return mass((*this)(l)); }
  // log of a drawn logit's share of the kept masses, from the logit itself: a rare token's mass has
  // few bits (weight 2^-40: three)
  __device__ __forceinline__ float log_share(float l, u64 total) const {
    const double z = l == top ? 0.0 : ((double)l - (double)top) * (c * 0.6931471805599453094);
    return (float)(z - log((double)total / MASS_ONE));
  }
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// sum over the block, in every thread
__device__ __forceinline__ u64 block_sum(u64 v, SampleShared& sh) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.warp_red[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 t = 0;
#pragma unroll
  for (int w = 0; w < SAMPLE_WARPS; ++w) t += sh.warp_red[w];
  return t;
}
// sum over the threads before this one
__device__ __forceinline__ u64 block_before(u64 v, SampleShared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 a = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += a;
  }
  __syncthreads();
  if (lane == 31) sh.warp_red[warp] = s;
  __syncthreads();
  u64 t = 0;
  for (int w = 0; w < warp; ++w) t += sh.warp_red[w];
  return t + s - v;
}

// p times a mass, rounded up: what a prefix has to reach (at least 1, so that the first
// element always stays)
__device__ __forceinline__ u64 part_of(double p, u64 mass) {
  const double x = ceil(p * (double)mass);
  if (!(x >= 1.0)) return 1;
  return x >= (double)mass ? mass : (u64)x;
}
// u * total as the whole number that the drawn running sum has to exceed
__device__ __forceinline__ u64 target_of(float u, u64 total) {
  const double x = (double)u * (double)total;
  if (!(x >= 1.0)) return 0;
  return x >= (double)total ? total - 1 : min((u64)x, total - 1);
}

// Bitonic sort of `size` (a power of two, at most two per thread) values in shared memory by
// the block. A thread holds two neighbours: distances up to 32 are a warp's own business
// (shuffles), only longer ones go through shared memory, twice at a time.
template <typename T, bool DESCENDING>
__device__ __forceinline__ void block_sort(T* v, int size) {
  static_assert(LIST_CAP == 2 * SAMPLE_THREADS, "two values per thread");
  __syncthreads();
  const int i0 = 2 * threadIdx.x;
  const bool live = i0 < size;
  T a = live ? v[i0] : T(0), b = live ? v[i0 + 1] : T(0);
  const auto better = [](T x, T y, bool first) {  // the value that the lower (first) or upper place keeps
    return (x > y) == (first == DESCENDING) ? x : y;
  };
  for (int k = 2; k <= size; k <<= 1) {
    const bool up = (i0 & k) == 0;  // a block of k in the wanted order, else reversed
    for (int j = k >> 1; j > 32; j >>= 1) {
      __syncthreads();
      if (live) v[i0] = a, v[i0 + 1] = b;
      __syncthreads();
      if (live) {
        const bool first = ((i0 & j) == 0) == up;
        a = better(a, v[i0 ^ j], first);
        b = better(b, v[(i0 ^ j) + 1], first);
      }
    }
    if (i0 - 2 * (int)(threadIdx.x & 31) < size) {  // the warp holds values
      for (int j = min(k >> 1, 32); j > 1; j >>= 1) {
        const bool first = ((i0 & j) == 0) == up;
        a = better(a, __shfl_xor_sync(0xffffffffu, a, j >> 1), first);
        b = better(b, __shfl_xor_sync(0xffffffffu, b, j >> 1), first);
      }
      const T x = better(a, b, up), y = better(a, b, !up);
      a = x;
      b = y;
    }
  }
  __syncthreads();
  if (live) v[i0] = a, v[i0 + 1] = b;
  __syncthreads();
}
__device__ __forceinline__ int power_of_two(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

// Sorts the leader's n <= LIST_CAP items and forms their masses.
__device__ __forceinline__ void sort_items(SampleShared& sh, int n, const Weights& wt) {
  const int size = power_of_two(n);
  __syncthreads();
  for (int i = threadIdx.x; i < size; i += SAMPLE_THREADS) sh.sorted[i] = i < n ? sh.item[i] : 0;
  block_sort<u64, true>(sh.sorted, size);
  for (int i = threadIdx.x; i < n; i += SAMPLE_THREADS) sh.weight[i] = wt.mass(logit_of(sh.sorted[i]));
  __syncthreads();
}

// The leader's block settles a row whose candidates are all in its sorted list: `keep` of them
// are within top-k; `want` > 0 is the mass that top-p has to reach, else it is formed here.
__device__ __forceinline__ void settle_list(const SampleArgs& a, SampleShared& sh, int row, int keep, bool cut_p,
                                            double top_p, u64 want, double min_p, float u, const Weights& wt) {
  const int i0 = 2 * threadIdx.x, i1 = i0 + 1;
  const u64 w0 = i0 < keep ? sh.weight[i0] : 0, w1 = i1 < keep ? sh.weight[i1] : 0;
  if (cut_p) {
    if (want == 0) want = part_of(top_p, block_sum(w0 + w1, sh));
    const u64 before = block_before(w0 + w1, sh);
    keep = (int)block_sum((u64)(i0 < keep && before < want) + (u64)(i1 < keep && before + w0 < want), sh);
  }
  if (min_p > 0) {
    const auto ok = [&](int i) { return i < keep && wt(logit_of(sh.sorted[i])) >= min_p; };
    keep = max(1, (int)block_sum((u64)ok(i0) + (u64)ok(i1), sh));
  }
  // in index order: (index, place) sorted, then a running sum
  const int size = power_of_two(keep);
  for (int i = threadIdx.x; i < size; i += SAMPLE_THREADS)
    sh.by_index[i] = i < keep ? ((uint32_t)index_of(sh.sorted[i]) << 10) | (uint32_t)i : 0xffffffffu;
  block_sort<uint32_t, false>(sh.by_index, size);
  static_assert(LIST_CAP == 1 << 10 && IDX_BITS + 10 <= 30, "index and place share a word");
  const u64 m0 = i0 < keep ? sh.weight[sh.by_index[i0] & 1023] : 0, m1 = i1 < keep ? sh.weight[sh.by_index[i1] & 1023] : 0;
  const u64 total = block_sum(m0 + m1, sh), before = block_before(m0 + m1, sh), target = target_of(u, total);
  if (before <= target && target < before + m0 + m1) {  // one thread
    const uint32_t drawn = sh.by_index[target >= before + m0 ? i1 : i0];
    a.token[row] = drawn >> 10;
    if (a.logprob) a.logprob[row] = wt.log_share(logit_of(sh.sorted[drawn & 1023]), total);
  }
}

// One block's share of a row, in steps of a warp: eight consecutive elements per lane. Places are
// counted from the 16-byte boundary at or before the row's start, so that whole vectors can be
// read. A warp's steps follow one another.
template <typename T>
struct Share {
  static constexpr int VEC = 16 / (int)sizeof(T), WORDS = 32 / VEC, PER = 4 / (int)sizeof(T);
  static constexpr int AHEAD = 1;  // steps that loads run ahead (more of them cost registers that the weights need)
  const T* src;
  int V, start;  // index of the share's first place (negative where the row begins behind it)
  int n_steps, per_warp;

  __device__ __forceinline__ int first() const { return min((int)(threadIdx.x >> 5) * per_warp, n_steps); }
  __device__ __forceinline__ int last() const { return min(first() + per_warp, n_steps); }
  __device__ __forceinline__ int index(int step) const { return start + step * BLOCK_ELEMS + (threadIdx.x & 31) * 8; }
  __device__ __forceinline__ float one(int i) const {
    if constexpr (sizeof(T) == 4) return src[i];
    else if constexpr (std::is_same<T, __half>::value) return __half2float(src[i]);
    else return __bfloat162float(src[i]);
  }
  struct Raw {  // eight elements as they lie in memory
    uint32_t w[WORDS];
  };
  __device__ __forceinline__ Raw load(int step) const {  // NaN outside the row
    const int i0 = index(step);
    Raw r;
    if (i0 >= 0 && i0 + 8 <= V) {
#pragma unroll
      for (int h = 0; h < WORDS / 4; ++h) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(src + i0) + h);
        r.w[4 * h] = v.x, r.w[4 * h + 1] = v.y, r.w[4 * h + 2] = v.z, r.w[4 * h + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < WORDS; ++e) {
        r.w[e] = 0xffffffffu;
#pragma unroll
        for (int x = 0; x < PER; ++x) {
          const int i = i0 + e * PER + x;
          if (i < 0 || i >= V) continue;
          if constexpr (sizeof(T) == 4) r.w[e] = __float_as_uint(src[i]);
          else r.w[e] = (r.w[e] & ~(0xffffu << 16 * x)) | (uint32_t)reinterpret_cast<const uint16_t*>(src)[i] << 16 * x;
        }
      }
    }
    return r;
  }
  static __device__ __forceinline__ float2 pair(const Raw& r, int x) {  // elements 2 x, 2 x + 1
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(r.w[2 * x]), __uint_as_float(r.w[2 * x + 1]));
    else if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&r.w[x]));
    else return make_float2(__uint_as_float(r.w[x] << 16), __uint_as_float(r.w[x] & 0xffff0000u));
  }
  // f(raw, first index) for the warp's steps
  template <typename F>
  __device__ __forceinline__ void steps(F&& f) const {
    const int s0 = first(), s1 = last();
    Raw next[AHEAD];
#pragma unroll
    for (int x = 0; x < AHEAD; ++x)
      if (s0 + x < s1) next[x] = load(s0 + x);
#pragma unroll 1
    for (int step = s0; step < s1; ++step) {
      const Raw now = next[0];
#pragma unroll
      for (int x = 0; x + 1 < AHEAD; ++x) next[x] = next[x + 1];
      if (step + AHEAD < s1) next[AHEAD - 1] = load(step + AHEAD);
      f(now, index(step));
    }
  }
  // f(four logits, index of the first) for the warp's elements, NaN outside the row
  template <typename F>
  __device__ __forceinline__ void fours(F&& f) const {
    steps([&](const Raw& r, int i0) {
#pragma unroll
      for (int x = 0; x < 4; x += 2) {
        const float2 a = pair(r, x), b = pair(r, x + 1);
        const float l[4] = {a.x, a.y, b.x, b.y};
        f(l, i0 + 2 * x);
      }
    });
  }
  // f(logit, index) for the warp's elements, NaN outside the row
  template <typename F>
  __device__ __forceinline__ void each(F&& f) const {
    steps([&](const Raw& r, int i0) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float2 l = pair(r, x);
        f(l.x, i0 + 2 * x);
        f(l.y, i0 + 2 * x + 1);
      }
    });
  }
};

// The passes over a share.
struct Bin {  // logits [low, high) (from low up where `top`), of elements at or above `cut`
  float low, high;
  bool top;
  u64 cut;
  __device__ __forceinline__ bool has(float l, int i) const {
    return l >= low && (top || l < high) && (cut == 0 || compose(l, i) >= cut);
  }
};
__device__ __forceinline__ float place_of(float l, float top, float inv_t) {  // grows as l falls, at least 0
  const float z = (top - l) * inv_t;
  return z == z ? z : 0.f;  // of +inf against +inf
}

template <typename T>
__device__ __forceinline__ float max_pass(Share<T> s) {
  float m = -INFINITY;
  s.each([&](float l, int) { m = fmaxf(m, l); });  // passes over NaN
  return m;
}
template <typename T>
__device__ __forceinline__ uint32_t first_pass(Share<T> s, float top) {  // lowest index of the largest logit
  uint32_t first = 0xffffffffu;
  s.each([&](float l, int i) {
    if (l == top) first = min(first, (uint32_t)i);
  });
  return first;
}
template <typename T>
__device__ __forceinline__ void bins_pass(Share<T> s, Weights wt, float inv_t, u64 cut, bool by_mass) {
  auto& priv = block_shared().priv;
#pragma unroll
  for (int b = 0; b < PBINS; ++b) priv[b][threadIdx.x] = 0;
  constexpr u64 ONE = 1ull << 52;
  // four elements at a time, and no branch: their chains of 64-bit instructions run side by side
  const auto put = [&](auto&& mass) {
    s.fours([&](const float (&l)[4], int i0) {
      u64 m[4];
      int b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        m[e] = mass(l[e], i0 + e);
        b[e] = (int)fminf(place_of(l[e], wt.top, inv_t), (float)(PBINS - 1));
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) priv[b[e]][threadIdx.x] += m[e];
    });
  };
  if (!by_mass) put([&](float l, int) { return l > -INFINITY ? ONE : 0; });
  else if (wt.only_top) put([&](float l, int i) { return l > -INFINITY && compose(l, i) >= cut ? ONE + wt.mass(l) : 0; });
  else if (cut == 0) put([&](float l, int) { const u64 m = ONE + Weights::mass(wt.finite(l)); return l > -INFINITY ? m : 0; });
  else put([&](float l, int i) {
    const u64 m = ONE + Weights::mass(wt.finite(l));
    return (l > -INFINITY) & (compose(l, i) >= cut) ? m : 0;
  });
}
template <typename T>
__device__ __forceinline__ int queue_pass(Share<T> s, Bin bin) {  // returns how many there are
  uint16_t* const queue = block_shared().queue[threadIdx.x >> 5];
  const int lane = threadIdx.x & 31, from = s.start + s.first() * BLOCK_ELEMS;
  int queued = 0;
  s.steps([&](const typename Share<T>::Raw& r, int i0) {
    uint32_t in = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float2 l = Share<T>::pair(r, x);
      in |= (bin.has(l.x, i0 + 2 * x) ? 1u : 0u) << (2 * x) | (bin.has(l.y, i0 + 2 * x + 1) ? 2u : 0u) << (2 * x);
    }
    const int cnt = __popc(in);
    int at = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += x;
    }
    const int all = __shfl_sync(0xffffffffu, at, 31);
    at += queued - cnt;
    for (; in; in &= in - 1, ++at)
      if (at < QUEUE) queue[at] = (uint16_t)(i0 + __ffs(in) - 1 - from);
    queued += all;
  });
  __syncwarp();
  return queued;
}
// f(logit, index) for the elements of the bin that this warp owns
template <typename T, typename F>
__device__ __forceinline__ void for_bin(const Share<T>& s, const Bin& bin, int queued, F&& f) {
  const uint16_t* const queue = block_shared().queue[threadIdx.x >> 5];
  if (queued <= QUEUE) {
    const int from = s.start + s.first() * BLOCK_ELEMS;
    for (int q = threadIdx.x & 31; q < queued; q += 4 * 32) {  // four loads under way
      float l[4];
      int i[4];
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (q + 32 * x < queued) {
          i[x] = from + (int)queue[q + 32 * x];
          l[x] = s.one(i[x]);
        }
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (q + 32 * x < queued) f(l[x], i[x]);
    }
  } else {
    s.each([&](float l, int i) {
      if (bin.has(l, i)) f(l, i);
    });
  }
}
// Parts of the bin for a histogram: 1024 of (m - l) / T from z0 on (shift < 0), or 2^shift
// composed numbers each from ceil_c down to floor_c.
struct Parts {
  float top, inv_t, z0, scale;
  int shift;
  u64 floor_c, ceil_c;
  __device__ __forceinline__ int operator()(float l, int i) const {  // -1: outside
    if (shift < 0) return (int)fminf((place_of(l, top, inv_t) - z0) * scale, (float)(NBINS - 1));
    const u64 c = compose(l, i);
    return c < floor_c || c > ceil_c ? -1 : (int)((ceil_c - c) >> shift);
  }
};
template <typename T>
__device__ __forceinline__ void histogram_pass(Share<T> s, Weights wt, Bin bin, Parts parts, bool by_mass, int queued) {
  SampleShared& sh = block_shared();
  for_bin(s, bin, queued, [&](float l, int i) {
    const int b = parts(l, i);
    if (b < 0) return;
    atomicAdd(&sh.count[b], 1u);
    if (by_mass) {
      const u64 w = wt.mass(l);
      atomicAdd(&sh.limb[0][b], (uint32_t)w & LIMB_MAX);
      atomicAdd(&sh.limb[1][b], (uint32_t)(w >> LIMB_BITS) & LIMB_MAX);
#pragma unroll
      for (int x = 2; x < LIMBS; ++x)  // of weights above 2^-15, and above 1/2
        if (w >> x * LIMB_BITS) atomicAdd(&sh.limb[x][b], (uint32_t)(w >> x * LIMB_BITS) & LIMB_MAX);
    }
  });
}
template <typename T>
__device__ __forceinline__ void range_pass(Share<T> s, Bin bin, Parts parts, int part, int queued, u64& first, u64& last) {
  u64 lo = ~0ull, hi = 0;
  for_bin(s, bin, queued, [&](float l, int i) {
    if (parts(l, i) != part) return;
    const u64 c = compose(l, i);
    lo = min(lo, c);
    hi = max(hi, c);
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  first = lo;
  last = hi;
}
// into the leader's list: all elements from `low` up; or those of one part of the bin
template <typename T>
__device__ __forceinline__ void list_pass(Share<T> s, float low, u64 cut, SampleShared* lead) {
  s.each([&](float l, int i) {
    if (!(l >= low) || l == -INFINITY || (cut != 0 && compose(l, i) < cut)) return;
    const uint32_t at = atomicAdd(&lead->n_items, 1u);
    if (at < LIST_CAP) lead->item[at] = compose(l, i);
  });
}
template <typename T>
__device__ __forceinline__ void list_part_pass(Share<T> s, Bin bin, Parts parts, int part, int queued, SampleShared* lead) {
  for_bin(s, bin, queued, [&](float l, int i) {
    if (parts(l, i) != part) return;
    const uint32_t at = atomicAdd(&lead->n_items, 1u);
    if (at < LIST_CAP) lead->item[at] = compose(l, i);
  });
}
// the warp's mass of what stays: of its queue, of its elements, of one step
struct Kept {
  Weights wt;
  u64 cut;
  double min_p;
  __device__ __forceinline__ u64 operator()(float l, int i) const {
    const double w = wt(l);
    return (min_p > 0 && !(w >= min_p)) || (cut != 0 && compose(l, i) < cut) || !(l > -INFINITY) ? 0 : wt.mass(w);
  }
};
template <typename T>
__device__ __forceinline__ u64 kept_queue_pass(Share<T> s, Kept kept, Bin bin, int queued) {
  u64 m = 0;
  for_bin(s, bin, queued, [&](float l, int i) { m += kept(l, i); });
  return warp_sum(m);
}
template <typename T>
__device__ __forceinline__ u64 kept_pass(Share<T> s, Kept kept) {
  u64 m = 0;
  if (kept.wt.only_top || !kept.wt.vanishing || kept.cut != 0 || kept.min_p > 0) s.each([&](float l, int i) { m += kept(l, i); });
  else s.each([&](float l, int) { m += Weights::mass(kept.wt.finite(l)); });  // nothing is cut
  return warp_sum(m);
}

static_assert(sizeof(SampleShared) <= (228 * 1024 - 2 * 1024) / 2, "two blocks per SM");

template <typename T>
__global__ void __launch_bounds__(SAMPLE_THREADS, 2) sample_kernel(SampleArgs a) {
  SampleShared& sh = block_shared();
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  SampleShared* lead = cluster.map_shared_rank(&sh, 0);

  const double top_p = a.top_p ? (double)a.top_p[row] : (double)a.top_p_v;
  const double min_p = a.min_p ? (double)a.min_p[row] : (double)a.min_p_v;
  // no weight reaches a min_p above 1, and the first of the order stays: what temperature 0 takes
  const float temp = min_p > 1.0 ? 0.f : a.temperature ? a.temperature[row] : a.temperature_v;
  const int top_k = a.top_k ? a.top_k[row] : a.top_k_v;
  const float u = a.u[row];
  const bool cut_k = top_k > 0 && top_k < a.V, cut_p = top_p < 1.0;

  Share<T> s;
  s.src = reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.row_stride;
  s.V = a.V;
  const int skew = (int)(((uintptr_t)s.src & 15) / sizeof(T));
  s.start = rank * a.share - skew;
  s.n_steps = (max(0, min(a.share, a.V - s.start)) + BLOCK_ELEMS - 1) / BLOCK_ELEMS;
  s.per_warp = (s.n_steps + SAMPLE_WARPS - 1) / SAMPLE_WARPS;

  // ---- the largest logit
  const float mine = max_pass<T>(s);
  float top = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (o == 4 && C < 8 && (lane & 7) == 0) sh.group_max[tid >> 3] = top;
    if (o == 8 && C == 8 && (lane & 15) == 0) sh.group_max[tid >> 4] = top;
  }
  const int groups = C < 8 ? 64 : 32;  // per block
  if (lane == 0) sh.warp_red[warp] = __float_as_uint(top);
  if (tid < 128) sh.exp2_128[tid] = exp2((double)tid / 128);
  if (tid == 0) {
    sh.first_index = 0xffffffffu;
    sh.n_items = 0;
  }
  const auto clear_bins = [&] {
    for (int i = tid; i < NBINS; i += SAMPLE_THREADS) sh.count[i] = sh.limb[0][i] = sh.limb[1][i] = sh.limb[2][i] = sh.limb[3][i] = 0;
  };
  clear_bins();
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SAMPLE_WARPS; ++w) top = fmaxf(top, __uint_as_float((uint32_t)sh.warp_red[w]));
  if (tid == 0) sh.best = top;
  cluster.sync();
#pragma unroll
  for (int r = 0; r < 8; ++r)
    if (r < C) top = fmaxf(top, cluster.map_shared_rank(&sh, r)->best);
  // a small top-k's bound: the k-th largest of the groups' maxima. (About -n ln(1 - k / n) elements lie
  // above it with n groups that hold elements: towards the smallest of them the bound falls off. k =
  // 200 of 256 in a row of 16384, where half of the warps have nothing, took 26.5 us, by the threads'
  // maxima 15.4; k = 64 takes 12.4 this way and 13.7 that way.)
  const int full = a.share / BLOCK_ELEMS, stretch = (full + SAMPLE_WARPS - 1) / SAMPLE_WARPS;
  const int filled = C * groups * ((full + stretch - 1) / stretch) / SAMPLE_WARPS;
  const bool small_k = cut_k && temp > 0.f && 5 * top_k <= 4 * filled;
  float bound = -INFINITY;
  if (small_k) {
    if (tid < C * groups) sh.all_max[tid] = cluster.map_shared_rank(&sh, tid / groups)->group_max[tid % groups];
    __syncthreads();
    if (tid < C * groups) {
      const float v = sh.all_max[tid];
      int before = 0;
#pragma unroll 8
      for (int i = 0; i < C * groups; ++i) before += sh.all_max[i] > v || (sh.all_max[i] == v && i < tid);
      if (before == top_k - 1) sh.bound = v;
    }
    __syncthreads();
    bound = sh.bound;
  }
  // every decision from here to the end is the same in all threads of the cluster
  if (!(temp > 0.f) || top == -INFINITY) {
    if (top > -INFINITY) {
      const uint32_t first = __reduce_min_sync(0xffffffffu, first_pass<T>(s, top));
      if (lane == 0 && first != 0xffffffffu) atomicMin(&lead->first_index, first);
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
      a.token[row] = top == -INFINITY ? 0 : sh.first_index;
      if (a.logprob) a.logprob[row] = top == -INFINITY ? -INFINITY : 0.f;
    }
    return;  // (the others' shared memory was last read before the barrier)
  }
  Weights wt;
  wt.top = top;
  wt.c = 1.4426950408889634 / (double)temp;
  // Where one step of fp32 below the largest logit is beyond 2^-900, a smaller slope says the same:
  // everything below has no mass, and 2^t stays a normal number down to the floor.
  const float below = nextafterf(top, -INFINITY);
  wt.only_top = top == INFINITY || below == -INFINITY;
  if (!wt.only_top) wt.c = fmin(wt.c, 900.0 / ((double)top - (double)below));
  wt.floor = fmaxf(fminf((float)((double)top + (double)MIN_LOG2 / wt.c), below), -3.402823466e38f);
  wt.vanishing = ((double)wt.floor - (double)top) * wt.c <= (double)MIN_LOG2 + 0.5;
  // 1 / T as a finite number, so that a difference of 0 is place 0 at any temperature
  const float inv_t = fminf((float)(1.0 / (double)temp), 3.402823466e38f);

  // the smallest logit whose place (m - l) / T lies below a bound, by a search of 32 steps at a time
  const auto lowest = [&](float bound) -> float {
    uint32_t lo = order_f32(-INFINITY), hi = order_f32(top);  // at or beyond the bound, below it
    while (hi - lo > 1) {
      const uint32_t step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
      const bool in = at >= hi || place_of(logit_of((u64)at << IDX_BITS), top, inv_t) < bound;
      const int f = __ffs(__ballot_sync(0xffffffffu, in)) - 1;  // the last lane's is at or above hi
      hi = min(hi, lo + (f + 1) * step);
      lo += f * step;
    }
    return logit_of((u64)hi << IDX_BITS);
  };
  u64 cut = 0;  // elements below it are dropped
  // ---- top-k by a bound from the threads' maxima
  const auto joint_bin = [&](float l) { return (int)fminf(place_of(l, top, inv_t) * (NBINS / BIN_SPAN), (float)(NBINS - 1)); };
  const auto join_bins = [&](bool by_mass) {  // each block joins its part of the bins into the leader
    cluster.sync();
    for (int b = rank * SAMPLE_THREADS + tid; b < NBINS; b += C * SAMPLE_THREADS) {
      uint32_t cnt = 0;
      u64 ms = 0;
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < C) {
          const SampleShared* o = cluster.map_shared_rank(&sh, r);
          cnt += o->count[b];
          if (by_mass) {
#pragma unroll
            for (int x = 0; x < LIMBS; ++x) ms += (u64)o->limb[x][b] << x * LIMB_BITS;
          }
        }
      lead->total[b] = cnt;
      lead->mass[b] = ms;
    }
    cluster.sync();
  };
  // the leader: the first bin whose running sum reaches `want`, else the last: result = bin and its
  // count, sum before it, elements up to and with it. (Where a bin is refined the sums reach it, unless
  // the logits are written to meanwhile.)
  const auto find_bin = [&](bool by_mass, u64 above, u64 want) {
    if (rank == 0) {
      const uint32_t c0 = sh.total[2 * tid], c1 = sh.total[2 * tid + 1];
      const u64 v0 = by_mass ? sh.mass[2 * tid] : c0, v1 = by_mass ? sh.mass[2 * tid + 1] : c1;
      const u64 before = above + block_before(v0 + v1, sh);
      const u64 cnt_before = block_before((u64)c0 + c1, sh);
      // one thread: the sums only grow
      if (before < want && (before + v0 + v1 >= want || tid == SAMPLE_THREADS - 1)) {
        const bool second = before + v0 < want;
        sh.result[0] = (u64)(2 * tid + second) | ((u64)(second ? c1 : c0) << 32);
        sh.result[1] = before + (second ? v0 : 0);
        sh.result[2] = cnt_before + c0 + (second ? c1 : 0);
      }
      if (tid == 0) sh.n_items = 0;
    }
    cluster.sync();
  };
  if (small_k) {
    list_pass<T>(s, bound, 0, lead);
    cluster.sync();
    const uint32_t m = lead->n_items;
    if (m <= LIST_CAP) {
      if (rank == 0) {
        sort_items(sh, (int)m, wt);
        settle_list(a, sh, row, min((int)m, top_k), cut_p, top_p, 0, min_p, u, wt);
      }
      cluster.sync();  // the leader's count may still be read
      return;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) sh.n_items = 0;
  } else if (cut_k && top_k <= LIST_CAP / 2 && top_k <= C * SAMPLE_THREADS / 4) {
    if (mine > -INFINITY) atomicAdd(&sh.count[joint_bin(mine)], 1u);
    join_bins(false);
    find_bin(false, 0, (u64)top_k);  // fewer maxima than k: the last bin, every element
    const int bin = (int)(uint32_t)lead->result[0];
    list_pass<T>(s, bin == NBINS - 1 ? -INFINITY : lowest((float)(bin + 1) / (NBINS / BIN_SPAN)), 0, lead);
    cluster.sync();
    const uint32_t m = lead->n_items;
    if (m <= LIST_CAP) {
      if (rank == 0) {
        sort_items(sh, (int)m, wt);
        settle_list(a, sh, row, min((int)m, top_k), cut_p, top_p, 0, min_p, u, wt);
      }
      cluster.sync();  // the leader's count may still be read
      return;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) sh.n_items = 0;
  }

  // ---- the cut of a wide top-k (by count), then of top-p (by mass)
  bool kept_known = false;  // sh.kept holds the mass that stays, per warp
  for (int pass = cut_k ? 0 : 1; pass < (cut_p ? 2 : 1); ++pass) {
    const bool by_mass = pass == 1;
    u64 want = by_mass ? 0 : (u64)top_k;  // the mass to reach is known once all masses are summed
    u64 above = 0, upto = 0, bin_elems = 0;
    __syncthreads();
    bins_pass<T>(s, wt, inv_t, cut, by_mass);
    __syncthreads();
    {
      // a thread for 16 of the 32 words of (bin, warp), from different banks; the pair joins
      const int b = tid >> 5, w = (tid & 31) >> 1, h = tid & 1;
      u64 ms = 0;
      uint32_t cnt = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const u64 v = sh.priv[b][w * 32 + h * 16 + ((i + w) & 15)];
        ms += v & 0xfffffffffffffull;
        cnt += (uint32_t)(v >> 52);
      }
      ms += __shfl_xor_sync(0xffffffffu, ms, 1);
      if (h == 0) sh.warp_bin[b][w] = ms;
      ms = warp_sum(ms) >> 1;  // every pair counts twice
      cnt = __reduce_add_sync(0xffffffffu, cnt);
      if (lane == 0) {
        sh.bin_mass[b] = ms;
        sh.bin_count[b] = cnt;
      }
    }
    cluster.sync();
    // every warp finds the bin for itself
    int bin0;
    {
      u64 ms = 0, cnt = 0;
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < C && lane < PBINS) {
          const SampleShared* o = cluster.map_shared_rank(&sh, r);
          ms += o->bin_mass[lane];
          cnt += o->bin_count[lane];
        }
      const u64 v = by_mass ? ms : cnt;
      if (want == 0) want = part_of(top_p, warp_sum(v));
      u64 sv = v;
      uint32_t sc = (uint32_t)cnt;
#pragma unroll
      for (int o = 1; o < PBINS; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, sv, o);
        const uint32_t y = __shfl_up_sync(0xffffffffu, sc, o);
        if (lane >= o) sv += x, sc += y;
      }
      const uint32_t reached = __ballot_sync(0xffffffffu, lane < PBINS && sv >= want);
      if (reached == 0) {  // fewer finite logits than k: nothing to cut
        cluster.sync();    // the others' sums may still be read
        continue;
      }
      bin0 = __ffs(reached) - 1;
      above = __shfl_sync(0xffffffffu, sv - v, bin0);
      upto = __shfl_sync(0xffffffffu, sc, bin0);  // elements up to and with the bin
    }
    // the bin [bin0, bin0 + 1) as a range of logits
    const Bin bin{bin0 == PBINS - 1 ? -3.402823466e38f : lowest((float)(bin0 + 1)), bin0 == 0 ? 0.f : lowest((float)bin0),
                  bin0 == 0, cut};
    if (upto <= LIST_CAP) {  // everything that can stay fits the list
      list_pass<T>(s, bin.low, cut, lead);
      cluster.sync();
      if (rank == 0) {
        const int m = min((int)sh.n_items, LIST_CAP);
        sort_items(sh, m, wt);
        settle_list(a, sh, row, by_mass ? m : min(m, top_k), cut_p, top_p, by_mass ? want : 0, min_p, u, wt);
      }
      return;  // (what is read of the others was read before the last barrier)
    }
    // ---- the bin's elements into the warps' queues; from here on only they are looked at
    const int queued = queue_pass<T>(s, bin);
    // a histogram over the bin's elements, joined in the leader: the part where `want` is reached
    const auto histogram = [&](const Parts& parts) {
      clear_bins();
      __syncthreads();
      histogram_pass<T>(s, wt, bin, parts, by_mass, queued);
      join_bins(by_mass);
      find_bin(by_mass, above, want);
      bin_elems = lead->result[0] >> 32;
      above = lead->result[1];
      return (int)(uint32_t)lead->result[0];
    };
    // 1024 parts (of the open last bin: 1/64 each; z - bin0 is exact, as z lies within a factor of two
    // of bin0 or bin0 is 0, and beyond that everything is in the last part)
    Parts parts{top, inv_t, (float)bin0, bin0 == PBINS - 1 ? 64.f : (float)NBINS, -1, 0, 0};
    int part = histogram(parts);
    if (bin_elems > LIST_CAP) {
      // ---- refine the part: bins of 2^shift composed numbers from ceil_c down
      u64 first, last;
      range_pass<T>(s, bin, parts, part, queued, first, last);
      __syncthreads();
      if (tid == 0) {
        sh.range[0] = ~0ull;
        sh.range[1] = 0;
      }
      __syncthreads();
      if (lane == 0) {
        atomicMin(&sh.range[0], first);
        atomicMax(&sh.range[1], last);
      }
      cluster.sync();
      for (int r = 0; r < C; ++r) {
        const SampleShared* o = cluster.map_shared_rank(&sh, r);
        first = min(first, o->range[0]);
        last = max(last, o->range[1]);
      }
      parts.floor_c = first;
      parts.ceil_c = last;
      while (bin_elems > LIST_CAP && parts.shift != 0) {  // with 0 a bin is one element
        // width >> shift < NBINS = 2^10
        parts.shift = max(0, 64 - __clzll((long long)(parts.ceil_c - parts.floor_c)) - 10);
        part = histogram(parts);
        parts.ceil_c -= (u64)part << parts.shift;
        const u64 size = 1ull << parts.shift;
        if (parts.ceil_c - parts.floor_c >= size) parts.floor_c = parts.ceil_c - size + 1;
        part = 0;  // of the narrowed range
      }
    }
    list_part_pass<T>(s, bin, parts, part, queued, lead);
    cluster.sync();
    // these elements decide: sort them, the cut is the one at which `want` is reached
    if (rank == 0) {
      const int m = min((int)sh.n_items, LIST_CAP);
      sort_items(sh, m, wt);
      if (tid == 0) sh.result[0] = m > 0 ? sh.sorted[m - 1] : 0;  // the last one, should none be found
      const int i0 = 2 * tid, i1 = i0 + 1;
      const u64 w0 = i0 < m ? (by_mass ? sh.weight[i0] : 1) : 0, w1 = i1 < m ? (by_mass ? sh.weight[i1] : 1) : 0;
      const u64 before = above + block_before(w0 + w1, sh);
      if (before < want && before + w0 + w1 >= want) {
        const bool second = before + w0 < want;
        sh.result[0] = sh.sorted[second ? i1 : i0];
      }
      __syncthreads();
      if (tid == 0) sh.n_items = 0;
    }
    cluster.sync();
    cut = lead->result[0];
    if (by_mass && !(min_p > 0)) {
      // the mass that stays: all of the bins before, of the bin what the queue holds from the cut on
      u64 m = kept_queue_pass<T>(s, Kept{wt, cut, 0.0}, bin, queued);
      for (int b = 0; b < bin0; ++b) m += sh.warp_bin[b][warp];
      if (lane == 0) sh.kept[warp] = m;
      kept_known = true;
    }
    if (!by_mass) cluster.sync();  // `result` may be written again
  }

  // ---- the draw: block, warp, step of 256 elements, element
  const Kept kept{wt, cut, min_p};
  if (!kept_known) {
    const u64 m = kept_pass<T>(s, kept);
    if (lane == 0) sh.kept[warp] = m;
  }
  __syncthreads();
  u64 share = 0;
#pragma unroll
  for (int w = 0; w < SAMPLE_WARPS; ++w) share += sh.kept[w];
  if (tid == 0) sh.share_mass = share;
  cluster.sync();
  u64 total = 0, before = 0;
#pragma unroll
  for (int r = 0; r < 8; ++r)
    if (r < C) {
      const u64 m = cluster.map_shared_rank(&sh, r)->share_mass;
      total += m;
      if (r < rank) before += m;
    }
  const u64 target = target_of(u, total);
  if (before <= target && target < before + share) {  // one block of the cluster
    int owner = 0;
    u64 b = before;
    while (owner < SAMPLE_WARPS - 1 && target >= b + sh.kept[owner]) b += sh.kept[owner++];
    const int first = min(owner * s.per_warp, s.n_steps), steps = min(first + s.per_warp, s.n_steps) - first;
    for (int step = warp; step < steps; step += SAMPLE_WARPS) {
      const int i0 = s.index(first + step);
      const typename Share<T>::Raw raw = s.load(first + step);
      u64 m = 0;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const float2 l = Share<T>::pair(raw, x);
        m += kept(l.x, i0 + 2 * x) + kept(l.y, i0 + 2 * x + 1);
      }
      m = warp_sum(m);
      if (lane == 0) sh.steps[step] = m;
    }
    __syncthreads();
    if (warp == 0) {
      int step = 0;
      while (step < steps - 1 && target >= b + sh.steps[step]) b += sh.steps[step++];
      const int i0 = s.index(first + step), i1 = min(i0 + 8, a.V);
      u64 lane_sum = 0;
#pragma unroll 1
      for (int i = max(i0, 0); i < i1; ++i) lane_sum += kept(s.one(i), i);
      u64 upto_lane = lane_sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, upto_lane, o);
        if (lane >= o) upto_lane += x;
      }
      b += upto_lane - lane_sum;
      if (b <= target && target < b + lane_sum) {  // one lane
#pragma unroll 1
        for (int i = max(i0, 0); i < i1; ++i) {
          const float l = s.one(i);
          const u64 m = kept(l, i);
          if (target < b + m) {
            a.token[row] = i;
            if (a.logprob) a.logprob[row] = wt.log_share(l, total);
            break;
          }
          b += m;
        }
      }
    }
  }
  cluster.sync();  // a block's shared memory stays until the others have read it
}

}  // namespace dsalt

using namespace dsalt;

extern "C" int dsalt_sample(const void* logits, int dtype, int64_t B, int64_t V, int64_t row_stride, const float* u,
                            const float* temperature, float temperature_value, const int32_t* top_k, int top_k_value,
                            const float* top_p, float top_p_value, const float* min_p, float min_p_value,
                            int64_t* token, float* logprob, void* stream) {
  if (B < 0 || V < 1 || row_stride < V) return fail(DSALT_ERR_INVALID, "sample: bad sizes");
  if (dtype != DSALT_F32 && dtype != DSALT_BF16 && dtype != DSALT_F16) return fail(DSALT_ERR_INVALID, "sample: dtype");
  if (V > (1 << IDX_BITS)) return fail(DSALT_ERR_UNSUPPORTED, "sample: vocabulary %lld above 2^20", (long long)V);
  if (B > (1 << 24)) return fail(DSALT_ERR_UNSUPPORTED, "sample: too many rows");
  if (B == 0) return DSALT_OK;
  if (!logits || !u || !token) return fail(DSALT_ERR_INVALID, "sample: null pointer");
  const int es = dtype == DSALT_F32 ? 4 : 2;
  if ((uintptr_t)logits % es) return fail(DSALT_ERR_INVALID, "sample: logits not aligned to their type");
  // Blocks per row: as many as leave every row's cluster resident at once (two blocks per SM; 64
  // rows of 151936, top-p 0.9, by 4 blocks 91 us, by 8 129), more where the decisive bin of a share
  // would overrun the warps' queues. A share below 2048 does not pay (a row of 4096, top-p 0.9, by
  // one block 28.0 us with shares of 2048, 30.6 with 512; a row of 50257 by shares of 8192 42.9
  // against 36.1).
  int C = 1;
  while (C < 8 && ((V / (2 * C) >= 2048 && B * (2 * C) <= 148 * 2) || V / C > 80000)) C *= 2;
  SampleArgs a;
  a.logits = logits;
  a.row_stride = row_stride;
  a.V = (int)V;
  a.share = (int)((V + 7 + (int64_t)C * BLOCK_ELEMS - 1) / ((int64_t)C * BLOCK_ELEMS) * BLOCK_ELEMS);  // 7: the skew
  if (a.share > MAX_SHARE) return fail(DSALT_ERR_UNSUPPORTED, "sample: share too long");
  a.u = u;
  a.temperature = temperature, a.top_k = top_k, a.top_p = top_p, a.min_p = min_p;
  a.temperature_v = temperature_value, a.top_k_v = top_k_value, a.top_p_v = top_p_value, a.min_p_v = min_p_value;
  a.token = token, a.logprob = logprob;
  const void* kernel = dtype == DSALT_F32   ? reinterpret_cast<const void*>(sample_kernel<float>)
                       : dtype == DSALT_F16 ? reinterpret_cast<const void*>(sample_kernel<__half>)
                                            : reinterpret_cast<const void*>(sample_kernel<__nv_bfloat16>);
  static std::atomic<uint64_t> ready[3];
  if (int rc = allow_dynamic_smem(kernel, (int)sizeof(SampleShared), ready[dtype])) return rc;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * C));
  cfg.blockDim = dim3(SAMPLE_THREADS);
  cfg.dynamicSmemBytes = sizeof(SampleShared);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[] = {&a};
  return check_cuda(cudaLaunchKernelExC(&cfg, kernel, args), "sample launch");
}
