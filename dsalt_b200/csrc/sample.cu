// Token sampling with temperature, top-k, top-p and min-p from given uniform numbers
// (dsalt_sample).
//
// Of a row of logits l, with m = max l and weights w = exp((l - m) / T):
//   top-k: the k first in the order (logit descending, index ascending)
//   top-p: of those the shortest prefix whose mass reaches p times theirs
//   min-p: of those the weights of at least min_p (the largest weight is 1)
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
//   top-p: masses and counts of 16 bins of (m - l) / T, then of 16 parts of the bin where p is
//          reached. Each thread has bins of its own (no atomics: a word per thread and bin), and
//          each warp keeps a queue of its elements in that bin: only they are looked at again.
// Otherwise the bin is refined by histograms over (key, index) until the cut is one element.
// The mass of what stays is then known per warp, and the draw goes down from block to warp to
// 256 elements to the token.
//
// Masses are whole numbers, w * 2^43 rounded from 64-bit arithmetic: their sums do not depend
// on the order in which threads arrive, so a row gives the same token in every batch and in
// every run, and a border lies within 2^20 roundings of 2^-44 (6e-8 of the largest weight at
// the very worst, about 1e-11 in practice) of where sums in 64-bit floating point put it.
//
// One cluster of C blocks owns a row, each a share of it. The row comes from HBM once; later
// passes find it in L1 or L2, which hold it for all rows under way.
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
constexpr int QUEUE = 1024;                   // elements of the decisive bin that a warp keeps
constexpr int MAX_GROUPS = 256;
constexpr double MASS_ONE = 8796093022208.0;  // 2^43: 2^20 of them stay below 2^63
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
      uint32_t count[NBINS], limb[3][NBINS];  // this block's joint histogram; masses as three limbs
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
  u64 bin_mass[2][PBINS];
  uint32_t bin_count[2][PBINS];
  u64 steps[MAX_STEPS];  // masses of the steps of the warp that holds the draw
  u64 kept[SAMPLE_WARPS];
  uint32_t n_items, first_index;
  float best, bound;
  float group_max[64], all_max[MAX_GROUPS];  // of 8 or 16 threads: this block's, the cluster's
  u64 share_mass, range[2], result[4];  // result: written by the leader only
  u64 warp_red[SAMPLE_WARPS];
  double exp2_16[16];  // 2^(j / 16)
};

// (key, index) as one number: larger comes first in the order of the filters
__device__ __forceinline__ u64 compose(float l, int idx) {
  return ((u64)order_f32(l + 0.0f) << IDX_BITS) | (u64)((1 << IDX_BITS) - 1 - idx);  // -0 as 0
}
__device__ __forceinline__ int index_of(u64 c) { return (1 << IDX_BITS) - 1 - (int)(c & ((1u << IDX_BITS) - 1)); }
__device__ __forceinline__ float logit_of(u64 c) {
  const uint32_t k = (uint32_t)(c >> IDX_BITS);
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}

// Weights of one row. 2^t, t = (l - m) log2(e) / T: t = k / 16 + g with |g| <= 1/32, then
// 2^(k/16) from a table of 16 and the exponent, 2^g by its Taylor series to the sixth power
// (the seventh term is below (ln 2 / 32)^7 / 7! = 4.4e-16).
struct Weights {
  float top, l_min;
  double c;
  const double* table;
  // no branch, so that several run side by side; 0 below l_min and for NaN
  __device__ __forceinline__ double operator()(float l) const {
    constexpr double MAGIC = 422212465065984.0;  // 1.5 * 2^48: adding it leaves steps of 1/16
    constexpr double C1 = 0.6931471805599453094, C2 = C1 * C1 / 2, C3 = C2 * C1 / 3, C4 = C3 * C1 / 4, C5 = C4 * C1 / 5,
                     C6 = C5 * C1 / 6;
    const double t = ((double)l - (double)top) * c, r = t + MAGIC;
    const int k = __double2loint(r);
    const double g = t - (r - MAGIC);
    double p = fma(g, C6, C5);
    p = fma(p, g, C4);
    p = fma(p, g, C3);
    p = fma(p, g, C2);
    p = fma(p, g, C1);
    p = fma(p, g, 1.0) * table[k & 15];
    p = __hiloint2double(__double2hiint(p) + ((k >> 4) << 20), __double2loint(p));
    p = l >= l_min ? p : 0.0;
    return l == top ? 1.0 : p;
  }
  __device__ __forceinline__ u64 mass(double w) const {  // w * 2^43 to the nearest whole number
    return (u64)__double_as_longlong(fma(w, MASS_ONE, 4503599627370496.0)) & 0xfffffffffffffull;  // + 2^52
  }
  __device__ __forceinline__ u64 mass(float l) const { return mass((*this)(l)); }
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

// bitonic sort of size (a power of two) values in shared memory by the block
template <typename T, bool DESCENDING>
__device__ __forceinline__ void block_sort(T* v, int size) {
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < size / 2; i += SAMPLE_THREADS) {
        const int x = 2 * i - (i & (j - 1)), y = x + j;
        const T a = v[x], b = v[y];
        if (((x & k) == 0) == (DESCENDING ? a < b : a > b)) {
          v[x] = b;
          v[y] = a;
        }
      }
    }
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
    const bool second = target >= before + m0;
    a.token[row] = sh.by_index[second ? i1 : i0] >> 10;
    if (a.logprob) a.logprob[row] = (float)log((double)(second ? m1 : m0) / (double)total);
  }
}

static_assert(sizeof(SampleShared) <= (228 * 1024 - 2 * 1024) / 2, "two blocks per SM");

template <typename T>
__global__ void __launch_bounds__(SAMPLE_THREADS, 2) sample_kernel(SampleArgs a) {
  extern __shared__ __align__(16) unsigned char dyn[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(dyn);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  SampleShared* lead = cluster.map_shared_rank(&sh, 0);
  const T* src = reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.row_stride;

  const float temp = a.temperature ? a.temperature[row] : a.temperature_v;
  const double top_p = a.top_p ? (double)a.top_p[row] : (double)a.top_p_v;
  const double min_p = a.min_p ? (double)a.min_p[row] : (double)a.min_p_v;
  const int top_k = a.top_k ? a.top_k[row] : a.top_k_v;
  const float u = a.u[row];
  const bool cut_k = top_k > 0 && top_k < a.V, cut_p = top_p < 1.0;

  // ---- the share, in steps of a warp: eight consecutive elements per lane. Places are counted
  // from the 16-byte boundary at or before the row's start, so that whole vectors can be read.
  constexpr int VEC = 16 / (int)sizeof(T);
  const int skew = (int)(((uintptr_t)src & 15) / sizeof(T));
  const int place0 = rank * a.share, n_steps = (max(0, min(a.share, a.V + skew - place0)) + BLOCK_ELEMS - 1) / BLOCK_ELEMS;
  const int per_warp = (n_steps + SAMPLE_WARPS - 1) / SAMPLE_WARPS;  // a warp's steps follow one another
  const int step0 = min(warp * per_warp, n_steps), step1 = min(step0 + per_warp, n_steps);
  const auto load_one = [&](int i) -> float {
    if constexpr (sizeof(T) == 4) return src[i];
    else if constexpr (std::is_same<T, __half>::value) return __half2float(src[i]);
    else return __bfloat162float(src[i]);
  };
  const auto load = [&](int step, float (&l)[8]) -> int {  // NaN outside the row; returns the first index
    const int i0 = place0 + step * BLOCK_ELEMS + lane * 8 - skew;
    if (i0 >= 0 && i0 + 8 <= a.V) {
#pragma unroll
      for (int h = 0; h < 8 / VEC; ++h) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(src + i0) + h);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (sizeof(T) == 4) {
            l[4 * h + e] = __uint_as_float(w[e]);
          } else if constexpr (std::is_same<T, __half>::value) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
            l[2 * e] = f.x, l[2 * e + 1] = f.y;
          } else {
            l[2 * e] = __uint_as_float(w[e] << 16), l[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
          }
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        l[e] = __int_as_float(0x7fffffff);
        if (i0 + e >= 0 && i0 + e < a.V) {
          l[e] = load_one(i0 + e);
        }
      }
    }
    return i0;
  };
  const auto for_each = [&](auto&& f) {  // every element of the share, NaN and places outside too
    for (int step = step0; step < step1; ++step) {
      float l[8];
      const int i0 = load(step, l);
#pragma unroll
      for (int e = 0; e < 8; ++e) f(l[e], i0 + e);
    }
  };

  // ---- the largest logit
  float mine = -INFINITY;
#pragma unroll 4
  for (int step = step0; step < step1; ++step) {
    float l[8];
    load(step, l);
#pragma unroll
    for (int e = 0; e < 8; ++e) mine = fmaxf(mine, l[e]);  // passes over NaN
  }
  float top = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (o == 4 && C < 8 && (lane & 7) == 0) sh.group_max[tid >> 3] = top;
    if (o == 8 && C == 8 && (lane & 15) == 0) sh.group_max[tid >> 4] = top;
  }
  const int groups = C < 8 ? 64 : 32;  // per block
  if (lane == 0) sh.warp_red[warp] = __float_as_uint(top);
  if (tid < 16) sh.exp2_16[tid] = exp2((double)tid / 16);
  if (tid == 0) {
    sh.first_index = 0xffffffffu;
    sh.n_items = 0;
  }
  const auto clear_bins = [&] {
    for (int i = tid; i < NBINS; i += SAMPLE_THREADS) sh.count[i] = sh.limb[0][i] = sh.limb[1][i] = sh.limb[2][i] = 0;
  };
  clear_bins();
  __syncthreads();
#pragma unroll
  for (int w = 0; w < SAMPLE_WARPS; ++w) top = fmaxf(top, __uint_as_float((uint32_t)sh.warp_red[w]));
  if (tid == 0) sh.best = top;
  cluster.sync();
  for (int r = 0; r < C; ++r) top = fmaxf(top, cluster.map_shared_rank(&sh, r)->best);
  // a small top-k's bound: the k-th largest of the groups' maxima. (Near the smallest of them
  // the bound would fall off, so the last few are left to the larger k's way.)
  const bool small_k = cut_k && temp > 0.f && top_k <= C * groups - C * groups / 8;
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
      uint32_t first = 0xffffffffu;
      for_each([&](float l, int i) {
        if (l == top) first = min(first, (uint32_t)i);
      });
      first = __reduce_min_sync(0xffffffffu, first);
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
  wt.l_min = top == INFINITY ? INFINITY : fmaxf((float)((double)top + (double)MIN_LOG2 / wt.c), -3.402823466e38f);
  wt.table = sh.exp2_16;
  const float inv_t = (float)(1.0 / (double)temp);
  const auto z_of = [&](float l) { return l == top ? 0.f : (top - l) * inv_t; };  // grows as l falls, at least 0

  u64 cut = 0;  // elements below it are dropped
  // A list of all that can stay, from `in` on: sorted and settled by the leader.
  const auto gather = [&](auto&& in) {
    for_each([&](float l, int i) {
      if (l > -INFINITY && in(l, i)) {
        const uint32_t at = atomicAdd(&lead->n_items, 1u);
        if (at < LIST_CAP) lead->item[at] = compose(l, i);
      }
    });
    cluster.sync();
  };

  // ---- top-k by a bound from the threads' maxima
  const auto joint_bin = [&](float l) { return (int)fminf(z_of(l) * (NBINS / BIN_SPAN), (float)(NBINS - 1)); };
  const auto join_bins = [&](bool by_mass) {  // each block joins its part of the bins into the leader
    cluster.sync();
    for (int b = rank * SAMPLE_THREADS + tid; b < NBINS; b += C * SAMPLE_THREADS) {
      uint32_t cnt = 0;
      u64 ms = 0;
      for (int r = 0; r < C; ++r) {
        const SampleShared* o = cluster.map_shared_rank(&sh, r);
        cnt += o->count[b];
        if (by_mass) ms += (u64)o->limb[0][b] + ((u64)o->limb[1][b] << 15) + ((u64)o->limb[2][b] << 30);
      }
      lead->total[b] = cnt;
      lead->mass[b] = ms;
    }
    cluster.sync();
  };
  // the leader: the first bin whose running sum reaches `want` (there is one): result = bin and its
  // count, sum before it, elements up to and with it
  const auto find_bin = [&](bool by_mass, u64 above, u64 want) {
    if (rank == 0) {
      const uint32_t c0 = sh.total[2 * tid], c1 = sh.total[2 * tid + 1];
      const u64 v0 = by_mass ? sh.mass[2 * tid] : c0, v1 = by_mass ? sh.mass[2 * tid + 1] : c1;
      const u64 before = above + block_before(v0 + v1, sh);
      const u64 cnt_before = block_before((u64)c0 + c1, sh);
      if (before < want && before + v0 + v1 >= want) {  // one thread: the sums only grow
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
    gather([&](float l, int) { return l >= bound; });
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
    if (rank == 0 && tid == 0) sh.result[0] = NBINS - 1;  // fewer maxima than k: every element
    join_bins(false);
    find_bin(false, 0, (u64)top_k);
    const int bin = (int)(uint32_t)lead->result[0];
    gather([&](float l, int) { return joint_bin(l) <= bin; });
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
    // bins of a level: every block adds up its own, the cluster's sums are found by each warp for
    // itself. Returns whether `want` is reached, and where.
    const auto find_private = [&](int level, int& bin) -> bool {
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
        if (level == 0 && h == 0) sh.warp_bin[b][w] = ms;
        ms = warp_sum(ms) >> 1;  // every pair counts twice
        cnt = __reduce_add_sync(0xffffffffu, cnt);
        if (lane == 0) {
          sh.bin_mass[level][b] = ms;
          sh.bin_count[level][b] = cnt;
        }
      }
      cluster.sync();
      u64 ms = 0, cnt = 0;
      if (lane < PBINS)
        for (int r = 0; r < C; ++r) {
          const SampleShared* o = cluster.map_shared_rank(&sh, r);
          ms += o->bin_mass[level][lane];
          cnt += o->bin_count[level][lane];
        }
      const u64 v = by_mass ? ms : cnt;
      if (want == 0) want = part_of(top_p, warp_sum(v));
      u64 sv = v, sc = cnt;
#pragma unroll
      for (int o = 1; o < PBINS; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, sv, o), y = __shfl_up_sync(0xffffffffu, sc, o);
        if (lane >= o) sv += x, sc += y;
      }
      const uint32_t reached = __ballot_sync(0xffffffffu, lane < PBINS && above + sv >= want);
      if (reached == 0) return false;
      bin = __ffs(reached) - 1;
      above += __shfl_sync(0xffffffffu, sv - v, bin);
      upto += __shfl_sync(0xffffffffu, sc - cnt, bin);  // elements before the bin
      bin_elems = __shfl_sync(0xffffffffu, cnt, bin);
      return true;
    };
    __syncthreads();
#pragma unroll
    for (int b = 0; b < PBINS; ++b) sh.priv[b][tid] = 0;
    __syncwarp();
    for (int step = step0; step < step1; ++step) {
      float l[8];
      const int i0 = load(step, l);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        u64 m = 1ull << 52;
        if (by_mass) m += wt.mass(l[e]);
        if (l[e] > -INFINITY && (cut == 0 || compose(l[e], i0 + e) >= cut))
          sh.priv[(int)fminf(z_of(l[e]), (float)(PBINS - 1))][tid] += m;
      }
    }
    int bin0 = 0, bin = 0;
    if (!find_private(0, bin0)) {  // fewer finite logits than k: nothing to cut
      cluster.sync();              // the others' sums may still be read
      continue;
    }
    const float z0 = (float)bin0;
    const bool last0 = bin0 == PBINS - 1;
    const auto settle = [&](auto&& in) {  // everything that can stay fits the list
      gather(in);
      if (rank == 0) {
        const int m = (int)sh.n_items;
        sort_items(sh, m, wt);
        settle_list(a, sh, row, by_mass ? m : min(m, top_k), cut_p, top_p, by_mass ? want : 0, min_p, u, wt);
      }
      // the others may leave: what is read of them was read before the last barrier
    };
    if (upto + bin_elems <= LIST_CAP) {
      settle([&](float l, int i) { return (last0 || z_of(l) < z0 + 1.f) && (cut == 0 || compose(l, i) >= cut); });
      return;
    }
    // ---- the bin's elements into the warps' queues; from here on only they are looked at
    const int stretch = place0 + step0 * BLOCK_ELEMS - skew;  // index of the warp's first place
    int queued = 0;
    for (int step = step0; step < step1; ++step) {
      float l[8];
      const int i0 = load(step, l);
      uint32_t in = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float z = z_of(l[e]);
        if (z >= z0 && (last0 || z < z0 + 1.f) && l[e] > -INFINITY && (cut == 0 || compose(l[e], i0 + e) >= cut))
          in |= 1u << e;
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
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (in >> e & 1) {
          if (at < QUEUE) sh.queue[warp][at] = (uint16_t)(i0 + e - stretch);
          ++at;
        }
      queued += all;
    }
    __syncwarp();
    const auto for_bin = [&](auto&& f) {  // every element of the bin that this warp owns
      if (queued <= QUEUE) {
        for (int q = lane; q < queued; q += 32) {
          const int i = stretch + (int)sh.queue[warp][q];
          f(load_one(i), i);
        }
      } else {
        for_each([&](float l, int i) {
          const float z = z_of(l);
          if (z >= z0 && (last0 || z < z0 + 1.f) && l > -INFINITY && (cut == 0 || compose(l, i) >= cut)) f(l, i);
        });
      }
    };
    __syncthreads();  // the first level's bins have been read
#pragma unroll
    for (int b = 0; b < PBINS; ++b) sh.priv[b][tid] = 0;
    // parts of 1/16: z - z0 is exact, as z lies within a factor of two of z0 (or z0 is 0)
    const auto part_bin = [&](float l) { return (int)fminf((z_of(l) - z0) * PBINS, (float)(PBINS - 1)); };
    for_bin([&](float l, int) { sh.priv[part_bin(l)][tid] += (1ull << 52) + (by_mass ? wt.mass(l) : 0); });
    find_private(1, bin);
    if (upto + bin_elems <= LIST_CAP) {
      const int to = bin;
      settle([&](float l, int i) {
        const float z = z_of(l);
        if (z < z0) return cut == 0 || compose(l, i) >= cut;
        return (last0 || z < z0 + 1.f) && part_bin(l) <= to && (cut == 0 || compose(l, i) >= cut);
      });
      return;
    }
    // ---- refine the part: bins of 2^shift composed numbers from ceil_c down
    u64 floor_c = 0, ceil_c = ~0ull;
    if (bin_elems > LIST_CAP) {
      u64 first = ~0ull, last = 0;
      for_bin([&](float l, int i) {
        if (part_bin(l) != bin) return;
        const u64 c = compose(l, i);
        first = min(first, c);
        last = max(last, c);
      });
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
        last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
      }
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
      floor_c = first;
      ceil_c = last;
      clear_bins();
      cluster.sync();  // `range` and the bins may be used again
      while (bin_elems > LIST_CAP) {
        const int shift = max(0, 64 - __clzll((long long)(ceil_c - floor_c)) - 10);  // width >> shift < NBINS = 2^10
        for_bin([&](float l, int i) {
          const u64 c = compose(l, i);
          if (c < floor_c || c > ceil_c) return;
          const int b = (int)((ceil_c - c) >> shift);
          atomicAdd(&sh.count[b], 1u);
          if (by_mass) {
            const u64 w = wt.mass(l);
            atomicAdd(&sh.limb[0][b], (uint32_t)(w & 0x7fff));
            atomicAdd(&sh.limb[1][b], (uint32_t)(w >> 15) & 0x7fff);
            atomicAdd(&sh.limb[2][b], (uint32_t)(w >> 30));
          }
        });
        join_bins(by_mass);
        clear_bins();  // for the next histogram
        find_bin(by_mass, above, want);
        bin_elems = lead->result[0] >> 32;
        above = lead->result[1];
        ceil_c -= (u64)(uint32_t)lead->result[0] << shift;
        const u64 size = 1ull << shift;
        if (ceil_c - floor_c >= size) floor_c = ceil_c - size + 1;
        cluster.sync();  // `result` may be written again
      }
    }
    const bool by_part = ceil_c == ~0ull;
    for_bin([&](float l, int i) {
      const u64 c = compose(l, i);
      if (by_part ? part_bin(l) == bin : c >= floor_c && c <= ceil_c) lead->item[atomicAdd(&lead->n_items, 1u)] = c;
    });
    cluster.sync();
    // these elements decide: sort them, the cut is the one at which `want` is reached
    if (rank == 0) {
      const int m = (int)sh.n_items;
      sort_items(sh, m, wt);
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
      u64 m = 0;
      for_bin([&](float l, int i) {
        if (compose(l, i) >= cut) m += wt.mass(l);
      });
      m = warp_sum(m);
      for (int b = 0; b < bin0; ++b) m += sh.warp_bin[b][warp];
      if (lane == 0) sh.kept[warp] = m;
      kept_known = true;
    }
    if (!by_mass) cluster.sync();  // `result` may be written again
  }

  // ---- the draw: block, warp, step of 256 elements, element
  const auto kept_mass = [&](float l, int i) -> u64 {
    const double w = wt(l);
    return w >= min_p && (cut == 0 || compose(l, i) >= cut) && l >= wt.l_min ? wt.mass(w) : 0;
  };
  if (!kept_known) {
    u64 m = 0;
    for_each([&](float l, int i) { m += kept_mass(l, i); });
    m = warp_sum(m);
    if (lane == 0) sh.kept[warp] = m;
  }
  __syncthreads();
  u64 share = 0;
#pragma unroll
  for (int w = 0; w < SAMPLE_WARPS; ++w) share += sh.kept[w];
  if (tid == 0) sh.share_mass = share;
  cluster.sync();
  u64 total = 0, before = 0;
  for (int r = 0; r < C; ++r) {
    const u64 m = cluster.map_shared_rank(&sh, r)->share_mass;
    total += m;
    if (r < rank) before += m;
  }
  const u64 target = target_of(u, total);
  if (before <= target && target < before + share) {  // one block of the cluster
    int owner = 0;
    u64 b = before;
    while (owner < SAMPLE_WARPS - 1 && target >= b + sh.kept[owner]) b += sh.kept[owner++];
    const int first = min(owner * per_warp, n_steps), steps = min(first + per_warp, n_steps) - first;
    for (int step = warp; step < steps; step += SAMPLE_WARPS) {
      float l[8];
      u64 m = 0;
      const int i0 = load(first + step, l);
#pragma unroll
      for (int e = 0; e < 8; ++e) m += kept_mass(l[e], i0 + e);
      m = warp_sum(m);
      if (lane == 0) sh.steps[step] = m;
    }
    __syncthreads();
    if (warp == 0) {
      int step = 0;
      while (step < steps - 1 && target >= b + sh.steps[step]) b += sh.steps[step++];
      float l[8];
      u64 m[8], lane_sum = 0;
      const int i0 = load(first + step, l);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        m[e] = kept_mass(l[e], i0 + e);
        lane_sum += m[e];
      }
      u64 s = lane_sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += x;
      }
      b += s - lane_sum;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (b <= target && target < b + m[e]) {
          a.token[row] = i0 + e;
          if (a.logprob) a.logprob[row] = (float)log((double)m[e] / (double)total);
        }
        b += m[e];
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
  // blocks per row: as many as leave every row's cluster resident at once (two blocks per
  // SM), more where the decisive bin of a share would overrun the warps' queues; a small row is
  // one block's
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
