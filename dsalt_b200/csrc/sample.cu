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
// (key, index) at which the row is cut, and it is found by histograms of counts or masses.
// Where at most LIST_CAP elements can matter they are gathered and settled in one block's
// shared memory; otherwise the histogram's bin is refined until the cut is one element, and
// the row is passed over again with it.
//
// Masses are whole numbers, w * 2^43 rounded from a 64-bit exp: their sums do not depend on
// the order in which threads arrive, so a row gives the same token in every batch and in
// every run, and a border lies within 2^20 roundings of 2^-44 (6e-8 of the largest weight at
// the very worst, about 1e-11 in practice) of where sums in 64-bit floating point put it.
//
// One cluster of C blocks owns a row; each block holds its share of the logits in shared
// memory, so the row is read from HBM once. Histograms and lists are joined through
// distributed shared memory.
#include <cooperative_groups.h>

#include "common.cuh"

namespace dsalt {

namespace cg = cooperative_groups;

constexpr int SAMPLE_THREADS = 512;
constexpr int SAMPLE_WARPS = SAMPLE_THREADS / 32;
constexpr int NBINS = 2 * SAMPLE_THREADS;     // two per thread where they are summed
constexpr int LIST_CAP = 2 * SAMPLE_THREADS;  // two per thread where they are ranked
constexpr int IDX_BITS = 20;                  // vocabulary of at most 2^20
constexpr int SAMPLE_MAX_SHARE = 131072;      // elements of one block: 2^17 limbs of 15 bits fit 32 bits
constexpr int SAMPLE_SMEM_SHARE = 160 * 1024;  // bytes of logits that one block keeps in shared memory
constexpr double MASS_ONE = 8796093022208.0;  // 2^43: 2^20 of them stay below 2^63
constexpr float BIN_SPAN = 32.f;              // (m - l) / T of the first histogram; its last bin takes the rest

typedef unsigned long long u64;

struct SampleArgs {
  const void* logits;
  int64_t row_stride;
  int V, share, in_smem;  // share: elements of one block
  const float* u;
  const float *temperature, *top_p, *min_p;  // per row, or null and the value below
  const int32_t* top_k;
  float temperature_v, top_p_v, min_p_v;
  int top_k_v;
  int64_t* token;
  float* logprob;
};

// The lists are formed after a histogram has been read, in its place.
struct SampleShared {
  union {
    struct {
      uint32_t count[NBINS], limb[3][NBINS];  // this block's histogram; masses as three limbs
    };
    struct {
      u64 sorted[LIST_CAP], weight[LIST_CAP];  // the leader's candidates in order, and their masses
    };
  };
  union {
    u64 mass[NBINS];     // joined over the cluster, in the leader's copy
    u64 item[LIST_CAP];  // candidates as they arrive, in the leader's copy
  };
  uint32_t total[NBINS];  // joined counts, in the leader's copy
  uint32_t n_items;
  // small exchanges; `result` is written by the leader only
  u64 best, share_mass, range[2], result[4];
  u64 warp_red[SAMPLE_WARPS];
};

// logits as unsigned keys that order as the logits do; NaN as -inf, -0 as 0
__device__ __forceinline__ uint32_t logit_key(float l) { return order_f32(l == l ? l + 0.0f : -INFINITY); }
__device__ __forceinline__ float key_logit(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}
// (key, index) as one number: larger comes first in the order of the filters
__device__ __forceinline__ u64 compose(uint32_t key, int idx) {
  return ((u64)key << IDX_BITS) | (u64)((1 << IDX_BITS) - 1 - idx);
}
__device__ __forceinline__ int index_of(u64 c) { return (1 << IDX_BITS) - 1 - (int)(c & ((1u << IDX_BITS) - 1)); }

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ double weight_of(float l, float top, double inv_t) {
  if (l == top) return 1.0;
  if (l == -INFINITY) return 0.0;  // at any temperature
  return exp(((double)l - (double)top) * inv_t);
}
__device__ __forceinline__ u64 mass_of(double w) { return (u64)__double2ull_rn(w * MASS_ONE); }

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

// Sorts the leader's n <= LIST_CAP items by counting the larger ones, and forms their masses.
__device__ void sort_items(SampleShared& sh, int n, float top, double inv_t) {
  __syncthreads();
  const u64 a = (int)threadIdx.x < n ? sh.item[threadIdx.x] : 0;
  const u64 b = (int)threadIdx.x + SAMPLE_THREADS < n ? sh.item[threadIdx.x + SAMPLE_THREADS] : 0;
  int ra = 0, rb = 0;
  for (int j = 0; j < n; ++j) {
    const u64 o = sh.item[j];
    ra += o > a;
    rb += o > b;
  }
  if ((int)threadIdx.x < n) {
    sh.sorted[ra] = a;
    sh.weight[ra] = mass_of(weight_of(key_logit((uint32_t)(a >> IDX_BITS)), top, inv_t));
  }
  if ((int)threadIdx.x + SAMPLE_THREADS < n) {
    sh.sorted[rb] = b;
    sh.weight[rb] = mass_of(weight_of(key_logit((uint32_t)(b >> IDX_BITS)), top, inv_t));
  }
  __syncthreads();
}

// u * total as the whole number that the drawn running sum has to exceed
__device__ __forceinline__ u64 target_of(float u, u64 total) {
  const double x = (double)u * (double)total;
  if (!(x >= 1.0)) return 0;
  return x >= (double)total ? total - 1 : min((u64)x, total - 1);
}

// The leader's block settles a row whose candidates are all in its list: `keep` of them in
// order are within top-k; `want` > 0 is the mass that top-p has to reach, else it is formed here.
__device__ void settle_list(const SampleArgs& a, SampleShared& sh, int row, int keep, bool cut_p, double top_p, u64 want,
                            double min_p, float u, float top, double inv_t) {
  const int i0 = 2 * threadIdx.x, i1 = i0 + 1;
  u64 w0 = i0 < keep ? sh.weight[i0] : 0, w1 = i1 < keep ? sh.weight[i1] : 0;
  if (cut_p) {
    if (want == 0) want = part_of(top_p, block_sum(w0 + w1, sh));
    const u64 before = block_before(w0 + w1, sh);
    keep = (int)block_sum((u64)(i0 < keep && before < want) + (u64)(i1 < keep && before + w0 < want), sh);
  }
  if (min_p > 0) {
    const auto ok = [&](int i) {
      return i < keep && weight_of(key_logit((uint32_t)(sh.sorted[i] >> IDX_BITS)), top, inv_t) >= min_p;
    };
    keep = max(1, (int)block_sum((u64)ok(i0) + (u64)ok(i1), sh));
  }
  const u64 total = block_sum((i0 < keep ? w0 : 0) + (i1 < keep ? w1 : 0), sh);
  const u64 target = target_of(u, total);
  // running sum in index order: a lower index is a larger low part of the item
  for (int i = threadIdx.x; i < keep; i += SAMPLE_THREADS) {
    const int mine = index_of(sh.sorted[i]);
    u64 before = 0;
    for (int j = 0; j < keep; ++j) before += index_of(sh.sorted[j]) < mine ? sh.weight[j] : 0;
    if (before <= target && target < before + sh.weight[i]) {
      a.token[row] = mine;
      if (a.logprob) a.logprob[row] = (float)log((double)sh.weight[i] / (double)total);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(SAMPLE_THREADS) sample_kernel(SampleArgs a) {
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ SampleShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  SampleShared* lead = cluster.map_shared_rank(&sh, 0);
  const int lo = min(rank * a.share, a.V), n = min(lo + a.share, a.V) - lo;
  const T* src = reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.row_stride + lo;

  const float temp = a.temperature ? a.temperature[row] : a.temperature_v;
  const double top_p = a.top_p ? (double)a.top_p[row] : (double)a.top_p_v;
  const double min_p = a.min_p ? (double)a.min_p[row] : (double)a.min_p_v;
  const int top_k = a.top_k ? a.top_k[row] : a.top_k_v;
  const float u = a.u[row];
  const bool cut_k = top_k > 0 && top_k < a.V, cut_p = top_p < 1.0;
  const double inv_t = 1.0 / (double)temp;
  const float bin_scale = (float)inv_t * (NBINS / BIN_SPAN);

  // ---- the share into shared memory; its first element in the order
  const T* val = src;
  u64 best = 0;
  auto see = [&](T v, int at) {
    const u64 c = compose(logit_key(as_float(v)), lo + at);
    best = c > best ? c : best;
  };
  if (a.in_smem) {
    constexpr int VEC = 16 / (int)sizeof(T);
    const int skew = (int)(((uintptr_t)src & 15) / sizeof(T));  // the copy keeps the source's alignment
    T* buf = reinterpret_cast<T*>(dyn) + skew;
    const int head = min(n, (VEC - skew) % VEC), body = (n - head) / VEC;
    for (int i = tid; i < body; i += SAMPLE_THREADS) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(src + head) + i);
      *reinterpret_cast<uint4*>(buf + head + i * VEC) = v;
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) see(e[j], head + i * VEC + j);
    }
    for (int i = tid; i < n - body * VEC; i += SAMPLE_THREADS) {
      const int at = i < head ? i : i + body * VEC;
      buf[at] = src[at];
      see(src[at], at);
    }
    val = buf;
  } else {
    for (int i = tid; i < n; i += SAMPLE_THREADS) see(src[i], i);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const u64 c = __shfl_xor_sync(0xffffffffu, best, o);
    best = c > best ? c : best;
  }
  if (lane == 0) sh.warp_red[warp] = best;
  auto clear_bins = [&] {
    for (int i = tid; i < NBINS; i += SAMPLE_THREADS) sh.count[i] = sh.limb[0][i] = sh.limb[1][i] = sh.limb[2][i] = 0;
  };
  clear_bins();
  __syncthreads();
  if (tid == 0) {
    u64 b = 0;
    for (int w = 0; w < SAMPLE_WARPS; ++w) b = sh.warp_red[w] > b ? sh.warp_red[w] : b;
    sh.best = b;
  }
  cluster.sync();
  for (int r = 0; r < C; ++r) {
    const u64 b = cluster.map_shared_rank(&sh, r)->best;
    best = b > best ? b : best;
  }
  const float top = key_logit((uint32_t)(best >> IDX_BITS));
  // every decision from here to the end is the same in all threads of the cluster
  if (!(temp > 0.f) || top == -INFINITY) {
    if (rank == 0 && tid == 0) {
      a.token[row] = top == -INFINITY ? 0 : index_of(best);
      if (a.logprob) a.logprob[row] = top == -INFINITY ? -INFINITY : 0.f;
    }
    cluster.sync();  // a block's shared memory stays until the others have read it
    return;
  }

  u64 cut = 0;  // elements below it are dropped
  bool listed = false;
  for (int pass = cut_k ? 0 : 1; pass < (cut_p ? 2 : 1) && !listed; ++pass) {
    const bool by_mass = pass == 1;
    u64 want = by_mass ? 0 : (u64)top_k;  // the mass to reach is known once all masses are summed
    u64 above = 0;                        // count or mass before the bins
    u64 floor_c = cut, ceil_c = ~0ull;
    int shift = -1;  // -1: bins of (m - l) / T; else bins of 2^shift composed numbers from ceil_c down
    int bin = 0;
    u64 bin_count = 0;
    auto first_bin = [&](float l) { return l == top ? 0 : (int)fminf((top - l) * bin_scale, (float)(NBINS - 1)); };
    while (true) {
      for (int i = tid; i < n; i += SAMPLE_THREADS) {
        const uint32_t key = logit_key(as_float(val[i]));
        const u64 c = compose(key, lo + i);
        if (c < floor_c || c > ceil_c) continue;
        const float l = key_logit(key);
        const int b = shift < 0 ? first_bin(l) : (int)((ceil_c - c) >> shift);
        atomicAdd(&sh.count[b], 1u);
        if (by_mass) {
          const u64 w = mass_of(weight_of(l, top, inv_t));
          atomicAdd(&sh.limb[0][b], (uint32_t)(w & 0x7fff));
          atomicAdd(&sh.limb[1][b], (uint32_t)(w >> 15) & 0x7fff);
          atomicAdd(&sh.limb[2][b], (uint32_t)(w >> 30));
        }
      }
      cluster.sync();
      // each block joins its part of the bins into the leader
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
      clear_bins();  // for the next histogram
      if (rank == 0) {
        // the first bin whose running sum reaches `want`
        const uint32_t c0 = sh.total[2 * tid], c1 = sh.total[2 * tid + 1];
        const u64 v0 = by_mass ? sh.mass[2 * tid] : c0, v1 = by_mass ? sh.mass[2 * tid + 1] : c1;
        if (want == 0) want = part_of(top_p, block_sum(v0 + v1, sh));
        const u64 before = above + block_before(v0 + v1, sh);
        const u64 cnt_before = block_before((u64)c0 + c1, sh);
        if (before < want && before + v0 + v1 >= want) {  // one thread: the sums only grow
          const bool second = before + v0 < want;
          sh.result[0] = (u64)(2 * tid + second) | ((u64)(second ? c1 : c0) << 32);
          sh.result[1] = before + (second ? v0 : 0);
          sh.result[2] = cnt_before + c0 + (second ? c1 : 0);  // elements up to and with the bin
          sh.result[3] = want;
        }
        if (tid == 0) sh.n_items = 0;
      }
      cluster.sync();
      bin = (int)(uint32_t)lead->result[0];
      bin_count = lead->result[0] >> 32;
      above = lead->result[1];
      want = lead->result[3];
      if (shift < 0) {
        if (lead->result[2] <= LIST_CAP) {
          listed = true;  // everything that can stay fits the list
          break;
        }
        // the composed numbers that the bin spans
        u64 first = ~0ull, last = 0;
        for (int i = tid; i < n; i += SAMPLE_THREADS) {
          const uint32_t key = logit_key(as_float(val[i]));
          const u64 c = compose(key, lo + i);
          if (c < floor_c || first_bin(key_logit(key)) != bin) continue;
          first = min(first, c);
          last = max(last, c);
        }
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
        cluster.sync();  // `range` may be used again
      } else {
        ceil_c -= (u64)bin << shift;
        const u64 size = 1ull << shift;
        if (ceil_c - floor_c >= size) floor_c = ceil_c - size + 1;
      }
      if (bin_count <= LIST_CAP) {
        // the bin's elements decide: sort them, the cut is the one at which `want` is reached
        for (int i = tid; i < n; i += SAMPLE_THREADS) {
          const u64 c = compose(logit_key(as_float(val[i])), lo + i);
          if (c >= floor_c && c <= ceil_c) lead->item[atomicAdd(&lead->n_items, 1u)] = c;
        }
        cluster.sync();
        if (rank == 0) {
          sort_items(sh, (int)bin_count, top, inv_t);
          const int i0 = 2 * tid, i1 = i0 + 1, m = (int)bin_count;
          const u64 w0 = i0 < m ? (by_mass ? sh.weight[i0] : 1) : 0, w1 = i1 < m ? (by_mass ? sh.weight[i1] : 1) : 0;
          const u64 before = above + block_before(w0 + w1, sh);
          if (before < want && before + w0 + w1 >= want) sh.result[0] = sh.sorted[before + w0 < want ? i1 : i0];
        }
        cluster.sync();
        cut = lead->result[0];
        clear_bins();  // the leader's held the list
        __syncthreads();
        break;
      }
      const u64 width = ceil_c - floor_c;
      shift = max(0, 64 - __clzll((long long)width) - 10);  // width >> shift < NBINS = 2^10
    }
    if (listed) {
      for (int i = tid; i < n; i += SAMPLE_THREADS) {
        const uint32_t key = logit_key(as_float(val[i]));
        const u64 c = compose(key, lo + i);
        if (c >= cut && first_bin(key_logit(key)) <= bin) lead->item[atomicAdd(&lead->n_items, 1u)] = c;
      }
      cluster.sync();
      if (rank == 0) {
        const int m = (int)sh.n_items;
        sort_items(sh, m, top, inv_t);
        settle_list(a, sh, row, by_mass ? m : min(m, top_k), cut_p, top_p, by_mass ? want : 0, min_p, u, top, inv_t);
      }
      // the others' shared memory is no longer read, theirs of the leader neither
      return;
    }
  }

  // ---- many elements stay: a pass over the row. Each thread sums a stretch of the share (an
  // odd number of elements, so that the threads' stretches start in different banks).
  const int per = ((n + SAMPLE_THREADS - 1) / SAMPLE_THREADS) | 1;
  const int from = min(tid * per, n), to = min(from + per, n);
  auto kept_mass = [&](int i) -> u64 {
    const uint32_t key = logit_key(as_float(val[i]));
    if (compose(key, lo + i) < cut) return 0;
    const double w = weight_of(key_logit(key), top, inv_t);
    return w >= min_p ? mass_of(w) : 0;
  };
  u64 sum = 0;
  for (int i = from; i < to; ++i) sum += kept_mass(i);
  const u64 share = block_sum(sum, sh);
  u64 before = block_before(sum, sh);
  if (tid == 0) sh.share_mass = share;
  cluster.sync();
  u64 total = 0;
  for (int r = 0; r < C; ++r) {
    const u64 m = cluster.map_shared_rank(&sh, r)->share_mass;
    total += m;
    if (r < rank) before += m;
  }
  const u64 target = target_of(u, total);
  if (before <= target && target < before + sum) {  // one thread of the cluster
    for (int i = from; i < to; ++i) {
      const u64 m = kept_mass(i);
      if (target < before + m) {
        a.token[row] = lo + i;
        if (a.logprob) a.logprob[row] = (float)log((double)m / (double)total);
        break;
      }
      before += m;
    }
  }
  cluster.sync();
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
  // SM), at least so many that a share fits; a small row is one block's
  int C = 1;
  while (C < 8 && (V / (2 * C) >= 2048 && B * (2 * C) <= 148 * 2)) C *= 2;
  while (C < 8 && ((V + C - 1) / C > SAMPLE_MAX_SHARE || (V + C - 1) / C * es > SAMPLE_SMEM_SHARE)) C *= 2;
  SampleArgs a;
  a.logits = logits;
  a.row_stride = row_stride;
  a.V = (int)V;
  a.share = (int)(((V + C - 1) / C + 7) / 8 * 8);
  a.in_smem = (int64_t)a.share * es <= SAMPLE_SMEM_SHARE + 64;
  a.u = u;
  a.temperature = temperature, a.top_k = top_k, a.top_p = top_p, a.min_p = min_p;
  a.temperature_v = temperature_value, a.top_k_v = top_k_value, a.top_p_v = top_p_value, a.min_p_v = min_p_value;
  a.token = token, a.logprob = logprob;
  const void* kernel = dtype == DSALT_F32   ? reinterpret_cast<const void*>(sample_kernel<float>)
                       : dtype == DSALT_F16 ? reinterpret_cast<const void*>(sample_kernel<__half>)
                                            : reinterpret_cast<const void*>(sample_kernel<__nv_bfloat16>);
  static std::atomic<uint64_t> ready[3];
  if (int rc = allow_dynamic_smem(kernel, SAMPLE_SMEM_SHARE + 256, ready[dtype])) return rc;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * C));
  cfg.blockDim = dim3(SAMPLE_THREADS);
  cfg.dynamicSmemBytes = a.in_smem ? (size_t)a.share * es + 32 : 0;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[] = {&a};
  return check_cuda(cudaLaunchKernelExC(&cfg, kernel, args), "sample launch");
}
