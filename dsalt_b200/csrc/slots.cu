// Block tables and slot maps of a paged key/value cache, built on the GPU from the request
// lengths (dsalt_reserve_slots, dsalt_release_slots).
//
// Row s holds len[s] tokens in ceil(len/P) pages and wants new[s] more:
//   have = ceil(len/P), want = ceil((len + new)/P), need = want - have (0 where the row's
//   table or the token budget does not hold it: refused)
//   upto = running sum of need over the rows; a row is granted when need = 0 or upto <= n_free
//   page number j of that running order is free[n_free - 1 - j]
//   slot of token r of row s = page(s, (len + r) / P) * P + (len + r) % P
// A granted row's first page number is upto - need, whatever becomes of the rows behind it,
// so no row waits for another: two running sums (need, new) over the rows and then one
// independent computation per token.
#include <cooperative_groups.h>

#include <atomic>

#include "common.cuh"

namespace dsalt {

namespace cg = cooperative_groups;

constexpr int SLOT_THREADS = 1024;
constexpr int SLOT_MAX_SEQS = 8192;  // three int32 per row in shared memory

struct Pair64 {
  long long a, b;
};

// inclusive sums of a pair over the block's threads
__device__ __forceinline__ Pair64 block_scan(Pair64 v, Pair64* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, v.a, o), b = __shfl_up_sync(0xffffffffu, v.b, o);
    if (lane >= o) {
      v.a += a;
      v.b += b;
    }
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    Pair64 s = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long a = __shfl_up_sync(0xffffffffu, s.a, o), b = __shfl_up_sync(0xffffffffu, s.b, o);
      if (lane >= o) {
        s.a += a;
        s.b += b;
      }
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  if (warp > 0) {
    v.a += warp_sums[warp - 1].a;
    v.b += warp_sums[warp - 1].b;
  }
  return v;
}

// One cluster. Every CTA forms the running sums of all rows for itself (they are a few
// loads and two shuffles deep; exchanging them would cost as much) and then fills its share
// of the tokens and table rows. The lengths and the free count may be updated in place:
// they are written behind a cluster barrier, after the last CTA has read them.
__global__ void __launch_bounds__(SLOT_THREADS) reserve_slots_kernel(
    int32_t* __restrict__ tables, int n_seqs, int max_pages, const int32_t* seq_lens, const int32_t* new_lens,
    const int32_t* __restrict__ free_pages, int free_cap, const int32_t* n_free_in, int page, int64_t n_tokens,
    int64_t* __restrict__ slots, int32_t* __restrict__ positions, int32_t* __restrict__ cu_new, uint8_t* granted,
    int32_t* seq_lens_out, int32_t* n_free_out) {
  extern __shared__ int32_t sm[];
  int32_t* s_cu = sm;                // [n_seqs + 1] first token of each row, at most n_tokens
  int32_t* s_old = s_cu + n_seqs + 1;  // [n_seqs] length before, -1 - length where the row is refused
  int32_t* s_first = s_old + n_seqs;   // [n_seqs] number of its first new page in the running order
  __shared__ Pair64 warp_sums[32];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), n_ranks = (int)cluster.num_blocks();
  const int tid = threadIdx.x;
  int n_free = *n_free_in;
  n_free = n_free < 0 ? 0 : (n_free > free_cap ? free_cap : n_free);
  Pair64 carry{0, 0};
  long long taken = 0;  // pages of granted rows, this thread's rows
  for (int base = 0; base < n_seqs; base += SLOT_THREADS) {
    const int s = base + tid;
    long long old = 0, add = 0;
    if (s < n_seqs) {
      old = max(seq_lens[s], 0);
      add = max(new_lens[s], 0);
    }
    // the token budget is judged on the running sum of the new tokens: that sum comes first
    const long long end = carry.b + block_scan(Pair64{0, add}, warp_sums).b;
    carry.b += warp_sums[31].b;
    __syncthreads();
    const long long have = (old + page - 1) / page, want = (old + add + page - 1) / page;
    const bool fits = want <= max_pages && end <= n_tokens && old + add <= 0x7fffffffLL;
    const long long need = s < n_seqs && fits ? want - have : 0;
    const long long upto = carry.a + block_scan(Pair64{need, 0}, warp_sums).a;
    carry.a += warp_sums[31].a;
    __syncthreads();
    const bool ok = fits && (need == 0 || upto <= n_free);
    if (s < n_seqs) {
      s_cu[s + 1] = (int32_t)min(end, (long long)n_tokens);
      s_old[s] = ok ? (int32_t)old : (int32_t)(-1 - old);
      s_first[s] = ok ? (int32_t)(upto - need) : 0;
      if (ok) taken += need;
    }
  }
  if (tid == 0) s_cu[0] = 0;
  block_scan(Pair64{taken, 0}, warp_sums);  // its barriers also publish s_cu, s_old, s_first
  const long long all_taken = warp_sums[31].a;
  // new table entries, a warp per row
  const int warp = tid >> 5, lane = tid & 31;
  for (int s = rank * (SLOT_THREADS / 32) + warp; s < n_seqs; s += n_ranks * (SLOT_THREADS / 32)) {
    const int old = s_old[s];
    if (old < 0) continue;
    const int add = s_cu[s + 1] - s_cu[s];
    const int have = (old + page - 1) / page, want = (int)(((long long)old + add + page - 1) / page);
    const int first = s_first[s];
    for (int c = have + lane; c < want; c += 32)
      tables[(int64_t)s * max_pages + c] = free_pages[n_free - 1 - (first + c - have)];
  }
  // slots and positions: four consecutive tokens per thread, one search for the first's row
  const int64_t quads = (n_tokens + 3) / 4;
  for (int64_t qd = (int64_t)rank * SLOT_THREADS + tid; qd < quads; qd += (int64_t)n_ranks * SLOT_THREADS) {
    const int64_t t0 = qd * 4;
    int lo = 0, hi = n_seqs;  // first row whose end lies behind t0
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (s_cu[mid + 1] > t0) hi = mid;
      else lo = mid + 1;
    }
    int s = lo;
    int64_t sl[4];
    int32_t ps[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t t = t0 + e;
      while (s < n_seqs && s_cu[s + 1] <= t) ++s;
      sl[e] = -1;
      ps[e] = 0;
      if (s < n_seqs && s_old[s] >= 0) {
        const int old = s_old[s];
        const int pos = old + (int)(t - s_cu[s]);
        const int col = pos / page, have = (old + page - 1) / page;
        const int id = col < have ? tables[(int64_t)s * max_pages + col]
                                  : free_pages[n_free - 1 - (s_first[s] + col - have)];
        ps[e] = pos;
        if (id >= 0) sl[e] = (int64_t)id * page + pos % page;
      }
    }
    if (t0 + 4 <= n_tokens) {
      reinterpret_cast<longlong2*>(slots + t0)[0] = make_longlong2(sl[0], sl[1]);
      reinterpret_cast<longlong2*>(slots + t0)[1] = make_longlong2(sl[2], sl[3]);
      *reinterpret_cast<int4*>(positions + t0) = make_int4(ps[0], ps[1], ps[2], ps[3]);
    } else {
      for (int e = 0; e < 4 && t0 + e < n_tokens; ++e) {
        slots[t0 + e] = sl[e];
        positions[t0 + e] = ps[e];
      }
    }
  }
  if (n_ranks > 1) cluster.sync();  // every CTA has read the lengths and the free count
  else __syncthreads();
  if (rank == 0) {
    for (int s = tid; s < n_seqs; s += SLOT_THREADS) {
      const int old = s_old[s];
      const bool ok = old >= 0;
      granted[s] = ok ? 1 : 0;
      // a granted row's tokens all lie within the budget: its share of s_cu is its new length
      seq_lens_out[s] = ok ? old + (s_cu[s + 1] - s_cu[s]) : -1 - old;
    }
    for (int s = tid; s <= n_seqs; s += SLOT_THREADS) cu_new[s] = s_cu[s];
    if (tid == 0) *n_free_out = n_free - (int)all_taken;
  }
}

// The pages of the flagged rows go back on the stack, in the order in which reserve_slots
// would take them again (page number j of the rows in order to free[n_free + total - 1 - j]);
// their table entries become -1 and their lengths 0.
__global__ void __launch_bounds__(SLOT_THREADS) release_slots_kernel(int32_t* __restrict__ tables, int n_seqs,
                                                                     int max_pages, int32_t* __restrict__ seq_lens,
                                                                     const uint8_t* __restrict__ release,
                                                                     int32_t* __restrict__ free_pages, int free_cap,
                                                                     int32_t* __restrict__ n_free_io, int page) {
  extern __shared__ int32_t s_upto[];  // [n_seqs] pages of the flagged rows up to and with s
  __shared__ Pair64 warp_sums[32];
  const int tid = threadIdx.x;
  int n_free = *n_free_io;
  n_free = n_free < 0 ? 0 : (n_free > free_cap ? free_cap : n_free);
  long long carry = 0;
  for (int base = 0; base < n_seqs; base += SLOT_THREADS) {
    const int s = base + tid;
    long long held = 0;
    if (s < n_seqs && release[s]) held = min(((long long)max(seq_lens[s], 0) + page - 1) / page, (long long)max_pages);
    const Pair64 p = block_scan(Pair64{held, 0}, warp_sums);
    if (s < n_seqs) s_upto[s] = (int32_t)(carry + p.a);
    carry += warp_sums[31].a;
    __syncthreads();
  }
  const int total = (int)carry;
  // every flagged page: number j, its row by search
  for (int j = tid; j < total; j += SLOT_THREADS) {
    int lo = 0, hi = n_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (s_upto[mid] > j) hi = mid;
      else lo = mid + 1;
    }
    const int col = j - (lo > 0 ? s_upto[lo - 1] : 0);
    int32_t* e = tables + (int64_t)lo * max_pages + col;
    const int64_t to = (int64_t)n_free + total - 1 - j;
    if (to < free_cap) free_pages[to] = *e;
    *e = -1;
  }
  for (int s = tid; s < n_seqs; s += SLOT_THREADS)
    if (release[s]) seq_lens[s] = 0;
  if (tid == 0) *n_free_io = (int)min((long long)n_free + total, (long long)free_cap);
}

static bool page_ok(int page) { return page == 16 || page == 32 || page == 64 || page == 128; }

}  // namespace dsalt

using namespace dsalt;

extern "C" {

int dsalt_reserve_slots(int32_t* block_tables, int n_seqs, int max_pages, const int32_t* seq_lens,
                        const int32_t* new_lens, const int32_t* free_pages, int64_t free_capacity,
                        const int32_t* n_free, int page_size, int64_t n_tokens, int64_t* slots, int32_t* positions,
                        int32_t* cu_new, uint8_t* granted, int32_t* seq_lens_out, int32_t* n_free_out, void* stream) {
  if (n_seqs < 1 || max_pages < 1 || n_tokens < 0 || free_capacity < 0)
    return fail(DSALT_ERR_INVALID, "reserve_slots: bad sizes");
  if (!page_ok(page_size)) return fail(DSALT_ERR_UNSUPPORTED, "reserve_slots: page size %d not in {16, 32, 64, 128}", page_size);
  if (n_seqs > SLOT_MAX_SEQS) return fail(DSALT_ERR_UNSUPPORTED, "reserve_slots: %d rows, at most %d", n_seqs, SLOT_MAX_SEQS);
  if (n_tokens > 0x7fffff00LL || free_capacity > 0x7fffff00LL)
    return fail(DSALT_ERR_UNSUPPORTED, "reserve_slots: token budget or pool too large");
  if (!block_tables || !seq_lens || !new_lens || (free_capacity > 0 && !free_pages) || !n_free || !cu_new || !granted ||
      !seq_lens_out || !n_free_out || (n_tokens > 0 && (!slots || !positions)))
    return fail(DSALT_ERR_INVALID, "reserve_slots: null pointer");
  if (((uintptr_t)slots | (uintptr_t)positions) & 15)
    return fail(DSALT_ERR_INVALID, "reserve_slots: slots and positions must be 16-byte aligned");
  const size_t smem = sizeof(int32_t) * (3 * (size_t)n_seqs + 1);
  static std::atomic<uint64_t> ready{0};
  if (int rc = allow_dynamic_smem(reinterpret_cast<const void*>(reserve_slots_kernel),
                                  (int)(sizeof(int32_t) * (3 * (size_t)SLOT_MAX_SEQS + 1)), ready))
    return rc;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  const unsigned ctas = n_tokens > 4 * SLOT_THREADS ? 8 : 1;  // one CTA covers a decode step's tokens in one go
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(SLOT_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, reserve_slots_kernel, block_tables, n_seqs, max_pages, seq_lens, new_lens,
                                       free_pages, (int)free_capacity, n_free, page_size, n_tokens, slots, positions,
                                       cu_new, granted, seq_lens_out, n_free_out),
                    "reserve_slots launch");
}

int dsalt_release_slots(int32_t* block_tables, int n_seqs, int max_pages, int32_t* seq_lens, const uint8_t* release,
                        int32_t* free_pages, int64_t free_capacity, int32_t* n_free, int page_size, void* stream) {
  if (n_seqs < 1 || max_pages < 1 || free_capacity < 0) return fail(DSALT_ERR_INVALID, "release_slots: bad sizes");
  if (!page_ok(page_size)) return fail(DSALT_ERR_UNSUPPORTED, "release_slots: page size %d not in {16, 32, 64, 128}", page_size);
  if (n_seqs > SLOT_MAX_SEQS) return fail(DSALT_ERR_UNSUPPORTED, "release_slots: %d rows, at most %d", n_seqs, SLOT_MAX_SEQS);
  if (free_capacity > 0x7fffff00LL) return fail(DSALT_ERR_UNSUPPORTED, "release_slots: pool too large");
  if (!block_tables || !seq_lens || !release || (free_capacity > 0 && !free_pages) || !n_free)
    return fail(DSALT_ERR_INVALID, "release_slots: null pointer");
  release_slots_kernel<<<1, SLOT_THREADS, sizeof(int32_t) * (size_t)n_seqs, reinterpret_cast<cudaStream_t>(stream)>>>(
      block_tables, n_seqs, max_pages, seq_lens, release, free_pages, (int)free_capacity, n_free, page_size);
  return check_cuda(cudaGetLastError(), "release_slots launch");
}

}  // extern "C"
