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
//
// Bound by latency throughout (a few KB of tables): 64 rows of a decode step 4.1 us on a B200, of
// which a launch is 2.5; 509 rows of 513 tokens (3 MB of slots and positions) and their release
// 22.8 us in three kernels.
#include <atomic>

#include "common.cuh"

namespace dsalt {

constexpr int SLOT_MAX_SEQS = 8192;  // three int32 per row in shared memory
constexpr int SLOT_THREADS = 1024;
constexpr int SLOT_FILL_MAX = 4096;  // tokens that the rows' block numbers itself: 4096 in 64 rows take 7.1 us
                                     // either way, 2048 in 4 rows 4.6 against 6.2, 8192 in 64 rows 9.9 against 7.3

struct Pair64 {
  long long a, b;
};

// inclusive sums of a pair over the block's threads, and the block's total
template <int THREADS>
__device__ __forceinline__ Pair64 block_scan(Pair64 v, Pair64* warp_sums, Pair64& all) {
  constexpr int WARPS = THREADS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, v.a, o), b = __shfl_up_sync(0xffffffffu, v.b, o);
    if (lane >= o) {
      v.a += a;
      v.b += b;
    }
  }
  __syncthreads();  // the sums of the call before have been read
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  Pair64 s = lane < WARPS ? warp_sums[lane] : Pair64{0, 0}, before{0, 0};
#pragma unroll
  for (int o = 1; o < WARPS; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, s.a, o), b = __shfl_up_sync(0xffffffffu, s.b, o);
    if (lane >= o) {
      s.a += a;
      s.b += b;
    }
  }
  all.a = __shfl_sync(0xffffffffu, s.a, WARPS - 1);
  all.b = __shfl_sync(0xffffffffu, s.b, WARPS - 1);
  before.a = __shfl_sync(0xffffffffu, s.a, warp > 0 ? warp - 1 : 0);
  before.b = __shfl_sync(0xffffffffu, s.b, warp > 0 ? warp - 1 : 0);
  if (warp > 0) {
    v.a += before.a;
    v.b += before.b;
  }
  return v;
}

// The rows: one block, which also numbers the tokens where they are few (FILL). Lengths and
// free count may be updated in place: each thread has read its rows, and everybody the free
// count, before the barriers that come before the writes.
template <int THREADS, bool FILL>
__global__ void __launch_bounds__(THREADS) reserve_slots_kernel(
    int32_t* __restrict__ tables, int n_seqs, int max_pages, const int32_t* seq_lens, const int32_t* new_lens,
    const int32_t* __restrict__ free_pages, int free_cap, const int32_t* n_free_in, int page_shift, int64_t n_tokens,
    int64_t* __restrict__ slots, int32_t* __restrict__ positions, int32_t* __restrict__ cu_new, uint8_t* granted,
    int32_t* seq_lens_out, int32_t* n_free_out) {
  extern __shared__ int32_t sm[];
  int32_t* s_cu = sm;                  // [n_seqs + 1] first token of each row, at most n_tokens
  int32_t* s_old = s_cu + n_seqs + 1;  // [n_seqs] length before, -1 - length where the row is refused
  int32_t* s_first = s_old + n_seqs;   // [n_seqs] number of its first new page in the running order
  __shared__ Pair64 warp_sums[THREADS / 32];
  __shared__ int s_taken;
  const int tid = threadIdx.x, page_mask = (1 << page_shift) - 1;
  int n_free = *n_free_in;
  n_free = n_free < 0 ? 0 : (n_free > free_cap ? free_cap : n_free);
  if (tid == 0) s_taken = 0;
  Pair64 carry{0, 0};
  for (int base = 0; base < n_seqs; base += THREADS) {
    const int s = base + tid;
    long long old = 0, add = 0;
    if (s < n_seqs) {
      old = max(seq_lens[s], 0);
      add = max(new_lens[s], 0);
    }
    // the token budget is judged on the running sum of the new tokens: that sum comes first
    Pair64 all;
    const long long end = carry.b + block_scan<THREADS>(Pair64{0, add}, warp_sums, all).b;
    carry.b += all.b;
    const long long have = (old + page_mask) >> page_shift, want = (old + add + page_mask) >> page_shift;
    const bool fits = want <= max_pages && end <= n_tokens && old + add <= 0x7fffffffLL;
    const long long need = s < n_seqs && fits ? want - have : 0;
    const long long upto = carry.a + block_scan<THREADS>(Pair64{need, 0}, warp_sums, all).a;
    carry.a += all.a;
    const bool ok = fits && (need == 0 || upto <= n_free);
    if (s < n_seqs) {
      s_cu[s + 1] = (int32_t)min(end, (long long)n_tokens);
      s_old[s] = ok ? (int32_t)old : (int32_t)(-1 - old);
      s_first[s] = ok ? (int32_t)(upto - need) : 0;
      // granted rows that need pages are the first that do: the last one's sum is what is taken
      if (ok && need > 0) atomicMax(&s_taken, (int)upto);
    }
  }
  if (tid == 0) s_cu[0] = 0;
  __syncthreads();
  // new table entries: of a row that gets few pages by a thread, of others by a warp
  const int warp = tid >> 5, lane = tid & 31;
  const auto enter = [&](int s, int from, int step, bool few) {
    const int old = s_old[s];
    if (old < 0) return;
    const int add = s_cu[s + 1] - s_cu[s], first = s_first[s];
    const int have = (int)(((long long)old + page_mask) >> page_shift), want = (int)(((long long)old + add + page_mask) >> page_shift);
    if ((want - have <= 4) != few) return;
    for (int c = have + from; c < want; c += step)
      tables[(int64_t)s * max_pages + c] = free_pages[n_free - 1 - (first + c - have)];
  };
  for (int s = tid; s < n_seqs; s += THREADS) enter(s, 0, 1, true);
  for (int s = warp; s < n_seqs; s += THREADS / 32) enter(s, lane, 32, false);
  for (int s = tid; s < n_seqs; s += THREADS) {
    const int old = s_old[s];
    const bool ok = old >= 0;
    granted[s] = ok ? 1 : 0;
    // a granted row's tokens all lie within the budget: its share of s_cu is its new length
    seq_lens_out[s] = ok ? old + (s_cu[s + 1] - s_cu[s]) : -1 - old;
  }
  for (int s = tid; s <= n_seqs; s += THREADS) cu_new[s] = s_cu[s];
  if (tid == 0) *n_free_out = n_free - s_taken;
  if (!FILL) return;
  for (int64_t t = tid; t < n_tokens; t += THREADS) {
    int lo = 0, hi = n_seqs;  // first row whose end lies behind t
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (s_cu[mid + 1] > t) hi = mid;
      else lo = mid + 1;
    }
    int64_t slot = -1;
    int pos = 0;
    if (lo < n_seqs && s_old[lo] >= 0) {
      const int old = s_old[lo], have = (int)(((long long)old + page_mask) >> page_shift);
      pos = old + (int)(t - s_cu[lo]);
      const int col = pos >> page_shift;
      // entries just written are read from where they came
      const int id = col < have ? tables[(int64_t)lo * max_pages + col]
                                : free_pages[n_free - 1 - (s_first[lo] + col - have)];
      if (id >= 0) slot = ((int64_t)id << page_shift) + (pos & page_mask);
    }
    slots[t] = slot;
    positions[t] = pos;
  }
}

// The tokens, where they are many: four consecutive ones per thread, one search for the first's
// row, from what the rows' kernel has written. (That kernel may still be under way when this one
// begins: its results are read by ordinary loads, not by those for constant data.)
__global__ void __launch_bounds__(256) fill_slots_kernel(const int32_t* tables, int n_seqs, int max_pages,
                                                         const int32_t* seq_lens, const int32_t* cu,
                                                         const uint8_t* granted, int page_shift, int64_t n_tokens,
                                                         int64_t* slots, int32_t* positions) {
  cudaGridDependencySynchronize();
  const int64_t t0 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (t0 >= n_tokens) return;
  int lo = 0, hi = n_seqs;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] > t0) hi = mid;
    else lo = mid + 1;
  }
  int s = lo;
  int64_t sl[4];
  int32_t ps[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int64_t t = t0 + e;
    while (s < n_seqs && cu[s + 1] <= t) ++s;
    sl[e] = -1;
    ps[e] = 0;
    if (s < n_seqs && granted[s]) {
      const int pos = seq_lens[s] - (int)(cu[s + 1] - t);
      const int id = tables[(int64_t)s * max_pages + (pos >> page_shift)];
      ps[e] = pos;
      if (id >= 0) sl[e] = ((int64_t)id << page_shift) + (pos & ((1 << page_shift) - 1));
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

// The pages of the flagged rows go back on the stack, in the order in which reserve_slots
// would take them again (page number j of the rows in order to free[n_free + total - 1 - j]);
// their table entries become -1 and their lengths 0.
__global__ void __launch_bounds__(SLOT_THREADS) release_slots_kernel(int32_t* __restrict__ tables, int n_seqs, int max_pages,
                                                                int32_t* __restrict__ seq_lens,
                                                                const uint8_t* __restrict__ release,
                                                                int32_t* __restrict__ free_pages, int free_cap,
                                                                int32_t* __restrict__ n_free_io, int page_shift) {
  extern __shared__ int32_t s_upto[];  // [n_seqs] pages of the flagged rows up to and with s
  __shared__ Pair64 warp_sums[SLOT_THREADS / 32];
  const int tid = threadIdx.x, page_mask = (1 << page_shift) - 1;
  int n_free = *n_free_io;
  n_free = n_free < 0 ? 0 : (n_free > free_cap ? free_cap : n_free);
  long long carry = 0;
  for (int base = 0; base < n_seqs; base += SLOT_THREADS) {
    const int s = base + tid;
    long long held = 0;
    if (s < n_seqs && release[s]) held = min(((long long)max(seq_lens[s], 0) + page_mask) >> page_shift, (long long)max_pages);
    Pair64 all;
    const Pair64 p = block_scan<SLOT_THREADS>(Pair64{held, 0}, warp_sums, all);
    if (s < n_seqs) s_upto[s] = (int32_t)(carry + p.a);
    carry += all.a;
  }
  __syncthreads();
  const int total = (int)carry;
  // every flagged page: number j, its row by search; four under way at a time
#pragma unroll 4
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
static int shift_of(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7; }

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
  const int most = (int)(sizeof(int32_t) * (3 * (size_t)SLOT_MAX_SEQS + 1));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int shift = shift_of(page_size);
  const bool fill = n_tokens <= SLOT_FILL_MAX;
  // one block of 256 threads is quicker round its barriers than one of 1024 (64 rows of a decode
  // step 3.8 against 4.6 us); with more rows or tokens than it takes at once the larger one is
  // (512 rows 7.4 against 21.8)
  const bool wide = n_seqs > 256 || n_tokens > 512;
  static std::atomic<uint64_t> ready[3];
  const auto kernel = !fill ? reserve_slots_kernel<SLOT_THREADS, false>
                      : wide ? reserve_slots_kernel<SLOT_THREADS, true>
                             : reserve_slots_kernel<256, true>;
  if (int rc = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), most, ready[!fill ? 0 : wide ? 1 : 2])) return rc;
  kernel<<<1, fill && !wide ? 256 : SLOT_THREADS, smem, st>>>(block_tables, n_seqs, max_pages, seq_lens, new_lens, free_pages,
                                        (int)free_capacity, n_free, shift, n_tokens, slots, positions, cu_new, granted,
                                        seq_lens_out, n_free_out);
  if (int rc = check_cuda(cudaGetLastError(), "reserve_slots launch")) return rc;
  if (fill) return DSALT_OK;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((n_tokens + 1023) / 1024));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, fill_slots_kernel, (const int32_t*)block_tables, n_seqs, max_pages,
                                       (const int32_t*)seq_lens_out, (const int32_t*)cu_new, (const uint8_t*)granted, shift,
                                       n_tokens, slots, positions),
                    "reserve_slots fill launch");
}

int dsalt_release_slots(int32_t* block_tables, int n_seqs, int max_pages, int32_t* seq_lens, const uint8_t* release,
                        int32_t* free_pages, int64_t free_capacity, int32_t* n_free, int page_size, void* stream) {
  if (n_seqs < 1 || max_pages < 1 || free_capacity < 0) return fail(DSALT_ERR_INVALID, "release_slots: bad sizes");
  if (!page_ok(page_size)) return fail(DSALT_ERR_UNSUPPORTED, "release_slots: page size %d not in {16, 32, 64, 128}", page_size);
  if (n_seqs > SLOT_MAX_SEQS) return fail(DSALT_ERR_UNSUPPORTED, "release_slots: %d rows, at most %d", n_seqs, SLOT_MAX_SEQS);
  if (free_capacity > 0x7fffff00LL) return fail(DSALT_ERR_UNSUPPORTED, "release_slots: pool too large");
  if (!block_tables || !seq_lens || !release || (free_capacity > 0 && !free_pages) || !n_free)
    return fail(DSALT_ERR_INVALID, "release_slots: null pointer");
  const size_t smem = sizeof(int32_t) * (size_t)n_seqs;  // at most 32 KB
  release_slots_kernel<<<1, SLOT_THREADS, smem, reinterpret_cast<cudaStream_t>(stream)>>>(
      block_tables, n_seqs, max_pages, seq_lens, release, free_pages, (int)free_capacity, n_free, shift_of(page_size));
  return check_cuda(cudaGetLastError(), "release_slots launch");
}

}  // extern "C"
