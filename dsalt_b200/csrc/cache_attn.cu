// Attention of one or a few query tokens per sequence over a paged cache held in 8 bits
// (dsalt_cache_attention).
//
// Query at position i of width w, head h: keys A = [max(0, i - w + 1), i] U {landmarks p of
// (h, sequence): 0 <= p < i - w + 1}, x_j = q.k_j / sqrt(D) (+ bias_p), out = sum softmax(x)_j
// v_j; without widths A = [0, i]. k_j = byte * 2^e of its page and kv head, v_j likewise.
//
// Bytes decide: 2 D per key and kv head are read once and give 4 D * (query rows of the kv
// head) operations, far below what the tensor cores do in that time; what has to be kept
// small are the instructions per byte. Eight query rows that share a kv head (the heads of a
// group, the tokens of a draft) are the narrow side of mma.sync m16n8k16, the keys and the
// channels the wide one: S^T = K Q^T (16 keys x 8 rows), O^T = V^T P^T (16 channels x 8 rows),
// with operands built in registers:
// * an e4m3 value is exact in fp16, so K and V are widened exactly; Q is scaled by a power of
//   two per row to a largest magnitude in [2^13, 2^14), which keeps bf16 and fp16 values
//   exact (those below 2^-27 of the row's largest fall short, under fp32's own rounding);
// * the contraction order of a product is free, so lane (g, t) takes 16 consecutive bytes of
//   a key for K Q^T and the D/8 bytes at D/8 g of four keys for V^T P^T, as they lie in the
//   cache; P alone is transposed, two movmatrix per 16 keys;
// * P is rounded to fp16 relative to the row's largest p * 2^e (half a step is 2^-11 of a
//   term, errors of either sign); fp32 queries take Q and P as two fp16 terms each (22 bits).
// * the tensor cores cut off what does not fit a sum's 24 bits, which over a long cache adds up
//   (3.4e-4 of the result after 4096 products in a row); so O is added up by them over
//   CA_CHAIN tiles at most and then, with rounding, to a sum in shared memory (local memory
//   where head_dim 128 leaves no room; 2e-6 remains), for fp32 queries over 16 keys only.
// The scales 2^e of V differ from page to page, so a row keeps two maxima: m of x for the
// denominator l = sum 2^(x - m), and M of x + e for the numerator O = sum 2^(x + e - M) byte;
// out = O 2^(M - m) / l. Neither can overflow whatever the scales are. The cache's own scales are
// powers of two; of others, written by another program, e is a logarithm good to 2^-22.
//
// The keys of an item (sequence, kv head, tile of 8 rows) are a list of tiles of 32: the
// window's, then the landmarks' of each head. Items are cut into units of about equal
// length, by the lengths found on the device (no host copy of them is needed and a captured
// call follows them); the parts of an item that was cut are joined by a second kernel.
// Within a unit each of two warps has its own stretch of tiles and its own ring of
// cp.async stages: nothing but the end is shared, so no warp waits for another.
//
// Measured on a B200 (device time): one row of 131072 keys over 16 heads of 64 in bf16, 268 MB,
// 53 us (5.1 TB/s; copying as much takes 41.6); 16 rows of up to 32768 keys, 8 heads to a kv head
// of 128, 174 MB, 40.6 us (4.3 TB/s); 64 rows with windows up to 512 and 128 landmarks 25 us.
// About 10 us of a call are the schedule and the queries (4), the warps' joining and the second
// kernel. Inside the loop no pipe is full (issue 39 %, ALU 40 %, tensor 15 %, DRAM 51 % of the
// 16 rows' time, shared by all of it): a tile of 32 keys is a chain of copy, widening, product,
// exponential and product that takes a warp about 1.5 us, and registers end the number of
// warps that could overlap it.
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace dsalt {

// Warps of a unit. Four (and half as many units) take 28.2 us against 25.1 for 64 rows with
// landmarks and 42.4 against 40.6 for 16 rows of 32768 keys, and win 1.7 us for a row alone.
constexpr int CA_WARPS = 2;
constexpr int CA_THREADS = 32 * CA_WARPS;
// tiles of 32 keys that a unit takes at least: four per warp (drafts of 23 rows: 24.3 us; 12 tiles
// 25.8, 16 tiles 27.7, before the join was made cheaper)
constexpr int CA_MIN_TILES = 8;
constexpr int CA_MAX_SEQS = 8192;
// Sequences, and query tokens beyond one of each, up to which every block makes the schedule for
// itself: 129 rows 30.8 us (by a kernel of its own 37.2), 200 rows 47.4 (48.3), 400 rows 103.9
// (84.5); 32 rows of 40 tokens 78.3 (48.4), 8 of 128 take 41 either way.
constexpr int CA_OWN_SCHED = 192;
constexpr int CA_OWN_ROWS = 1024;
constexpr int CA_ERR_PAGE = 41;        // device status: a page number outside the pool was met
constexpr float CA_P_SHIFT = 14.f;     // P is held times 2^14: fp16 stays normal down to 2^-28
constexpr int CA_CHAIN = 64;           // tiles that O is added up over by the tensor cores alone
constexpr float CA_SLACK = 1.f;        // P may exceed 2^14 by 2^1 before its reference moves (fp16 ends at 2^16)

// Blocks per SM that registers and rings allow; one round of them is the number of units wanted.
// Two stages: a third costs blocks, and at head_dim 64 with 7 of them one row of 131072 keys
// takes 57.1 us against 54.2, with 6 of them 52.2 but 64 rows 33.9 against 25.2; at head_dim 128
// with 4 of them 41.9 us against 40.8. Nine blocks of head_dim 64 leave 112 registers: 69 us.
template <int D>
struct Shape {
  static constexpr int OCC = D == 64 ? 8 : 6;
  static constexpr int STAGES = 2;
  static constexpr int SLOTS = 148 * OCC;
};
constexpr int CA_ROWS = 8;
constexpr int CA_MAX_SLOTS = 148 * 8;

struct CacheAttnArgs {
  const void* q;
  int64_t q_stride;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int32_t* tables;
  int max_pages, n_pages;
  const int32_t *seq_lens, *cu_q, *w, *lmk;
  const float* bias;
  int k_lmk, n_seqs, T, H, Hkv, G, page_shift;
  float scale_log2;
  void* out;
  int out_dtype;
  float* lse;
  float* part_o;   // [cut units][8][D]
  float* part_s;   // [cut units][8][4]: m, l, M
  int2* row_part;  // [T * H] first part of the row and how many there are
  int2* sched;     // many sequences or tokens: {chunk, units}, then {units, parts} before each sequence; else null
  struct SeqPlan* plans;  // with sched: [n_seqs]
  int* err;
};

struct RowState {
  float m, l, M;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// cp.async of 16 bytes, zeros when !ok
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(__cvta_generic_to_global(src)) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src, bool ok) { cp_async_16(dst, src, ok ? 16 : 0); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// two e4m3 bytes -> two fp16
__device__ __forceinline__ uint32_t widen_lo(uint32_t v) {
  uint32_t r;
  asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, l;}" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t widen_hi(uint32_t v) {
  uint32_t r;
  asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, h;}" : "=r"(r) : "r"(v));
  return r;
}
// log2 of a scale; of 0 (a page never written) -127: its exponent (put into the significand of 2^23, and
// 2^23 + 127 taken off), and the logarithm of its significand, exactly 0 for a power of two
__device__ __forceinline__ float scale_log(float s) {
  const uint32_t u = __float_as_uint(s);
  float f;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(f) : "f"(__uint_as_float((u & 0x7fffffu) | 0x3f800000u)));
  return __uint_as_float(0x4b000000u + (u >> 23)) - 8388735.f + f;
}

// query of sequence s: tokens, keys and the tiles of 32 that they make
struct SeqPlan {
  int q0, n_q, len, n_window, n_lmk;  // tiles of one row tile, at most
};
__device__ __forceinline__ int first_key(const CacheAttnArgs& a, int t, int pos) {
  if (!a.w) return 0;
  const int w = max(a.w[t], 1);
  return max(pos - w + 1, 0);  // no overflow: pos < 2^31, w >= 1
}
// The rows of a kv head go head by head, each head's tokens after one another: a tile meets the
// landmarks of few heads, where token by token it would meet those of all. From 8 tokens on a
// head has tiles of its own, each with the windows of 8 neighbours.
__device__ __forceinline__ int head_rows(int n_q) { return n_q < CA_ROWS ? n_q : (n_q + CA_ROWS - 1) & ~(CA_ROWS - 1); }
__device__ __forceinline__ int tile_heads(const CacheAttnArgs& a, int n_q) {  // of one tile, at most
  if (n_q <= 1) return n_q <= 0 ? 0 : min(a.G, CA_ROWS);
  return n_q >= CA_ROWS ? 1 : min(a.G, n_q == 2 || n_q == 4 ? CA_ROWS / n_q : (CA_ROWS - 2) / n_q + 2);
}
// (lane, lanes: who looks at which of the tokens; the lanes' findings are joined)
__device__ __forceinline__ SeqPlan plan_of(const CacheAttnArgs& a, int s, int lane = 0, int lanes = 1) {
  SeqPlan p;
  p.q0 = a.cu_q ? min(max(a.cu_q[s], 0), a.T) : s;
  p.n_q = a.cu_q ? max(min(a.cu_q[s + 1], a.T) - p.q0, 0) : 1;
  p.len = min(max(a.seq_lens[s], 0), a.max_pages << a.page_shift);
  int lo = p.len, top = 0, span = 0;
  if (!a.w) lo = 0;
  else for (int r = lane; r < p.n_q; r += lanes) {
    const int w = max(__ldg(a.w + p.q0 + r), 1);  // on its way beside the lengths
    const int pos = p.len - p.n_q + r;
    if (pos < 0) continue;
    const int f = max(pos - w + 1, 0);
    lo = min(lo, f);
    top = max(top, f);
    span = max(span, pos + 1 - f);
  }
  if (lanes > 1) {
    lo = __reduce_min_sync(0xffffffffu, lo);
    top = __reduce_max_sync(0xffffffffu, top);
    span = __reduce_max_sync(0xffffffffu, span);
  }
  // tiles of 32 keys from the first key on, to the sequence's last; 8 neighbours have at most
  // span + 7 keys
  p.n_window = p.n_q > 0 && p.len > 0 ? (p.len - (lo & ~31) + 31) >> 5 : 0;
  if (a.w && p.n_q >= CA_ROWS) p.n_window = min(p.n_window, (span + (CA_ROWS - 1) + 30) / 32 + 1);
  p.n_lmk = a.k_lmk > 0 && top > 0 ? tile_heads(a, p.n_q) * ((a.k_lmk + 31) >> 5) : 0;  // none lies before a window from 0
  return p;
}
__device__ __forceinline__ int row_tiles(const CacheAttnArgs& a, int n_q) { return (head_rows(n_q) * a.G + CA_ROWS - 1) / CA_ROWS; }

// sums of two numbers over the block's threads, exclusive; totals in `all`
template <int WARPS>
__device__ __forceinline__ int2 block_before2(int2 v, int2* red, int2& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int2 s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, s.x, o), y = __shfl_up_sync(0xffffffffu, s.y, o);
    if (lane >= o) s.x += x, s.y += y;
  }
  __syncthreads();
  if (lane == 31) red[warp] = s;
  __syncthreads();
  int2 before = make_int2(0, 0);
  all = make_int2(0, 0);
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    if (i < warp) before.x += red[i].x, before.y += red[i].y;
    all.x += red[i].x, all.y += red[i].y;
  }
  return make_int2(before.x + s.x - v.x, before.y + s.y - v.y);
}

// Tiles that a unit takes. Cutting adds at most one unit per item: where the items leave room,
// all units run at once; where they do not, only items above an average slot's load are cut.
__device__ __forceinline__ int chunk_of(long long tiles, long long items, int slots) {
  const long long want = items < slots ? max(slots - items, (long long)slots / 4) : slots;
  return (int)min(max((tiles + want - 1) / want, (long long)CA_MIN_TILES), 0x7fffffffLL);
}

__device__ __forceinline__ int parts_of(int tiles, int chunk) { return max(1, (tiles + chunk - 1) / chunk); }

// The schedule of many sequences or tokens, made once: for few, each block's own takes less time
// than a launch; its time grows with their number, in every block.
constexpr int CP_THREADS = 1024;
__global__ void __launch_bounds__(CP_THREADS) cache_attn_plan_kernel(CacheAttnArgs a, int slots) {
  __shared__ long long s_sum[CP_THREADS / 32][2];
  __shared__ int2 red[CP_THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int MINE = CA_MAX_SEQS / CP_THREADS;  // sequences of one thread
  int len[MINE], count[MINE];
  long long tiles = 0, items = 0;
  for (int s = warp; s < a.n_seqs; s += CP_THREADS / 32) {
    const SeqPlan p = plan_of(a, s, lane, 32);
    if (lane == 0) a.plans[s] = p;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    const int s = i * CP_THREADS + tid;
    len[i] = count[i] = 0;
    if (s < a.n_seqs) {
      const SeqPlan p = a.plans[s];
      len[i] = p.n_window + p.n_lmk;
      count[i] = row_tiles(a, p.n_q) * a.Hkv;
      tiles += (long long)len[i] * count[i];
      items += count[i];
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    items += __shfl_xor_sync(0xffffffffu, items, o);
  }
  if (lane == 0) s_sum[warp][0] = tiles, s_sum[warp][1] = items;
  __syncthreads();
  tiles = items = 0;
  for (int w = 0; w < CP_THREADS / 32; ++w) tiles += s_sum[w][0], items += s_sum[w][1];
  const int chunk = chunk_of(tiles, items, slots);
  int2 carry = make_int2(0, 0);
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    if (i * CP_THREADS >= a.n_seqs) break;
    const int s = i * CP_THREADS + tid;
    const int splits = parts_of(len[i], chunk);
    const int2 v = make_int2(count[i] * splits, splits > 1 ? count[i] * splits : 0);
    int2 all;
    const int2 b = block_before2<CP_THREADS / 32>(v, red, all);
    if (s < a.n_seqs) a.sched[1 + s] = make_int2(carry.x + b.x, carry.y + b.y);
    carry.x += all.x;
    carry.y += all.y;
  }
  if (tid == 0) a.sched[0] = make_int2(chunk, carry.x);
}

// One stage of a warp's ring: 32 keys. K and V rows of D bytes, their 16-byte chunks placed so
// that a warp's fragment loads meet no bank twice, and {scale of K, scale of V, bias, position
// or -1}: of landmarks per key, of a window tile per half at keys 0 and 16.
template <int D>
struct Stage {
  static constexpr int V = 32 * D, META = 64 * D, BYTES = 64 * D + 512;
  static __device__ __forceinline__ int k_at(int r, int c) {
    return D == 64 ? ((r ^ (r >> 2 & 1)) * 64 + c * 16) : (r * 128 + ((c ^ (r & 4)) * 16));
  }
  static __device__ __forceinline__ int v_at(int r, int c) {
    return V + (D == 64 ? r * 64 + ((c ^ (r & 2)) * 16) : r * 128 + ((c ^ (r & 3) << 1) * 16));
  }
};
// Which key of eight is row n of S^T: so chosen that the keys 2t, 2t+1 (and 8 on) of P^T that
// lane t contracts are t, t+4 (and 8 on), whose V rows lie together.
__device__ __forceinline__ int slot_of(int n) { return (n >> 1) + 4 * (n & 1); }
// transposes an 8 x 8 matrix of 16-bit values: lane (g, t) gives [g][2t, 2t+1] and gets [2t, 2t+1][g]
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ uint32_t nan_bytes(uint32_t v) {  // 0xff where a byte is an e4m3 NaN
  return __vcmpeq4(v & 0x7f7f7f7fu, 0x7f7f7f7fu);
}

// NS: fp16 terms that Q and P are held in (2 for fp32 queries)
template <typename T, int D, int NS>
__global__ void __launch_bounds__(CA_THREADS, Shape<D>::OCC) cache_attn_kernel(CacheAttnArgs a) {
  constexpr int KS = D / 16, MT = D / 16, STAGES = Shape<D>::STAGES;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ int2 red[CA_WARPS];
  __shared__ long long s_sum[CA_WARPS][2];
  __shared__ float s_m[CA_WARPS][CA_ROWS], s_l[CA_WARPS][CA_ROWS], s_M[CA_WARPS][CA_ROWS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  __shared__ struct {
    SeqPlan plan;
    int s, local, splits, cut;  // sequence, unit within it, parts of its items, parts of cut items before it
  } s_job;
  SeqPlan* s_plans = reinterpret_cast<SeqPlan*>(dyn);  // [n_seqs], before the rings
  float* s_o = reinterpret_cast<float*>(dyn);  // [warps][8][D], after the rings

  const int unit = blockIdx.x;
  int n_units;
  if (a.sched) {
    // ---- the schedule is there: the last sequence whose units begin at or before this one
    const int2 head = a.sched[0];
    n_units = head.y;
    if (warp == 0 && unit < n_units) {
      int lo = 0, hi = a.n_seqs;  // sched[1 + lo].x <= unit, sched[1 + hi].x > unit (or hi is the end)
      while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const uint32_t in = __ballot_sync(0xffffffffu, at < hi && a.sched[1 + at].x <= unit);  // lane 0 always
        const int f = 31 - __clz(in);
        hi = min(hi, lo + (f + 1) * step);
        lo += f * step;
      }
      if (lane == 0) {
        const int2 from = a.sched[1 + lo];
        s_job.plan = a.plans[lo];
        s_job.s = lo;
        s_job.local = unit - from.x;
        s_job.splits = parts_of(s_job.plan.n_window + s_job.plan.n_lmk, head.x);
        s_job.cut = from.y;
      }
    }
  } else {
    // ---- schedule: every block derives the same one from the lengths
    // tiles and items of the call; both stay below 2^40
    long long mine = 0, count = 0;
    const auto add = [&](int s, const SeqPlan& p) {
      const int items = row_tiles(a, p.n_q) * a.Hkv;
      s_plans[s] = p;
      mine += (long long)(p.n_window + p.n_lmk) * items;
      count += items;
    };
    if (a.w && a.T >= 32 * a.n_seqs) {  // many tokens each: a warp looks at their widths
      for (int s = warp; s < a.n_seqs; s += CA_WARPS) {
        const SeqPlan p = plan_of(a, s, lane, 32);
        if (lane == 0) add(s, p);
      }
    } else {
      for (int s = tid; s < a.n_seqs; s += CA_THREADS) add(s, plan_of(a, s));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      mine += __shfl_xor_sync(0xffffffffu, mine, o);
      count += __shfl_xor_sync(0xffffffffu, count, o);
    }
    if (lane == 0) s_sum[warp][0] = mine, s_sum[warp][1] = count;
    __syncthreads();
    long long total = 0, items = 0;
#pragma unroll
    for (int w = 0; w < CA_WARPS; ++w) total += s_sum[w][0], items += s_sum[w][1];
    const int chunk = chunk_of(total, items, Shape<D>::SLOTS);
    int2 carry = make_int2(0, 0);
    for (int base = 0; base < a.n_seqs; base += CA_THREADS) {
      const int s = base + tid;
      int2 v = make_int2(0, 0), all;
      int splits = 1;
      if (s < a.n_seqs) {
        const SeqPlan& p = s_plans[s];
        splits = parts_of(p.n_window + p.n_lmk, chunk);
        v.x = row_tiles(a, p.n_q) * a.Hkv * splits;
        v.y = splits > 1 ? v.x : 0;
      }
      const int2 b = block_before2<CA_WARPS>(v, red, all);
      const int from = carry.x + b.x;
      if (unit >= from && unit < from + v.x) {  // one thread, if any
        s_job.plan = s_plans[s];
        s_job.s = s;
        s_job.local = unit - from;
        s_job.splits = splits;
        s_job.cut = carry.y + b.y;
      }
      carry.x += all.x;
      carry.y += all.y;
    }
    n_units = carry.x;
  }
  __syncthreads();
  cudaTriggerProgrammaticLaunchCompletion();  // the join may take its places; it waits for this grid's end
  // rows behind the last sequence's: zero, log-sum-exp -inf
  if (a.cu_q) {
    const int64_t rows0 = (int64_t)min(max(a.cu_q[a.n_seqs], 0), a.T) * a.H, rows1 = (int64_t)a.T * a.H;
    for (int64_t r = rows0 + unit; r < rows1; r += gridDim.x) {
      for (int d = tid; d < D; d += CA_THREADS) {
        if (a.out_dtype == DSALT_F32) reinterpret_cast<float*>(a.out)[r * D + d] = 0.f;
        else reinterpret_cast<uint16_t*>(a.out)[r * D + d] = 0;
      }
      if (tid == 0) {
        if (a.lse) a.lse[r] = -INFINITY;
        a.row_part[r] = make_int2(0, 1);
      }
    }
  }
  if (unit >= n_units) return;
  const SeqPlan p = s_job.plan;
  const int s = s_job.s, splits = s_job.splits, tiles = p.n_window + p.n_lmk;
  const int split = s_job.local % splits, item = s_job.local / splits;
  const int hk = item % a.Hkv, tile = item / a.Hkv;
  const int part0 = s_job.cut + item * splits;
  const int each = (tiles + splits - 1) / splits;
  const int t_begin = min(split * each, tiles), t_end = min(t_begin + each, tiles);

  // row r of the tile: head head0 + head_of(tok0 + r), token what is left
  const int per_head = head_rows(p.n_q), n_rows = min(per_head * a.G - tile * CA_ROWS, CA_ROWS);
  const int head0 = tile * CA_ROWS / per_head, tok0 = tile * CA_ROWS - head0 * per_head;
  const int inverse = per_head < CA_ROWS ? (255 + per_head) / per_head : 0;  // exact for quotients of 14 and less
  const auto head_of = [&](int x) { return per_head < CA_ROWS ? x * inverse >> 8 : 0; };
  const int n_heads = head_of(tok0 + n_rows - 1) + 1;
  // ---- rows 2t, 2t+1 of the tile are this lane's in S^T and O^T
  int row_lo[2], row_hi[2], row_head[2];
  unsigned row_span[2], row_before[2];  // keys of the window; positions before it, where landmarks count
  bool row_ok[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int x = tok0 + 2 * t + c, head = head_of(x), tok = x - head * per_head;
    row_ok[c] = 2 * t + c < n_rows && tok < p.n_q;
    const int pos = p.len - p.n_q + tok;
    const bool keys = row_ok[c] && pos >= 0;
    row_lo[c] = keys ? first_key(a, p.q0 + tok, pos) : 0x7fffffff;
    row_hi[c] = keys ? pos + 1 : 0;
    row_head[c] = head;
    row_span[c] = keys ? row_hi[c] - row_lo[c] : 0;
    row_before[c] = keys ? row_lo[c] : 0;
  }
  // keys that every row of the tile attends to need no mask
  int lo_min = min(row_lo[0], row_lo[1]), hi_max = max(row_hi[0], row_hi[1]);
  int lo_max = max(row_ok[0] ? row_lo[0] : 0, row_ok[1] ? row_lo[1] : 0);
  int hi_min = min(row_ok[0] ? row_hi[0] : 0x7fffffff, row_ok[1] ? row_hi[1] : 0x7fffffff);
#pragma unroll
  for (int x = 1; x < 4; x <<= 1) {
    lo_max = max(lo_max, __shfl_xor_sync(0xffffffffu, lo_max, x));
    hi_min = min(hi_min, __shfl_xor_sync(0xffffffffu, hi_min, x));
    lo_min = min(lo_min, __shfl_xor_sync(0xffffffffu, lo_min, x));
    hi_max = max(hi_max, __shfl_xor_sync(0xffffffffu, hi_max, x));
  }
  const int page_mask = (1 << a.page_shift) - 1;
  const int* table = a.tables + (int64_t)s * a.max_pages;
  const int lmk32 = max((a.k_lmk + 31) >> 5, 1);
  bool bad_page = false;

  // ---- this warp's share of the unit: a stretch of window tiles, then one of landmark tiles
  const int w0 = min(t_begin, p.n_window), w1 = min(t_end, p.n_window);
  const int l1 = min(max(t_end - p.n_window, 0), n_heads * lmk32), l0 = min(max(t_begin - p.n_window, 0), l1);
  const int wq = (w1 - w0 + CA_WARPS - 1) / CA_WARPS, lq = (l1 - l0 + CA_WARPS - 1) / CA_WARPS;
  const int wb = min(w0 + warp * wq, w1);
  int we = min(wb + wq, w1);
  const int lb = min(l0 + warp * lq, l1), le = min(lb + lq, l1);
  const int lo32 = lo_min < p.len ? lo_min & ~31 : 0;  // window tiles begin here
  we = min(we, max(wb, (hi_max - lo32 + 31) >> 5));
  const int n_w = we - wb, n = n_w + le - lb;

  // where keys lie: of 16 window tiles ahead a lane per half, of the next landmark tile a lane per key
  struct Where {
    int key, page;  // -1 where none
    float add;
  };
  const auto page_of = [&](int key) { return key >= 0 && key < p.len ? __ldg(table + (key >> a.page_shift)) : -1; };
  // cache row of a key, or -1 (also for a page that does not exist)
  const auto row_of = [&](const Where& o) -> int {
    if (o.key < 0 || o.key >= p.len) return -1;
    if ((unsigned)o.page >= (unsigned)a.n_pages) {
      bad_page = true;
      return -1;
    }
    return ((o.page * a.Hkv + hk) << a.page_shift) + (o.key & page_mask);
  };
  auto find_window = [&](int i) {  // lane: half lane & 1 of tile wb + i + lane / 2
    Where o;
    o.add = 0.f;
    o.key = i + (lane >> 1) < n_w ? lo32 + (wb + i) * 32 + lane * 16 : -1;
    o.page = page_of(o.key);
    return o;
  };
  auto find_lmk = [&](int i) {  // lane: key `lane` of tile lb + i
    Where o;
    o.add = 0.f;
    o.key = -1;
    const int l = lb + i, c = (l % lmk32) * 32 + lane;
    if (l < le && c < a.k_lmk) {
      const int64_t at = ((int64_t)(hk * a.G + head0 + l / lmk32) * a.n_seqs + s) * a.k_lmk + c;
      o.key = a.lmk[at];
      if (a.bias) o.add = a.bias[at] * 1.4426950408889634f;
    }
    o.page = page_of(o.key);
    return o;
  };
  Where ww = find_window(0), wn = ww, ln = ww;
  if (n_w > 16) wn = find_window(16);
  if (le > lb) ln = find_lmk(0);
  // ---- Q of row g: the 16 consecutive elements at 16 t of each 64, on their way while the first
  // tiles are asked for
  constexpr int QV = (int)sizeof(T);  // vectors of 16 bytes per 64 channels
  uint4 q_raw[D / 64][QV];
  {
    const int head = head_of(tok0 + g), tok = tok0 + g - head * per_head;
    const bool live = g < n_rows && tok < p.n_q;
    const T* src = reinterpret_cast<const T*>(a.q) + (int64_t)(p.q0 + (live ? tok : 0)) * a.q_stride +
                   (int64_t)(hk * a.G + head0 + (live ? head : 0)) * D + t * 16;
#pragma unroll
    for (int b = 0; b < D / 64; ++b)
#pragma unroll
      for (int j = 0; j < QV; ++j) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(src + b * 64) + j);
        q_raw[b][j] = live ? v : make_uint4(0, 0, 0, 0);
      }
  }
  uint8_t* ring = dyn + warp * (STAGES * Stage<D>::BYTES);
  const uint32_t ring_s = smem_u32(ring);
  int ww_row = -1;                  // row of ww's key
  int in_stage = 0, out_stage = 0;  // byte offsets of the stages written and read next
  constexpr int CPR = D / 16, RPI = 32 / CPR;  // 16-byte chunks per row, rows per step of the warp
  const int my_row = lane / CPR, my_chunk = lane % CPR;
  // places of this lane's chunks and fragments in a stage; whole steps and halves are added (the
  // swizzle looks at the lowest bits of the row alone, save one bit that K's odd steps flip)
  const int k_put = Stage<D>::k_at(my_row, my_chunk), v_put = Stage<D>::v_at(my_row, my_chunk);
  const auto k_step = [&](int x) { return D == 64 ? k_put + x * RPI * D : (k_put ^ (x & 1) * 64) + x * RPI * D; };
  const int k_get = Stage<D>::k_at(slot_of(g), t), v_get = D == 64 ? Stage<D>::v_at(t, g >> 1) + (g & 1) * 8 : Stage<D>::v_at(t, g);
  // scales come with the keys, by cp.async: nothing waits for them here
  const auto put_meta = [&](uint32_t st_s, float4* meta, int slot, int row, const Where& o) {
    const int head = max(row, 0) >> a.page_shift;
    const uint32_t at = st_s + Stage<D>::META + slot * 16;
    cp_async_4(at, a.ks + head, row >= 0 ? 4 : 0);
    cp_async_4(at + 4, a.vs + head, row >= 0 ? 4 : 0);
    *reinterpret_cast<float2*>(&meta[slot].z) = make_float2(o.add, __int_as_float(row >= 0 ? o.key : -1));
  };
  auto issue = [&](int i) {
    if (i < n) {
      const uint32_t st_s = ring_s + in_stage;
      float4* meta = reinterpret_cast<float4*>(ring + in_stage + Stage<D>::META);
      if (i < n_w) {
        const int b = i & 15;
        if (b == 0 && i > 0) {
          ww = wn;
          if (i + 16 < n_w) wn = find_window(i + 16);
        }
        if (b == 0) ww_row = row_of(ww);
        if ((lane >> 1) == b) put_meta(st_s, meta, (lane & 1) * 16, ww_row, ww);
        const int key = __shfl_sync(0xffffffffu, ww.key, 2 * b);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = __shfl_sync(0xffffffffu, ww_row, 2 * b + h);
          const int left = row < 0 ? 0 : p.len - key - h * 16;  // rows from here that hold keys
          const int64_t at = (int64_t)max(row, 0) * D + lane * 16;
          const uint8_t *ksrc = a.kc + at, *vsrc = a.vc + at;
          if (left >= 16) {
#pragma unroll
            for (int x = 0; x < 16 / RPI; ++x) {
              copy16(st_s + k_step(x) + h * 16 * D, ksrc + x * 512);
              copy16(st_s + v_put + (h * 16 + x * RPI) * D, vsrc + x * 512);
            }
          } else {
#pragma unroll
            for (int x = 0; x < 16 / RPI; ++x) {
              copy16(st_s + k_step(x) + h * 16 * D, ksrc + x * 512, x * RPI + my_row < left);
              copy16(st_s + v_put + (h * 16 + x * RPI) * D, vsrc + x * 512, x * RPI + my_row < left);
            }
          }
        }
      } else {
        const Where lw = ln;
        if (i + 1 < n) ln = find_lmk(i + 1 - n_w);
        const int mine = row_of(lw);
        put_meta(st_s, meta, lane, mine, lw);
#pragma unroll
        for (int x = 0; x < 32 / RPI; ++x) {
          const int r = x * RPI + my_row, row = __shfl_sync(0xffffffffu, mine, r);
          const int64_t at = (int64_t)max(row, 0) * D + my_chunk * 16;
          copy16(st_s + k_step(x), a.kc + at, row >= 0);
          copy16(st_s + v_put + x * RPI * D, a.vc + at, row >= 0);
        }
      }
      in_stage = in_stage == (STAGES - 1) * Stage<D>::BYTES ? 0 : in_stage + Stage<D>::BYTES;
    }
    copies_commit();
  };
  // (the schedule's memory becomes the rings: it was last read before the barrier behind it)
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue(i);
  uint32_t qb[NS][KS][2];
  float row_f[2];
  {
    float x[D / 4];
#pragma unroll
    for (int b = 0; b < D / 64; ++b)
#pragma unroll
      for (int j = 0; j < QV; ++j) {
        const uint4 u = q_raw[b][j];
        const uint32_t wd[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (sizeof(T) == 4) {
            x[b * 16 + j * 4 + e] = __uint_as_float(wd[e]);
          } else {
            float2 f;
            if constexpr (std::is_same<T, __half>::value) f = __half22float2(*reinterpret_cast<const __half2*>(&wd[e]));
            else f = make_float2(__uint_as_float(wd[e] << 16), __uint_as_float(wd[e] & 0xffff0000u));
            x[b * 16 + j * 8 + 2 * e] = f.x;
            x[b * 16 + j * 8 + 2 * e + 1] = f.y;
          }
        }
      }
    float big = 0.f;
#pragma unroll
    for (int j = 0; j < D / 4; ++j) big = fmaxf(big, fabsf(x[j]));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    const int eb = (int)(__float_as_uint(big) >> 23);  // biased exponent; 255: an infinity
    const int up = eb == 255 ? 0 : min(max(13 - (eb - 127), -126), 126);
    const float mul = __uint_as_float((uint32_t)(up + 127) << 23);
    const float f = a.scale_log2 * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
    for (int c = 0; c < 2; ++c) row_f[c] = __shfl_sync(0xffffffffu, f, (2 * t + c) * 4);
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float lo = x[4 * k + 2 * h] * mul, hi = x[4 * k + 2 * h + 1] * mul;
        qb[0][k][h] = pack_f16x2(lo, hi);
        if constexpr (NS == 2) {
          const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&qb[0][k][h]));
          qb[1][k][h] = pack_f16x2(lo - b.x, hi - b.y);
        }
      }
  }

  float o[MT][4];  // channels D/8 g + 2 i (0, 1) and one on (2, 3) of rows 2t, 2t+1
#pragma unroll
  for (int i = 0; i < MT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  RowState st[2] = {{-INFINITY, 0.f, -INFINITY}, {-INFINITY, 0.f, -INFINITY}};

  // m and M are references, not exact maxima: they move when a lane's logit passes them by the
  // slack, which after the first tiles is rare, and only then are maxima formed over the lanes
  const auto raise = [&](const float (&lm)[2], const float (&lM)[2]) {
    if (!__any_sync(0xffffffffu, lm[0] > st[0].m + CA_SLACK || lM[0] > st[0].M + CA_SLACK || lm[1] > st[1].m + CA_SLACK ||
                                     lM[1] > st[1].M + CA_SLACK))
      return;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float gm = lm[c], gM = lM[c];
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, x));
        gM = fmaxf(gM, __shfl_xor_sync(0xffffffffu, gM, x));
      }
      const float m = fmaxf(st[c].m, gm), M = fmaxf(st[c].M, gM);
      st[c].l *= m == -INFINITY ? 1.f : ex2_approx(st[c].m - m);
      const float corr = M == -INFINITY ? 1.f : ex2_approx(st[c].M - M);
      st[c].m = m;
      st[c].M = M;
#pragma unroll
      for (int x = 0; x < MT; ++x) {
        o[x][c] *= corr;
        o[x][2 + c] *= corr;
      }
    }
  };

  // o to the sum over the tiles before; that sum, in o, with `all`
  [[maybe_unused]] volatile float far_o[D == 64 ? 1 : MT][4];
  [[maybe_unused]] float* const far_s =
      reinterpret_cast<float*>(dyn + CA_WARPS * STAGES * Stage<D>::BYTES) + warp * (MT * 4 * 32) + lane;
  [[maybe_unused]] const auto far_get = [&](int x, int e) -> float {
    if constexpr (D == 64) return far_s[(x * 4 + e) * 32];
    else return far_o[x][e];
  };
  [[maybe_unused]] const auto far_put = [&](int x, int e, float v) {
    if constexpr (D == 64) far_s[(x * 4 + e) * 32] = v;
    else far_o[x][e] = v;
  };
  [[maybe_unused]] float far_M[2];
  [[maybe_unused]] const auto put_by = [&](bool first, bool all) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float corr = first || st[c].M == -INFINITY ? 1.f : ex2_approx(far_M[c] - st[c].M);
#pragma unroll
      for (int x = 0; x < MT; ++x)
#pragma unroll
        for (int e = c; e < 4; e += 2) {
          if (!first) o[x][e] = fmaf(far_get(x, e), corr, o[x][e]);
          if (!all) {
            far_put(x, e, o[x][e]);
            o[x][e] = 0.f;
          }
        }
      far_M[c] = st[c].M;
    }
  };

  for (int i = 0; i < n; ++i) {
    if constexpr (NS == 1)
      if (i % CA_CHAIN == 0 && i > 0) put_by(i == CA_CHAIN, false);
    copies_wait<STAGES - 2>();
    __syncwarp();  // every lane's copies of stage i are there, and stage i - 1 is read
    issue(i + STAGES - 1);
    const uint8_t* stage = ring + out_stage;
    out_stage = out_stage == (STAGES - 1) * Stage<D>::BYTES ? 0 : out_stage + Stage<D>::BYTES;
    const float4* meta = reinterpret_cast<const float4*>(stage + Stage<D>::META);
    const bool window = i < n_w;
    // ---- S^T = K Q^T
    float sc[2][4];  // half h: keys g (0, 1) and 8 on (2, 3) of rows 2t, 2t+1
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sc[h][0] = sc[h][1] = sc[h][2] = sc[h][3] = 0.f;
#pragma unroll
      for (int b = 0; b < D / 64; ++b) {
        const uint4 ka = *reinterpret_cast<const uint4*>(stage + (k_get ^ b * 64) + h * 16 * D);
        const uint4 kb = *reinterpret_cast<const uint4*>(stage + (k_get ^ b * 64) + (h * 16 + 8) * D);
        const uint32_t k0[4] = {ka.x, ka.y, ka.z, ka.w}, k1[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a0 = widen_lo(k0[k]), a1 = widen_lo(k1[k]), a2 = widen_hi(k0[k]), a3 = widen_hi(k1[k]);
#pragma unroll
          for (int x = 0; x < NS; ++x) mma_f16(sc[h], a0, a1, a2, a3, qb[x][b * 4 + k][0], qb[x][b * 4 + k][1]);
        }
      }
    }
    // ---- P = 2^(x + e - M + 14), l += 2^(x - m)
    const int key0 = lo32 + (wb + i) * 32, slot = slot_of(g);
    float4 mh[2] = {meta[0], meta[16]};  // of a window tile's halves; .y: exponent of V's scale
    const bool whole = window && key0 >= lo_max && key0 + 32 <= hi_min && __float_as_int(mh[0].w) >= 0 &&
                       __float_as_int(mh[1].w) >= 0;  // every row attends to every key
    const int head = window ? 0 : (lb + i - n_w) / lmk32;
    // does row c attend to this lane's key b of half h?
    const auto attends = [&](int h, int b, int c) -> bool {
      if (window)
        return (unsigned)(key0 + h * 16 + b * 8 + slot - row_lo[c]) < (__float_as_int(mh[h].w) >= 0 ? row_span[c] : 0u);
      return __float_as_uint(meta[h * 16 + b * 8 + slot].w) < (head == row_head[c] ? row_before[c] : 0u);
    };
    float ve[2][2];
    bool formed = !window;  // sc holds logits
    if (window) {
      mh[0].y = scale_log(mh[0].y);
      mh[1].y = scale_log(mh[1].y);
      if (!whole) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int c = 0; c < 2; ++c)
              if (!attends(h, b, c)) sc[h][2 * b + c] = -INFINITY;
      }
      // one exponential per element: the sum of P is brought to l's reference
      float f[2][2], lm[2][2], top[2], top_e[2], mu[2], Mu[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f[c][h] = fmaxf(mh[h].x * row_f[c], 1.17549435e-38f);  // above 0, so that -inf stays what it is
          lm[c][h] = f[c][h] * fmaxf(sc[h][c], sc[h][2 + c]);
        }
        top[c] = fmaxf(lm[c][0], lm[c][1]);
        top_e[c] = fmaxf(lm[c][0] + mh[0].y, lm[c][1] + mh[1].y);
      }
      raise(top, top_e);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        mu[c] = st[c].m == -INFINITY ? 0.f : st[c].m;
        Mu[c] = st[c].M == -INFINITY ? 0.f : st[c].M;
      }
      // where V's scale is so small that P of a logit near m would vanish, l needs its own exponentials
      const float e_min = fminf(mh[0].y, mh[1].y);
      formed = __any_sync(0xffffffffu, !(fminf(mu[0] - Mu[0], mu[1] - Mu[1]) + e_min > -90.f));
      if (!formed) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float shift = mh[h].y - Mu[c] + CA_P_SHIFT;
            sc[h][c] = ex2_approx(fmaf(sc[h][c], f[c][h], shift));
            sc[h][2 + c] = ex2_approx(fmaf(sc[h][2 + c], f[c][h], shift));
            st[c].l = fmaf(sc[h][c] + sc[h][2 + c], ex2_approx(-shift - mu[c]), st[c].l);
          }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          ve[h][0] = ve[h][1] = mh[h].y;
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[h][e] *= f[e & 1][h];
        }
      }
    } else {
      float lm[2] = {-INFINITY, -INFINITY}, lM[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const float4 mt = meta[h * 16 + b * 8 + slot];
          ve[h][b] = scale_log(mt.y);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float& x = sc[h][2 * b + c];
            x = attends(h, b, c) ? fmaf(x, mt.x * row_f[c], mt.z) : -INFINITY;
            lm[c] = fmaxf(lm[c], x);
            lM[c] = fmaxf(lM[c], x + ve[h][b]);
          }
        }
      raise(lm, lM);
    }
    if (formed) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float mu = st[c].m == -INFINITY ? 0.f : st[c].m, Mu = st[c].M == -INFINITY ? 0.f : st[c].M;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const float x = sc[h][2 * b + c];
            st[c].l += ex2_approx(x - mu);
            sc[h][2 * b + c] = ex2_approx(x + ve[h][b] - Mu + CA_P_SHIFT);
          }
      }
    }
    // ---- O^T += V^T P^T, 16 keys at a time
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t pb[NS][2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const float lo = sc[h][2 * b], hi = sc[h][2 * b + 1];
        const uint32_t first = pack_f16x2(lo, hi);
        pb[0][b] = transpose8(first);
        if constexpr (NS == 2) {
          const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&first));
          pb[1][b] = transpose8(pack_f16x2(lo - x.x, hi - x.y));
        }
      }
      uint32_t v[4][D / 32];  // keys t, t + 4, t + 8, t + 12
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint8_t* at = stage + v_get + (h * 16 + 4 * x) * D;
        if constexpr (D == 64) {
          const uint2 y = *reinterpret_cast<const uint2*>(at);
          v[x][0] = y.x, v[x][1] = y.y;
        } else {
          const uint4 y = *reinterpret_cast<const uint4*>(at);
          v[x][0] = y.x, v[x][1] = y.y, v[x][2] = y.z, v[x][3] = y.w;
        }
      }
      bool nans = false;
      if (!whole) {
        uint32_t hit = 0;  // 0x7f, the only NaN, is what a carry takes to the eighth bit
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
          for (int y = 0; y < D / 32; ++y) hit |= (v[x][y] & 0x7f7f7f7fu) + 0x01010101u;
        nans = __any_sync(0xffffffffu, (hit & 0x80808080u) != 0);
      }
      if (nans) {
        // P = 0 must not spread a NaN: count, per channel and row, the NaNs among the keys that the
        // row attends to (a product of ones), and take the NaNs themselves out
        uint32_t ones[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          ones[b] = transpose8((attends(h, b, 0) ? 0x3c00u : 0u) | (attends(h, b, 1) ? 0x3c000000u : 0u));
        }
#pragma unroll
        for (int x = 0; x < D / 32; ++x) {
          uint32_t nb[4];
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            nb[y] = nan_bytes(v[y][x]);
            v[y][x] &= ~nb[y];
          }
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t sel = y ? 0x7362 : 0x5140;
            const uint32_t b0 = __byte_perm(nb[0], nb[1], sel), b1 = __byte_perm(nb[2], nb[3], sel);
            float cnt[4] = {0.f, 0.f, 0.f, 0.f};
            // 0xff per NaN -> fp16 1.0
            mma_f16(cnt, __byte_perm(b0, 0, 0x1100) & 0x3c003c00u, __byte_perm(b0, 0, 0x3322) & 0x3c003c00u,
                    __byte_perm(b1, 0, 0x1100) & 0x3c003c00u, __byte_perm(b1, 0, 0x3322) & 0x3c003c00u, ones[0], ones[1]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (cnt[e] > 0.f) o[2 * x + y][e] = __int_as_float(0x7fffffff);
          }
        }
      }
#pragma unroll
      for (int x = 0; x < D / 32; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const uint32_t sel = y ? 0x7362 : 0x5140;
          const uint32_t b0 = __byte_perm(v[0][x], v[1][x], sel), b1 = __byte_perm(v[2][x], v[3][x], sel);
          const uint32_t a0 = widen_lo(b0), a1 = widen_hi(b0), a2 = widen_lo(b1), a3 = widen_hi(b1);
          if constexpr (NS == 1) {
            mma_f16(o[2 * x + y], a0, a1, a2, a3, pb[0][0], pb[0][1]);
          } else {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
            mma_f16(c, a0, a1, a2, a3, pb[1][0], pb[1][1]);
            mma_f16(c, a0, a1, a2, a3, pb[0][0], pb[0][1]);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[2 * x + y][e] += c[e];
          }
        }
    }
  }
  if constexpr (NS == 1)
    if (n > CA_CHAIN) put_by(false, true);
  if (bad_page) report_device_error(a.err, CA_ERR_PAGE);

  // ---- the warps' parts into one
  copies_wait<0>();
  __syncthreads();  // the rings' memory becomes the parts
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float l = st[c].l;
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
    if (g == 0) {
      s_m[warp][2 * t + c] = st[c].m;
      s_l[warp][2 * t + c] = l;
      s_M[warp][2 * t + c] = st[c].M;
    }
    float* dst = s_o + (warp * CA_ROWS + 2 * t + c) * D + g * (D / 8);
#pragma unroll
    for (int i = 0; i < MT; ++i) *reinterpret_cast<float2*>(dst + 2 * i) = make_float2(o[i][c], o[i][2 + c]);
  }
  __syncthreads();
  for (int e = tid; e < CA_ROWS * D; e += CA_THREADS) {
    const int r = e / D, d = e % D;
    const int head = head_of(tok0 + r), tok = tok0 + r - head * per_head, h = hk * a.G + head0 + head;
    if (r >= n_rows || tok >= p.n_q) continue;
    float m = -INFINITY, M = -INFINITY;
#pragma unroll
    for (int x = 0; x < CA_WARPS; ++x) {
      m = fmaxf(m, s_m[x][r]);
      M = fmaxf(M, s_M[x][r]);
    }
    const float mu = m == -INFINITY ? 0.f : m, Mu = M == -INFINITY ? 0.f : M;
    float l = 0.f, v = 0.f;
#pragma unroll
    for (int x = 0; x < CA_WARPS; ++x) {
      l += s_l[x][r] * ex2_approx(s_m[x][r] - mu);
      v += s_o[(x * CA_ROWS + r) * D + d] * ex2_approx(s_M[x][r] - Mu);
    }
    const int64_t row = (int64_t)(p.q0 + tok) * a.H + h;
    if (splits == 1) {
      const float res = l == 0.f ? 0.f : v * ex2_approx(Mu - mu - CA_P_SHIFT) / l;
      if (a.out_dtype == DSALT_F32) reinterpret_cast<float*>(a.out)[row * D + d] = res;
      else if (a.out_dtype == DSALT_BF16) reinterpret_cast<__nv_bfloat16*>(a.out)[row * D + d] = __float2bfloat16_rn(res);
      else reinterpret_cast<__half*>(a.out)[row * D + d] = __float2half_rn(res);
      if (d == 0) {
        if (a.lse) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        a.row_part[row] = make_int2(0, 1);
      }
    } else {
      const int64_t part = part0 + split;
      a.part_o[(part * CA_ROWS + r) * D + d] = v;
      if (d == 0) {
        float* ps = a.part_s + (part * CA_ROWS + r) * 4;
        ps[0] = m, ps[1] = l, ps[2] = M;
        if (split == 0) a.row_part[row] = make_int2(part0 * CA_ROWS + r, splits);
      }
    }
  }
}

// Joins the parts of the rows that were cut: of few parts by a warp, of many by the block, one row
// after another. (256 rows of 27 parts, a block each: 40.8 us with the attention, by warps 43.5;
// 2576 rows of two parts, five to a block: 24.1 us, by warps 22.0.) The order of every sum is
// fixed by the parts' numbers: the result does not depend on which finished first.
constexpr int CJ_THREADS = 256;
template <int D>
__global__ void __launch_bounds__(CJ_THREADS) cache_attn_join_kernel(CacheAttnArgs a, int rows_per_block) {
  constexpr int TPP = D / 4, GROUPS = CJ_THREADS / TPP;  // threads per part, parts at a time
  __shared__ float s_w[2 * CA_MAX_SLOTS];
  __shared__ float s_red[3][CJ_THREADS / 32];
  __shared__ float4 s_v[GROUPS][TPP];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cudaGridDependencySynchronize();
  const int64_t rows = (int64_t)a.T * a.H, row0 = (int64_t)blockIdx.x * rows_per_block;
  // which of the block's rows were cut. One part: already written. Anything else than parts of
  // this call: a row of no sequence.
  __shared__ int2 s_part[CJ_THREADS];
  bool cut = false;
  if (tid < rows_per_block && row0 + tid < rows) {
    const int2 rp = a.row_part[row0 + tid];
    cut = rp.y > 1 && rp.x >= 0 && rp.y <= 2 * CA_MAX_SLOTS && rp.x / CA_ROWS + rp.y <= 2 * CA_MAX_SLOTS;
    s_part[tid] = cut ? rp : make_int2(0, 0);
  }
  if (!__syncthreads_or(cut)) return;
  const auto put = [&](int64_t at, float v) {
    if (a.out_dtype == DSALT_F32) reinterpret_cast<float*>(a.out)[at] = v;
    else if (a.out_dtype == DSALT_BF16) reinterpret_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
    else reinterpret_cast<__half*>(a.out)[at] = __float2half_rn(v);
  };
  const int here = (int)min((int64_t)rows_per_block, rows - row0), few = min(32, 8 * rows_per_block);
  for (int r = warp; r < here; r += CJ_THREADS / 32) {
    const int2 rp = s_part[r];
    if (rp.y == 0 || rp.y > few) continue;
    float4 v = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
    if (lane < rp.y) v = reinterpret_cast<const float4*>(a.part_s)[rp.x + lane * CA_ROWS];
    float m = v.x, M = v.z;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    }
    const float mu = m == -INFINITY ? 0.f : m, Mu = M == -INFINITY ? 0.f : M;
    float l = v.y * ex2_approx(v.x - mu);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    const float weight = ex2_approx(v.z - Mu);
    const float2* po = reinterpret_cast<const float2*>(a.part_o + (int64_t)rp.x * D) + lane;
    float2 sum[D / 64];
#pragma unroll
    for (int d = 0; d < D / 64; ++d) sum[d] = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int x = 0; x < rp.y; ++x) {
      const float w = __shfl_sync(0xffffffffu, weight, x);
#pragma unroll
      for (int d = 0; d < D / 64; ++d) {
        const float2 y = po[(int64_t)x * (CA_ROWS * D / 2) + d * 32];
        sum[d].x += y.x * w, sum[d].y += y.y * w;
      }
    }
    const float f = l == 0.f ? 0.f : ex2_approx(Mu - mu - CA_P_SHIFT) / l;
    const int64_t row = row0 + r;
#pragma unroll
    for (int d = 0; d < D / 64; ++d) {
      put(row * D + d * 64 + 2 * lane, l == 0.f ? 0.f : sum[d].x * f);
      put(row * D + d * 64 + 2 * lane + 1, l == 0.f ? 0.f : sum[d].y * f);
    }
    if (lane == 0 && a.lse) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
  }
  for (int64_t row = row0; row < row0 + here; ++row) {
    const int2 rp = s_part[row - row0];
    if (rp.y <= few) continue;
    const float4* ps = reinterpret_cast<const float4*>(a.part_s) + rp.x;
    float m = -INFINITY, M = -INFINITY;
    for (int x = tid; x < rp.y; x += CJ_THREADS) {
      const float4 v = ps[(int64_t)x * CA_ROWS];
      m = fmaxf(m, v.x);
      M = fmaxf(M, v.z);
      s_w[x] = v.z;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    }
    if (lane == 0) s_red[0][warp] = m, s_red[1][warp] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < CJ_THREADS / 32; ++w) {
      m = fmaxf(m, s_red[0][w]);
      M = fmaxf(M, s_red[1][w]);
    }
    const float mu = m == -INFINITY ? 0.f : m, Mu = M == -INFINITY ? 0.f : M;
    float l = 0.f;
    for (int x = tid; x < rp.y; x += CJ_THREADS) {
      const float4 v = ps[(int64_t)x * CA_ROWS];
      l += v.y * ex2_approx(v.x - mu);
      s_w[x] = ex2_approx(s_w[x] - Mu);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) s_red[2][warp] = l;
    __syncthreads();
    l = 0.f;
#pragma unroll
    for (int w = 0; w < CJ_THREADS / 32; ++w) l += s_red[2][w];
    const float4* po = reinterpret_cast<const float4*>(a.part_o + (int64_t)rp.x * D) + tid % TPP;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int x = tid / TPP; x < rp.y; x += GROUPS) {
      const float4 y = po[(int64_t)x * (CA_ROWS * TPP)];
      const float w = s_w[x];
      v.x += y.x * w, v.y += y.y * w, v.z += y.z * w, v.w += y.w * w;
    }
    s_v[tid / TPP][tid % TPP] = v;
    __syncthreads();
    if (tid < D) {
      float sum = 0.f;
#pragma unroll
      for (int x = 0; x < GROUPS; ++x) sum += reinterpret_cast<const float*>(&s_v[x][0])[tid];
      put(row * D + tid, l == 0.f ? 0.f : sum * ex2_approx(Mu - mu - CA_P_SHIFT) / l);
    }
    if (tid == 0 && a.lse) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    __syncthreads();  // the shared arrays are used again
  }
}

static inline size_t ca_a256(size_t v) { return (v + 255) & ~(size_t)255; }
// is the schedule made by a kernel of its own?
static inline bool ca_plans(int64_t T, int n_seqs) { return n_seqs > CA_OWN_SCHED || T - n_seqs > CA_OWN_ROWS; }
// items of the kernel at most: from 8 tokens on a sequence's heads are filled up to whole tiles
static inline int64_t ca_items(int64_t T, int n_seqs, int G, int Hkv) {
  return ((T * G + (CA_ROWS - 1) * (n_seqs + G * std::min<int64_t>(n_seqs, T / CA_ROWS))) / CA_ROWS + 1) * Hkv;
}

template <typename T, int D, int NS>
static int launch_cache_attn(const CacheAttnArgs& a, unsigned grid, bool join, cudaStream_t stream) {
  constexpr size_t RING = (size_t)CA_WARPS * Shape<D>::STAGES * Stage<D>::BYTES;
  constexpr size_t SMEM = RING + (NS == 1 && D == 64 ? sizeof(float) * CA_THREADS * D / 4 : 0);
  static_assert(RING >= sizeof(float) * CA_WARPS * CA_ROWS * D, "the parts take the rings' place");
  static_assert(RING >= sizeof(SeqPlan) * CA_OWN_SCHED, "so does the schedule");
  static std::atomic<uint64_t> ready{0};
  if (int rc = allow_dynamic_smem(reinterpret_cast<const void*>(cache_attn_kernel<T, D, NS>), (int)SMEM, ready)) return rc;
  if (a.sched) {
    cache_attn_plan_kernel<<<1, CP_THREADS, 0, stream>>>(a, Shape<D>::SLOTS);
    if (int rc = check_cuda(cudaGetLastError(), "cache_attention plan launch")) return rc;
  }
  cache_attn_kernel<T, D, NS><<<grid, CA_THREADS, SMEM, stream>>>(a);
  if (int rc = check_cuda(cudaGetLastError(), "cache_attention launch")) return rc;
  if (!join) return DSALT_OK;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  // a block per row up to one round of blocks; where there are more rows, few of them are cut
  const int64_t rows = (int64_t)a.T * a.H;
  const int per = (int)std::min<int64_t>((rows + 148 * 4 - 1) / (148 * 4), CJ_THREADS);
  cfg.gridDim = dim3((unsigned)((rows + per - 1) / per));
  cfg.blockDim = dim3(CJ_THREADS);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, cache_attn_join_kernel<D>, a, per), "cache_attention join launch");
}

}  // namespace dsalt

using namespace dsalt;

extern "C" {

size_t dsalt_cache_attention_workspace_bytes(int64_t T, int n_seqs, int n_heads, int n_kv, int head_dim) {
  if (T < 0 || n_seqs < 1 || n_heads < 1 || n_kv < 1 || head_dim < 1) return 0;
  // cut items: two parts or more each of more than half the wanted length, so at most twice as many as slots
  return ca_a256(sizeof(int2) * (size_t)T * n_heads) + ca_a256(sizeof(float) * 2 * CA_MAX_SLOTS * CA_ROWS * 4) +
         ca_a256(sizeof(float) * 2 * CA_MAX_SLOTS * CA_ROWS * (size_t)head_dim) +
         (ca_plans(T, n_seqs) ? ca_a256(sizeof(int2) * (size_t)(n_seqs + 1)) + ca_a256(sizeof(SeqPlan) * (size_t)n_seqs) : 0);
}

int dsalt_cache_attention(const void* q, int dtype, int64_t T, int n_heads, int n_kv, int head_dim, int64_t q_stride,
                          const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale,
                          int64_t n_pages, int page_size, const int32_t* block_tables, int max_pages,
                          const int32_t* seq_lens, int n_seqs, const int32_t* cu_q, const int32_t* w,
                          const int32_t* lmk, const float* lmk_bias, int k_lmk, void* out, int out_dtype, float* lse,
                          void* workspace, size_t workspace_bytes, void* stream) {
  if (T < 0 || n_heads < 1 || n_kv < 1 || n_heads % n_kv || n_seqs < 1 || max_pages < 1 || n_pages < 0 || k_lmk < 0)
    return fail(DSALT_ERR_INVALID, "cache_attention: bad sizes");
  if ((dtype != DSALT_F32 && dtype != DSALT_BF16 && dtype != DSALT_F16) ||
      (out_dtype != DSALT_F32 && out_dtype != DSALT_BF16 && out_dtype != DSALT_F16))
    return fail(DSALT_ERR_INVALID, "cache_attention: dtype");
  if (head_dim != 64 && head_dim != 128)
    return fail(DSALT_ERR_UNSUPPORTED, "cache_attention: head_dim %d not in {64, 128}", head_dim);
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
    return fail(DSALT_ERR_UNSUPPORTED, "cache_attention: page size %d not in {16, 32, 64, 128}", page_size);
  if (n_seqs > CA_MAX_SEQS) return fail(DSALT_ERR_UNSUPPORTED, "cache_attention: %d sequences, at most %d", n_seqs, CA_MAX_SEQS);
  if (!cu_q && T != n_seqs) return fail(DSALT_ERR_INVALID, "cache_attention: without cu_q there is one query per sequence");
  if (q_stride < (int64_t)n_heads * head_dim) return fail(DSALT_ERR_INVALID, "cache_attention: token stride smaller than heads x head_dim");
  if (k_lmk > 0 && !w) return fail(DSALT_ERR_INVALID, "cache_attention: landmarks need window widths");
  if (T == 0) return DSALT_OK;
  if (!q || !k_cache || !v_cache || !k_scale || !v_scale || !block_tables || !seq_lens || !out || !workspace ||
      (k_lmk > 0 && !lmk))
    return fail(DSALT_ERR_INVALID, "cache_attention: null pointer");
  if (T * n_heads > 0x7fffff00LL || n_pages * n_kv * page_size > 0x7fffff00LL ||
      (int64_t)max_pages * page_size > 0x7fffff00LL)
    return fail(DSALT_ERR_UNSUPPORTED, "cache_attention: sizes above 2^31");
  const int es = dtype == DSALT_F32 ? 4 : 2;
  if ((((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) || (q_stride * es) % 16)
    return fail(DSALT_ERR_INVALID, "cache_attention: rows must be 16-byte aligned");
  const size_t need = dsalt_cache_attention_workspace_bytes(T, n_seqs, n_heads, n_kv, head_dim);
  if (workspace_bytes < need) return fail(DSALT_ERR_WORKSPACE, "cache_attention: workspace %zu < %zu", workspace_bytes, need);
  CacheAttnArgs a;
  a.q = q, a.q_stride = q_stride;
  a.kc = reinterpret_cast<const uint8_t*>(k_cache), a.vc = reinterpret_cast<const uint8_t*>(v_cache);
  a.ks = k_scale, a.vs = v_scale;
  a.tables = block_tables, a.max_pages = max_pages, a.n_pages = (int)n_pages;
  a.seq_lens = seq_lens, a.cu_q = cu_q, a.w = w, a.lmk = lmk, a.bias = lmk_bias;
  a.k_lmk = k_lmk, a.n_seqs = n_seqs, a.T = (int)T, a.H = n_heads, a.Hkv = n_kv, a.G = n_heads / n_kv;
  a.page_shift = page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : 7;
  a.scale_log2 = (float)(1.4426950408889634 / sqrt((double)head_dim));
  a.out = out, a.out_dtype = out_dtype, a.lse = lse;
  char* ws = reinterpret_cast<char*>(workspace);
  a.row_part = reinterpret_cast<int2*>(ws);
  ws += ca_a256(sizeof(int2) * (size_t)T * n_heads);
  a.part_s = reinterpret_cast<float*>(ws);
  ws += ca_a256(sizeof(float) * 2 * CA_MAX_SLOTS * CA_ROWS * 4);
  a.part_o = reinterpret_cast<float*>(ws);
  ws += ca_a256(sizeof(float) * 2 * CA_MAX_SLOTS * CA_ROWS * (size_t)head_dim);
  a.sched = ca_plans(T, n_seqs) ? reinterpret_cast<int2*>(ws) : nullptr;
  ws += ca_a256(sizeof(int2) * (size_t)(n_seqs + 1));
  a.plans = reinterpret_cast<SeqPlan*>(ws);
  a.err = device_status_ptr();
  const int64_t items = ca_items(T, n_seqs, a.G, n_kv);
  const int64_t grid = items + CA_MAX_SLOTS;
  if (grid > 0x7fffff00LL) return fail(DSALT_ERR_UNSUPPORTED, "cache_attention: too many rows");
  // tables too short for any item to be cut: nothing to join
  const int64_t most = (((int64_t)max_pages * page_size + 31) >> 5) + (int64_t)a.G * ((k_lmk + 31) >> 5);
  const bool join = most > CA_MIN_TILES;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
#define DSALT_CA(TT, NS)                                                              \
  (head_dim == 64 ? launch_cache_attn<TT, 64, NS>(a, (unsigned)grid, join, st)        \
                  : launch_cache_attn<TT, 128, NS>(a, (unsigned)grid, join, st))
  if (dtype == DSALT_F32) return DSALT_CA(float, 2);
  if (dtype == DSALT_F16) return DSALT_CA(__half, 1);
  return DSALT_CA(__nv_bfloat16, 1);
#undef DSALT_CA
}

}  // extern "C"
