// Attention of one or a few query tokens per sequence over a paged cache held in 8 bits
// (dsalt_cache_attention).
//
// Query at position i of width w, head h: keys A = [max(0, i - w + 1), i] U {landmarks p of
// (h, sequence): 0 <= p < i - w + 1}, x_j = q.k_j / sqrt(D) (+ bias_p), out = sum softmax(x)_j
// v_j; without widths A = [0, i]. k_j = byte * 2^e of its page and kv head, v_j likewise.
//
// Bytes decide: 2 D per key and kv head are read once and give 4 D * (query rows of the kv
// head) operations, far below what the tensor cores do in that time. So every query row that
// shares a kv head (the heads of a group, the tokens of a draft) goes into one 16-row tile of
// mma.sync m16n8k16, whose operands can be built in registers straight from global loads:
// * an e4m3 value is exact in fp16, so K and V are widened exactly; Q is scaled by a power of
//   two per row to a largest magnitude in [2^13, 2^14), which keeps bf16 and fp16 values
//   exact (those below 2^-27 of the row's largest fall short, under fp32's own rounding);
// * the contraction order of a product is free, so lane (g, t) takes 16 consecutive bytes of
//   key g for Q K^T and the D/8 bytes at D/8 g of keys 2t, 2t+1, 2t+8, 2t+9 for P V: whole
//   sectors, no shared memory, no shuffles of data;
// * P is rounded to fp16 relative to the row's largest p * 2^e (half a step is 2^-12, under
//   the 2^-9 of a bf16 result and as large as an fp16 result's own); fp32 queries take Q and
//   P as two fp16 terms each (22 bits).
// The scales of V differ from page to page, so a row keeps two maxima: m of x for the
// denominator l = sum 2^(x - m), and M of x + e for the numerator O = sum 2^(x + e - M) byte;
// out = O 2^(M - m) / l. Neither can overflow whatever the scales are.
//
// The keys of an item (sequence, kv head, tile of 16 rows) are a list of groups of 16: the
// window's, then the landmarks' of each head. Items are cut into units of about equal
// length, by the lengths found on the device (no host copy of them is needed and a captured
// call follows them); the parts of an item that was cut are joined by a second kernel.
#include <type_traits>

#include "common.cuh"

namespace dsalt {

constexpr int CA_WARPS = 4;
constexpr int CA_THREADS = 32 * CA_WARPS;
constexpr int CA_TARGET = 148 * 4;     // units wanted where the keys can be cut into as many
constexpr int CA_MIN_GROUPS = 16;      // groups of 16 keys that a unit takes at least
constexpr int CA_MAX_SEQS = 8192;
constexpr int CA_ERR_PAGE = 41;        // device status: a page number outside the pool was met
constexpr float CA_P_SHIFT = 14.f;     // P is held times 2^14: fp16 stays normal down to 2^-28

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
  float* part_o;   // [cut units][16][D]
  float* part_s;   // [cut units][16][4]: m, l, M
  int2* row_part;  // [T * H] first part of the row and how many there are
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
__device__ __forceinline__ float exp2_fast(float x) { return ex2_approx(x); }
// e of a scale 2^e, as a float; 0 (a page never written) as the lowest
__device__ __forceinline__ float scale_log(float s) { return (float)((int)(__float_as_uint(s) >> 23 & 0xff) - 127); }

// query of sequence s: tokens, keys and the groups of 16 that they make
struct SeqPlan {
  int q0, n_q, len, lo16, n_window, n_lmk;  // lo16: first key of the first group
};
__device__ __forceinline__ int first_key(const CacheAttnArgs& a, int t, int pos) {
  if (!a.w) return 0;
  const int w = max(a.w[t], 1);
  return max(pos - w + 1, 0);  // no overflow: pos < 2^31, w >= 1
}
__device__ __forceinline__ SeqPlan plan_of(const CacheAttnArgs& a, int s) {
  SeqPlan p;
  p.q0 = a.cu_q ? min(max(a.cu_q[s], 0), a.T) : s;
  p.n_q = a.cu_q ? max(min(a.cu_q[s + 1], a.T) - p.q0, 0) : 1;
  p.len = min(max(a.seq_lens[s], 0), a.max_pages << a.page_shift);
  int lo = p.len, top = 0;
  if (!a.w) lo = 0;
  else for (int r = 0; r < p.n_q; ++r) {
    const int pos = p.len - p.n_q + r;
    if (pos < 0) continue;
    const int f = first_key(a, p.q0 + r, pos);
    lo = min(lo, f);
    top = max(top, f);
  }
  // the last key is the sequence's last: groups behind a tile's own rows are passed over
  p.lo16 = lo & ~15;
  p.n_window = p.n_q > 0 && p.len > 0 ? (p.len - p.lo16 + 15) >> 4 : 0;
  p.n_lmk = a.k_lmk > 0 && top > 0 ? a.G * ((a.k_lmk + 15) >> 4) : 0;  // none lies before a window from 0
  return p;
}
__device__ __forceinline__ int tiles_of(const CacheAttnArgs& a, int n_q) { return (n_q * a.G + 15) >> 4; }

// sums of two numbers over the block's 128 threads, exclusive; totals in `all`
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
  for (int i = 0; i < CA_WARPS; ++i) {
    if (i < warp) before.x += red[i].x, before.y += red[i].y;
    all.x += red[i].x, all.y += red[i].y;
  }
  return make_int2(before.x + s.x - v.x, before.y + s.y - v.y);
}

template <int D>
struct Frag {
  uint32_t k[2][D / 16];   // key g of either half: D/4 bytes of this lane
  uint32_t v[4][D / 32];   // keys 2t, 2t+1, 2t+8, 2t+9: D/8 bytes each
};

// D/4 bytes of K (16 at 16 t of each 64) and D/8 bytes of V (at D/8 g) of one cache row
template <int D>
__device__ __forceinline__ void load_k(uint32_t (&r)[D / 16], const uint8_t* base, int row, int t, bool ok) {
#pragma unroll
  for (int i = 0; i < D / 64; ++i) {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (ok) x = __ldg(reinterpret_cast<const uint4*>(base + (int64_t)row * D + i * 64 + t * 16));
    r[4 * i] = x.x, r[4 * i + 1] = x.y, r[4 * i + 2] = x.z, r[4 * i + 3] = x.w;
  }
}
template <int D>
__device__ __forceinline__ void load_v(uint32_t (&r)[D / 32], const uint8_t* base, int row, int g, bool ok) {
  if constexpr (D == 64) {
    uint2 x = make_uint2(0, 0);
    if (ok) x = __ldg(reinterpret_cast<const uint2*>(base + (int64_t)row * D + g * 8));
    r[0] = x.x, r[1] = x.y;
  } else {
    uint4 x = make_uint4(0, 0, 0, 0);
    if (ok) x = __ldg(reinterpret_cast<const uint4*>(base + (int64_t)row * D + g * 16));
    r[0] = x.x, r[1] = x.y, r[2] = x.z, r[3] = x.w;
  }
}
__device__ __forceinline__ uint32_t nan_bytes(uint32_t v) {  // 0xff where a byte is an e4m3 NaN
  return __vcmpeq4(v & 0x7f7f7f7fu, 0x7f7f7f7fu);
}

// NS: fp16 terms that Q and P are held in (2 for fp32 queries)
template <typename T, int D, int NS>
__global__ void __launch_bounds__(CA_THREADS) cache_attn_kernel(CacheAttnArgs a) {
  constexpr int KS = D / 16, NT = D / 8;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ int2 red[CA_WARPS];
  __shared__ float s_m[CA_WARPS][16], s_l[CA_WARPS][16], s_M[CA_WARPS][16];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  int* s_base = reinterpret_cast<int*>(dyn);  // [n_seqs] units of the sequences before s
  int* s_cut = s_base + a.n_seqs;             // [n_seqs] parts of cut items before s
  float* s_o = reinterpret_cast<float*>(dyn);  // [warps][16][D], after the schedule has been read

  // ---- schedule: every block derives the same one from the lengths
  int2 all;
  int chunk;
  {
    long long mine = 0;
    for (int s = tid; s < a.n_seqs; s += CA_THREADS) {
      const SeqPlan p = plan_of(a, s);
      mine += (long long)(p.n_window + p.n_lmk) * tiles_of(a, p.n_q) * a.Hkv;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    __shared__ long long s_sum[CA_WARPS];
    if (lane == 0) s_sum[warp] = mine;
    __syncthreads();
    const long long total = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
    chunk = (int)min(max((total + CA_TARGET - 1) / CA_TARGET, (long long)CA_MIN_GROUPS), 0x7fffffffLL);
  }
  int2 carry = make_int2(0, 0);
  for (int base = 0; base < a.n_seqs; base += CA_THREADS) {
    const int s = base + tid;
    int2 v = make_int2(0, 0);
    if (s < a.n_seqs) {
      const SeqPlan p = plan_of(a, s);
      const int splits = max(1, (p.n_window + p.n_lmk + chunk - 1) / chunk);
      v.x = tiles_of(a, p.n_q) * a.Hkv * splits;
      v.y = splits > 1 ? v.x : 0;
    }
    const int2 b = block_before2(v, red, all);
    if (s < a.n_seqs) {
      s_base[s] = carry.x + b.x;
      s_cut[s] = carry.y + b.y;
    }
    carry.x += all.x;
    carry.y += all.y;
  }
  __syncthreads();
  const int unit = blockIdx.x;
  // rows behind the last sequence's: zero, log-sum-exp -inf
  if (a.cu_q) {
    const int64_t rows0 = (int64_t)min(max(a.cu_q[a.n_seqs], 0), a.T) * a.H, rows1 = (int64_t)a.T * a.H;
    for (int64_t r = rows0 + unit; r < rows1; r += gridDim.x) {
      if (tid < D) {
        if (a.out_dtype == DSALT_F32) reinterpret_cast<float*>(a.out)[r * D + tid] = 0.f;
        else reinterpret_cast<uint16_t*>(a.out)[r * D + tid] = 0;
      }
      if (tid == 0) {
        if (a.lse) a.lse[r] = -INFINITY;
        if (a.row_part) a.row_part[r] = make_int2(0, 1);
      }
    }
  }
  if (unit >= carry.x) return;
  int s = 0;
  {
    int lo = 0, hi = a.n_seqs - 1;  // the last sequence whose units begin at or before this one
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_base[mid] <= unit) lo = mid;
      else hi = mid - 1;
    }
    s = lo;
  }
  const SeqPlan p = plan_of(a, s);
  const int groups = p.n_window + p.n_lmk, splits = max(1, (groups + chunk - 1) / chunk);
  const int local = unit - s_base[s];
  const int split = local % splits, item = local / splits;
  const int hk = item % a.Hkv, tile = item / a.Hkv;
  const int part0 = s_cut[s] + item * splits;
  __syncthreads();  // the schedule's memory is used again below
  const int each = (groups + splits - 1) / splits;
  const int g_begin = split * each, g_end = min(g_begin + each, groups);

  // ---- this lane's two query rows
  int row_lo[2], row_hi[2], row_head[2];
  int64_t row_q[2];
  float row_f[2];
  bool row_ok[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = tile * 16 + g + r * 8, tok = i / a.G, h = hk * a.G + i % a.G;
    row_ok[r] = tok < p.n_q;
    const int pos = p.len - p.n_q + tok;
    const bool keys = row_ok[r] && pos >= 0;
    row_lo[r] = keys ? first_key(a, p.q0 + tok, pos) : 0x7fffffff;
    row_hi[r] = keys ? pos + 1 : 0;
    row_head[r] = i % a.G;
    row_q[r] = (int64_t)(p.q0 + tok) * a.H + h;
    row_f[r] = 0.f;
  }
  uint32_t qa[NS][KS][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    // 16 consecutive elements at 16 t of each 64
    float x[D / 4];
#pragma unroll
    for (int i = 0; i < D / 4; ++i) x[i] = 0.f;
    if (row_ok[r]) {
      const int i = tile * 16 + g + r * 8;
      const T* src = reinterpret_cast<const T*>(a.q) + (int64_t)(p.q0 + i / a.G) * a.q_stride +
                     (int64_t)(hk * a.G + i % a.G) * D + t * 16;
#pragma unroll
      for (int b = 0; b < D / 64; ++b) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 f = __ldg(reinterpret_cast<const float4*>(src + b * 64) + j);
            x[b * 16 + 4 * j] = f.x, x[b * 16 + 4 * j + 1] = f.y, x[b * 16 + 4 * j + 2] = f.z, x[b * 16 + 4 * j + 3] = f.w;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(src + b * 64) + j);
            const uint32_t wd[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float2 f;
              if constexpr (std::is_same<T, __half>::value) f = __half22float2(*reinterpret_cast<const __half2*>(&wd[e]));
              else f = make_float2(__uint_as_float(wd[e] << 16), __uint_as_float(wd[e] & 0xffff0000u));
              x[b * 16 + j * 8 + 2 * e] = f.x;
              x[b * 16 + j * 8 + 2 * e + 1] = f.y;
            }
          }
        }
      }
    }
    float big = 0.f;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) big = fmaxf(big, fabsf(x[i]));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
    const int eb = (int)(__float_as_uint(big) >> 23);  // biased exponent; 255: an infinity
    const int up = eb == 255 ? 0 : min(max(13 - (eb - 127), -126), 126);
    const float mul = __uint_as_float((uint32_t)(up + 127) << 23);
    row_f[r] = a.scale_log2 * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float lo = x[4 * k + 2 * h] * mul, hi = x[4 * k + 2 * h + 1] * mul;
        const uint32_t first = pack_f16x2(lo, hi);
        qa[0][k][2 * h + r] = first;
        if constexpr (NS == 2) {
          const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&first));
          qa[1][k][2 * h + r] = pack_f16x2(lo - b.x, hi - b.y);
        }
      }
  }
  // keys that every row of the tile attends to need no mask
  int lo_min = min(row_lo[0], row_lo[1]), hi_max = max(row_hi[0], row_hi[1]);
  int lo_max = max(row_ok[0] ? row_lo[0] : 0, row_ok[1] ? row_lo[1] : 0);
  int hi_min = min(row_ok[0] ? row_hi[0] : 0x7fffffff, row_ok[1] ? row_hi[1] : 0x7fffffff);
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    lo_max = max(lo_max, __shfl_xor_sync(0xffffffffu, lo_max, o));
    hi_min = min(hi_min, __shfl_xor_sync(0xffffffffu, hi_min, o));
    lo_min = min(lo_min, __shfl_xor_sync(0xffffffffu, lo_min, o));
    hi_max = max(hi_max, __shfl_xor_sync(0xffffffffu, hi_max, o));
  }

  float o[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  RowState st[2] = {{-INFINITY, 0.f, -INFINITY}, {-INFINITY, 0.f, -INFINITY}};
  const int page_mask = (1 << a.page_shift) - 1;
  const int* table = a.tables + (int64_t)s * a.max_pages;
  const int lmk16 = (a.k_lmk + 15) >> 4;
  bool bad_page = false;

  for (int gi = g_begin + warp; gi < g_end; gi += CA_WARPS) {
    const bool window = gi < p.n_window;
    const int key0 = p.lo16 + gi * 16;
    if (window && (key0 + 16 <= lo_min || key0 >= hi_max)) continue;  // keys of the sequence's other tiles
    // slot j = lane & 15 of the group: its cache row (or -1), scales, position
    int key, row = -1, slot_head = 0;
    float add = 0.f, ks = 0.f, ve = 0.f;
    const int j = lane & 15;
    if (window) key = key0 + j;
    else {
      const int l = gi - p.n_window, c = (l % lmk16) * 16 + j;
      slot_head = l / lmk16;
      key = -1;
      if (c < a.k_lmk) {
        const int64_t at = ((int64_t)(hk * a.G + slot_head) * a.n_seqs + s) * a.k_lmk + c;
        key = a.lmk[at];
        if (a.bias) add = a.bias[at] * 1.4426950408889634f;
      }
      if (key >= p.len) key = -1;  // no row attends to it, and it may lie outside the table
    }
    if (key >= 0 && key < p.len) {
      const int id = __ldg(table + (key >> a.page_shift));
      if ((unsigned)id < (unsigned)a.n_pages) {
        const int64_t head = (int64_t)id * a.Hkv + hk;
        row = (int)(head << a.page_shift) + (key & page_mask);
        ks = __ldg(a.ks + head);
        ve = scale_log(__ldg(a.vs + head));
      } else {
        bad_page = true;
      }
    }
    // valid for any row of the tile?  (a masked key's bytes are not looked at)
    Frag<D> f;
    {
      const int r0 = __shfl_sync(0xffffffffu, row, g), r1 = __shfl_sync(0xffffffffu, row, g + 8);
      load_k<D>(f.k[0], a.kc, r0, t, r0 >= 0);
      load_k<D>(f.k[1], a.kc, r1, t, r1 >= 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int rv = __shfl_sync(0xffffffffu, row, (i & 1) + 2 * t + (i >> 1) * 8);
        load_v<D>(f.v[i], a.vc, rv, g, rv >= 0);
      }
    }
    // ---- S = Q K^T
    float sc[2][4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const uint32_t b0 = widen_lo(f.k[nt][k]), b1 = widen_hi(f.k[nt][k]);
#pragma unroll
        for (int n = 0; n < NS; ++n) mma_f16(sc[nt], qa[n][k][0], qa[n][k][1], qa[n][k][2], qa[n][k][3], b0, b1);
      }
    }
    // ---- logits (base 2) of this lane's columns: keys 2t, 2t+1 of either half
    const bool plain = window && key0 >= lo_max && key0 + 16 <= hi_min && !__any_sync(0xffffffffu, row < 0);
    float ve_col[2][2];
    uint32_t valid = 0;  // bit 4 nt + 2 r + c: row r attends to column c of half nt
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int from = nt * 8 + 2 * t + c;
        const float kscale = __shfl_sync(0xffffffffu, ks, from), badd = __shfl_sync(0xffffffffu, add, from);
        ve_col[nt][c] = __shfl_sync(0xffffffffu, ve, from);
        const int kk = __shfl_sync(0xffffffffu, key, from), rr = __shfl_sync(0xffffffffu, row, from);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float x = fmaf(sc[nt][2 * r + c], kscale * row_f[r], badd);
          const bool ok = plain || (rr >= 0 && (window ? kk >= row_lo[r] && kk < row_hi[r]
                                                       : kk < row_lo[r] && kk < row_hi[r] && slot_head == row_head[r]));
          if (ok) valid |= 1u << (4 * nt + 2 * r + c);
          sc[nt][2 * r + c] = ok ? x : -INFINITY;
        }
      }
    // ---- online softmax with the two maxima
    float pr[2][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float gm = -INFINITY, gM = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          gm = fmaxf(gm, sc[nt][2 * r + c]);
          gM = fmaxf(gM, sc[nt][2 * r + c] + ve_col[nt][c]);
        }
#pragma unroll
      for (int x = 1; x < 4; x <<= 1) {
        gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, x));
        gM = fmaxf(gM, __shfl_xor_sync(0xffffffffu, gM, x));
      }
      const float m = fmaxf(st[r].m, gm), M = fmaxf(st[r].M, gM);
      const float mu = m == -INFINITY ? 0.f : m, Mu = M == -INFINITY ? 0.f : M;
      const float cl = exp2_fast(st[r].m - mu), cO = exp2_fast(st[r].M - Mu);
      float l = st[r].l * cl;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float x = sc[nt][2 * r + c];
          l += exp2_fast(x - mu);
          pr[nt][2 * r + c] = exp2_fast(x + ve_col[nt][c] - Mu + CA_P_SHIFT);
        }
      st[r].m = m;
      st[r].M = M;
      st[r].l = l;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        o[i][2 * r] *= cO;
        o[i][2 * r + 1] *= cO;
      }
    }
    // ---- O += P V
    uint32_t pa[NS][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int nt = i >> 1, r = i & 1;
      const float lo = pr[nt][2 * r], hi = pr[nt][2 * r + 1];
      pa[0][i] = pack_f16x2(lo, hi);
      if constexpr (NS == 2) {
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&pa[0][i]));
        pa[1][i] = pack_f16x2(lo - b.x, hi - b.y);
      }
    }
    bool nans = false;
    if (!plain) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < D / 32; ++x) nans |= nan_bytes(f.v[i][x]) != 0;
    }
    nans = !plain && __any_sync(0xffffffffu, nans);
    uint32_t va[4] = {0, 0, 0, 0};
    if (nans) {  // 1.0 where a row attends to a key: counts its NaNs, which P = 0 must not spread
#pragma unroll
      for (int i = 0; i < 4; ++i)
        va[i] = (valid >> (4 * (i >> 1) + 2 * (i & 1)) & 1 ? 0x3c00u : 0u) |
                (valid >> (4 * (i >> 1) + 2 * (i & 1) + 1) & 1 ? 0x3c000000u : 0u);
    }
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
      uint32_t v0 = f.v[0][x], v1 = f.v[1][x], v2 = f.v[2][x], v3 = f.v[3][x];
      uint32_t n0 = 0, n1 = 0, n2 = 0, n3 = 0;
      if (nans) {
        n0 = nan_bytes(v0), n1 = nan_bytes(v1), n2 = nan_bytes(v2), n3 = nan_bytes(v3);
        v0 &= ~n0, v1 &= ~n1, v2 &= ~n2, v3 &= ~n3;
      }
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint32_t sel = y ? 0x7362 : 0x5140;
        const uint32_t b0 = __byte_perm(v0, v1, sel), b1 = __byte_perm(v2, v3, sel);
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const int nt = 4 * x + 2 * y + z;
          const uint32_t w0 = z ? widen_hi(b0) : widen_lo(b0), w1 = z ? widen_hi(b1) : widen_lo(b1);
#pragma unroll
          for (int n = 0; n < NS; ++n) mma_f16(o[nt], pa[n][0], pa[n][1], pa[n][2], pa[n][3], w0, w1);
          if (nans) {
            // bytes 0xff -> fp16 1.0
            const uint32_t m0 = __byte_perm(__byte_perm(n0, n1, sel), 0, z ? 0x3322 : 0x1100);
            const uint32_t m1 = __byte_perm(__byte_perm(n2, n3, sel), 0, z ? 0x3322 : 0x1100);
            float cnt[4] = {0.f, 0.f, 0.f, 0.f};
            mma_f16(cnt, va[0], va[1], va[2], va[3], m0 & 0x3c003c00u, m1 & 0x3c003c00u);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (cnt[e] > 0.f) o[nt][e] = __int_as_float(0x7fffffff);
          }
        }
      }
    }
  }
  if (bad_page) report_device_error(a.err, CA_ERR_PAGE);

  // ---- the warps' parts into one
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float l = st[r].l;
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0) {
      s_m[warp][g + 8 * r] = st[r].m;
      s_l[warp][g + 8 * r] = l;
      s_M[warp][g + 8 * r] = st[r].M;
    }
    float* dst = s_o + (warp * 16 + g + 8 * r) * D + t * (D / 4);  // columns D/8 (2t) + i and D/8 (2t + 1) + i
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      dst[i] = o[i][2 * r];
      dst[NT + i] = o[i][2 * r + 1];
    }
  }
  __syncthreads();
  for (int e = tid; e < 16 * D; e += CA_THREADS) {
    const int r = e / D, d = e % D;
    const int i = tile * 16 + r, tok = i / a.G, h = hk * a.G + i % a.G;
    if (tok >= p.n_q) continue;
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
      l += s_l[x][r] * exp2_fast(s_m[x][r] - mu);
      v += s_o[(x * 16 + r) * D + d] * exp2_fast(s_M[x][r] - Mu);
    }
    const int64_t row = (int64_t)(p.q0 + tok) * a.H + h;
    if (splits == 1) {
      const float res = l == 0.f ? 0.f : v * exp2_fast(Mu - mu - CA_P_SHIFT) / l;
      if (a.out_dtype == DSALT_F32) reinterpret_cast<float*>(a.out)[row * D + d] = res;
      else if (a.out_dtype == DSALT_BF16) reinterpret_cast<__nv_bfloat16*>(a.out)[row * D + d] = __float2bfloat16_rn(res);
      else reinterpret_cast<__half*>(a.out)[row * D + d] = __float2half_rn(res);
      if (d == 0) {
        if (a.lse) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        if (a.row_part) a.row_part[row] = make_int2(0, 1);
      }
    } else {
      const int64_t part = part0 + split;
      a.part_o[(part * 16 + r) * D + d] = v;
      if (d == 0) {
        float* ps = a.part_s + (part * 16 + r) * 4;
        ps[0] = m, ps[1] = l, ps[2] = M;
        if (split == 0) a.row_part[row] = make_int2(part0 * 16 + r, splits);
      }
    }
  }
}

// Joins the parts of the rows that were cut, a block of four warps per (token, head). Parts
// are added in their order: the result does not depend on which finished first.
template <int D>
__global__ void __launch_bounds__(128) cache_attn_join_kernel(CacheAttnArgs a) {
  cudaGridDependencySynchronize();
  const int64_t row = blockIdx.x;
  const int2 rp = a.row_part[row];
  // one part: already written. Anything else than parts of this call: a row of no sequence.
  if (rp.y <= 1 || rp.x < 0 || rp.y > 2 * CA_TARGET || rp.x / 16 + rp.y > 2 * CA_TARGET) return;
  __shared__ float s_red[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float* ps = a.part_s + (int64_t)rp.x * 4;
  float m = -INFINITY, M = -INFINITY;
  for (int x = tid; x < rp.y; x += 128) {
    m = fmaxf(m, ps[(int64_t)x * 64]);
    M = fmaxf(M, ps[(int64_t)x * 64 + 2]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  }
  if (lane == 0) s_red[warp] = m, s_red[4 + warp] = M;
  __syncthreads();
  m = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  M = fmaxf(fmaxf(s_red[4], s_red[5]), fmaxf(s_red[6], s_red[7]));
  const float mu = m == -INFINITY ? 0.f : m, Mu = M == -INFINITY ? 0.f : M;
  float l = 0.f;
  for (int x = 0; x < rp.y; ++x) l += ps[(int64_t)x * 64 + 1] * exp2_fast(ps[(int64_t)x * 64] - mu);
  if (tid < D) {
    float v = 0.f;
    for (int x = 0; x < rp.y; ++x)
      v += a.part_o[((int64_t)rp.x + (int64_t)x * 16) * D + tid] * exp2_fast(ps[(int64_t)x * 64 + 2] - Mu);
    const float res = l == 0.f ? 0.f : v * exp2_fast(Mu - mu - CA_P_SHIFT) / l;
    if (a.out_dtype == DSALT_F32) reinterpret_cast<float*>(a.out)[row * D + tid] = res;
    else if (a.out_dtype == DSALT_BF16) reinterpret_cast<__nv_bfloat16*>(a.out)[row * D + tid] = __float2bfloat16_rn(res);
    else reinterpret_cast<__half*>(a.out)[row * D + tid] = __float2half_rn(res);
  }
  if (tid == 0 && a.lse) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

static inline size_t ca_a256(size_t v) { return (v + 255) & ~(size_t)255; }
static inline int64_t ca_items(int64_t T, int n_seqs, int G, int Hkv) { return ((T * G + 15 * (int64_t)n_seqs) / 16 + 1) * Hkv; }

template <typename T, int D, int NS>
static int launch_cache_attn(const CacheAttnArgs& a, unsigned grid, bool join, cudaStream_t stream) {
  size_t smem = 2 * sizeof(int) * (size_t)a.n_seqs;
  const size_t merge = sizeof(float) * CA_WARPS * 16 * D;
  if (smem < merge) smem = merge;
  static std::atomic<uint64_t> ready{0};
  if (int rc = allow_dynamic_smem(reinterpret_cast<const void*>(cache_attn_kernel<T, D, NS>),
                                  (int)(2 * sizeof(int) * CA_MAX_SEQS), ready))
    return rc;
  cache_attn_kernel<T, D, NS><<<grid, CA_THREADS, smem, stream>>>(a);
  if (int rc = check_cuda(cudaGetLastError(), "cache_attention launch")) return rc;
  if (!join) return DSALT_OK;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((int64_t)a.T * a.H));
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, cache_attn_join_kernel<D>, a), "cache_attention join launch");
}

}  // namespace dsalt

using namespace dsalt;

extern "C" {

size_t dsalt_cache_attention_workspace_bytes(int64_t T, int n_seqs, int n_heads, int n_kv, int head_dim) {
  if (T < 0 || n_seqs < 1 || n_heads < 1 || n_kv < 1 || head_dim < 1) return 0;
  // a cut item has at least two units of at least half the wanted length: at most twice the target
  return ca_a256(sizeof(int2) * (size_t)T * n_heads) + ca_a256(sizeof(float) * 2 * CA_TARGET * 64) +
         ca_a256(sizeof(float) * 2 * CA_TARGET * 16 * (size_t)head_dim);
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
  ws += ca_a256(sizeof(float) * 2 * CA_TARGET * 64);
  a.part_o = reinterpret_cast<float*>(ws);
  a.err = device_status_ptr();
  const int64_t items = ca_items(T, n_seqs, a.G, n_kv);
  const int64_t grid = items + CA_TARGET;
  if (grid > 0x7fffff00LL) return fail(DSALT_ERR_UNSUPPORTED, "cache_attention: too many rows");
  // tables too short for any item to be cut: nothing to join
  const int64_t most = ((int64_t)max_pages * page_size >> 4) + (int64_t)a.G * ((k_lmk + 15) >> 4);
  const bool join = most > CA_MIN_GROUPS;
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
