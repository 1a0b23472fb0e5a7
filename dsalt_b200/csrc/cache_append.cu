// Appends the keys and values of new tokens to a paged cache held in 8 bits
// (dsalt_append_cache).
//
// A page holds P tokens of every kv head, [kv head][token][head_dim] in e4m3, with one scale
// 2^e per (page, kv head) for keys and one for values; an element is byte * 2^e. e is the
// smallest exponent with amax <= 448 * 2^e over what the page holds: it starts afresh with
// the page's first token, never falls while the page fills, and the bytes already there are
// rewritten when it grows. Scales are powers of two because e4m3 is a floating-point
// format: a finer scale gives no more significant bits, while a power of two multiplies
// exactly, so that rewriting rounds only values that sink below 2^-6 (subnormal bytes), the
// choice of e is a comparison of bits, and the result does not depend on the order of
// anything. An infinity is stored as the largest value of its page (448 * 2^e) and does not
// enter amax, a NaN as NaN.
//
// A run is the tokens of one page among `page` consecutive tokens of the call, beginning with
// the first of them. One group of lanes owns a run of one head: it takes amax, settles e,
// rewrites the older bytes if e grew and writes the new ones, so nothing is exchanged between
// groups. A decode step is all runs of one token: D/8 lanes each, so that a warp holds
// 4 (2) heads at once. A prompt is runs of P tokens: a warp each, which reads a run in chunks of
// 8 vectors per lane (4 of fp32), keeps the last one between the two passes and takes the others
// from L1 or L2 again.
//
// Measured on a B200 (device time): 4 prompts of 8192 tokens, 12 heads of 64 in bf16 with pages of
// 64 (132 MB: the prompts are ragged) 30.0 us (4.4 TB/s; copying as much takes 20.5): bound by memory and by the chain
// that each block goes through (slots, runs, first pass, second pass), which the other two
// blocks of an SM cover; without the fetches to L2 it takes 34.1 us. 64 decode rows of 16 heads
// 3.0 us, next to nothing of which is bytes.
#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace dsalt {

constexpr int APPEND_THREADS = 256;
constexpr int APPEND_WARPS = APPEND_THREADS / 32;
constexpr int APPEND_MAX_WINDOW = 64;  // tokens whose runs one block looks for
constexpr int APPEND_MAX_PAGE = 128;
constexpr int SCALE_E_MIN = -110;  // 2^-110 times the smallest byte is still a normal fp32

struct AppendSide {  // k or v
  const void* src;
  uint8_t* cache;
  float* scale;
  int64_t token_stride, head_stride;
};
struct AppendArgs {
  AppendSide k, v;
  const int64_t* slots;
  int64_t T, n_pages;
  int n_kv, page_shift, window;
};

__device__ __forceinline__ float pow2f(int e) {  // 2^e, -126 <= e <= 127
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
// smallest e >= SCALE_E_MIN with amax <= 448 * 2^e = 1.75 * 2^(e + 8); amax finite, >= 0
__device__ __forceinline__ int need_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - ((u & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return max(e, SCALE_E_MIN);
}
__device__ __forceinline__ int scale_exponent(float s) {  // of a stored scale; anything else counts as none
  const uint32_t u = __float_as_uint(s);
  const int e = (int)(u >> 23) - 127;  // a negative number or a NaN comes out above 127
  return e > 127 ? SCALE_E_MIN : max(e, SCALE_E_MIN);
}
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {  // a in the lowest byte
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
__device__ __forceinline__ float2 from_e4m3x2(uint16_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(v));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}
__device__ __forceinline__ uint32_t rescale_e4m3x4(uint32_t v, float f) {
  const float2 a = from_e4m3x2((uint16_t)v), b = from_e4m3x2((uint16_t)(v >> 16));
  return to_e4m3x4(a.x * f, a.y * f, b.x * f, b.y * f);
}
// a vector of eight elements, as loaded
template <typename T>
struct Vec8 {
  uint4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Vec8<T> load8(const T* p) {
  Vec8<T> v;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) v.w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  return v;
}
template <typename T>
__device__ __forceinline__ void widen8(const Vec8<T>& v, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      x[4 * i] = __uint_as_float(v.w[i].x), x[4 * i + 1] = __uint_as_float(v.w[i].y);
      x[4 * i + 2] = __uint_as_float(v.w[i].z), x[4 * i + 3] = __uint_as_float(v.w[i].w);
    }
  } else {
    const uint32_t w[4] = {v.w[0].x, v.w[0].y, v.w[0].z, v.w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 f;
      if constexpr (std::is_same<T, __half>::value) f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      else f = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}
// Largest magnitude, as ordered bits: 16-bit types two to a word. Infinities and NaN come out
// above every finite number and are looked for afterwards.
template <typename T>
__device__ __forceinline__ uint32_t max8(const Vec8<T>& v, uint32_t m) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      m = max(m, max(v.w[i].x & 0x7fffffffu, v.w[i].y & 0x7fffffffu));
      m = max(m, max(v.w[i].z & 0x7fffffffu, v.w[i].w & 0x7fffffffu));
    }
  } else {
    m = __vmaxu2(m, __vmaxu2(v.w[0].x & 0x7fff7fffu, v.w[0].y & 0x7fff7fffu));
    m = __vmaxu2(m, __vmaxu2(v.w[0].z & 0x7fff7fffu, v.w[0].w & 0x7fff7fffu));
  }
  return m;
}
// the same over finite numbers alone
template <typename T>
__device__ __forceinline__ uint32_t max8_finite(const Vec8<T>& v, uint32_t m) {
  float x[8];
  widen8<T>(v, x);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float f = fabsf(x[j]);
    if (!(f < INFINITY)) continue;
    if constexpr (sizeof(T) == 4) m = max(m, __float_as_uint(f));
    else if constexpr (std::is_same<T, __half>::value) m = __vmaxu2(m, __half_as_ushort(__float2half_rn(f)));
    else m = __vmaxu2(m, __float_as_uint(f) >> 16);
  }
  return m;
}
template <typename T>
__device__ __forceinline__ uint32_t fold(uint32_t m) {  // the larger of the two halves
  return sizeof(T) == 4 ? m : max(m & 0xffffu, m >> 16);
}
template <typename T>
__device__ __forceinline__ bool finite_bits(uint32_t m) {
  return m < (sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u);
}
template <typename T>
__device__ __forceinline__ float bits_value(uint32_t m) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(m);
  else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)m));
  else return __uint_as_float(m << 16);
}

// exponent of a run of one head, and the rewriting of the page's older bytes by the warp
// where it grew (`own`: this lane holds the decision of its group; one group at a time)
__device__ __forceinline__ void rewrite_page(uint8_t* bytes, int n16, int shrink) {
  const float f = shrink < -126 ? 0.f : pow2f(shrink);
  uint4* p = reinterpret_cast<uint4*>(bytes);
  for (int i = threadIdx.x & 31; i < n16; i += 32) {
    uint4 v = p[i];
    v.x = rescale_e4m3x4(v.x, f);
    v.y = rescale_e4m3x4(v.y, f);
    v.z = rescale_e4m3x4(v.z, f);
    v.w = rescale_e4m3x4(v.w, f);
    p[i] = v;
  }
}
template <typename T>
__device__ __forceinline__ uint2 quantise8(const Vec8<T>& v, float inv) {
  float x[8];
  widen8<T>(v, x);
  return make_uint2(to_e4m3x4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv),
                    to_e4m3x4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv));
}

// grid: (window of tokens, share of the 2 n_kv planes: heads of k, then of v)
template <typename T, int D>
__global__ void __launch_bounds__(APPEND_THREADS, 3) append_cache_kernel(AppendArgs a) {
  constexpr int VPT = D / 8, STEP = 32 / VPT;          // lanes per token, tokens (or heads) per warp
  constexpr int KEEP = sizeof(T) == 4 ? 4 : 8;         // vectors of a lane in one chunk
  __shared__ int32_t s_page[APPEND_MAX_WINDOW + 2 * APPEND_MAX_PAGE];  // page of each token near the window, -1: none
  __shared__ int16_t s_in[APPEND_MAX_WINDOW + 2 * APPEND_MAX_PAGE];    // its offset in the page
  __shared__ int16_t s_one[APPEND_MAX_WINDOW], s_run[APPEND_MAX_WINDOW], s_len[APPEND_MAX_WINDOW];
  __shared__ int16_t s_cand[APPEND_MAX_WINDOW];
  __shared__ int s_cands, s_ones, s_runs;
  const int64_t t0 = (int64_t)blockIdx.x * a.window;
  const int page = 1 << a.page_shift, back = (int)min((int64_t)page - 1, t0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int have = (int)min((int64_t)(back + a.window + page - 1), a.T - t0 + back);
  if (threadIdx.x == 0) s_cands = s_ones = s_runs = 0;
  const int planes = 2 * a.n_kv, share = (planes + gridDim.y - 1) / gridDim.y;
  const int p0 = blockIdx.y * share, p1 = min(p0 + share, planes), n_planes = max(p1 - p0, 0);
  for (int i = threadIdx.x; i < have; i += APPEND_THREADS) {
    const int64_t s = a.slots[t0 - back + i];
    const int64_t id = s >> a.page_shift;
    s_page[i] = id < a.n_pages ? (int32_t)max(id, (int64_t)-1) : -1;  // outside the pool: not written
    s_in[i] = (int16_t)(s & (page - 1));
  }
  // the rows are on their way to L2 while the runs are looked for
  if (a.window > 8) {
    constexpr int LINES = D * (int)sizeof(T) / 128;
    const int n = (int)min((int64_t)a.window, a.T - t0);
    for (int i = threadIdx.x; i < n * n_planes; i += APPEND_THREADS) {
      const int y = i / n_planes, pl = p0 + i % n_planes;
      const bool is_v = pl >= a.n_kv;
      const int64_t token = t0 + y, at = is_v ? token * a.v.token_stride + (pl - a.n_kv) * a.v.head_stride
                                             : token * a.k.token_stride + pl * a.k.head_stride;
      const T* p = reinterpret_cast<const T*>(is_v ? a.v.src : a.k.src) + at;
#pragma unroll
      for (int l = 0; l < LINES; ++l) asm volatile("prefetch.global.L2 [%0];" ::"l"(p + l * (128 / (int)sizeof(T))));
    }
  }
  __syncthreads();
  // a run begins where none of the `page - 1` tokens before lies in the same page, and spans the
  // last of the `page - 1` tokens behind that does; s_len: its length, 0x100 where it holds the
  // page's first token, 0x200 where its tokens follow one another without gaps
  // (in a prompt most tokens follow one of their page: only the others are looked at closely)
  if ((int)threadIdx.x < a.window) {
    const int x = back + threadIdx.x;
    if (x < have && s_page[x] >= 0 && (x == 0 || s_page[x - 1] != s_page[x]))
      s_cand[atomicAdd(&s_cands, 1)] = (int16_t)x;
  }
  __syncthreads();
  for (int i = warp; i < s_cands; i += APPEND_WARPS) {
    const int x = s_cand[i], id = s_page[x];
    bool older = false;
    for (int y = x - 2 - lane; y >= max(0, x - page + 1); y -= 32) older |= s_page[y] == id;
    if (__any_sync(0xffffffffu, older)) continue;
    bool fresh = false, dense = true;
    int len = 0;
    for (int y = x + lane; y < min(have, x + page); y += 32)
      if (s_page[y] == id) {
        len = y - x + 1;
        fresh |= s_in[y] == 0;
        dense &= s_in[y] - s_in[x] == y - x && s_page[y - (y > x)] == id;
      }
    len = __reduce_max_sync(0xffffffffu, len);
    fresh = __any_sync(0xffffffffu, fresh);
    dense = __all_sync(0xffffffffu, dense);
    if (lane == 0) {
      if (len == 1) {
        s_one[atomicAdd(&s_ones, 1)] = (int16_t)x;
      } else {
        const int r = atomicAdd(&s_runs, 1);
        s_run[r] = (int16_t)x;
        s_len[r] = (int16_t)(len | (fresh ? 0x100 : 0) | (dense ? 0x200 : 0));
      }
    }
  }
  __syncthreads();
  const int64_t tok0 = t0 - back;

  // ---- runs of one token: D/8 lanes each
  const int per_one = (n_planes + STEP - 1) / STEP, ones = s_ones * per_one;
  for (int w = warp; w < ones; w += APPEND_WARPS) {
    const int x = s_one[w / per_one], pl = p0 + (w % per_one) * STEP + lane / VPT;
    const bool live = pl < p1;
    const bool is_v = pl >= a.n_kv;
    const AppendSide side = is_v ? a.v : a.k;
    const int head = is_v ? pl - a.n_kv : pl;
    const int id = s_page[x], off = s_in[x];
    const int64_t at = (int64_t)id * a.n_kv + head;
    Vec8<T> v;
    uint32_t top = 0;
    float old = 0.f;
    if (live) {
      old = side.scale[at];
      v = load8(reinterpret_cast<const T*>(side.src) + (tok0 + x) * side.token_stride +
                head * side.head_stride + (lane % VPT) * 8);
      top = fold<T>(max8<T>(v, 0));
      if (!finite_bits<T>(top)) top = fold<T>(max8_finite<T>(v, 0));
    }
#pragma unroll
    for (int o = VPT / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float amax = bits_value<T>(top);
    const int e_old = off == 0 ? SCALE_E_MIN : scale_exponent(old);
    const int e = max(e_old, need_exponent(amax));
    uint8_t* bytes = side.cache + (at << a.page_shift) * D;
    uint32_t grown = __ballot_sync(0xffffffffu, live && off != 0 && e > e_old && lane % VPT == 0);
    while (grown) {  // the warp rewrites the pages one after another
      const int from = __ffs(grown) - 1;
      grown &= grown - 1;
      rewrite_page(reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(bytes), from)),
                   (D << a.page_shift) / 16, __shfl_sync(0xffffffffu, e_old - e, from));
    }
    __syncwarp();  // the new bytes lie in the range just rewritten; every lane has read the old scale
    if (live) {
      *reinterpret_cast<uint2*>(bytes + off * D + (lane % VPT) * 8) = quantise8<T>(v, pow2f(-e));
      if (lane % VPT == 0) side.scale[at] = pow2f(e);
    }
  }

  // ---- longer runs: a warp each
  for (int w = warp; w < s_runs * n_planes; w += APPEND_WARPS) {
    const int r = w / n_planes, x0 = s_run[r], n = s_len[r] & 0xff, pl = p0 + w % n_planes;
    const bool fresh = s_len[r] & 0x100, dense = s_len[r] & 0x200;
    const bool is_v = pl >= a.n_kv;
    const AppendSide side = is_v ? a.v : a.k;
    const int head = is_v ? pl - a.n_kv : pl;
    const int id = s_page[x0], first = lane / VPT;
    const int64_t at = (int64_t)id * a.n_kv + head, stride = side.token_stride;
    const T* src = reinterpret_cast<const T*>(side.src) + (tok0 + x0 + first) * stride + head * side.head_stride +
                   (lane % VPT) * 8;
    const float old = side.scale[at];
    uint8_t* bytes = side.cache + (at << a.page_shift) * D;
    uint8_t* dst = bytes + (lane % VPT) * 8;
    // Chunks of KEEP vectors: all of a chunk's loads are under way at once. The last chunk stays in
    // registers for the second pass, which takes the others from L1 or L2 again. A run with gaps
    // or out of order goes token by token.
    constexpr int CHUNK = KEEP * STEP;
    const int chunks = dense ? (n + CHUNK - 1) / CHUNK : 0;
    Vec8<T> keep[KEEP];
    const auto load_chunk = [&](int c) {
      const T* p = src + (int64_t)c * CHUNK * stride;
      const int left = n - first - c * CHUNK;
#pragma unroll
      for (int i = 0; i < KEEP; ++i) {
        if (i * STEP < left) keep[i] = load8(p);
        p += STEP * stride;
      }
      return left;
    };
    const auto sparse = [&](auto&& f) {
      for (int y = first; !dense && y < n; y += STEP)
        if (s_page[x0 + y] == id) f(load8(src + (y - first) * stride), s_in[x0 + y]);
    };
    uint32_t top = 0;
    for (int c = 0; c < chunks; ++c) {
      const int left = load_chunk(c);
#pragma unroll
      for (int i = 0; i < KEEP; ++i)
        if (i * STEP < left) top = max8<T>(keep[i], top);
    }
    sparse([&](const Vec8<T>& v, int) { top = max8<T>(v, top); });
    top = __reduce_max_sync(0xffffffffu, fold<T>(top));
    if (!finite_bits<T>(top)) {
      uint32_t m = 0;
      for (int y = first; y < n; y += STEP)
        if (s_page[x0 + y] == id) m = max8_finite<T>(load8(src + (y - first) * stride), m);
      top = __reduce_max_sync(0xffffffffu, fold<T>(m));
    }
    const int e_old = fresh ? SCALE_E_MIN : scale_exponent(old);
    const int e = max(e_old, need_exponent(bits_value<T>(top)));
    if (!fresh && e > e_old) rewrite_page(bytes, (D << a.page_shift) / 16, e_old - e);
    __syncwarp();  // as above
    const float inv = pow2f(-e);
    uint8_t* out = dst + (s_in[x0] + first) * D;
    for (int c = chunks - 1; c >= 0; --c) {
      const int left = c == chunks - 1 ? n - first - c * CHUNK : load_chunk(c);
#pragma unroll
      for (int i = 0; i < KEEP; ++i)
        if (i * STEP < left) *reinterpret_cast<uint2*>(out + (c * CHUNK + i * STEP) * D) = quantise8<T>(keep[i], inv);
    }
    sparse([&](const Vec8<T>& v, int off) { *reinterpret_cast<uint2*>(dst + off * D) = quantise8<T>(v, inv); });
    if (lane == 0) side.scale[at] = pow2f(e);
  }
}

}  // namespace dsalt

using namespace dsalt;

extern "C" int dsalt_append_cache(const void* k, const void* v, int dtype, int64_t T, int n_kv, int head_dim,
                                  int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                                  int64_t v_head_stride, void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                                  int64_t n_pages, int page_size, const int64_t* slots, void* stream) {
  if (T < 0 || n_kv < 1 || n_pages < 0) return fail(DSALT_ERR_INVALID, "append_cache: bad sizes");
  if (dtype != DSALT_F32 && dtype != DSALT_BF16 && dtype != DSALT_F16)
    return fail(DSALT_ERR_INVALID, "append_cache: dtype");
  if (head_dim != 64 && head_dim != 128)
    return fail(DSALT_ERR_UNSUPPORTED, "append_cache: head_dim %d not in {64, 128}", head_dim);
  if (page_size != 16 && page_size != 32 && page_size != 64 && page_size != 128)
    return fail(DSALT_ERR_UNSUPPORTED, "append_cache: page size %d not in {16, 32, 64, 128}", page_size);
  if (n_kv > 65535 || T > 0x7fffff00LL || n_pages > 0x7fffff00LL) return fail(DSALT_ERR_UNSUPPORTED, "append_cache: too many heads, tokens or pages");
  if (T == 0) return DSALT_OK;
  if (!k || !v || !k_cache || !v_cache || !k_scale || !v_scale || !slots)
    return fail(DSALT_ERR_INVALID, "append_cache: null pointer");
  const int64_t es = dtype == DSALT_F32 ? 4 : 2;
  if ((((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) ||
      ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) * es) % 16)
    return fail(DSALT_ERR_INVALID, "append_cache: rows must be 16-byte aligned");
  AppendArgs a;
  a.k = {k, reinterpret_cast<uint8_t*>(k_cache), k_scale, k_token_stride, k_head_stride};
  a.v = {v, reinterpret_cast<uint8_t*>(v_cache), v_scale, v_token_stride, v_head_stride};
  a.slots = slots, a.T = T, a.n_pages = n_pages, a.n_kv = n_kv;
  a.page_shift = page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : 7;
  // few tokens: small windows, so that a decode step's runs spread over the GPU (512 rows of 12 heads
  // 4.6 us, in windows of 64 13.2); many: larger ones, so that fewer blocks find no run (4096
  // tokens of a prompt 6.2 us, in windows of 8 9.7). Planes are shared out until there are blocks enough
  // (or each has no more planes than warps).
  a.window = T <= 2048 ? 8 : page_size >= 64 ? 64 : 32;
  const int64_t windows = (T + a.window - 1) / a.window;
  const int planes = 2 * n_kv, most = a.window == 8 ? (planes + 256 / head_dim - 1) / (256 / head_dim) : planes;
  const int64_t shares = std::min<int64_t>(most, std::max<int64_t>((148 * 2 + windows - 1) / windows, (planes + 7) / 8));
  const dim3 grid((unsigned)windows, (unsigned)shares);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
#define DSALT_APPEND(TT)                                                                    \
  (head_dim == 64 ? append_cache_kernel<TT, 64><<<grid, APPEND_THREADS, 0, s>>>(a)         \
                  : append_cache_kernel<TT, 128><<<grid, APPEND_THREADS, 0, s>>>(a))
  if (dtype == DSALT_F32) DSALT_APPEND(float);
  else if (dtype == DSALT_F16) DSALT_APPEND(__half);
  else DSALT_APPEND(__nv_bfloat16);
#undef DSALT_APPEND
  return check_cuda(cudaGetLastError(), "append_cache launch");
}
