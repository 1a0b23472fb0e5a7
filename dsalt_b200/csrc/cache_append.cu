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
// the first of them. One group of threads owns a run of one head: it takes amax, settles e,
// rewrites the older bytes if e grew and writes the new ones, so nothing is exchanged between
// groups. A decode step is all runs of one token (a warp each), a prompt is runs of P
// tokens (a block each).
#include <type_traits>

#include "common.cuh"

namespace dsalt {

constexpr int APPEND_THREADS = 256;
constexpr int APPEND_MAX_WINDOW = 64;  // tokens whose runs one block looks for
constexpr int APPEND_MAX_PAGE = 128;
constexpr int SCALE_E_MIN = -110;  // 2^-110 times the smallest byte is still a normal fp32

struct AppendArgs {
  const void* src[2];  // k, v
  uint8_t* cache[2];
  float* scale[2];
  int64_t token_stride[2], head_stride[2];
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
template <typename T>
__device__ __forceinline__ float amax8(const Vec8<T>& v, float amax) {
  float x[8];
  widen8<T>(v, x);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float m = fabsf(x[j]);
    amax = m < INFINITY ? fmaxf(amax, m) : amax;  // false for NaN as well
  }
  return amax;
}

// One run of one head by the threads of a warp (BLOCK = false) or of the block: n tokens of
// the call from `tok` on, those whose slot lies in page `id`; s_off: their offsets in the page,
// -1 for the others.
template <typename T, int D, bool BLOCK>
__device__ __forceinline__ void append_run(const AppendArgs& a, int which, int head, int64_t tok, int n, int id,
                                           bool fresh, const int16_t* s_off, float* s_red) {
  constexpr int N = BLOCK ? APPEND_THREADS : 32;
  constexpr int VPT = D / 8;  // vectors per token
  constexpr int KEEP = sizeof(T) == 4 ? 2 : 4;
  const int me = BLOCK ? (int)threadIdx.x : (int)(threadIdx.x & 31);
  const int64_t stride = a.token_stride[which];
  // N is a multiple of VPT: a thread keeps its place within the rows and steps by whole tokens
  const T* src = reinterpret_cast<const T*>(a.src[which]) + tok * stride + head * a.head_stride[which] + (me % VPT) * 8;
  const int64_t at = (int64_t)id * a.n_kv + head;
  uint8_t* page_bytes = a.cache[which] + (at << a.page_shift) * D;
  float* scale = a.scale[which] + at;
  const float old_scale = *scale;
  constexpr int STEP = N / VPT;  // tokens per step
  const int first = me / VPT;
  // the first KEEP of a thread's vectors stay in registers between the passes
  Vec8<T> keep[KEEP];
  int off[KEEP];
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const int x = first + i * STEP;
    off[i] = x < n ? s_off[x] : -1;
    if (off[i] >= 0) keep[i] = load8(src + x * stride);
  }
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if (off[i] >= 0) amax = amax8<T>(keep[i], amax);
  for (int x = first + KEEP * STEP; x < n; x += STEP)
    if (s_off[x] >= 0) amax = amax8<T>(load8(src + x * stride), amax);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (BLOCK) {
    if ((threadIdx.x & 31) == 0) s_red[threadIdx.x >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < APPEND_THREADS / 32; ++w) amax = fmaxf(amax, s_red[w]);
  }
  const int e_old = fresh ? SCALE_E_MIN : scale_exponent(old_scale);
  const int e = max(e_old, need_exponent(amax));
  if (!fresh && e > e_old) {
    const float f = e_old - e < -126 ? 0.f : pow2f(e_old - e);
    uint4* p = reinterpret_cast<uint4*>(page_bytes);
    for (int i = me; i < (D << a.page_shift) / 16; i += N) {
      uint4 v = p[i];
      v.x = rescale_e4m3x4(v.x, f);
      v.y = rescale_e4m3x4(v.y, f);
      v.z = rescale_e4m3x4(v.z, f);
      v.w = rescale_e4m3x4(v.w, f);
      p[i] = v;
    }
    // the new tokens' bytes lie in the range just rewritten, by other threads
    if (BLOCK) __syncthreads();
    else __syncwarp();
  }
  const float inv = pow2f(-e);
  uint8_t* dst = page_bytes + (me % VPT) * 8;
  auto put = [&](int o, const Vec8<T>& v) {
    float x[8];
    widen8<T>(v, x);
    uint2 b;
    b.x = to_e4m3x4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    b.y = to_e4m3x4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv);
    *reinterpret_cast<uint2*>(dst + o * D) = b;
  };
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
    if (off[i] >= 0) put(off[i], keep[i]);
  for (int x = first + KEEP * STEP; x < n; x += STEP)
    if (s_off[x] >= 0) put(s_off[x], load8(src + x * stride));
  __syncwarp();  // every lane has read the old scale
  if (me == 0) *scale = pow2f(e);
}

// grid: (window of tokens, kv head, k | v)
template <typename T, int D>
__global__ void __launch_bounds__(APPEND_THREADS) append_cache_kernel(AppendArgs a) {
  __shared__ int32_t s_page[APPEND_MAX_WINDOW + 2 * APPEND_MAX_PAGE];  // page of each token near the window, -1: none
  __shared__ int16_t s_in[APPEND_MAX_WINDOW + 2 * APPEND_MAX_PAGE];    // its offset in the page
  __shared__ int16_t s_off[APPEND_THREADS / 32][APPEND_MAX_PAGE];      // per warp: offsets of a run's tokens
  __shared__ int16_t s_len[APPEND_MAX_WINDOW];  // tokens that a run spans (0: none begins here), negative: afresh
  __shared__ float s_red[APPEND_THREADS / 32];
  const int64_t t0 = (int64_t)blockIdx.x * a.window;
  const int page = 1 << a.page_shift, back = (int)min((int64_t)page - 1, t0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int have = (int)min((int64_t)(back + a.window + page - 1), a.T - t0 + back);
  for (int i = threadIdx.x; i < have; i += APPEND_THREADS) {
    const int64_t s = a.slots[t0 - back + i];
    const int64_t id = s >> a.page_shift;
    s_page[i] = id < a.n_pages ? (int32_t)max(id, (int64_t)-1) : -1;  // outside the pool: not written
    s_in[i] = (int16_t)(s & (page - 1));
  }
  __syncthreads();
  // a run begins where none of the `page - 1` tokens before lies in the same page, and spans the
  // last of the `page - 1` tokens behind that does
  for (int i = warp; i < a.window; i += APPEND_THREADS / 32) {
    const int x = back + i;
    int len = 0;
    if (x < have && s_page[x] >= 0) {
      const int id = s_page[x];
      bool older = false;
      for (int y = x - 1 - lane; !__any_sync(0xffffffffu, older) && __any_sync(0xffffffffu, y >= max(0, x - page + 1)); y -= 32)
        older = y >= max(0, x - page + 1) && s_page[y] == id;
      if (!__any_sync(0xffffffffu, older)) {
        bool fresh = false;
        for (int y = x + lane; __any_sync(0xffffffffu, y < min(have, x + page)); y += 32) {
          const bool mine = y < min(have, x + page) && s_page[y] == id;
          fresh |= mine && s_in[y] == 0;
          if (mine) len = y - x + 1;
        }
        len = __reduce_max_sync(0xffffffffu, len);
        if (__any_sync(0xffffffffu, fresh)) len = -len;
      }
    }
    if (lane == 0) s_len[i] = (int16_t)len;
  }
  __syncthreads();
  const int head = blockIdx.y, which = blockIdx.z;
  // up to what a warp keeps in registers: a warp each; longer ones: the block, one after another
  constexpr int SHORT = 32 * (sizeof(T) == 4 ? 2 : 4) * 8 / D;
  for (int i = warp; i < a.window; i += APPEND_THREADS / 32) {
    const int n = abs(s_len[i]);
    if (n == 0 || n > SHORT) continue;
    const int x = back + i, id = s_page[x];
    __syncwarp();
    if (lane < n) s_off[warp][lane] = s_page[x + lane] == id ? s_in[x + lane] : -1;
    __syncwarp();
    append_run<T, D, false>(a, which, head, t0 + i, n, id, s_len[i] < 0, s_off[warp], s_red);
  }
  for (int i = 0; i < a.window; ++i) {
    const int n = abs(s_len[i]);
    if (n <= SHORT) continue;
    const int x = back + i, id = s_page[x];
    __syncthreads();  // s_off and s_red are used again
    for (int y = threadIdx.x; y < n; y += APPEND_THREADS) s_off[0][y] = s_page[x + y] == id ? s_in[x + y] : -1;
    __syncthreads();
    append_run<T, D, true>(a, which, head, t0 + i, n, id, s_len[i] < 0, s_off[0], s_red);
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
  a.src[0] = k, a.src[1] = v;
  a.cache[0] = reinterpret_cast<uint8_t*>(k_cache), a.cache[1] = reinterpret_cast<uint8_t*>(v_cache);
  a.scale[0] = k_scale, a.scale[1] = v_scale;
  a.token_stride[0] = k_token_stride, a.token_stride[1] = v_token_stride;
  a.head_stride[0] = k_head_stride, a.head_stride[1] = v_head_stride;
  a.slots = slots, a.T = T, a.n_pages = n_pages, a.n_kv = n_kv;
  a.page_shift = page_size == 16 ? 4 : page_size == 32 ? 5 : page_size == 64 ? 6 : 7;
  // few tokens: windows of a warp per token, so that a decode step fills the GPU; many: windows
  // of 64, so that a prompt's blocks find about one run each
  a.window = (T + 7) / 8 * n_kv * 2 <= 148 * 16 ? 8 : APPEND_MAX_WINDOW;
  const dim3 grid((unsigned)((T + a.window - 1) / a.window), (unsigned)n_kv, 2);
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
