// Activations in 8 bits (dsalt_pack8, dsalt_unpack8): GROUP8 = 32 neighbouring values of a row share
// a power-of-two scale 2^(s - 127), kept as the byte s, and are held as whole numbers of -127..127.
//
//   E = exponent field of the group's largest magnitude (fp32), s = max(E - 6, 1)
//   code = clamp(rint(x * 2^(127 - s)), -127, 127),  value = code * 2^(s - 127)
//
// The largest magnitude lies in [64, 128) steps, so a value is off by half a step at most (2^-7 of
// the group's largest), or by a whole one where it is above 127 steps. The product with a power
// of two is exact: codes are the same on every path that computes them from the same 32-bit values.
// A value is at most 127/128 of the power of two above the group's largest, which every type that
// holds the largest holds too: unpacking cannot overflow. A group
// with a NaN or an infinity gets s = 255 and reads as NaN as a whole. Two groups of 32 instead of
// one of 64 or 128: 3 % more bytes for a step that is 1.2 to 1.4 times finer on normal data.
//
// Bound by memory: a thread takes 32 bytes of a row, the lanes of a group share its maximum by
// shuffles. Rows that 32-byte accesses do not fit take a lane per value.
// 32768 x 2048 in bf16: to codes 38 us, back 30, together 5.9 TB/s of the bytes they have to move.
#include "pack8.cuh"

namespace dsalt {
namespace {

constexpr int THREADS = 256;
constexpr int64_t MAX_CHUNKS = 1ll << 31;  // of a launch: 64 GB and more

__device__ __forceinline__ void ld32(uint32_t (&u)[8], const void* p) {
  asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
               : "l"(__cvta_generic_to_global(p)));
}
__device__ __forceinline__ void st32(void* p, const uint32_t (&u)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(__cvta_generic_to_global(p)), "r"(u[0]),
               "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
               : "memory");
}

template <typename T>
__device__ __forceinline__ void widen(const uint32_t (&u)[8], float (&f)[32 / sizeof(T)]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(u[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) widen2<T>(u[i], f[2 * i], f[2 * i + 1]);
  }
}

// rows of n values in chunks of 32 bytes, a chunk per thread; a row's chunk count is rounded up
// to whole groups, so that the lanes of a group are neighbours in a warp. Chunks are counted in 32 bits, whose
// division is a few instructions; the host calls for as many rows as that allows
template <typename T>
__global__ void __launch_bounds__(THREADS) pack_rows_kernel(const T* __restrict__ x, uint32_t rows, int n,
                                                            int64_t x_stride, int8_t* __restrict__ codes,
                                                            uint8_t* __restrict__ exps, int groups) {
  constexpr int N = 32 / (int)sizeof(T), LANES = GROUP8 / N;
  const uint32_t chunks = groups * LANES, total = rows * chunks;
  for (uint32_t i = blockIdx.x * THREADS + threadIdx.x; i - threadIdx.x % 32 < total; i += gridDim.x * THREADS) {
    const bool in = i < total;
    const uint32_t at_row = in ? i / chunks : 0;
    const int64_t row = at_row;
    const int chunk = in ? (int)(i - at_row * chunks) : 0, col = chunk * N;
    const bool held = in && col < n;
    uint32_t u[8] = {};
    if (held) ld32(u, x + row * x_stride + col);
    float f[N];
    widen<T>(u, f);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    const uint32_t s = scale_byte(top);
    uint32_t w[N / 4];
    pack_codes<N>(f, s, w);
    if (held) {
      int8_t* at = codes + row * n + col;
      if constexpr (N == 16) *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
      else *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
      if (chunk % LANES == 0) exps[row * groups + chunk / LANES] = (uint8_t)s;
    }
  }
}

// a lane per value, a warp per group
template <typename T>
__global__ void __launch_bounds__(THREADS) pack_any_kernel(const T* __restrict__ x, int64_t rows, int n,
                                                           int64_t x_stride, int8_t* __restrict__ codes,
                                                           uint8_t* __restrict__ exps, int groups) {
  const int lane = threadIdx.x % 32;
  const int64_t total = rows * groups;
  for (int64_t i = ((int64_t)blockIdx.x * THREADS + threadIdx.x) / 32; i < total;
       i += (int64_t)gridDim.x * (THREADS / 32)) {
    const int64_t row = i / groups;
    const int col = (int)(i - row * groups) * GROUP8 + lane;
    float f[1] = {col < n ? to_float(x[row * x_stride + col]) : 0.f};
    const uint32_t s = scale_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(f[0]) & 0x7fffffffu));
    if (col < n) codes[row * n + col] = (int8_t)code_of(f[0], s);
    if (lane == 0) exps[i] = (uint8_t)s;
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) unpack_rows_kernel(const int8_t* __restrict__ codes,
                                                              const uint8_t* __restrict__ exps, uint32_t rows, int n,
                                                              int groups, T* __restrict__ out) {
  constexpr int N = 32 / (int)sizeof(T);
  const uint32_t chunks = n / N, total = rows * chunks;
  for (uint32_t i = blockIdx.x * THREADS + threadIdx.x; i < total; i += gridDim.x * THREADS) {
    const uint32_t at_row = i / chunks;
    const int64_t row = at_row;
    const int col = (int)(i - at_row * chunks) * N;
    const float scale = scale_of(exps[row * groups + col / GROUP8]);
    uint32_t w[N / 4];
    if constexpr (N == 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(codes + row * n + col);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
      const uint2 v = *reinterpret_cast<const uint2*>(codes + row * n + col);
      w[0] = v.x, w[1] = v.y;
    }
    float f[N];
    unpack_codes<N>(w, scale, f);
    uint32_t u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (sizeof(T) == 4) u[j] = __float_as_uint(f[j]);
      else u[j] = narrow2<T>(f[2 * j], f[2 * j + 1]);
    }
    st32(out + row * n + col, u);
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) unpack_any_kernel(const int8_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ exps, int64_t rows, int n,
                                                             int groups, T* __restrict__ out) {
  const int64_t total = rows * n;
  for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < total; i += (int64_t)gridDim.x * THREADS) {
    const int64_t row = i / n;
    const int col = (int)(i - row * n);
    out[i] = from_float<T>((float)codes[i] * scale_of(exps[row * groups + col / GROUP8]));
  }
}

int blocks_for(int64_t threads) {
  const int64_t b = (threads + THREADS - 1) / THREADS;
  return (int)(b < 148 * 8 * 4 ? b : 148 * 8 * 4);  // 8 blocks an SM, four rounds
}

bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

template <typename T>
int pack(const T* x, int64_t rows, int n, int64_t x_stride, int8_t* codes, uint8_t* exps, cudaStream_t stream) {
  constexpr int N = 32 / (int)sizeof(T);
  const int groups = (n + GROUP8 - 1) / GROUP8;
  if (n % N || x_stride % N || !aligned(x, 32) || !aligned(codes, 16)) {
    pack_any_kernel<T><<<blocks_for(rows * groups * 32), THREADS, 0, stream>>>(x, rows, n, x_stride, codes, exps, groups);
    return check_cuda(cudaGetLastError(), "pack8 launch");
  }
  const int64_t most = MAX_CHUNKS / (groups * (GROUP8 / N));
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t part = rows - r < most ? rows - r : most;
    pack_rows_kernel<T><<<blocks_for(part * groups * (GROUP8 / N)), THREADS, 0, stream>>>(
        x + r * x_stride, (uint32_t)part, n, x_stride, codes + r * n, exps + r * groups, groups);
    if (int rc = check_cuda(cudaGetLastError(), "pack8 launch")) return rc;
  }
  return DSALT_OK;
}

template <typename T>
int unpack(const int8_t* codes, const uint8_t* exps, int64_t rows, int n, T* out, cudaStream_t stream) {
  constexpr int N = 32 / (int)sizeof(T);
  const int groups = (n + GROUP8 - 1) / GROUP8;
  if (n % N || !aligned(out, 32) || !aligned(codes, 16)) {
    unpack_any_kernel<T><<<blocks_for(rows * n), THREADS, 0, stream>>>(codes, exps, rows, n, groups, out);
    return check_cuda(cudaGetLastError(), "unpack8 launch");
  }
  const int64_t most = MAX_CHUNKS / (n / N);
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t part = rows - r < most ? rows - r : most;
    unpack_rows_kernel<T><<<blocks_for(part * (n / N)), THREADS, 0, stream>>>(codes + r * n, exps + r * groups, (uint32_t)part,
                                                                              n, groups, out + r * n);
    if (int rc = check_cuda(cudaGetLastError(), "unpack8 launch")) return rc;
  }
  return DSALT_OK;
}

int check_sizes(const char* fn, int dtype, int64_t rows, int64_t cols) {
  if (dtype != DSALT_F32 && dtype != DSALT_BF16 && dtype != DSALT_F16) return fail(DSALT_ERR_INVALID, "%s: bad dtype %d", fn, dtype);
  if (rows < 0 || cols < 0) return fail(DSALT_ERR_INVALID, "%s: bad sizes (%lld rows, %lld columns)", fn, (long long)rows, (long long)cols);
  if (cols > (1 << 30)) return fail(DSALT_ERR_UNSUPPORTED, "%s: rows of more than 2^30 values", fn);
  return DSALT_OK;
}

}  // namespace

int launch_pack8(const void* x, int dtype, int64_t rows, int64_t cols, int64_t x_stride, int8_t* codes, uint8_t* exps,
                 cudaStream_t stream) {
  if (dtype == DSALT_F32) return pack(static_cast<const float*>(x), rows, (int)cols, x_stride, codes, exps, stream);
  if (dtype == DSALT_BF16) return pack(static_cast<const __nv_bfloat16*>(x), rows, (int)cols, x_stride, codes, exps, stream);
  return pack(static_cast<const __half*>(x), rows, (int)cols, x_stride, codes, exps, stream);
}

int launch_unpack8(const int8_t* codes, const uint8_t* exps, int64_t rows, int64_t cols, void* out, int dtype,
                   cudaStream_t stream) {
  if (dtype == DSALT_F32) return unpack(codes, exps, rows, (int)cols, static_cast<float*>(out), stream);
  if (dtype == DSALT_BF16) return unpack(codes, exps, rows, (int)cols, static_cast<__nv_bfloat16*>(out), stream);
  return unpack(codes, exps, rows, (int)cols, static_cast<__half*>(out), stream);
}

}  // namespace dsalt

using namespace dsalt;

extern "C" {

int dsalt_pack8(const void* x, int dtype, int64_t rows, int64_t cols, int64_t x_stride, int8_t* codes, uint8_t* exps,
                void* stream) {
  if (int rc = check_sizes("pack8", dtype, rows, cols)) return rc;
  if (rows > 1 && x_stride < cols) return fail(DSALT_ERR_INVALID, "pack8: rows overlap");
  if (rows == 0 || cols == 0) return DSALT_OK;
  if (!x || !codes || !exps) return fail(DSALT_ERR_INVALID, "pack8: null pointer");
  return launch_pack8(x, dtype, rows, cols, x_stride, codes, exps, static_cast<cudaStream_t>(stream));
}

int dsalt_unpack8(const int8_t* codes, const uint8_t* exps, int64_t rows, int64_t cols, void* out, int dtype,
                  void* stream) {
  if (int rc = check_sizes("unpack8", dtype, rows, cols)) return rc;
  if (rows == 0 || cols == 0) return DSALT_OK;
  if (!codes || !exps || !out) return fail(DSALT_ERR_INVALID, "unpack8: null pointer");
  return launch_unpack8(codes, exps, rows, cols, out, dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
