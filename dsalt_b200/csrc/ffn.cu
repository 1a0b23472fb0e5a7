// The gated feed-forward block y = (act(x Wg^T) * (x Wu^T)) Wd^T and its gradients
// (dsalt_gated_ffn, dsalt_gated_ffn_bwd): arguments, workspaces, and the path for what the tensor
// cores do not take: fp32 inputs, and sizes that are not multiples of 8. That path is plain: products on the
// CUDA cores in fp32 (128 x 128 tiles, 8 x 8 outputs a thread), the activation and its gradient as kernels of their
// own between them.
#include "ffn.cuh"

namespace dsalt {
namespace ffn {
namespace {

constexpr int BM = 128, BN = 128, BK = 16, THREADS = 256;

// C[m, n] = sum over both segments and k of A(m, k) B(n, k), in fp32
struct Operand {
  const void* p;
  int64_t row, k;  // strides in elements
};
struct Product {
  Operand a[2], b[2];
  int segments;
  int64_t M;
  int N;
  int64_t K;
  int64_t c_stride;
};

template <typename T>
__device__ __forceinline__ void load_tile(float (&s)[BK][BM + 4], const Operand& o, int64_t row0, int64_t rows, int64_t k0,
                                          int64_t K) {
  const T* p = static_cast<const T*>(o.p);
  const bool along_k = o.k == 1;
#pragma unroll
  for (int i = 0; i < BM * BK / THREADS; ++i) {
    const int e = i * THREADS + threadIdx.x;
    const int r = along_k ? e / BK : e % BM, k = along_k ? e % BK : e / BM;
    const bool in = row0 + r < rows && k0 + k < K;
    s[k][r] = in ? to_float(p[(row0 + r) * o.row + (k0 + k) * o.k]) : 0.f;
  }
}

template <typename T, typename TO>
__global__ void __launch_bounds__(THREADS) product_kernel(const Product p, TO* __restrict__ c) {
  __shared__ __align__(16) float as[BK][BM + 4], bs[BK][BN + 4];
  const int64_t m0 = (int64_t)blockIdx.y * BM;
  const int64_t n0 = (int64_t)blockIdx.x * BN;
  const int tm = threadIdx.x / 16 * 8, tn = threadIdx.x % 16 * 8;
  float acc[8][8] = {};
  for (int seg = 0; seg < p.segments; ++seg)
    for (int64_t k0 = 0; k0 < p.K; k0 += BK) {
      load_tile<T>(as, p.a[seg], m0, p.M, k0, p.K);
      load_tile<T>(bs, p.b[seg], n0, p.N, k0, p.K);
      __syncthreads();
#pragma unroll
      for (int k = 0; k < BK; ++k) {
        float a[8], b[8];
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          *reinterpret_cast<float4*>(a + i) = *reinterpret_cast<const float4*>(&as[k][tm + i]);
          *reinterpret_cast<float4*>(b + i) = *reinterpret_cast<const float4*>(&bs[k][tn + i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
      }
      __syncthreads();
    }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (m0 + tm + i < p.M && n0 + tn + j < p.N) c[(m0 + tm + i) * p.c_stride + n0 + tn + j] = from_float<TO>(acc[i][j]);
}

// a warp per 32 columns of a row: h and what is kept (of fp32: g and u lie there already, but for the columns behind F)
template <typename T, int ACT>
__global__ void __launch_bounds__(THREADS) act_kernel(const float* g, const float* u, int64_t T_,
                                                      int F, int64_t pitch, T* __restrict__ h, void* kept,
                                                      uint8_t* __restrict__ exps, int keep) {
  const int lane = threadIdx.x % 32;
  const int64_t groups = pitch / GROUP8, total = T_ * groups, plane = T_ * pitch;
  for (int64_t i = ((int64_t)blockIdx.x * THREADS + threadIdx.x) / 32; i < total;
       i += (int64_t)gridDim.x * (THREADS / 32)) {
    const int64_t at = i * GROUP8 + lane;
    const bool in = at % pitch < F;
    const float a = in ? g[at] : 0.f, b = in ? u[at] : 0.f;
    h[at] = from_float<T>(activate<ACT, false>(a) * b);
    if (sizeof(T) == 4 && keep == DSALT_KEEP_INPUT) {
      if (!in) static_cast<float*>(kept)[at] = static_cast<float*>(kept)[plane + at] = 0.f;
    } else if (keep == DSALT_KEEP_INPUT) {
      uint16_t* to = static_cast<uint16_t*>(kept) + at;
      to[0] = (uint16_t)upper_halves(a, 0.f);
      to[plane] = (uint16_t)upper_halves(b, 0.f);
      to[2 * plane] = (uint16_t)third_bytes(a, b);
    } else if (keep == DSALT_KEEP_8BIT) {
      const uint32_t sa = scale_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(a) & 0x7fffffffu));
      const uint32_t sb = scale_byte(__reduce_max_sync(0xffffffffu, __float_as_uint(b) & 0x7fffffffu));
      static_cast<int8_t*>(kept)[at] = (int8_t)code_of(a, sa);
      static_cast<int8_t*>(kept)[plane + at] = (int8_t)code_of(b, sb);
      if (lane == 0) {
        exps[i % groups * T_ + i / groups] = (uint8_t)sa;
        exps[(groups + i % groups) * T_ + i / groups] = (uint8_t)sb;
      }
    }
  }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(THREADS) act_grad_kernel(const float* __restrict__ dh, int64_t T_, int F, int64_t pitch,
                                                           const void* kept, const uint8_t* __restrict__ exps, int keep,
                                                           T* __restrict__ h,  // nullable: it was kept
                                                           T* __restrict__ dg, T* __restrict__ du) {
  const int64_t total = T_ * pitch;
  for (int64_t at = (int64_t)blockIdx.x * THREADS + threadIdx.x; at < total; at += (int64_t)gridDim.x * THREADS) {
    float a, b;
    if (sizeof(T) == 4 && keep == DSALT_KEEP_INPUT) {
      a = static_cast<const float*>(kept)[at];
      b = static_cast<const float*>(kept)[total + at];
    } else if (keep == DSALT_KEEP_INPUT) {
      const uint16_t* w = static_cast<const uint16_t*>(kept) + at;
      a = held24<0>(w[0], w[2 * total]).x;
      b = held24<1>(w[total], w[2 * total]).x;
    } else {
      const int8_t* c = static_cast<const int8_t*>(kept);
      const int64_t scale = at % pitch / GROUP8 * T_ + at / pitch;
      a = (float)c[at] * scale_of(exps[scale]);
      b = (float)c[total + at] * scale_of(exps[pitch / GROUP8 * T_ + scale]);
    }
    const float d = at % pitch < F ? dh[at] : 0.f;
    float v, dv;
    activate_grad<ACT, false>(a, v, dv);
    if (h) h[at] = from_float<T>(v * b);
    dg[at] = from_float<T>(d * b * dv);
    du[at] = from_float<T>(d * v);
  }
}

template <typename T, typename TO>
int product(const Product& p, TO* c, cudaStream_t stream, const char* what) {
  const int64_t rows = (p.M + BM - 1) / BM;
  // grid.y holds 65535 row tiles; longer products go in parts
  for (int64_t r = 0; r < rows; r += 65535) {
    Product q = p;
    const int64_t skip = r * BM;
    for (int s = 0; s < p.segments; ++s) q.a[s].p = static_cast<const T*>(p.a[s].p) + skip * p.a[s].row;
    q.M = p.M - skip;
    const int64_t n = rows - r < 65535 ? rows - r : 65535;
    product_kernel<T, TO><<<dim3((p.N + BN - 1) / BN, (unsigned)n), THREADS, 0, stream>>>(q, c + skip * p.c_stride);
    if (int rc = check_cuda(cudaGetLastError(), what)) return rc;
  }
  return DSALT_OK;
}

int blocks_for(int64_t threads) {
  const int64_t b = (threads + THREADS - 1) / THREADS;
  return (int)(b < 148 * 32 ? b : 148 * 32);
}

// whether the product of gate and up, the last product's operand, is kept, or formed again by the backward pass
bool keeps_h(int dtype, int keep) { return dtype == DSALT_F32 && keep == DSALT_KEEP_INPUT; }

template <typename T, int ACT>
int forward_plain(const Ffn& f) {
  // of fp32 inputs that keep their activations the sums are formed where they are kept
  float* g = keeps_h(f.dtype, f.keep) ? static_cast<float*>(f.kept) : f.wide;
  float* u = g + f.T * f.pitch;
  int rc;
  for (int i = 0; i < 2; ++i) {
    const Product p = {{{f.x, f.x_stride, 1}}, {{i ? f.w_up : f.w_gate, f.d, 1}}, 1, f.T, f.F, f.d, f.pitch};
    if ((rc = product<T, float>(p, i ? u : g, f.stream, "gated_ffn product launch"))) return rc;
  }
  act_kernel<T, ACT><<<blocks_for(f.T * f.pitch), THREADS, 0, f.stream>>>(g, u, f.T, f.F, f.pitch, static_cast<T*>(f.h),
                                                                         f.kept, f.exps, f.keep);
  if ((rc = check_cuda(cudaGetLastError(), "gated_ffn activation launch"))) return rc;
  const Product p = {{{f.h, f.pitch, 1}}, {{f.w_down, f.F, 1}}, 1, f.T, f.d_out, f.F, f.d_out};
  return product<T, T>(p, static_cast<T*>(f.y), f.stream, "gated_ffn product launch");
}

template <typename T, int ACT>
int backward_plain(const Ffn& f) {
  int rc;
  const Product dh = {{{f.dy, f.dy_stride, 1}}, {{f.w_down, 1, f.F}}, 1, f.T, f.F, f.d_out, f.pitch};
  if ((rc = product<T, float>(dh, f.wide, f.stream, "gated_ffn_bwd product launch"))) return rc;
  act_grad_kernel<T, ACT><<<blocks_for(f.T * f.pitch), THREADS, 0, f.stream>>>(
      f.wide, f.T, f.F, f.pitch, f.kept, f.exps, f.keep, keeps_h(f.dtype, f.keep) ? nullptr : static_cast<T*>(f.h),
      static_cast<T*>(f.dg), static_cast<T*>(f.du));
  if ((rc = check_cuda(cudaGetLastError(), "gated_ffn_bwd activation launch"))) return rc;
  if (f.dx) {
    const Product p = {{{f.dg, f.pitch, 1}, {f.du, f.pitch, 1}}, {{f.w_gate, 1, f.d}, {f.w_up, 1, f.d}}, 2, f.T, f.d, f.F, f.d};
    if ((rc = product<T, T>(p, static_cast<T*>(f.dx), f.stream, "gated_ffn_bwd product launch"))) return rc;
  }
  if (f.dw_gate)
    for (int i = 0; i < 2; ++i) {
      const Product p = {{{i ? f.du : f.dg, 1, f.pitch}}, {{f.x, 1, f.x_stride}}, 1, f.F, f.d, f.T, f.d};
      if ((rc = product<T, T>(p, static_cast<T*>(i ? f.dw_up : f.dw_gate), f.stream, "gated_ffn_bwd product launch"))) return rc;
    }
  if (f.dw_down) {
    const Product p = {{{f.dy, 1, f.dy_stride}}, {{f.h, 1, f.pitch}}, 1, f.d_out, f.F, f.T, f.F};
    if ((rc = product<T, T>(p, static_cast<T*>(f.dw_down), f.stream, "gated_ffn_bwd product launch"))) return rc;
  }
  return DSALT_OK;
}

template <typename T>
int run_plain(const Ffn& f, bool backward) {
  if (f.act == DSALT_ACT_SILU) return backward ? backward_plain<T, DSALT_ACT_SILU>(f) : forward_plain<T, DSALT_ACT_SILU>(f);
  return backward ? backward_plain<T, DSALT_ACT_GELU>(f) : forward_plain<T, DSALT_ACT_GELU>(f);
}

bool tensor_cores(int dtype, int d, int F, int d_out);

int run(const Ffn& f, bool backward) {
  if (tensor_cores(f.dtype, f.d, f.F, f.d_out)) return run_tensor_cores(f, backward);
  if (f.dtype == DSALT_F32) return run_plain<float>(f, backward);
  if (f.dtype == DSALT_BF16) return run_plain<__nv_bfloat16>(f, backward);
  return run_plain<__half>(f, backward);
}

size_t a256(size_t v) { return (v + 255) & ~(size_t)255; }
size_t elem_bytes(int dtype) { return dtype == DSALT_F32 ? 4 : 2; }
// whether the caller has to give a place for scales (with 24 bits nothing is written there)
bool scaled(int dtype, int keep) { return keep == DSALT_KEEP_8BIT || (keep == DSALT_KEEP_INPUT && dtype != DSALT_F32); }
// what the tensor cores take; their operands' rows have to be 16-byte aligned
bool tensor_cores(int dtype, int d, int F, int d_out) { return dtype != DSALT_F32 && d % 8 == 0 && F % 8 == 0 && d_out % 8 == 0; }
int check_rows(const char* fn, const Ffn& f) {
  if (!tensor_cores(f.dtype, f.d, f.F, f.d_out)) return DSALT_OK;
  for (const void* p : {f.x, f.dy, f.w_gate, f.w_up, f.w_down, (const void*)f.y, (const void*)f.dx, (const void*)f.dw_gate,
                        (const void*)f.dw_up, (const void*)f.dw_down})
    if (reinterpret_cast<uintptr_t>(p) & 15) return fail(DSALT_ERR_INVALID, "%s: operands must be 16-byte aligned", fn);
  if ((f.x && f.x_stride % 8) || (f.dy && f.dy_stride % 8))
    return fail(DSALT_ERR_INVALID, "%s: rows must be 16-byte aligned", fn);
  return DSALT_OK;
}
bool off256(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 255) != 0; }
bool known_dtype(int dt) { return dt == DSALT_F32 || dt == DSALT_BF16 || dt == DSALT_F16; }

int check(const char* fn, int dtype, int64_t T, int d, int F, int d_out, int act, int keep) {
  if (!known_dtype(dtype)) return fail(DSALT_ERR_INVALID, "%s: bad dtype %d", fn, dtype);
  if (T < 0 || d < 1 || F < 1 || d_out < 1) return fail(DSALT_ERR_INVALID, "%s: bad sizes (%lld tokens, %d -> %d -> %d)", fn, (long long)T, d, F, d_out);
  if (act != DSALT_ACT_SILU && act != DSALT_ACT_GELU) return fail(DSALT_ERR_INVALID, "%s: bad activation %d", fn, act);
  if (keep != DSALT_KEEP_NONE && keep != DSALT_KEEP_INPUT && keep != DSALT_KEEP_8BIT) return fail(DSALT_ERR_INVALID, "%s: bad keep %d", fn, keep);
  if (T > (1 << 27) || d > (1 << 20) || F > (1 << 20) || d_out > (1 << 20))
    return fail(DSALT_ERR_UNSUPPORTED, "%s: more than 2^27 tokens or 2^20 channels", fn);
  return DSALT_OK;
}

}  // namespace
}  // namespace ffn
}  // namespace dsalt

using namespace dsalt;
using namespace dsalt::ffn;

extern "C" {

int64_t dsalt_gated_ffn_pitch(int d_ff) { return d_ff < 1 ? 0 : pitch_of(d_ff); }

size_t dsalt_gated_ffn_workspace_bytes(int dtype, int64_t T, int d_model, int d_ff, int d_out) {
  return dsalt_gated_ffn_keep_workspace_bytes(dtype, T, d_model, d_ff, d_out, DSALT_KEEP_NONE);
}

size_t dsalt_gated_ffn_keep_workspace_bytes(int dtype, int64_t T, int d_model, int d_ff, int d_out, int keep) {
  if (check("gated_ffn", dtype, T, d_model, d_ff, d_out, 0, keep)) return 0;
  if (keeps_h(dtype, keep)) return 256;
  const size_t n = (size_t)T * pitch_of(d_ff);
  return a256(n * elem_bytes(dtype)) + (tensor_cores(dtype, d_model, d_ff, d_out) ? 0 : a256(2 * n * sizeof(float))) + 256;
}

int dsalt_gated_ffn(const void* x, int dtype, int64_t T, int d_model, int64_t x_stride, const void* w_gate,
                    const void* w_up, const void* w_down, int d_ff, int d_out, int activation, int keep, void* kept,
                    uint8_t* kept_exps, void* y, void* workspace, size_t workspace_bytes, void* stream) {
  constexpr const char* FN = "gated_ffn";
  if (int rc = check(FN, dtype, T, d_model, d_ff, d_out, activation, keep)) return rc;
  if (T == 0) return DSALT_OK;
  if (T > 1 && x_stride < d_model) return fail(DSALT_ERR_INVALID, "%s: rows overlap", FN);
  if (!x || !w_gate || !w_up || !w_down || !y || !workspace || (keep && !kept) || (scaled(dtype, keep) && !kept_exps))
    return fail(DSALT_ERR_INVALID, "%s: null pointer", FN);
  if (off256(kept) || off256(workspace)) return fail(DSALT_ERR_INVALID, "%s: kept and workspace must be 256-byte aligned", FN);
  if (workspace_bytes < dsalt_gated_ffn_keep_workspace_bytes(dtype, T, d_model, d_ff, d_out, keep))
    return fail(DSALT_ERR_WORKSPACE, "%s: workspace of %zu bytes is too small", FN, workspace_bytes);
  Ffn f{};
  f.dtype = dtype, f.act = activation, f.keep = keep, f.T = T, f.d = d_model, f.F = d_ff, f.d_out = d_out;
  f.pitch = pitch_of(d_ff);
  f.w_gate = w_gate, f.w_up = w_up, f.w_down = w_down, f.x = x, f.x_stride = T > 1 ? x_stride : d_model, f.kept = kept, f.exps = kept_exps;
  f.y = y;
  f.h = keeps_h(dtype, keep) ? static_cast<char*>(kept) + 2 * T * f.pitch * elem_bytes(dtype) : workspace;
  f.wide = reinterpret_cast<float*>(static_cast<char*>(workspace) + a256((size_t)T * f.pitch * elem_bytes(dtype)));
  f.stream = static_cast<cudaStream_t>(stream);
  if (int rc = check_rows(FN, f)) return rc;
  return run(f, false);
}

size_t dsalt_gated_ffn_bwd_workspace_bytes(int dtype, int64_t T, int d_model, int d_ff, int d_out, int keep) {
  if (check("gated_ffn_bwd", dtype, T, d_model, d_ff, d_out, 0, keep)) return 0;
  const size_t n = (size_t)T * pitch_of(d_ff);
  // dg and du, h where it was not kept; x where it was kept in 8 bits; the plain path's dh
  return (keeps_h(dtype, keep) ? 2 : 3) * a256(n * elem_bytes(dtype)) +
         (keep == DSALT_KEEP_8BIT ? a256((size_t)T * d_model * elem_bytes(dtype)) : 0) +
         (tensor_cores(dtype, d_model, d_ff, d_out) ? 0 : a256(n * sizeof(float))) + 256;
}

int dsalt_gated_ffn_bwd(const void* dy, int dtype, int64_t T, int d_model, int64_t dy_stride, const void* x,
                        int64_t x_stride, const uint8_t* x_exps, const void* w_gate, const void* w_up,
                        const void* w_down, int d_ff, int d_out, int activation, int keep, const void* kept,
                        const uint8_t* kept_exps, void* dx, void* dw_gate, void* dw_up, void* dw_down, void* workspace,
                        size_t workspace_bytes, void* stream) {
  constexpr const char* FN = "gated_ffn_bwd";
  if (int rc = check(FN, dtype, T, d_model, d_ff, d_out, activation, keep)) return rc;
  if (keep == DSALT_KEEP_NONE) return fail(DSALT_ERR_INVALID, "%s: the forward pass has to keep its activations", FN);
  if ((dw_gate == nullptr) != (dw_up == nullptr)) return fail(DSALT_ERR_INVALID, "%s: the gate's and up's gradients go together", FN);
  const size_t es = elem_bytes(dtype), w_bytes = (size_t)d_ff * d_model * es;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (T == 0) {  // no tokens: the weights' gradients are zero
    int rc = DSALT_OK;
    if (dw_gate && ((rc = check_cuda(cudaMemsetAsync(dw_gate, 0, w_bytes, s), "clear dw_gate")) ||
                    (rc = check_cuda(cudaMemsetAsync(dw_up, 0, w_bytes, s), "clear dw_up"))))
      return rc;
    if (dw_down) rc = check_cuda(cudaMemsetAsync(dw_down, 0, (size_t)d_ff * d_out * es, s), "clear dw_down");
    return rc;
  }
  const bool coded = keep == DSALT_KEEP_8BIT;
  if (T > 1 && (dy_stride < d_out || (!coded && x_stride < d_model))) return fail(DSALT_ERR_INVALID, "%s: rows overlap", FN);
  if (!dy || (dw_gate && (!x || (coded && !x_exps))) || !w_gate || !w_up || !w_down || !kept || (scaled(dtype, keep) && !kept_exps) || !workspace)
    return fail(DSALT_ERR_INVALID, "%s: null pointer", FN);
  if (off256(kept) || off256(workspace)) return fail(DSALT_ERR_INVALID, "%s: kept and workspace must be 256-byte aligned", FN);
  if (workspace_bytes < dsalt_gated_ffn_bwd_workspace_bytes(dtype, T, d_model, d_ff, d_out, keep))
    return fail(DSALT_ERR_WORKSPACE, "%s: workspace of %zu bytes is too small", FN, workspace_bytes);
  Ffn f{};
  f.dtype = dtype, f.act = activation, f.keep = keep, f.T = T, f.d = d_model, f.F = d_ff, f.d_out = d_out;
  f.pitch = pitch_of(d_ff);
  f.w_gate = w_gate, f.w_up = w_up, f.w_down = w_down;
  f.kept = const_cast<void*>(kept), f.exps = const_cast<uint8_t*>(kept_exps);
  f.dy = dy, f.dy_stride = T > 1 ? dy_stride : d_out, f.dx = dx, f.dw_gate = dw_gate, f.dw_up = dw_up, f.dw_down = dw_down;
  f.stream = s;
  const size_t n = a256((size_t)T * f.pitch * es);
  char* ws = static_cast<char*>(workspace);
  f.dg = ws, f.du = ws + n;
  const bool kept_h = keeps_h(dtype, keep);
  char* wide_x = ws + (kept_h ? 2 : 3) * n;
  f.wide = reinterpret_cast<float*>(coded ? wide_x + a256((size_t)T * d_model * es) : wide_x);
  f.h = kept_h ? static_cast<char*>(f.kept) + 2 * T * f.pitch * es : ws + 2 * n;
  f.x = coded ? nullptr : x, f.x_stride = T > 1 ? x_stride : d_model;
  if (int rc = check_rows(FN, f)) return rc;
  if (coded && dw_gate) {
    if (int rc = launch_unpack8(static_cast<const int8_t*>(x), x_exps, T, d_model, wide_x, dtype, s)) return rc;
    f.x = wide_x, f.x_stride = d_model;
  }
  return run(f, true);
}

}  // extern "C"
