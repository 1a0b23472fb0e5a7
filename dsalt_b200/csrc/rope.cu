// Norm of each query and key head with the rotation of its position, and the gradients
// (dsalt_qk_norm_rope, dsalt_qk_norm_rope_bwd).
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = w * (x r)           (without weights: n = x)
//   out = (n_a cos - n_b sin, n_b cos + n_a sin)            a, b: the halves of the head
// backward, with dn = the gradient turned back:
//   dn = (d_a cos + d_b sin, d_b cos - d_a sin),  dw = sum dn (x r)
//   dx = r (w dn - (x r) mean(w dn (x r)))
//
// Everything between the load and the store is fp32; a result is rounded once. The backward pass
// forms r again from x: one more pass over registers instead of 4 bytes a head kept and read.
//
// Bound by memory: an element is read once (backward: x and its gradient) and written once. A lane
// holds 16 bytes of each half of a head, so that the rotation needs no exchange and the norm a sum over
// G lanes (4 for 64 values of 16 bits); its angles, 4 bytes a value, are read once for several
// heads of the token, whose loads are all under way before the first is used. Queries and keys
// are two sides of one launch: a block works on one of them, so that a thread's share of the
// weights' gradient stays in registers until the block ends. The blocks' sums are joined by a second
// kernel in the blocks' order: results repeat bit for bit.
// 131072 tokens, 16 + 16 heads of 64 in bf16: forward 190 us, 5.8 TB/s; a forward and a backward pass over 24000
// tokens of 12 + 12 heads 80 us: 30 and 44 for the bytes, 6 for the sums of the weights' gradient.
#include "pack8.cuh"

namespace dsalt {
namespace {

constexpr int THREADS = 256;
constexpr int MAX_HEAD_DIM = 256;

// Heads whose loads are under way at once, and blocks an SM has room for. Measured at 131072 tokens, 16 + 16
// heads of 64 in bf16 (forward / backward us; the bytes take 164 / 246): 4 and 2 heads, two blocks 186 / 291;
// 2 and 2, three and two blocks 196 / 300; 4 and 4, two and one block 187 / 358; whatever makes registers spill
// (three backward blocks and more) 400 to 500 backward.
constexpr int FWD_HEADS = 4, BWD_HEADS = 2, PER_SM = 2;
constexpr int FWD_BLOCKS = 148 * 8, BWD_BLOCKS = 148 * PER_SM;  // backward: one share of the weights' gradient a block

struct Side {
  const void* x;
  const void* d;        // gradient of the output (backward)
  void* out;            // output, or the gradient of x
  const void* w;        // nullable
  int64_t x_token, x_head, d_token, d_head;
  int heads, chunks;    // chunks of HEADS heads in a token
  uint32_t items;       // tokens * chunks
};
struct Args {
  Side side[2];
  const float* cos;
  const float* sin;
  int64_t table_stride;
  const int32_t* pos;   // nullable: row t of the tables
  int64_t table_rows;
  float eps;
  int w_dtype, D;
  int q_blocks;         // blocks of the queries' side; the others are the keys'
  float* partial;       // [blocks, D] sums of the weights' gradients
  int* err;
};

template <typename T, int V>
__device__ __forceinline__ void widen16(float (&f)[V], const uint4& u) {
  if constexpr (sizeof(T) == 4) {
    f[0] = __uint_as_float(u.x), f[1] = __uint_as_float(u.y), f[2] = __uint_as_float(u.z), f[3] = __uint_as_float(u.w);
  } else {
    widen2<T>(u.x, f[0], f[1]);
    widen2<T>(u.y, f[2], f[3]);
    widen2<T>(u.z, f[4], f[5]);
    widen2<T>(u.w, f[6], f[7]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store16(T* p, const float (&f)[V]) {
  uint4 u;
  if constexpr (sizeof(T) == 4) {
    u = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  } else {
    u = make_uint4(narrow2<T>(f[0], f[1]), narrow2<T>(f[2], f[3]), narrow2<T>(f[4], f[5]), narrow2<T>(f[6], f[7]));
  }
  *reinterpret_cast<uint4*>(p) = u;
}
template <int V>
__device__ __forceinline__ void load_f32(float (&f)[V], const float* p) {
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    const float4 v = *reinterpret_cast<const float4*>(p + i);
    f[i] = v.x, f[i + 1] = v.y, f[i + 2] = v.z, f[i + 3] = v.w;
  }
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// G lanes to a head, of which those below D / (2 V) hold values; a warp takes 32 / G chunks at a time
template <typename T, int G, bool BWD>
__global__ void __launch_bounds__(THREADS, PER_SM) qk_norm_rope_kernel(const __grid_constant__ Args a) {
  constexpr int V = 16 / (int)sizeof(T), SLOTS = THREADS / G, HEADS = BWD ? BWD_HEADS : FWD_HEADS;
  const int which = (int)blockIdx.x >= a.q_blocks;
  const Side& s = a.side[which];
  const int block = which ? blockIdx.x - a.q_blocks : blockIdx.x, blocks = which ? gridDim.x - a.q_blocks : a.q_blocks;
  const int lane = threadIdx.x % G, half = a.D / 2, col = lane * V;
  const bool held = col < half;
  const bool norm = s.w != nullptr;
  float wa[V], wb[V], ga[V], gb[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    wa[i] = norm && held ? load_elem(s.w, col + i, a.w_dtype) : 1.f;
    wb[i] = norm && held ? load_elem(s.w, half + col + i, a.w_dtype) : 1.f;
    ga[i] = gb[i] = 0.f;
  }
  const float inv_d = 1.f / (float)a.D;
  const uint32_t first = block * SLOTS + threadIdx.x / G;
  // the lanes of a warp leave the loop together: the sums over a head need them all
  for (uint32_t item = first; item - (threadIdx.x % 32) / G < s.items; item += blocks * SLOTS) {
    const bool in = item < s.items;
    const int64_t t = in ? item / (uint32_t)s.chunks : 0;
    const int h0 = in ? (int)(item - (uint32_t)t * s.chunks) * HEADS : 0;
    const int n = in && held ? min(HEADS, s.heads - h0) : 0;
    int64_t p = a.pos && n > 0 ? __ldg(a.pos + t) : t;
    const T* x = static_cast<const T*>(s.x) + t * s.x_token + h0 * s.x_head + col;
    uint4 xr[HEADS][2] = {}, dr[HEADS][2] = {};
#pragma unroll
    for (int j = 0; j < HEADS; ++j)
      if (j < n) {
        xr[j][0] = __ldg(reinterpret_cast<const uint4*>(x + j * s.x_head));
        xr[j][1] = __ldg(reinterpret_cast<const uint4*>(x + j * s.x_head + half));
      }
    if constexpr (BWD) {
      const T* d = static_cast<const T*>(s.d) + t * s.d_token + h0 * s.d_head + col;
#pragma unroll
      for (int j = 0; j < HEADS; ++j)
        if (j < n) {
          dr[j][0] = __ldg(reinterpret_cast<const uint4*>(d + j * s.d_head));
          dr[j][1] = __ldg(reinterpret_cast<const uint4*>(d + j * s.d_head + half));
        }
    }
    float c[V] = {}, sn[V] = {};
    if (n > 0) {
      if (p < 0 || p >= a.table_rows) {  // reported, and read as the table's first row
        report_device_error(a.err, 51);
        p = 0;
      }
      load_f32<V>(c, a.cos + p * a.table_stride + col);
      load_f32<V>(sn, a.sin + p * a.table_stride + col);
    }
    T* out = static_cast<T*>(s.out) + (t * s.heads + h0) * a.D + col;
#pragma unroll
    for (int j = 0; j < HEADS; ++j) {
      float xa[V], xb[V], r = 1.f;
      widen16<T, V>(xa, xr[j][0]);
      widen16<T, V>(xb, xr[j][1]);
      if (norm) {
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) q += xa[i] * xa[i] + xb[i] * xb[i];
        r = 1.f / sqrtf(group_sum<G>(q) * inv_d + a.eps);
        if (j >= n) r = 0.f;  // no head here: with eps = 0 an infinity, which would reach the weights' sums as NaN
      }
      float oa[V], ob[V];
      if constexpr (!BWD) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float na = xa[i] * r * wa[i], nb = xb[i] * r * wb[i];
          oa[i] = na * c[i] - nb * sn[i];
          ob[i] = nb * c[i] + na * sn[i];
        }
      } else {
        float da[V], db[V], dot = 0.f;
        widen16<T, V>(da, dr[j][0]);
        widen16<T, V>(db, dr[j][1]);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          oa[i] = da[i] * c[i] + db[i] * sn[i];
          ob[i] = db[i] * c[i] - da[i] * sn[i];
          if (norm) {
            xa[i] *= r;
            xb[i] *= r;
            ga[i] += oa[i] * xa[i];
            gb[i] += ob[i] * xb[i];
            oa[i] *= wa[i];
            ob[i] *= wb[i];
            dot += oa[i] * xa[i] + ob[i] * xb[i];
          }
        }
        if (norm) {
          dot = group_sum<G>(dot) * inv_d;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            oa[i] = r * (oa[i] - xa[i] * dot);
            ob[i] = r * (ob[i] - xb[i] * dot);
          }
        }
      }
      if (j < n) {
        store16<T, V>(out + j * a.D, oa);
        store16<T, V>(out + j * a.D + half, ob);
      }
    }
  }
  if constexpr (BWD) {
    if (!norm) return;
    // the block's sum: over the heads of a warp, then over the warps in their order
    __shared__ float sums[THREADS / 32][MAX_HEAD_DIM];
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int o = G; o < 32; o <<= 1) {
        ga[i] += __shfl_xor_sync(0xffffffffu, ga[i], o);
        gb[i] += __shfl_xor_sync(0xffffffffu, gb[i], o);
      }
    }
    if (threadIdx.x % 32 < G && held) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        sums[threadIdx.x / 32][col + i] = ga[i];
        sums[threadIdx.x / 32][half + col + i] = gb[i];
      }
    }
    __syncthreads();
    if ((int)threadIdx.x < a.D) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < THREADS / 32; ++w) v += sums[w][threadIdx.x];
      a.partial[(int64_t)blockIdx.x * a.D + threadIdx.x] = v;
    }
  }
}

// block (32 columns, side): 32 columns x 32 runs of partial sums
__global__ void __launch_bounds__(1024) weight_grad_kernel(const float* __restrict__ partial, int q_blocks, int blocks,
                                                          int D, void* dwq, void* dwk, int dtype) {
  __shared__ float sums[32][33];
  const int run = threadIdx.x / 32;
  int col = blockIdx.x * 32 + threadIdx.x % 32;
  const int lo = blockIdx.y ? q_blocks : 0, hi = blockIdx.y ? blocks : q_blocks;
  void* out = blockIdx.y ? dwk : dwq;
  float v = 0.f;
  if (col < D) {
#pragma unroll 8
    for (int b = lo + run; b < hi; b += 32) v += partial[b * D + col];
  }
  sums[threadIdx.x % 32][run] = v;
  __syncthreads();
  // a warp per column
  v = sums[run][threadIdx.x % 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  col = blockIdx.x * 32 + run;
  if (threadIdx.x % 32 == 0 && col < D) {
    if (dtype == DSALT_F32) static_cast<float*>(out)[col] = v;
    else if (dtype == DSALT_BF16) static_cast<__nv_bfloat16*>(out)[col] = __float2bfloat16_rn(v);
    else static_cast<__half*>(out)[col] = __float2half_rn(v);
  }
}

int elem_bytes(int dtype) { return dtype == DSALT_F32 ? 4 : 2; }
int lanes_for(int D, int es) {
  int g = 1;
  while (g * (16 / es) < D / 2) g *= 2;
  return g;
}

template <typename T, bool BWD, int G>
int launch(const Args& a, int blocks, int lanes, cudaStream_t stream) {
  if constexpr (G * (16 / (int)sizeof(T)) < MAX_HEAD_DIM / 2)
    if (lanes > G) return launch<T, BWD, 2 * G>(a, blocks, lanes, stream);
  qk_norm_rope_kernel<T, G, BWD><<<blocks, THREADS, 0, stream>>>(a);
  return check_cuda(cudaGetLastError(), BWD ? "qk_norm_rope_bwd launch" : "qk_norm_rope launch");
}

template <bool BWD>
int launch_typed(const Args& a, int blocks, int G, int dtype, cudaStream_t stream) {
  if (dtype == DSALT_F32) return launch<float, BWD, 1>(a, blocks, G, stream);
  if (dtype == DSALT_BF16) return launch<__nv_bfloat16, BWD, 1>(a, blocks, G, stream);
  return launch<__half, BWD, 1>(a, blocks, G, stream);
}

// blocks of both sides, as many as their items need (at most `most`), shared in proportion to their heads
int share_blocks(Args& a, const char* fn, int64_t T, int G, int heads, int most, int& blocks) {
  const int slots = THREADS / G;
  int64_t need[2];
  for (int i = 0; i < 2; ++i) {
    Side& s = a.side[i];
    s.chunks = (s.heads + heads - 1) / heads;
    if (T * s.chunks > 1ll << 30) return fail(DSALT_ERR_UNSUPPORTED, "%s: more than 2^30 groups of %d heads", fn, heads);
    s.items = (uint32_t)(T * s.chunks);
    need[i] = ((int64_t)s.items + slots - 1) / slots;
  }
  if (need[0] + need[1] > most) {
    const int64_t q = most * need[0] / (need[0] + need[1]);
    need[0] = q < 1 ? 1 : (q > most - 1 ? most - 1 : q);
    need[1] = most - need[0];
  }
  a.q_blocks = (int)need[0];
  blocks = (int)(need[0] + need[1]);
  return DSALT_OK;
}

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

int check(const char* fn, int dtype, int w_dtype, int64_t T, int H, int Hk, int D, const void* wq, const void* wk,
          const float* cos, const float* sin, int64_t table_rows, int64_t table_stride, const int32_t* pos, float eps) {
  auto known = [](int dt) { return dt == DSALT_F32 || dt == DSALT_BF16 || dt == DSALT_F16; };
  if (!known(dtype) || !known(w_dtype)) return fail(DSALT_ERR_INVALID, "%s: bad dtype", fn);
  if (T < 0 || H < 1 || Hk < 1 || D < 1 || table_rows < 1 || table_stride < D / 2)
    return fail(DSALT_ERR_INVALID, "%s: bad sizes", fn);
  const int unit = 32 / elem_bytes(dtype);
  if (D % unit != 0 || D > MAX_HEAD_DIM)
    return fail(DSALT_ERR_UNSUPPORTED, "%s: head_dim %d (a multiple of %d up to %d is taken)", fn, D, unit, MAX_HEAD_DIM);
  if (H > 4096 || Hk > 4096) return fail(DSALT_ERR_UNSUPPORTED, "%s: more than 4096 heads", fn);
  if (!pos && table_rows < T) return fail(DSALT_ERR_INVALID, "%s: tables of %lld rows for %lld tokens", fn, (long long)table_rows, (long long)T);
  if ((wq == nullptr) != (wk == nullptr)) return fail(DSALT_ERR_INVALID, "%s: weights for one of queries and keys", fn);
  if (!(eps >= 0.f)) return fail(DSALT_ERR_INVALID, "%s: eps must not be negative", fn);
  if (T == 0) return DSALT_OK;
  if (!cos || !sin) return fail(DSALT_ERR_INVALID, "%s: null pointer", fn);
  if (off16(cos) || off16(sin) || table_stride % 4 != 0)
    return fail(DSALT_ERR_INVALID, "%s: rows of the tables must be 16-byte aligned", fn);
  return DSALT_OK;
}

int check_rows(const char* fn, const void* p, int dtype, int64_t token, int64_t head) {
  if (!p) return fail(DSALT_ERR_INVALID, "%s: null pointer", fn);
  const int64_t unit = 16 / elem_bytes(dtype);
  if (off16(p) || token % unit != 0 || head % unit != 0)
    return fail(DSALT_ERR_INVALID, "%s: rows of heads must be 16-byte aligned", fn);
  return DSALT_OK;
}

}  // namespace
}  // namespace dsalt

using namespace dsalt;

extern "C" {

int dsalt_qk_norm_rope(const void* q, const void* k, int dtype, int64_t T, int n_heads, int n_kv, int head_dim,
                       int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride, int64_t k_head_stride,
                       const void* q_weight, const void* k_weight, int w_dtype, float eps, const float* cos,
                       const float* sin, int64_t table_rows, int64_t table_stride, const int32_t* positions, void* q_out,
                       void* k_out, void* stream) {
  constexpr const char* FN = "qk_norm_rope";
  int rc = check(FN, dtype, w_dtype, T, n_heads, n_kv, head_dim, q_weight, k_weight, cos, sin, table_rows, table_stride,
                 positions, eps);
  if (rc || T == 0) return rc;
  if ((rc = check_rows(FN, q, dtype, q_token_stride, q_head_stride)) ||
      (rc = check_rows(FN, k, dtype, k_token_stride, k_head_stride)) || (rc = check_rows(FN, q_out, dtype, 0, 0)) ||
      (rc = check_rows(FN, k_out, dtype, 0, 0)))
    return rc;
  Args a{};
  a.side[0] = {q, nullptr, q_out, q_weight, q_token_stride, q_head_stride, 0, 0, n_heads, 0, 0};
  a.side[1] = {k, nullptr, k_out, k_weight, k_token_stride, k_head_stride, 0, 0, n_kv, 0, 0};
  a.cos = cos, a.sin = sin, a.table_stride = table_stride, a.pos = positions, a.table_rows = table_rows;
  a.eps = eps, a.w_dtype = w_dtype, a.D = head_dim, a.err = device_status_ptr();
  const int G = lanes_for(head_dim, elem_bytes(dtype));
  int blocks;
  if ((rc = share_blocks(a, FN, T, G, FWD_HEADS, FWD_BLOCKS, blocks))) return rc;
  return launch_typed<false>(a, blocks, G, dtype, static_cast<cudaStream_t>(stream));
}

size_t dsalt_qk_norm_rope_bwd_workspace_bytes(int head_dim) {
  return head_dim < 1 ? 0 : ((size_t)BWD_BLOCKS * head_dim * sizeof(float) + 255) & ~(size_t)255;
}

int dsalt_qk_norm_rope_bwd(const void* q, const void* k, const void* dq_out, const void* dk_out, int dtype, int64_t T,
                           int n_heads, int n_kv, int head_dim, int64_t q_token_stride, int64_t q_head_stride,
                           int64_t k_token_stride, int64_t k_head_stride, int64_t dq_token_stride,
                           int64_t dq_head_stride, int64_t dk_token_stride, int64_t dk_head_stride,
                           const void* q_weight, const void* k_weight, int w_dtype, float eps, const float* cos,
                           const float* sin, int64_t table_rows, int64_t table_stride, const int32_t* positions,
                           void* dq, void* dk, void* dq_weight, void* dk_weight, void* workspace,
                           size_t workspace_bytes, void* stream) {
  constexpr const char* FN = "qk_norm_rope_bwd";
  int rc = check(FN, dtype, w_dtype, T, n_heads, n_kv, head_dim, q_weight, k_weight, cos, sin, table_rows, table_stride,
                 positions, eps);
  if (rc) return rc;
  const bool norm = q_weight != nullptr;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (norm && (!dq_weight || !dk_weight)) return fail(DSALT_ERR_INVALID, "%s: null pointer", FN);
  if (T == 0) {  // no tokens: the weights' gradients are zero
    const size_t n = (size_t)head_dim * elem_bytes(w_dtype);
    if (norm && ((rc = check_cuda(cudaMemsetAsync(dq_weight, 0, n, s), "clear dq_weight")) ||
                 (rc = check_cuda(cudaMemsetAsync(dk_weight, 0, n, s), "clear dk_weight"))))
      return rc;
    return DSALT_OK;
  }
  if ((rc = check_rows(FN, q, dtype, q_token_stride, q_head_stride)) ||
      (rc = check_rows(FN, k, dtype, k_token_stride, k_head_stride)) ||
      (rc = check_rows(FN, dq_out, dtype, dq_token_stride, dq_head_stride)) ||
      (rc = check_rows(FN, dk_out, dtype, dk_token_stride, dk_head_stride)) || (rc = check_rows(FN, dq, dtype, 0, 0)) ||
      (rc = check_rows(FN, dk, dtype, 0, 0)))
    return rc;
  if (norm && !workspace) return fail(DSALT_ERR_INVALID, "%s: null pointer", FN);
  if (norm && workspace_bytes < dsalt_qk_norm_rope_bwd_workspace_bytes(head_dim))
    return fail(DSALT_ERR_WORKSPACE, "%s: workspace of %zu bytes is too small", FN, workspace_bytes);
  Args a{};
  a.side[0] = {q, dq_out, dq, q_weight, q_token_stride, q_head_stride, dq_token_stride, dq_head_stride, n_heads, 0, 0};
  a.side[1] = {k, dk_out, dk, k_weight, k_token_stride, k_head_stride, dk_token_stride, dk_head_stride, n_kv, 0, 0};
  a.cos = cos, a.sin = sin, a.table_stride = table_stride, a.pos = positions, a.table_rows = table_rows;
  a.eps = eps, a.w_dtype = w_dtype, a.D = head_dim, a.err = device_status_ptr();
  a.partial = static_cast<float*>(workspace);
  const int G = lanes_for(head_dim, elem_bytes(dtype));
  int blocks;
  if ((rc = share_blocks(a, FN, T, G, BWD_HEADS, BWD_BLOCKS, blocks))) return rc;
  if ((rc = launch_typed<true>(a, blocks, G, dtype, s)) || !norm) return rc;
  weight_grad_kernel<<<dim3((head_dim + 31) / 32, 2), 1024, 0, s>>>(a.partial, a.q_blocks, blocks, head_dim, dq_weight,
                                                                   dk_weight, w_dtype);
  return check_cuda(cudaGetLastError(), "qk_norm_rope_bwd weights launch");
}

}  // extern "C"
