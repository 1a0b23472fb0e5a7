// The gated feed-forward block for up to sixteen tokens (bf16, fp16): a stream of weights past them.
//
//   h = act(x Wg^T) (x Wu^T), then y = h Wd^T
//
// Bound by reading the weights once, and at these sizes as much by latency: nothing is staged. A warp
// holds 16 rows of weights (of gate and of up) and a part of K as operands of mma.sync m16n8k16: the order
// of K in a product is free, so a lane takes 16 consecutive bytes of a row, which are its share of two
// products, and the same 16 bytes of a token. All loads of BATCH x 32 values of K are under way before the
// first is used. The warps of a block, and the blocks of a cluster, take parts of K; their sums are
// added in the order of their ranks (results repeat bit for bit). The second product is launched while the
// first one runs and loads its first weights before it waits for h. One token in bf16, weights from
// memory: 1024 -> 4096 (25 MB) 8.8 us, 2048 -> 11008 (135 MB) 27 us, 5 TB/s.
#include "ffn_tc.cuh"

namespace dsalt {
namespace ffn {
namespace {

constexpr int ROWS = 16, MAX_SPLIT = 8;
// The second product has few rows and a long K: twice the warps to a block, each with twice the loads under
// way, so that one token's weights wait in registers for h and clusters are rarely needed
template <bool GATED>
struct Block {
  static constexpr int WARPS = GATED ? 8 : 16, THREADS = 32 * WARPS, BATCH = GATED ? 4 : 8;
};

struct TokenArgs {
  const void* w[2];
  const void* x;
  void* out;
  int64_t x_stride, out_stride;
  int T, rows, K, split;
};

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load_once(const void* p) {  // weights: not kept in L1
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(__cvta_generic_to_global(p)));
  return v;
}

// NT: groups of 8 tokens
template <bool GATED, int NT, typename T, int ACT>
__global__ void __launch_bounds__(Block<GATED>::THREADS) ffn_token_kernel(const __grid_constant__ TokenArgs a) {
  constexpr int WARPS = Block<GATED>::WARPS, THREADS = Block<GATED>::THREADS, BATCH = Block<GATED>::BATCH;
  constexpr int MATS = GATED ? 2 : 1, TOKENS = 8 * NT, SUMS = MATS * ROWS * TOKENS;
  __shared__ float part[WARPS][SUMS];
  float* total = part[0];  // of all warps
  if constexpr (GATED) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int rank = a.split > 1 ? (int)cluster_rank() : 0, f0 = blockIdx.x / a.split * ROWS;
  // this warp's part of K, in chunks of 32 values
  const int chunks = (a.K + 31) / 32, parts = a.split * WARPS, id = rank * WARPS + warp;
  const int lo = (int)((int64_t)id * chunks / parts), hi = (int)((int64_t)(id + 1) * chunks / parts);

  const T* row[MATS][2];
#pragma unroll
  for (int m = 0; m < MATS; ++m)
#pragma unroll
    for (int i = 0; i < 2; ++i)  // rows behind the last are read as the last and not stored
      row[m][i] = static_cast<const T*>(a.w[m]) + (int64_t)min(f0 + g + 8 * i, a.rows - 1) * a.K + 8 * t;

  float acc[MATS][NT][4] = {};
  bool waited = false;
  for (int c0 = lo; c0 < hi; c0 += BATCH) {
    uint4 w[BATCH][MATS][2] = {};
#pragma unroll
    for (int b = 0; b < BATCH; ++b)
      if (c0 + b < hi && (c0 + b) * 32 + 8 * t < a.K) {
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
          for (int i = 0; i < 2; ++i) w[b][m][i] = load_once(row[m][i] + (c0 + b) * 32);
      }
    if (!GATED && !waited) {
      asm volatile("griddepcontrol.wait;" ::: "memory");  // the tokens' rows are made by the first product
      waited = true;
    }
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int k = (c0 + b) * 32 + 8 * t;
      const bool in = c0 + b < hi && k < a.K;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint4 x = {};
        if (in && 8 * n + g < a.T)
          x = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + (8 * n + g) * a.x_stride + k);
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
          mma_16816<T>(acc[m][n], w[b][m][0].x, w[b][m][1].x, w[b][m][0].y, w[b][m][1].y, x.x, x.y);
          mma_16816<T>(acc[m][n], w[b][m][0].z, w[b][m][1].z, w[b][m][0].w, w[b][m][1].w, x.z, x.w);
        }
      }
    }
  }
  if (!GATED && !waited) asm volatile("griddepcontrol.wait;" ::: "memory");

  // sums as [matrix][token][row]
#pragma unroll
  for (int m = 0; m < MATS; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        part[warp][(m * TOKENS + 8 * n + 2 * t + (i & 1)) * ROWS + g + 8 * (i >> 1)] = acc[m][n][i];
  __syncthreads();
  for (int i = threadIdx.x; i < SUMS; i += THREADS) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += part[w][i];
    total[i] = v;
  }
  if (a.split > 1) cluster_sync();
  else __syncthreads();
  for (int i = rank * THREADS + threadIdx.x; i < TOKENS * ROWS; i += a.split * THREADS) {
    float v = total[i], u = GATED ? total[TOKENS * ROWS + i] : 0.f;
    if (a.split > 1) {
      float x[MAX_SPLIT][MATS];
#pragma unroll
      for (int c = 0; c < MAX_SPLIT; ++c)
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
          x[c][m] = 0.f;
          if (c < a.split)
            asm volatile("ld.shared::cluster.f32 %0, [%1];"
                         : "=f"(x[c][m])
                         : "r"(in_cta(smem_u32(total + m * TOKENS * ROWS + i), c))
                         : "memory");
        }
      v = u = 0.f;
#pragma unroll
      for (int c = 0; c < MAX_SPLIT; ++c) v += x[c][0], u += x[c][MATS - 1];
    }
    const int tok = i / ROWS, f = f0 + i % ROWS;
    if constexpr (GATED) v = activate<ACT, true>(v) * u;
    if (tok < a.T && f < a.rows) static_cast<T*>(a.out)[tok * a.out_stride + f] = from_float<T>(v);
  }
  if (a.split > 1) cluster_sync();  // the others' reads of this block's sums
}

template <bool GATED, int NT, typename T, int ACT>
int launch_token(TokenArgs& a, const Ffn& f, const char* what) {
  const int tiles = ceil_div(a.rows, ROWS);
  // clusters where the tiles would leave more than half of the SMs idle and every warp has several batches
  a.split = 1;
  while (a.split < MAX_SPLIT && a.split * tiles < 64 && 2 * a.split * Block<GATED>::WARPS * Block<GATED>::BATCH * 32 <= a.K)
    a.split *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(tiles * a.split);
  cfg.blockDim = dim3(Block<GATED>::THREADS);
  cfg.stream = f.stream;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = GATED ? 1 : 2;
  return check_cuda(cudaLaunchKernelEx(&cfg, ffn_token_kernel<GATED, NT, T, ACT>, a), what);
}

template <int NT, typename T, int ACT>
int tokens(const Ffn& f) {
  TokenArgs a{{f.w_gate, f.w_up}, f.x, f.h, f.x_stride, f.pitch, (int)f.T, f.F, f.d, 1};
  if (int rc = launch_token<true, NT, T, ACT>(a, f, "gated_ffn gate and up launch")) return rc;
  TokenArgs b{{f.w_down, f.w_down}, f.h, f.y, f.pitch, f.d_out, (int)f.T, f.d_out, f.F, 1};
  return launch_token<false, NT, T, 0>(b, f, "gated_ffn down launch");
}

template <typename T, int ACT>
int tokens_n(const Ffn& f) {
  return f.T <= 8 ? tokens<1, T, ACT>(f) : tokens<2, T, ACT>(f);
}

template <typename T>
int tokens_typed(const Ffn& f) {
  return f.act == DSALT_ACT_SILU ? tokens_n<T, DSALT_ACT_SILU>(f) : tokens_n<T, DSALT_ACT_GELU>(f);
}

}  // namespace

int forward_tokens(const Ffn& f) {
  return f.dtype == DSALT_BF16 ? tokens_typed<__nv_bfloat16>(f) : tokens_typed<__half>(f);
}

}  // namespace ffn
}  // namespace dsalt
