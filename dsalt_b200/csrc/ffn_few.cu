// The gated feed-forward block for few tokens (bf16, fp16): weights are the wide side of the product.
//
//   h = act(x Wg^T) (x Wu^T), then y = h Wd^T, as D = W x^T: up to 128 rows of weights (those of gate and the
//   same of up) by up to 256 tokens a CTA
//
// Bound by reading the weights once, so every SM has to read an equal share of them. The first product has
// many rows: a tile is as many as make the SMs' shares equal, and takes all of K. The second has few rows
// and a long K: the CTAs of a cluster share 128 rows and take equal parts of K, and add up their fp32 sums
// through each other's shared memory in the order of their ranks (results repeat bit for bit). It is
// launched while the first one runs and asks for its first weights before it waits for h. 64 tokens, 2048 ->
// 11008 in bf16 (135 MB of weights): 34 to 35 us in a row, 3.9 TB/s; memory's own rate gives 21.
#include "ffn_tc.cuh"

namespace dsalt {
namespace ffn {
namespace {

constexpr int ROWS = 128, KB = 64, THREADS = 128, MAX_STAGES = 12, MAX_SPLIT = 8, MAX_SMEM = 226 * 1024;
constexpr int HALF_SMEM = 228 * 1024 / 2 - 1024 - 256;  // of two CTAs an SM, beside what each keeps for itself

struct FewArgs {
  CUtensorMap w[2], x;      // weights (gate's and up's, or one twice) and tokens
  void* out;
  int64_t out_stride;
  int64_t T;
  int rows;                 // of the output's features
  int box;                  // rows of weights in a load; a tile is two of them
  int tokens, stages, blocks, split;
  int smem;
  uint32_t idesc, tmem_cols;
  int* err;
};

struct FewBars {
  uint64_t full[MAX_STAGES], empty[MAX_STAGES], acc_full;
  uint32_t tmem;
};

__device__ __forceinline__ float2 load_peer2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ float2 load_own2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

template <bool GATED, typename T, int ACT>
__global__ void __launch_bounds__(THREADS) ffn_few_kernel(const __grid_constant__ FewArgs a) {
  extern __shared__ uint8_t raw[];
  __shared__ FewBars bars;
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = (int)cluster_rank(), tile = blockIdx.x / a.split;
  const int f0 = tile * (GATED ? a.box : 2 * a.box), t0 = blockIdx.y * a.tokens;
  const int lo = rank * a.blocks / a.split, n = (rank + 1) * a.blocks / a.split - lo;
  const uint32_t w_bytes = 2 * a.box * KB * 2, stage_bytes = w_bytes + a.tokens * KB * 2;

  if (threadIdx.x == 96) {
    tma_prefetch_desc(&a.w[0]);
    tma_prefetch_desc(&a.w[1]);
    tma_prefetch_desc(&a.x);
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], 1);
    }
    mbar_init(&bars.acc_full, 1);
    fence_barrier_init();
  }
  if (warp == 2) {
    tmem_alloc(&bars.tmem, a.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  if constexpr (GATED) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (warp == 0 && lane == 0) {
    auto weights = [&](int i, int s) {
      const uint32_t at = base + s * stage_bytes;
      mbar_arrive_expect_tx(&bars.full[s], stage_bytes);
      load_own_2d(at, &a.w[0], &bars.full[s], (lo + i) * KB, f0);
      load_own_2d(at + w_bytes / 2, &a.w[1], &bars.full[s], (lo + i) * KB, GATED ? f0 : f0 + a.box);
    };
    auto tokens = [&](int i, int s) {
      load_own_2d(base + s * stage_bytes + w_bytes, &a.x, &bars.full[s], (lo + i) * KB, t0);
    };
    const int first = min(n, a.stages);
    for (int i = 0; i < first; ++i) weights(i, i);
    asm volatile("griddepcontrol.wait;" ::: "memory");  // h, where the first product made it
    for (int i = 0; i < first; ++i) tokens(i, i);
    int s = 0;
    uint32_t phase = 0;
    for (int i = first; i < n; ++i) {
      if (!mbar_wait(&bars.empty[s], phase, a.err, 66)) break;
      weights(i, s);
      tokens(i, s);
      if (++s == a.stages) {
        s = 0;
        phase ^= 1;
      }
    }
  } else if (warp == 1 && lane == 0) {
    int s = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      if (!(ok = mbar_wait(&bars.full[s], phase, a.err, 67))) break;
      tc_fence_after();
      const uint32_t w = base + s * stage_bytes;
      // 128 rows are read whatever the tile has: those behind it are some other operand's, and the sums
      // that they give are not looked at
#pragma unroll
      for (int ks = 0; ks < KB / 16; ++ks)
        umma_ss(tmem, sw128_desc(w + ks * 32, 16, 1024), sw128_desc(w + w_bytes + ks * 32, 16, 1024), a.idesc, i | ks);
      umma_commit(&bars.empty[s]);
      if (++s == a.stages) {
        s = 0;
        phase ^= 1;
      }
    }
    if (ok) umma_commit(&bars.acc_full);
  }
  __syncwarp();

  // sums of this part of K, as [token][row of weights], where the operands were (every load has arrived: its
  // product is done)
  const int here = (int)min((int64_t)a.tokens, a.T - t0);
  if (mbar_wait(&bars.acc_full, 0, a.err, 68)) {
    tc_fence_after();
    for (int c = 0; c < here; c += 16) {
      uint32_t r[16];
      float f[16];
      ask_acc<16>(tmem + c + ((uint32_t)(warp * 32) << 16), r);
      take_acc<16>(r, f);
#pragma unroll
      for (int i = 0; i < 16; ++i)
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(base + ((c + i) * ROWS + warp * 32 + lane) * 4), "f"(f[i]) : "memory");
    }
  }
  tc_fence_before();
  if constexpr (GATED) __syncthreads();
  else cluster_sync();

  if constexpr (GATED) {  // all of K is here
    constexpr int BATCH = 4;  // tokens whose sums are asked for at once
    const int r = 2 * lane;
    if (r < a.box && f0 + r < a.rows)
      for (int t = warp; t < here; t += 4 * BATCH) {
        float2 g[BATCH], u[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
          if (t + 4 * i < here) {
            g[i] = load_own2(base + ((t + 4 * i) * ROWS + r) * 4);
            u[i] = load_own2(base + ((t + 4 * i) * ROWS + a.box + r) * 4);
          }
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
          if (t + 4 * i < here)
            *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + (t0 + t + 4 * i) * a.out_stride + f0 + r) =
                narrow2<T>(activate<ACT, true>(g[i].x) * u[i].x, activate<ACT, true>(g[i].y) * u[i].y);
      }
  } else {
    for (int t = rank * 4 + warp; t < here; t += 4 * a.split) {
      T* out = static_cast<T*>(a.out) + (t0 + t) * a.out_stride + f0;
      float2 v[2][MAX_SPLIT];
#pragma unroll
      for (int c = 0; c < MAX_SPLIT; ++c)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          v[i][c] = c < a.split ? load_peer2(in_cta(base + (t * ROWS + 64 * i + 2 * lane) * 4, c)) : float2{0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 64 * i + 2 * lane;
#pragma unroll
        for (int c = 1; c < MAX_SPLIT; ++c) v[i][0].x += v[i][c].x, v[i][0].y += v[i][c].y;
        if (f0 + r < a.rows) *reinterpret_cast<uint32_t*>(out + r) = narrow2<T>(v[i][0].x, v[i][0].y);
      }
    }
  }
  if constexpr (GATED) __syncthreads();
  else cluster_sync();  // the others' reads of this CTA's sums
  if (warp == 2) tmem_dealloc(tmem, a.tmem_cols);
}

// ---------------------------------------------------------------- host side
// How a product of `rows` features, T tokens and K is cut: tiles of weights and of tokens, parts of K, stages.
//
// Two CTAs an SM, where the sums leave room for that: the second product's first loads, and clusters of eight,
// find room beside others (one CTA an SM with twice the stages took 16 % longer at 64 tokens, 2048 -> 11008).
// Tokens are cut as finely as lets all CTAs run at once, to 48 (second product: 64) of them: weights that several CTAs read
// come from L2, and what a CTA does for each of its tokens after its products is seen by nobody else. (One tile
// of up to 256 tokens | so cut, us: 64 tokens 768 -> 2048 13.9 | 12.6, 128 tokens 1024 -> 4096 20.8 | 17.8, 192
// tokens 2048 -> 5504 44 | 29, 128 tokens 2048 -> 11008 41 | 36.4.)
void cut(FewArgs& a, bool gated, int rows, int64_t T, int K, int& tiles, int& token_tiles) {
  constexpr int SMS = 148;
  tiles = ceil_div(rows, gated ? ROWS / 2 : ROWS);
  const int most = 2 * SMS / tiles, wanted = ceil_div(T, gated ? 48 : 64), least = ceil_div(T, 256);
  token_tiles = wanted < most ? wanted : most;
  if (token_tiles < least) token_tiles = least;
  a.tokens = ceil_div(ceil_div(T, token_tiles), 16) * 16;
  token_tiles = ceil_div(T, a.tokens);
  a.tmem_cols = 32;
  while ((int)a.tmem_cols < a.tokens) a.tmem_cols *= 2;
  a.rows = rows;
  a.blocks = ceil_div(K, KB);
  a.box = ROWS / 2;
  a.split = 1;
  if (gated) {
    // An SM reads its tiles' weights from memory and the tokens, at about twice the rate, from L2; each two
    // tiles that it works on at once have a start and an end besides, of some thousand cycles (here in rows of
    // weights, which take K / 12 cycles each)
    int best = 1 << 30;
    for (int box = ROWS / 2; box >= 8; box -= 8) {
      const int n = ceil_div((int64_t)ceil_div(rows, box) * token_tiles, SMS);
      const int cost = n * (2 * box + a.tokens / 2) + (n + 1) / 2 * ((2000 + 15 * a.tokens) * 12 / K);
      if (cost < best) best = cost, a.box = box;
    }
    tiles = ceil_div(rows, a.box);
  } else {
    // clusters that all run at once: 36 of 8 or 72 of 4, two CTAs an SM, do not (16 us against 21 at 384 tokens,
    // 768 -> 2048)
    while (a.split < MAX_SPLIT && 2 * a.split * tiles * token_tiles <= 256 && 8 * a.split <= a.blocks) a.split *= 2;
  }
  // the products read 128 rows from the start of the last stage on; the stages later hold the sums
  const int stage = (2 * a.box + a.tokens) * KB * 2, behind = (ROWS - 2 * a.box) * KB * 2, sums = a.tokens * ROWS * 4;
  const bool two = 1024 + (sums > 2 * stage + behind ? sums : 2 * stage + behind) <= HALF_SMEM;
  a.stages = ((two ? HALF_SMEM : MAX_SMEM) - 1024 - behind) / stage;
  a.stages = a.stages < MAX_STAGES ? a.stages : MAX_STAGES;
  a.smem = 1024 + a.stages * stage + behind;
  if (a.smem < 1024 + sums) a.smem = 1024 + sums;
}

template <bool GATED, typename T, int ACT>
int launch_few(FewArgs& a, const Ffn& f, int tiles, int token_tiles, const char* what) {
  static std::atomic<uint64_t> ready{0};
  auto kernel = ffn_few_kernel<GATED, T, ACT>;
  if (int rc = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), MAX_SMEM, ready)) return rc;
  a.idesc = umma_idesc_f16(f.dtype == DSALT_BF16 ? 1 : 0, 0, 0, ROWS, a.tokens);
  a.err = device_status_ptr();
  a.T = f.T;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(tiles * a.split, token_tiles);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = a.smem;
  cfg.stream = f.stream;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = a.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = GATED ? 1 : 2;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, a), what);
}

template <typename T, int ACT>
int few(const Ffn& f) {
  int rc, tiles, token_tiles;
  {
    FewArgs a{};
    cut(a, true, f.F, f.T, f.d, tiles, token_tiles);
    if ((rc = make_map(&a.w[0], f.w_gate, f.dtype, f.F, f.d, f.d, a.box, KB)) ||
        (rc = make_map(&a.w[1], f.w_up, f.dtype, f.F, f.d, f.d, a.box, KB)) ||
        (rc = make_map(&a.x, f.x, f.dtype, f.T, f.d, f.x_stride, a.tokens, KB)))
      return rc;
    a.out = f.h, a.out_stride = f.pitch;
    if ((rc = launch_few<true, T, ACT>(a, f, tiles, token_tiles, "gated_ffn gate and up launch"))) return rc;
  }
  FewArgs a{};
  cut(a, false, f.d_out, f.T, f.F, tiles, token_tiles);
  if ((rc = make_map(&a.w[0], f.w_down, f.dtype, f.d_out, f.F, f.F, a.box, KB)) ||
      (rc = make_map(&a.x, f.h, f.dtype, f.T, f.F, f.pitch, a.tokens, KB)))
    return rc;
  a.w[1] = a.w[0];
  a.out = f.y, a.out_stride = f.d_out;
  return launch_few<false, T, 0>(a, f, tiles, token_tiles, "gated_ffn down launch");
}

template <typename T>
int few_typed(const Ffn& f) {
  return f.act == DSALT_ACT_SILU ? few<T, DSALT_ACT_SILU>(f) : few<T, DSALT_ACT_GELU>(f);
}

}  // namespace

int forward_few(const Ffn& f) {
  return f.dtype == DSALT_BF16 ? few_typed<__nv_bfloat16>(f) : few_typed<__half>(f);
}

}  // namespace ffn
}  // namespace dsalt
