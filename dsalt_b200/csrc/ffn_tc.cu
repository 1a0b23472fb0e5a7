// The gated feed-forward block on the tensor cores (bf16, fp16): one persistent matrix kernel whose
// epilogue is the activation, its gradient, or a plain store.
//
//   forward    gate, up = x [Wg | Wu]^T -> epilogue: h = act(gate) up, gate and up kept if a gradient
//              will be wanted;  y = h Wd^T
//   backward   dh = dy Wd -> epilogue: dg = dh up act'(gate), du = dh act(gate), and h again;
//              dx = dg Wg + du Wu (one sum over both);  dWg = dg^T x, dWu = du^T x, dWd = dy^T h, all
//              in one launch
//
// Two CTAs share a tile of 256 x 256 outputs (tcgen05.mma of the pair: each holds 128 rows of A
// and 128 of B, and reads the other's B through it), 64 values of K and 32 KB a CTA in a stage. The
// accumulators of two tiles lie in TMEM (2 x 256 columns), so that a tile's epilogue runs under the
// next one's products. A tile of the first product is 128 columns of gate beside the same 128 of up:
// one CTA of the pair loads gate's rows, the other up's, and a thread finds both in its row. Operands whose
// K runs along memory rows or across them (weights and gradients as they lie) are both read as they
// are, by the major-ness of the matrix descriptors; nothing is transposed in memory.
//
// Bound by what an SM can take from L2, 64 bytes a cycle: a stage of 32 KB feeds 512 cycles of products, so
// at the tensor cores' full rate the operands alone fill that path (85 to 90 % of the rate is reached),
// and what an epilogue writes and reads (up to 8 and 6 bytes for each of T x d_ff values) comes on top. Long runs
// are bound by the power limit, under which the clock falls from 1.9 to 1.3 GHz. Measured, bf16, a call alone and in a row: 32768 x
// 2048 -> 11008 forward 2.9 ms (1530 TFLOP/s) and 3.3 (1330); 32768 x 768 -> 2048 forward, 16 bits kept, and backward
// 0.78 and 0.94 (1180 and 990); 16384 x 1024 -> 4096, 8 bits kept, 0.96 and 1.12 (1290 and 1100); 1999 x 768 -> 2048 30 us.
#include "ffn_tc.cuh"

namespace dsalt {
namespace ffn {
namespace {

constexpr int SUMS_COL = 128 * 4;  // bytes of a column of partial sums
constexpr int PAIR_M = 256, CTA_M = 128, PAIR_N = 256, KB = 64;
constexpr int OPERAND_BYTES = CTA_M * KB * 2, STAGE_BYTES = 2 * OPERAND_BYTES;
constexpr int BOX = 32, BOX_BYTES = 32 * BOX * 2;  // a warp's staged outputs: 32 rows of 32 columns
constexpr int EPI_WARPS = 8, THREADS = 32 * (4 + EPI_WARPS);  // 16 warps in the first epilogue: no faster
constexpr uint32_t TMEM_COLS = 512;
constexpr int PAIRS = 74;  // of SMs
constexpr int64_t HALF_L2 = 60 << 20;

enum Order { ALONG = 0, ACROSS = 1, BY_JOB = 2 };  // how K of A lies: along its rows, across them
enum Epilogue { PLAIN = 0, GATE_UP = 1, GRADS = 2 };

struct alignas(64) Job {
  CUtensorMap a[2], b[2];  // of both segments of K; the first product: gate's and up's rows
  CUtensorMap c[3];
  int tiles_m, tiles_n, blocks0, blocks;  // blocks of K in the first segment and in all
  int group;                              // tiles of 256 rows whose A stays in L2 while N is walked
  int rows, cols;                         // of the outputs
  int a_across;                           // K of A lies across its rows (where jobs differ)
  void* out;                              // of c[0], for a plain store's sums of several parts
};
struct Kept {
  void* p;           // gate's and up's codes [2, T, pitch], or their 24 bits [3, T, pitch]
  uint8_t* exps;     // their scales [2, pitch / 32, T]: the lanes of a warp, rows of a tile, find theirs side by side
  void* h;           // [T, pitch]
  int64_t T, pitch;
};
template <int NJ>
struct Args {
  Job job[NJ];
  CUtensorMap kept_map[2];  // gate's and up's, where they are read
  Kept kept;
  // Tiles are dealt round robin, or (of two kinds of jobs) the first `dealt` are, then each pair takes its extra
  // ones of the others and then `rounds` in turn with the other pairs
  int dealt, rounds, extra[PAIRS + 1];
  int tiles, split;  // split > 1: a cluster of so many pairs shares a tile, each takes a part of K
  uint32_t idesc;
  int* err;
};

// ---------------------------------------------------------------- pair-wide forms
// relaxed: it says that the accumulator has been read (tcgen05.wait::ld has returned); a release would wait for the
// thread's stores to memory, some 1600 cycles a tile
__device__ __forceinline__ void arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// load into this CTA's shared memory, counted on a barrier of the pair
__device__ __forceinline__ void load_2d(uint32_t dst, const void* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], "
      "[%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
// bytes of this CTA's shared memory to another's, counted on a barrier there
__device__ __forceinline__ void copy_to_cta(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "r"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void store_2d(const void* map, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src),
               "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// arrives on the barrier at this offset in both CTAs of the pair (ranks leader, leader + 1) once the
// thread's products so far are done
__device__ __forceinline__ void pair_commit(uint64_t* bar, uint32_t leader) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)(3u << leader))
      : "memory");
}

// ---------------------------------------------------------------- shared memory
// What an epilogue keeps in shared memory, and the stages that this leaves for the operands. The first
// product's writes its rows from registers. A plain store stages its output for the store engine, in four
// sets of boxes. The backward's has what was kept brought in by the load engine, a warp's 32 rows x 32
// columns of gate and of up at a time, three of them under way (hidden gradients of
// 32768 x 768 -> 2048: read row by row by the threads 165 us, so 148, and 123 since accumulators are given back
// early, with two codes of 16 bits a value; 162 with 24 bits each and h formed again, 850 MB of memory traffic where there were
// 558). The upper halves of 24 bits are replaced by the gradients where they lie, the third bytes and h go
// through registers; codes of 8 bits have a set of boxes for three outputs besides.
template <int EPI, int KEEP>
struct Shape {
  static constexpr bool IN_PLACE = EPI == GRADS && KEEP == DSALT_KEEP_INPUT;
  static constexpr int OUTPUTS = EPI == GATE_UP ? 0 : EPI == PLAIN ? 1 : IN_PLACE ? 2 : 3;
  static constexpr int SETS = EPI == PLAIN ? 4 : IN_PLACE ? 0 : 1, STAGES = EPI == GATE_UP ? 6 : EPI == GRADS ? 4 : 5;
  static constexpr int KEPT_SETS = EPI == GRADS ? 3 : 0, KEPT_BOX = BOX * BOX * (KEEP == DSALT_KEEP_8BIT ? 1 : 2);
  static constexpr int SET_BYTES = OUTPUTS * BOX_BYTES, WARP_BYTES = SETS * SET_BYTES + KEPT_SETS * 2 * KEPT_BOX;
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + EPI_WARPS * WARP_BYTES + 512;
  // columns of the accumulator that a warp works on (of the first product: as many of gate and of up)
  static constexpr int COLS = (EPI == GATE_UP ? PAIR_N / 2 : PAIR_N) / (EPI_WARPS / 4);
};
template <int STAGES>
struct Bars {
  uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2], kept_full[EPI_WARPS][3], sums;
  uint32_t tmem;
};

struct Tile {
  int job, m, n;
};
// the i-th tile of a pair, or -1
template <int NJ>
__device__ __forceinline__ int tile_of(const Args<NJ>& a, int pair, int pairs, int i) {
  const int t = pair + i * pairs;
  if (t < a.dealt) return t;
  if (a.dealt == a.tiles) return -1;
  int k = i - (pair < a.dealt ? (a.dealt - pair + pairs - 1) / pairs : 0);
  const int n = a.extra[pair + 1] - a.extra[pair];
  if (k < n) return a.dealt + a.rounds * pairs + a.extra[pair] + k;
  k -= n;
  return k < a.rounds ? a.dealt + k * pairs + pair : -1;
}
template <int NJ>
__device__ __forceinline__ Tile find_tile(const Args<NJ>& a, int t) {
  int j = 0;
#pragma unroll
  for (int i = 0; i + 1 < NJ; ++i) {
    const int n = a.job[i].tiles_m * a.job[i].tiles_n;
    if (j == i && t >= n) {
      t -= n;
      ++j;
    }
  }
  const int tm = a.job[j].tiles_m, tn = a.job[j].tiles_n;
  const int high = a.job[j].group, group = t / (high * tn), first = group * high, rows = min(high, tm - first);
  const int r = t - group * high * tn;
  return {j, first + r % rows, r / rows};
}

// N values of a row as fp32 from column `first` of the warp's box (64 bytes a row, 16-byte pieces
// swizzled as the store's map has it: piece ^ row / 2)
template <typename T, int N>
__device__ __forceinline__ void stage_row(uint32_t box, int lane, const float (&f)[N], int first) {
#pragma unroll
  for (int c = 0; c < N / 8; ++c) {
    const uint32_t at = box + lane * 64 + (((c + first / 8) ^ ((lane >> 1) & 3)) << 4);
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(narrow2<T>(f[8 * c], f[8 * c + 1])),
                 "r"(narrow2<T>(f[8 * c + 2], f[8 * c + 3])), "r"(narrow2<T>(f[8 * c + 4], f[8 * c + 5])),
                 "r"(narrow2<T>(f[8 * c + 6], f[8 * c + 7]))
                 : "memory");
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_row(T* p, const float (&f)[N]) {
#pragma unroll
  for (int c = 0; c < N / 16; ++c)
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(__cvta_generic_to_global(p + 16 * c)),
                 "r"(narrow2<T>(f[16 * c], f[16 * c + 1])), "r"(narrow2<T>(f[16 * c + 2], f[16 * c + 3])),
                 "r"(narrow2<T>(f[16 * c + 4], f[16 * c + 5])), "r"(narrow2<T>(f[16 * c + 6], f[16 * c + 7])),
                 "r"(narrow2<T>(f[16 * c + 8], f[16 * c + 9])), "r"(narrow2<T>(f[16 * c + 10], f[16 * c + 11])),
                 "r"(narrow2<T>(f[16 * c + 12], f[16 * c + 13])), "r"(narrow2<T>(f[16 * c + 14], f[16 * c + 15]))
                 : "memory");
}
__device__ __forceinline__ void store_32b(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(__cvta_generic_to_global(p)), "r"(w[0]), "r"(w[1]),
               "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
// bits of the largest magnitude of 32, NaN if there is one
__device__ __forceinline__ uint32_t largest_of(const float (&f)[GROUP8]) {
  float top[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) top[i] = fabsf(f[i]);
#pragma unroll
  for (int i = 4; i < GROUP8; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top[i % 4]) : "f"(fabsf(f[i])));
#pragma unroll
  for (int i = 1; i < 4; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top[0]) : "f"(top[i]));
  return __float_as_uint(top[0]) & 0x7fffffffu;
}
// 32 bytes of what the forward pass kept
__device__ __forceinline__ void load_32b(uint32_t (&w)[8], const void* p) {
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(__cvta_generic_to_global(p)));
}

__device__ __forceinline__ uint4 load_shared(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
// values 16 half .. 16 half + 15 of a row of a box of codes, as the load engine wrote it
__device__ __forceinline__ void coded_values(uint32_t box, int lane, int half, float scale, float (&f)[16]) {
  const uint4 v = load_shared(box + lane * 32 + half * 16);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  unpack_codes<16>(w, scale, f);
}
// the same of a box of upper halves, with their third bytes
template <int UP>
__device__ __forceinline__ void held_values(uint32_t box, int lane, int half, const uint32_t (&third)[8], float (&f)[16]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 v = load_shared(box + lane * 64 + (((2 * half + i) ^ ((lane >> 1) & 3)) << 4));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 v = held24<UP>(w[j], third[4 * i + j]);
      f[8 * i + 2 * j] = v.x, f[8 * i + 2 * j + 1] = v.y;
    }
  }
}

// ---------------------------------------------------------------- the kernel
template <int EPI, int A_ORDER, bool B_MN, typename T, int ACT, int KEEP, int NJ>
__global__ void __launch_bounds__(THREADS, 1)
    ffn_pair_kernel(const __grid_constant__ Args<NJ> args) {
  using S = Shape<EPI, KEEP>;
  constexpr int STAGES = S::STAGES;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t staging = base + STAGES * STAGE_BYTES;
  Bars<STAGES>& bars = *reinterpret_cast<Bars<STAGES>*>(raw + (staging + EPI_WARPS * S::WARP_BYTES - smem_u32(raw)));
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t cta = cluster_rank(), rank = cta & 1u, leader = cta & ~1u;
  const int part = EPI == PLAIN ? (int)cta / 2 : 0, split = EPI == PLAIN ? args.split : 1;
  const int pair = blockIdx.x / 2 / split, pairs = gridDim.x / 2 / split;  // or cluster and clusters
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  if (threadIdx.x == 96) {  // of the first tile
    const Job& job = args.job[find_tile<NJ>(args, pair).job];
    tma_prefetch_desc(&job.a[0]);
    tma_prefetch_desc(&job.b[EPI == GATE_UP ? rank : 0]);
    if constexpr (EPI != GATE_UP) tma_prefetch_desc(&job.c[0]);
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.acc_full[i], 1);
      mbar_init(&bars.acc_empty[i], 2 * EPI_WARPS);
    }
    mbar_init(&bars.sums, 1);
    if constexpr (EPI == GRADS)
      for (int i = 0; i < EPI_WARPS * 3; ++i) mbar_init(&bars.kept_full[i / 3][i % 3], 1);
    fence_barrier_init();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem)),
                 "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // a product before this one may still be running

  if (warp == 0) {
    if (lane == 0) {  // loads of this CTA's halves of A and B
      int s = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = 0, t; ok && (t = tile_of<NJ>(args, pair, pairs, i)) >= 0; ++i) {
        const Tile tile = find_tile<NJ>(args, t);
        const Job& job = args.job[tile.job];
        const int m0 = tile.m * PAIR_M + (int)rank * CTA_M;
        const int n0 = EPI == GATE_UP ? tile.n * (PAIR_N / 2) : tile.n * PAIR_N + (int)rank * (PAIR_N / 2);
        const int last = (part + 1) * job.blocks / split;
        for (int kb = part * job.blocks / split; kb < last; ++kb) {
          if (!mbar_wait(&bars.empty[s], phase ^ 1, args.err, 61)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(&bars.full[s], 2 * STAGE_BYTES);
          const uint32_t full = in_cta(smem_u32(&bars.full[s]), leader);
          const int seg = kb >= job.blocks0, k = (seg ? kb - job.blocks0 : kb) * KB;
          const uint32_t a = base + s * STAGE_BYTES, b = a + OPERAND_BYTES;
          const CUtensorMap* ma = &job.a[seg];
          const CUtensorMap* mb = &job.b[EPI == GATE_UP ? (int)rank : seg];
          if (A_ORDER == ACROSS || (A_ORDER == BY_JOB && job.a_across)) {
            load_2d(a, ma, full, m0, k);
            load_2d(a + OPERAND_BYTES / 2, ma, full, m0 + 64, k);
          } else {
            load_2d(a, ma, full, k, m0);
          }
          if constexpr (B_MN) {
            load_2d(b, mb, full, n0, k);
            load_2d(b + OPERAND_BYTES / 2, mb, full, n0 + 64, k);
          } else {
            load_2d(b, mb, full, k, n0);
          }
          if (++s == STAGES) {
            s = 0;
            phase ^= 1;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && lane == 0) {  // products of the pair
      int s = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int t; ok && (t = tile_of<NJ>(args, pair, pairs, it)) >= 0; ++it) {
        const Tile tile = find_tile<NJ>(args, t);
        const int all = args.job[tile.job].blocks, blocks = (part + 1) * all / split - part * all / split, acc = it & 1;
        if (!mbar_wait(&bars.acc_empty[acc], ((it >> 1) & 1) ^ 1, args.err, 62)) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * PAIR_N;
        const bool across = A_ORDER == ACROSS || (A_ORDER == BY_JOB && args.job[tile.job].a_across);
        const uint32_t idesc = args.idesc | (across ? 1u << 15 : 0u);
        for (int kb = 0; kb < blocks; ++kb) {
          if (!mbar_wait(&bars.full[s], phase, args.err, 63)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = base + s * STAGE_BYTES, b = a + OPERAND_BYTES;
#pragma unroll
          for (int ks = 0; ks < KB / 16; ++ks) {
            // K along rows of 128 bytes: 16 values are 32 bytes on; across: 16 rows of 128 bytes
            const uint64_t da = across ? sw128_desc(a + ks * 2048, OPERAND_BYTES / 2, 1024) : sw128_desc(a + ks * 32, 16, 1024);
            const uint64_t db = B_MN ? sw128_desc(b + ks * 2048, OPERAND_BYTES / 2, 1024) : sw128_desc(b + ks * 32, 16, 1024);
            pair_mma(d, da, db, idesc, kb | ks);
          }
          pair_commit(&bars.empty[s], leader);
          if (++s == STAGES) {
            s = 0;
            phase ^= 1;
          }
        }
        if (ok) pair_commit(&bars.acc_full[acc], leader);
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int quad = warp % 4, side = (warp - 4) / 4;  // 32 rows, a share of the columns
    const uint32_t boxes = staging + (warp - 4) * S::WARP_BYTES;
    int it = 0, set = 0;
    // The backward's first epilogue: a warp's chunks of 32 columns are numbered through its tiles. What was
    // kept of the two or three after the present one is under way, in this tile or the next.
    constexpr int CHUNKS = S::COLS / 32;
    uint64_t* kept_full = bars.kept_full[warp - 4];
    const uint32_t kept_boxes = boxes + S::SETS * S::SET_BYTES;
    int rows[2] = {0, 0}, cols[2] = {0, 0};  // of this tile and the next
    bool more = pair < args.tiles;           // whether there is a next one
    auto look_ahead = [&](int t) {
      more = t < args.tiles;
      if (more) {
        const Tile tile = find_tile<NJ>(args, t);
        rows[1] = tile.m * PAIR_M + (int)rank * CTA_M + quad * 32;
        cols[1] = tile.n * PAIR_N + side * S::COLS;
      }
    };
    auto ask_kept = [&](int n, int c) {  // by lane 0: chunk number n, the c-th of this tile
      const bool next = c >= CHUNKS;
      if (next && !more) return;
      const int row = next ? rows[1] : rows[0], col = (next ? cols[1] - CHUNKS * 32 : cols[0]) + c * 32;
      const uint32_t to = kept_boxes + n % 3 * 2 * S::KEPT_BOX;
      mbar_arrive_expect_tx(&kept_full[n % 3], 2 * S::KEPT_BOX);
      load_own_2d(to, &args.kept_map[0], &kept_full[n % 3], col, row);
      load_own_2d(to + S::KEPT_BOX, &args.kept_map[1], &kept_full[n % 3], col, row);
    };
    // of codes the scales of a chunk, of 24 bits the third bytes of half of one, which are asked for a chunk ahead
    uint32_t sg = 127, su = 127, third[2][8] = {};
    auto ask_third = [&](int c, int half) {
      const bool next = c >= CHUNKS;
      const int64_t row = (next ? rows[1] : rows[0]) + lane, col = (next ? cols[1] - CHUNKS * 32 : cols[0]) + c * 32;
      if ((!next || more) && row < args.kept.T && col < args.kept.pitch)
        load_32b(third[half],
                 static_cast<const uint16_t*>(args.kept.p) + (2 * args.kept.T + row) * args.kept.pitch + col + 16 * half);
    };
    auto ask_scales = [&](int c) {
      const bool next = c >= CHUNKS;
      const int64_t row = (next ? rows[1] : rows[0]) + lane, group = ((next ? cols[1] - CHUNKS * 32 : cols[0]) + c * 32) / GROUP8;
      sg = su = 127;
      if ((!next || more) && row < args.kept.T && group < args.kept.pitch / GROUP8) {
        const uint8_t* at = args.kept.exps + group * args.kept.T + row;
        sg = __ldg(at);
        su = __ldg(at + args.kept.pitch / GROUP8 * args.kept.T);
      }
    };
    if constexpr (EPI == GRADS) {
      look_ahead(pair);
      if constexpr (KEEP == DSALT_KEEP_8BIT) {
        ask_scales(CHUNKS);
      } else {
        ask_third(CHUNKS, 0);
        ask_third(CHUNKS, 1);
      }
      if (lane == 0)
        for (int n = 0; n < (S::IN_PLACE ? 2 : 3); ++n) ask_kept(n, CHUNKS + n);
      __syncwarp();
    }
    for (int t; (t = tile_of<NJ>(args, pair, pairs, it)) >= 0; ++it) {
      const Tile tile = find_tile<NJ>(args, t);
      const Job& job = args.job[tile.job];
      const int acc = it & 1;
      const int row0 = tile.m * PAIR_M + (int)rank * CTA_M + quad * 32;
      const uint32_t ta = tmem + acc * PAIR_N + ((uint32_t)(quad * 32) << 16);
      // the next set of boxes, once the stores that read it are done
      auto next_boxes = [&]() {
        set = set + 1 == S::SETS ? 0 : set + 1;
        if (lane == 0) store_wait_read<(S::SETS > 0 ? S::SETS - 1 : 0)>();
        __syncwarp();
        return boxes + set * S::SET_BYTES;
      };
      auto send = [&](uint32_t to, int col) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (row0 < job.rows && col < job.cols)
#pragma unroll
            for (int i = 0; i < S::OUTPUTS; ++i) store_2d(&job.c[i], to + i * BOX_BYTES, col, row0);
          store_commit();
        }
      };
      const uint32_t mine = ta + side * S::COLS;
      auto acc_read = [&]() {  // the accumulator may be overwritten
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_remote(in_cta(smem_u32(&bars.acc_empty[acc]), leader));
      };
      if constexpr (EPI == GRADS) {
        rows[0] = rows[1], cols[0] = cols[1];
        look_ahead(t + pairs);
        if (!mbar_wait(&bars.acc_full[acc], (it >> 1) & 1, args.err, 64)) break;
        tc_fence_after();
        uint32_t r[32];
        ask_acc<32>(mine, r);
        bool ok = true;
#pragma unroll 1
        for (int c = 0; c < S::COLS; c += 32) {
          const int n = it * CHUNKS + c / 32;
          const uint32_t from = kept_boxes + n % 3 * 2 * S::KEPT_BOX;
          const float scale_g = scale_of(sg), scale_u = scale_of(su);
          if constexpr (KEEP == DSALT_KEEP_8BIT) ask_scales(c / 32 + 1);
          if (!(ok = mbar_wait(&kept_full[n % 3], n / 3 & 1, args.err, 65))) break;
          float d[32];
          take_acc<32>(r, d);
          if (c + 32 < S::COLS) ask_acc<32>(mine + c + 32, r);
          else acc_read();
          uint32_t to = from;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float a[16], b[16], e[16];
            if constexpr (KEEP == DSALT_KEEP_8BIT) {
              coded_values(from, lane, half, scale_g, a);
              coded_values(from + S::KEPT_BOX, lane, half, scale_u, b);
            } else {
              held_values<0>(from, lane, half, third[half], a);
              held_values<1>(from + S::KEPT_BOX, lane, half, third[half], b);
              ask_third(c / 32 + 1, half);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float v, dv;
              activate_grad<ACT, true>(a[i], v, dv);
              a[i] = d[16 * half + i] * b[i] * dv;
              b[i] *= v;
              e[i] = d[16 * half + i] * v;
            }
            if constexpr (!S::IN_PLACE)
              if (half == 0) to = next_boxes();
            stage_row<T, 16>(to, lane, a, 16 * half);
            stage_row<T, 16>(to + BOX_BYTES, lane, e, 16 * half);
            if constexpr (S::IN_PLACE) {
              const int64_t row = row0 + lane;
              if (row < args.kept.T && cols[0] + c < args.kept.pitch)
                store_row<T, 16>(static_cast<T*>(args.kept.h) + row * args.kept.pitch + cols[0] + c + 16 * half, b);
            } else {
              stage_row<T, 16>(to + 2 * BOX_BYTES, lane, b, 16 * half);
            }
          }
          send(to, cols[0] + c);
          if (lane == 0) {
            if constexpr (S::IN_PLACE) {
              store_wait_read<1>();  // the chunk before this one has left its boxes
              ask_kept(n + 2, c / 32 + 2);
            } else {
              ask_kept(n + 3, c / 32 + 3);  // every lane has read this one's
            }
          }
          __syncwarp();
        }
        if (!ok) break;
      } else if constexpr (EPI == GATE_UP) {
        if (!mbar_wait(&bars.acc_full[acc], (it >> 1) & 1, args.err, 64)) break;
        tc_fence_after();
        const int col = tile.n * (PAIR_N / 2) + side * S::COLS;
        const int64_t row = row0 + lane, at = row * args.kept.pitch + col, plane = args.kept.T * args.kept.pitch;
        uint32_t rg[32], ru[32];
        ask_acc<32>(mine, rg);
        ask_acc<32>(mine + PAIR_N / 2, ru);
#pragma unroll
        for (int half = 0; half < S::COLS / 32; ++half) {
          float g[32], u[32];
          take_acc<32>(rg, g);
          take_acc<32>(ru, u);
          if (half + 1 < S::COLS / 32) {
            ask_acc<32>(mine + 32, rg);
            ask_acc<32>(mine + PAIR_N / 2 + 32, ru);
          } else {
            acc_read();
          }
          const bool in = row < args.kept.T && col + 32 * half < args.kept.pitch;
          if constexpr (KEEP == DSALT_KEEP_8BIT) {
            uint32_t c[8];
            char* codes = static_cast<char*>(args.kept.p) + at + 32 * half;
            uint32_t s = scale_byte(largest_of(g));
            pack_codes<GROUP8>(g, s, c);
            if (in) {
              store_32b(codes, c);
              args.kept.exps[(col / GROUP8 + half) * args.kept.T + row] = (uint8_t)s;
            }
            s = scale_byte(largest_of(u));
            pack_codes<GROUP8>(u, s, c);
            if (in) {
              store_32b(codes + plane, c);
              args.kept.exps[((args.kept.pitch + col) / GROUP8 + half) * args.kept.T + row] = (uint8_t)s;
            }
          } else if constexpr (KEEP == DSALT_KEEP_INPUT) {
            uint16_t* to = static_cast<uint16_t*>(args.kept.p) + at + 32 * half;
#pragma unroll
            for (int i = 0; i < 32; i += 16) {
              uint32_t wg[8], wu[8], w3[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const int k = i + 2 * j;
                wg[j] = upper_halves(g[k], g[k + 1]);
                wu[j] = upper_halves(u[k], u[k + 1]);
                w3[j] = __byte_perm(third_bytes(g[k], u[k]), third_bytes(g[k + 1], u[k + 1]), 0x5410);
              }
              if (in) {
                store_32b(to + i, wg);
                store_32b(to + plane + i, wu);
                store_32b(to + 2 * plane + i, w3);
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) g[i] = activate<ACT, true>(g[i]) * u[i];
          if (in) store_row<T, 32>(static_cast<T*>(args.kept.h) + at + 32 * half, g);
        }
      } else {
        if (!mbar_wait(&bars.acc_full[acc], (it >> 1) & 1, args.err, 64)) break;
        tc_fence_after();
        const int col0 = tile.n * PAIR_N + side * S::COLS;
        uint32_t r[BOX];
        ask_acc<BOX>(mine, r);
#pragma unroll 1
        for (int c = 0; c < S::COLS; c += BOX) {
          float d[BOX];
          take_acc<BOX>(r, d);
          if (c + BOX < S::COLS) ask_acc<BOX>(mine + c + BOX, r);
          else acc_read();
          if (split > 1) {  // sums of this part of K, column by column, where the operands were
#pragma unroll
            for (int i = 0; i < BOX; ++i)
              asm volatile("st.shared.f32 [%0], %1;" ::"r"(base + (side * S::COLS + c + i) * SUMS_COL + (quad * 32 + lane) * 4),
                           "f"(d[i])
                           : "memory");
            continue;
          }
          const uint32_t to = next_boxes();
          stage_row<T, BOX>(to, lane, d, 0);
          send(to, col0 + c);
        }
      }
    }
    if (lane == 0) store_wait_read<0>();
    __syncwarp();
  }
  tc_fence_before();
  if constexpr (EPI == PLAIN) {
    if (split > 1) {
      // Each pair adds up and stores its share of the columns: the others' sums of it are copied over,
      // whole columns at a time, behind its own (threads that read them where they are took 7000 cycles).
      fence_proxy_async_smem();
      cluster_sync();  // every part has its sums, and no operand is read any more
      auto first = [&](int p) { return p * 32 / split; };  // groups of 8 columns
      const int lo = first(part), groups = first(part + 1) - lo;
      const uint32_t inbox = base + PAIR_N * SUMS_COL;
      if (threadIdx.x == 0) {
        mbar_arrive_expect_tx(&bars.sums, (split - 1) * groups * 8 * SUMS_COL);
        for (int p = 0; p < split; ++p)
          if (p != part) {
            const int n = first(p + 1) - first(p), place = part < p ? part : part - 1;
            copy_to_cta(in_cta(inbox + place * n * 8 * SUMS_COL, 2 * p + rank), base + first(p) * 8 * SUMS_COL, n * 8 * SUMS_COL,
                        in_cta(smem_u32(&bars.sums), 2 * p + rank));
          }
      }
      const Tile tile = find_tile<NJ>(args, pair);
      const Job& job = args.job[tile.job];
      const int row = warp % 4 * 32 + lane, m = tile.m * PAIR_M + (int)rank * CTA_M + row;
      if (mbar_wait(&bars.sums, 0, args.err, 60))
        for (int g = warp / 4; g < groups; g += THREADS / 128) {
          float v[8] = {};
          for (int p = 0; p < split; ++p) {  // in the order of the parts
            const uint32_t from =
                (p == part ? base + lo * 8 * SUMS_COL : inbox + (p < part ? p : p - 1) * groups * 8 * SUMS_COL) + row * 4;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              float x;
              asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(from + (g * 8 + i) * SUMS_COL) : "memory");
              v[i] += x;
            }
          }
          const int n = tile.n * PAIR_N + (lo + g) * 8;
          if (m < job.rows && n < job.cols)
            *reinterpret_cast<uint4*>(static_cast<T*>(job.out) + (int64_t)m * job.cols + n) = make_uint4(
                narrow2<T>(v[0], v[1]), narrow2<T>(v[2], v[3]), narrow2<T>(v[4], v[5]), narrow2<T>(v[6], v[7]));
        }
    }
  }
  __syncthreads();
  cluster_sync();  // the other CTAs' barriers, operands and sums are not touched after this
  if (warp == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
}

// ---------------------------------------------------------------- host side
// an operand: K along its rows (128 rows of 64 values of K), or across them (64 rows of K, 64 columns)
int operand(CUtensorMap* m, const void* p, const Ffn& f, int64_t rows, int64_t cols, int64_t stride, bool across) {
  return make_map(m, p, f.dtype, rows, cols, stride, across ? KB : CTA_M, 64);
}
int output(CUtensorMap* m, void* p, const Ffn& f, int64_t rows, int64_t cols, int64_t stride) {
  return make_map(m, p, f.dtype, rows, cols, stride, 32, BOX);
}
void size_job(Job& j, int64_t M, int64_t N, int64_t K, int tile_n) {
  j.tiles_m = ceil_div(M, PAIR_M);
  j.tiles_n = ceil_div(N, tile_n);
  j.blocks0 = j.blocks = ceil_div(K, KB);
  // Columns of tiles are walked once for every `group` of 256 rows. Where the walked operand (the first product's:
  // gate's and up's) is more than half of L2, it comes from memory each time, so that it should be seldom: 32768 x
  // 2048 -> 11008 in a row, which the power limit bounds, on one GPU 3.71 ms with 4, 3.61 with 8, 3.49 with 16, 3.55 with 24 (3.3
  // with 16 on others). Smaller ones stay in L2, and 4, which share A among more pairs, are as fast or faster (16384 x 1024 ->
  // 4096, training: 1105 us against 1125 with 16). Of x's gradient one of the two segments counts: with both, 16384 x
  // 2048 -> 11008, 16384 x 1536 -> 12288 and 8192 x 2048 -> 8192 would get 16, and their training steps take as long
  // (5.6, 5.1, 2.1 ms either way).
  j.group = N * K * (tile_n == PAIR_N ? 2 : 4) > HALF_L2 ? 16 : 4;
  j.rows = (int)M;
  j.cols = (int)N;
}

// Where a plain store's tiles leave half of the pairs idle, K is split over 2 to 4 pairs of a cluster, as far as
// all clusters run at once: of 4, 6 and 8 CTAs of this size the GPU holds 33, 22 and 15 (its processing
// clusters have odd numbers of SMs left over). 1999 x 768 -> 2048 (24 tiles of
// K = 2048 in the second product), both launches: one part 40 us, two 33, three 43.
int split_for(int tiles, int blocks) {
  constexpr int AT_ONCE[5] = {0, PAIRS, 33, 22, 15};
  int split = 1;
  while (split < 4 && tiles <= AT_ONCE[split + 1] && 4 * (split + 1) <= blocks) ++split;
  return split;
}
// blocks of K that the longest-working pair goes through
int64_t rounds_of(int tiles, int blocks) {
  const int split = split_for(tiles, blocks);
  return split > 1 ? ceil_div(blocks, split) : (int64_t)ceil_div(tiles, PAIRS) * blocks;
}

// Of the weights' and x's gradients, which differ in length: the longer tiles are dealt round robin, the shorter
// ones so that all pairs end together. (Two launches leave pairs idle at the end of each: 341 us against 332 at
// 32768 x 768 -> 2048.)
void deal(Args<4>& a) {
  const Job& x = a.job[a.job[0].a_across ? 3 : 0];
  const Job* first_w = a.job + (a.job[0].a_across ? 0 : 1);
  const Job& w = first_w[first_w->tiles_m ? 0 : 1];
  const int x_tiles = x.tiles_m * x.tiles_n, w_tiles = a.tiles - x_tiles;
  if (!x_tiles || !w_tiles) return;
  const bool x_first = &x == &a.job[0];
  // what a tile costs: its blocks of K and about eight more for its epilogue
  const int64_t first_cost = (x_first ? x : w).blocks + 8, cost = (x_first ? w : x).blocks + 8;
  a.dealt = x_first ? x_tiles : w_tiles;
  const int others = a.tiles - a.dealt;
  int64_t load[PAIRS], low = 0, high = 0;
  for (int p = 0; p < PAIRS; ++p) {
    load[p] = (p < a.dealt ? (a.dealt - p + PAIRS - 1) / PAIRS : 0) * first_cost;
    high = load[p] > high ? load[p] : high;
  }
  high += (others / PAIRS + 1) * cost;
  auto fits = [&](int64_t level, int p) { return level > load[p] ? (int)((level - load[p]) / cost) : 0; };
  while (low < high) {  // the lowest level at which all find a place
    const int64_t level = (low + high) / 2;
    int64_t n = 0;
    for (int p = 0; p < PAIRS; ++p) n += fits(level, p);
    if (n >= others) high = level;
    else low = level + 1;
  }
  int counts[PAIRS], left = -others;
  for (int p = 0; p < PAIRS; ++p) left += counts[p] = fits(low, p);
  for (int p = 0; left > 0; p = (p + 1) % PAIRS)
    if (counts[p] > 0) --counts[p], --left;
  a.rounds = counts[0];
  for (int p = 1; p < PAIRS; ++p) a.rounds = counts[p] < a.rounds ? counts[p] : a.rounds;
  for (int p = 0; p < PAIRS; ++p) a.extra[p + 1] = a.extra[p] + counts[p] - a.rounds;
}
template <int NJ>
void deal(Args<NJ>&) {}

// `after`: the launch before it in the stream is one of this call, whose end it may overlap
template <int EPI, int A_ORDER, bool B_MN, typename T, int ACT, int KEEP, int NJ>
int launch_pair(Args<NJ>& a, const Ffn& f, bool after, const char* what) {
  static std::atomic<uint64_t> ready{0};
  constexpr int bytes = Shape<EPI, KEEP>::SMEM_BYTES;
  static_assert(sizeof(Bars<6>) <= 512 && bytes <= 232448, "shared memory of a block");
  static_assert(EPI != PLAIN || bytes >= 1024 + 512 + (PAIR_N + 3 * PAIR_N / 4) * SUMS_COL, "the sums of a part do not fit");
  auto kernel = ffn_pair_kernel<EPI, A_ORDER, B_MN, T, ACT, KEEP, NJ>;
  if (int rc = allow_dynamic_smem(reinterpret_cast<const void*>(kernel), bytes, ready)) return rc;
  a.tiles = 0;
  for (int i = 0; i < NJ; ++i) a.tiles += a.job[i].tiles_m * a.job[i].tiles_n;
  if (a.split < 1) a.split = EPI == PLAIN ? split_for(a.tiles, a.job[0].blocks) : 1;
  a.idesc = umma_idesc_f16(f.dtype == DSALT_BF16 ? 1 : 0, 0, B_MN, PAIR_M, PAIR_N);
  a.dealt = a.tiles;
  if (NJ == 4 && a.split == 1 && a.tiles > PAIRS) deal(a);
  a.err = device_status_ptr();
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * a.split * (a.split > 1 || a.tiles < PAIRS ? a.tiles : PAIRS));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = f.stream;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2 * a.split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = after ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, a), what);
}

template <typename T, int ACT, int KEEP>
int gate_up(const Ffn& f) {
  Args<1> a{};
  Job& j = a.job[0];
  size_job(j, f.T, f.F, f.d, PAIR_N / 2);
  int rc;
  if ((rc = operand(&j.a[0], f.x, f, f.T, f.d, f.x_stride, false)) || (rc = operand(&j.b[0], f.w_gate, f, f.F, f.d, f.d, false)) ||
      (rc = operand(&j.b[1], f.w_up, f, f.F, f.d, f.d, false)))
    return rc;
  a.kept = {f.kept, f.exps, f.h, f.T, f.pitch};
  return launch_pair<GATE_UP, ALONG, false, T, ACT, KEEP, 1>(a, f, false, "gated_ffn gate and up launch");
}

template <typename T, int ACT>
int forward(const Ffn& f) {
  int rc = f.keep == DSALT_KEEP_NONE ? gate_up<T, ACT, DSALT_KEEP_NONE>(f)
           : f.keep == DSALT_KEEP_INPUT ? gate_up<T, ACT, DSALT_KEEP_INPUT>(f)
                                        : gate_up<T, ACT, DSALT_KEEP_8BIT>(f);
  if (rc) return rc;
  Args<1> a{};
  Job& j = a.job[0];
  size_job(j, f.T, f.d_out, f.F, PAIR_N);
  if ((rc = operand(&j.a[0], f.h, f, f.T, f.F, f.pitch, false)) ||
      (rc = operand(&j.b[0], f.w_down, f, f.d_out, f.F, f.F, false)) || (rc = output(&j.c[0], f.y, f, f.T, f.d_out, f.d_out)))
    return rc;
  j.out = f.y;
  return launch_pair<PLAIN, ALONG, false, T, 0, 0, 1>(a, f, true, "gated_ffn down launch");
}

template <typename T, int ACT, int KEEP>
int grads(const Ffn& f) {
  Args<1> a{};
  Job& j = a.job[0];
  size_job(j, f.T, f.F, f.d_out, PAIR_N);
  int rc;
  if ((rc = operand(&j.a[0], f.dy, f, f.T, f.d_out, f.dy_stride, false)) ||
      (rc = operand(&j.b[0], f.w_down, f, f.d_out, f.F, f.F, true)) || (rc = output(&j.c[0], f.dg, f, f.T, f.F, f.pitch)) ||
      (rc = output(&j.c[1], f.du, f, f.T, f.F, f.pitch)) || (KEEP == DSALT_KEEP_8BIT && (rc = output(&j.c[2], f.h, f, f.T, f.F, f.pitch))))
    return rc;
  a.kept = {f.kept, f.exps, f.h, f.T, f.pitch};
  for (int i = 0; i < 2; ++i) {
    const char* p = static_cast<const char*>(f.kept) + i * f.T * f.pitch * (KEEP == DSALT_KEEP_8BIT ? 1 : 2);
    if ((rc = KEEP == DSALT_KEEP_8BIT ? make_map(&a.kept_map[i], p, DTYPE_BYTES, f.T, f.pitch, f.pitch, 32, 32)
                                      : make_map(&a.kept_map[i], p, f.dtype, f.T, f.pitch, f.pitch, 32, BOX)))
      return rc;
  }
  return launch_pair<GRADS, ALONG, true, T, ACT, KEEP, 1>(a, f, false, "gated_ffn_bwd hidden gradients launch");
}

int weight_job(Job& j, const Ffn& f, const void* a, int64_t M, int64_t a_stride, const void* b, int64_t N, int64_t b_stride,
               void* c) {
  size_job(j, M, N, f.T, PAIR_N);
  j.a_across = 1;
  int rc;
  if ((rc = operand(&j.a[0], a, f, f.T, M, a_stride, true)) || (rc = operand(&j.b[0], b, f, f.T, N, b_stride, true))) return rc;
  j.out = c;
  return output(&j.c[0], c, f, M, N, N);
}

template <typename T, int ACT>
int backward(const Ffn& f) {
  int rc = f.keep == DSALT_KEEP_8BIT ? grads<T, ACT, DSALT_KEEP_8BIT>(f) : grads<T, ACT, DSALT_KEEP_INPUT>(f);
  if (rc) return rc;
  if (!f.dx && !f.dw_gate && !f.dw_down) return DSALT_OK;
  // x's gradient, of 2 d_ff, and the weights', of T values of K: in one launch, the longer ones first, or in two
  // where the few long tiles of one would outlast the rest. That and the cut of K, and with it the sums' order,
  // are the same whichever gradients are wanted.
  const int x_blocks = 2 * ceil_div(f.F, KB), w_blocks = ceil_div(f.T, KB), F_tiles = ceil_div(f.F, PAIR_N);
  const int x_tiles = ceil_div(f.T, PAIR_M) * ceil_div(f.d, PAIR_N);
  const int w_tiles = ceil_div(f.d_out, PAIR_M) * F_tiles + 2 * F_tiles * ceil_div(f.d, PAIR_N);
  const int tiles = x_tiles + w_tiles, longest = x_blocks > w_blocks ? x_blocks : w_blocks;
  const int split = split_for(tiles, x_blocks < w_blocks ? x_blocks : w_blocks);
  const int64_t even = ((int64_t)x_tiles * x_blocks + (int64_t)w_tiles * w_blocks) / PAIRS;
  const int64_t one = split > 1 ? ceil_div(longest, split) : tiles > PAIRS && even > longest ? even : longest;
  const bool together = one <= rounds_of(x_tiles, x_blocks) + rounds_of(w_tiles, w_blocks) + 16;  // 16: a launch
  const bool x_first = x_blocks > w_blocks;
  for (int launch = 0; launch < (together ? 1 : 2); ++launch) {
    Args<4> a{};
    const bool xs = f.dx && (together || launch == 0), ws = (f.dw_down || f.dw_gate) && (together || launch == 1);
    if (!xs && !ws) continue;
    a.split = together ? split : launch == 0 ? split_for(x_tiles, x_blocks) : split_for(w_tiles, w_blocks);
    Job* w = a.job + (x_first ? 1 : 0);
    for (int i = 0; i < 3; ++i) w[i].a_across = 1;
    if (xs) {
      Job& j = a.job[x_first ? 0 : 3];
      size_job(j, f.T, f.d, f.F, PAIR_N);
      j.blocks = 2 * j.blocks0;
      j.out = f.dx;
      if ((rc = operand(&j.a[0], f.dg, f, f.T, f.F, f.pitch, false)) || (rc = operand(&j.a[1], f.du, f, f.T, f.F, f.pitch, false)) ||
          (rc = operand(&j.b[0], f.w_gate, f, f.F, f.d, f.d, true)) || (rc = operand(&j.b[1], f.w_up, f, f.F, f.d, f.d, true)) ||
          (rc = output(&j.c[0], f.dx, f, f.T, f.d, f.d)))
        return rc;
    }
    if (ws && f.dw_down && (rc = weight_job(w[0], f, f.dy, f.d_out, f.dy_stride, f.h, f.F, f.pitch, f.dw_down))) return rc;
    if (ws && f.dw_gate && ((rc = weight_job(w[1], f, f.dg, f.F, f.pitch, f.x, f.d, f.x_stride, f.dw_gate)) ||
                            (rc = weight_job(w[2], f, f.du, f.F, f.pitch, f.x, f.d, f.x_stride, f.dw_up))))
      return rc;
    if ((rc = launch_pair<PLAIN, BY_JOB, true, T, 0, 0, 4>(a, f, true, "gated_ffn_bwd gradients launch"))) return rc;
  }
  return DSALT_OK;
}

template <typename T>
int run_typed(const Ffn& f, bool back) {
  if (f.act == DSALT_ACT_SILU) return back ? backward<T, DSALT_ACT_SILU>(f) : forward<T, DSALT_ACT_SILU>(f);
  return back ? backward<T, DSALT_ACT_GELU>(f) : forward<T, DSALT_ACT_GELU>(f);
}

}  // namespace

int run_tensor_cores(const Ffn& f, bool back) {
  // the tensor maps are made by the driver, which wants the thread's context: a thread that autograd
  // started has the device set, but no context until the runtime is told so
  int dev = 0;
  int rc;
  if ((rc = check_cuda(cudaGetDevice(&dev), "current device")) || (rc = check_cuda(cudaSetDevice(dev), "current device"))) return rc;
  // Measured (us in a row, weights not in L2), a stream past tokens | tiles for few tokens | this file, at
  //   512 -> 1408:   256 tokens - | 12.7 | 20; 1024 tokens - | 15.6 | 21; 1536 - | 19 | 22; 2560 - | 27 | 25
  //   768 -> 2048:   16 tokens 7.5 | 11.7 | 21; 64 tokens - | 12.6 | 21; 256 - | 15.6 | 23; 1024 - | 22 | 25; 1536 - | 31 | 28
  //   1024 -> 4096:  16 tokens 10.4 | 14.8 | 25; 64 tokens - | 15.9 | 26; 256 - | 20 | 26; 512 - | 24 | 28; 896 - | 42 | 35
  //   2048 -> 5504:  64 tokens - | 24 | 34; 256 - | 32 | 35; 384 - | 39 | 46; 544 - | 61 | 49
  //   2048 -> 11008: 16 tokens 36 | 29.7 | 54; 64 tokens - | 33 | 54; 192 - | 45 | 54; 224 - | 58 | 54
  //   4096 -> 28672: 64 tokens - | 131 | 169; 128 - | 139 | 170; 160 - | 175 | 171
  // Nine to sixteen tokens, stream | tiles by millions of weights: 19 M 12.7 | 17.0, 25 M 14.4 | 20.0 (d_ff = 2 d) and 18.6 | 19.2,
  // 34 M 21.6 | 22.2, 41 M 23.5 | 23.7 (16 tokens 24.4 | 24.0), 53 M 33 | 27.5: they meet at 40 M. The tiles for few tokens win
  // over this file's while their CTAs run at once, two an SM with some 128 tokens each: that is T d_ff (measured for d_ff
  // of 2.7 to 7 times d only).
  if (!back && f.keep == DSALT_KEEP_NONE) {
    const int64_t weights = (int64_t)f.F * (2 * f.d + f.d_out);
    if (f.T <= 8 || (f.T <= 16 && weights <= 40000000)) return forward_tokens(f);
    if (f.T <= 128 || (f.T <= 2048 && f.T * f.F <= 2300000)) return forward_few(f);
  }
  return f.dtype == DSALT_BF16 ? run_typed<__nv_bfloat16>(f, back) : run_typed<__half>(f, back);
}

}  // namespace ffn
}  // namespace dsalt
