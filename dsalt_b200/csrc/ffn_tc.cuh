// Shared by the tensor-core kernels of the gated feed-forward block: clusters, accumulators, tensor maps.
#pragma once

#include <cuda.h>

#include "ffn.cuh"

namespace dsalt {
namespace ffn {

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t in_cta(uint32_t smem_addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// N columns of the accumulator, in flight until take_acc
template <int N>
__device__ __forceinline__ void ask_acc(uint32_t taddr, uint32_t (&r)[N]) {
  if constexpr (N == 32) {
    DSALT_TMEM_LD32(taddr, r);
  } else {
    DSALT_TMEM_LD16(taddr, r);
  }
}
// waits for what was asked; the registers pass through the wait, so that nothing reads them before it
template <int N>
__device__ __forceinline__ void take_acc(uint32_t (&r)[N], float (&f)[N]) {
  if constexpr (N == 32) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
  } else {
    static_assert(N == 16, "16 or 32 columns");
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
  }
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = __uint_as_float(r[i]);
}
// load into this CTA's shared memory, counted on its own barrier
__device__ __forceinline__ void load_own_2d(uint32_t dst, const void* map, uint64_t* bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
          dst),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}
inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn get_encode() {
  static const EncodeTiledFn fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
                    q == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<EncodeTiledFn>(ptr) : nullptr;
  }();
  return fn;
}

// rows x cols values of 16 bits, `stride` values from row to row, in boxes of box_rows x box_cols (as wide as
// the swizzle: 64 or 32 columns), or DTYPE_BYTES in boxes of 32 columns without a swizzle
constexpr int DTYPE_BYTES = -1;
inline int make_map(CUtensorMap* m, const void* p, int dtype, int64_t rows, int64_t cols, int64_t stride, int box_rows,
                    int box_cols) {
  const EncodeTiledFn enc = get_encode();
  if (!enc) return fail(DSALT_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const bool bytes = dtype == DTYPE_BYTES;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)stride * (bytes ? 1 : 2)};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  const cuuint32_t step[2] = {1, 1};
  const CUresult r = enc(m,
                         bytes                 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                         : dtype == DSALT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                               : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                         2, const_cast<void*>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         bytes            ? CU_TENSOR_MAP_SWIZZLE_NONE
                         : box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B
                                          : CU_TENSOR_MAP_SWIZZLE_64B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(DSALT_ERR_CUDA, "gated_ffn: cuTensorMapEncodeTiled failed (%d)", (int)r);
  return DSALT_OK;
}
}  // namespace ffn
}  // namespace dsalt
