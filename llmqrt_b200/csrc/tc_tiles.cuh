// What the tcgen05 GEMMs share besides the instructions: cluster ranks, stores, tile order, tensor maps.
#pragma once
#include <mutex>

#include "tc_primitives.cuh"

namespace llmqrt {
namespace {

constexpr int kRowBytes = 128;     // bytes of K per stage row (one swizzle span)

__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// 32 bytes from registers to global memory (an address that is a multiple of 32): every lane writes a whole sector.
__device__ __forceinline__ void st_global_256(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
               "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// A 2-D tile from shared memory to global memory; the issuing thread's stores are counted in bulk groups.
__device__ __forceinline__ void tma_store_2d(const void* tensor_map, uint32_t src_smem, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];\n\t"
               "cp.async.bulk.commit_group;" ::"l"(tensor_map), "r"(src_smem), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void tma_stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Tile order: the weight tiles are walked in groups of kPairGroup; inside a group the token tile
// changes fastest.  The clusters that run at the same time then share a few weight tiles and a few
// token tiles, and a weight group (8 x 256 rows) stays in L2 until every token tile has used it -- with
// the weight tile changing fastest instead, a weight matrix larger than L2 (gate_up of Qwen2-7B: 136 MB)
// is streamed from HBM once per token tile.
constexpr int kPairGroup = 8;
__device__ __forceinline__ void pair_tile_coords(int tile, int tiles_p, int tiles_q, int& tp, int& tq) {
  const int per_group = tiles_p * kPairGroup;
  const int group = tile / per_group, within = tile - group * per_group;
  const int gw = min(kPairGroup, tiles_q - group * kPairGroup);         // weight tiles in this group
  tp = within / gw;
  tq = group * kPairGroup + within - tp * gw;
}

// ---- host side -------------------------------------------------------------------------------

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_tiled_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// 2-D K-major operand [rows, K] with `ld` elements between rows; box = 128 bytes x box_rows.
inline int make_operand_map(CUtensorMap* map, const void* base, int elt_bytes, int64_t rows, int64_t K, int64_t ld,
                     int box_rows) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return set_error(LLMQRT_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)(ld * elt_bytes)};
  cuuint32_t box[2] = {(cuuint32_t)(kRowBytes / elt_bytes), (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, elt_bytes == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2,
                  const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(LLMQRT_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", (int)r);
  return LLMQRT_OK;
}

// 2-D output [rows, cols] with `ld` elements between rows; box = 128 bytes x 32 rows, the two-CTA kernel's staging tile.
inline int make_output_map(CUtensorMap* map, void* base, int elt_bytes, int64_t rows, int64_t cols, int64_t ld) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return set_error(LLMQRT_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)(ld * elt_bytes)};
  cuuint32_t box[2] = {(cuuint32_t)(128 / elt_bytes), 32};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(map, elt_bytes == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, base, dims, strides, box,
                  estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(LLMQRT_ERR_CUDA, "cuTensorMapEncodeTiled (output) failed with code %d", (int)r);
  return LLMQRT_OK;
}

}  // namespace
}  // namespace llmqrt
