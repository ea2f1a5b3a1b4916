// Tensor maps for TMA loads (the driver's encoder, looked up at run time so the library links against cudart only).
#pragma once
#include <cuda.h>
#include <cuda_runtime_api.h>

#include <atomic>
#include <cstdint>

namespace mkb {

// 16-bit values [rows][heads][width], rows `ld` values apart, heads `width` apart: boxes of `box_rows` rows of `box_heads`
// heads of `box_width` values, 128-byte swizzle, zeros outside. base 16-byte aligned, ld % 8 == 0. 0 or a CUDA error.
inline int make_map3(CUtensorMap* map, bool bf16, const void* base, int width, int heads, int64_t rows, int64_t ld,
                     int box_width, int box_rows, int box_heads = 1) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<Encode> known{nullptr};  // calls from several host threads may look it up at once
  Encode encode = known.load(std::memory_order_acquire);
  if (!encode) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found);
    if (e != cudaSuccess) return e;
    if (found != cudaDriverEntryPointSuccess || !f) return cudaErrorNotSupported;
    encode = reinterpret_cast<Encode>(f);
    known.store(encode, std::memory_order_release);
  }
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(width), static_cast<cuuint64_t>(heads),
                              static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(width) * 2, static_cast<cuuint64_t>(ld) * 2};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(box_width), static_cast<cuuint32_t>(box_heads),
                             static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t step[3] = {1, 1, 1};
  const CUresult r = encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                            const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : static_cast<int>(cudaErrorInvalidValue);
}

}  // namespace mkb
