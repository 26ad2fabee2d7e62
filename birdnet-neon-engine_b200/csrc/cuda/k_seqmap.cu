// Host side of tc16.cuh: the TMA maps of the operators over sequences.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <mutex>

#include "tc16.cuh"

static PFN_cuTensorMapEncodeTiled_v12000 seq_encode_fn(void) {
  static std::once_flag once;
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  std::call_once(once, [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult qr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qr) == cudaSuccess &&
        qr == cudaDriverEntryPointSuccess)
      fn = (PFN_cuTensorMapEncodeTiled_v12000)p;
  });
  return fn;
}

int bnn::encode_heads(CUtensorMap *m, const void *base, int bf16, int width, int heads, long long rows, long long rs,
                      int box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = seq_encode_fn();
  if (!enc) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {(cuuint64_t)width, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)width * 2, (cuuint64_t)rs * 2};
  const cuuint32_t box[3] = {64, 1, (cuuint32_t)box_rows}, es[3] = {1, 1, 1};
  return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(base),
             dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
             ? cudaErrorInvalidValue
             : 0;
}

int bnn::encode_rows16(CUtensorMap *m, const void *base, int bf16, int width, long long rows, long long rs, int box_w,
                       int box_rows, int sw) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = seq_encode_fn();
  if (!enc) return cudaErrorNotSupported;
  const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)rs * 2};
  const cuuint32_t box[2] = {(cuuint32_t)box_w, (cuuint32_t)box_rows}, es[2] = {1, 1};
  return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(base),
             dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             sw == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : sw == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
             ? cudaErrorInvalidValue
             : 0;
}

int bnn::encode_slots16(CUtensorMap *m, const void *base, int bf16, int width, int rows, int slots, int box_w,
                        int box_rows) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = seq_encode_fn();
  if (!enc) return cudaErrorNotSupported;
  const cuuint64_t dims[3] = {(cuuint64_t)width, (cuuint64_t)rows, (cuuint64_t)slots};
  const cuuint64_t strides[2] = {(cuuint64_t)width * 2, (cuuint64_t)width * 2 * rows};
  const cuuint32_t box[3] = {(cuuint32_t)box_w, (cuuint32_t)box_rows, 1}, es[3] = {1, 1, 1};
  return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(base),
             dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             box_w == 64   ? CU_TENSOR_MAP_SWIZZLE_128B
             : box_w == 32 ? CU_TENSOR_MAP_SWIZZLE_64B
             : box_w == 16 ? CU_TENSOR_MAP_SWIZZLE_32B
                           : CU_TENSOR_MAP_SWIZZLE_NONE,
             CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE)
             ? cudaErrorInvalidValue
             : 0;
}
