// Tensor-map encoding through the driver entry point (no link-time
// dependency on libcuda).
#include <cudaTypedefs.h>

#include "decode.h"
#include "tma.h"

namespace wgx {

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  if (!fn) {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q{};
    check_cuda(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q),
               "cuTensorMapEncodeTiled entry point");
    if (q != cudaDriverEntryPointSuccess || !p) fail("cuTensorMapEncodeTiled is unavailable");
    fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }
  return fn;
}

void encode_nchw_tmap(CUtensorMap *map, const void *base, int B, int C, int HW, int box_c) {
  if ((reinterpret_cast<uintptr_t>(base) & 15) || HW % 8 || box_c < 1 || box_c > 256)
    fail("conv2d: tensor map needs a 16-byte aligned base and HW % 8 == 0");
  const cuuint64_t dims[3] = {cuuint64_t(HW), cuuint64_t(C), cuuint64_t(B)};
  const cuuint64_t strides[2] = {cuuint64_t(HW) * 2, cuuint64_t(C) * HW * 2};
  const cuuint32_t box[3] = {64, cuuint32_t(box_c), 1};
  const cuuint32_t estride[3] = {1, 1, 1};
  const CUresult r = encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(base),
                                 dims, strides, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) fail("conv2d: cuTensorMapEncodeTiled failed (" + std::to_string(int(r)) + ")");
}

bool encode_rows_tmap(CUtensorMap *map, const void *base, const wgx_kv_cache &c, int64_t page_stride,
                      int64_t head_stride, int64_t slot_stride, int panels, int rows) {
  const bool half = c.dtype == WGX_FLOAT16;
  const int64_t es = half ? 2 : 4, panel = 128 / es;
  const cuuint64_t dims[5] = {cuuint64_t(panels > 1 ? panel : c.head_dim), cuuint64_t(c.page_size),
                              cuuint64_t(panels), cuuint64_t(c.kv_heads), cuuint64_t(c.pages)};
  const int64_t bytes[4] = {slot_stride * es, 128, head_stride * es, page_stride * es};
  cuuint64_t strides[4];
  for (int i = 0; i < 4; ++i) {
    // (an extent of one is never stepped over: any stride will do)
    const int64_t s = dims[i + 1] == 1 ? 128 : bytes[i];
    if (s <= 0 || s % 16 || s >= int64_t(1) << 40) return false;
    strides[i] = cuuint64_t(s);
  }
  const cuuint32_t box[5] = {cuuint32_t(panel), cuuint32_t(rows), cuuint32_t(panels), 1, 1};
  const cuuint32_t estride[5] = {1, 1, 1, 1, 1};
  return encode_fn()(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 5,
                     const_cast<void *>(base), dims, strides, box, estride, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace wgx
