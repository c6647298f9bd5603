// Dispatch of the products whose weights a row chooses (rows_kernel.cuh; one file per form, so that they compile side by side).
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "gemm_tile.h"
#include "rows.h"

namespace sb {

namespace {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn g_rows_encode = nullptr;

}  // namespace

bool rows_map(CUtensorMap* map, const void* ptr, int64_t rows, int64_t cols, int64_t pitch, bool fp8, int box_rows) {
    const int eb = fp8 ? 1 : 2;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)pitch * eb};
    const cuuint32_t box[2] = {(cuuint32_t)(128 / eb), (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return g_rows_encode(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides,
                         box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool rows_out_map(CUtensorMap* map, void* ptr, int64_t rows, int64_t cols, int64_t pitch, bool f32, int row_bytes) {
    const int eb = f32 ? 4 : 2;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)pitch * eb};
    const cuuint32_t box[2] = {(cuuint32_t)(row_bytes / eb), 32};
    const cuuint32_t estr[2] = {1, 1};
    return g_rows_encode(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, ptr, dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, row_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

cudaError_t rows_configure(const char** why) {
    if (!g_rows_encode) {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
        if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !fn) {
            if (why) *why = "cuTensorMapEncodeTiled is not available from the driver";
            return e != cudaSuccess ? e : cudaErrorNotSupported;
        }
        g_rows_encode = reinterpret_cast<EncodeTiledFn>(fn);
    }
    for (cudaError_t (*set)() : {rows_grouped_configure, rows_gathered_configure, rows_adapters_configure, rows_few_configure, adapter_down_configure}) {
        const cudaError_t e = set();
        if (e != cudaSuccess) {
            if (why) *why = "shared-memory opt-in for the row products failed";
            return e;
        }
    }
    return cudaSuccess;
}

cudaError_t rows_launch(const RowsArgs& g, int sm_count, int* d_error, cudaStream_t stream) {
    if (!g_rows_encode) return cudaErrorNotReady;
    if (g.M <= 0) return cudaSuccess;
    // few rows a group: gathers fetch only those, a box always 128
    const bool picked = g.rows || (int64_t)g.M < (int64_t)g.n_groups * 64;
    const RowsTileShape t = rows_tile(g.M, g.N, g.n_groups, g.out_mode != kOutBf16, picked, sm_count);
    if (rows_few(g)) return rows_few_launch(g, t, sm_count, d_error, stream);
    if (g.row_adapter) return rows_adapters_launch(g, t, sm_count, d_error, stream);
    if (picked) return rows_gathered_launch(g, t, sm_count, d_error, stream);
    return rows_grouped_launch(g, t, sm_count, d_error, stream);
}

}  // namespace sb
