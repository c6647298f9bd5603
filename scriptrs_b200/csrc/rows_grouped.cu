// Products of groups of rows (rows_kernel.cuh).
#include "rows_kernel.cuh"

namespace sb {

cudaError_t rows_grouped_configure() {
    const cudaError_t e = rows_set_all<false, kGrouped>();
    return e != cudaSuccess ? e : rows_set_all<true, kGrouped>();
}

cudaError_t rows_grouped_launch(const RowsArgs& g, RowsTileShape t, int sm_count, int* d_error, cudaStream_t stream) {
    return g.fp8 ? rows_pick<true, kGrouped>(g, t, sm_count, d_error, stream) : rows_pick<false, kGrouped>(g, t, sm_count, d_error, stream);
}

}  // namespace sb
