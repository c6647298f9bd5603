// Products of groups of rows that an index picks (rows_kernel.cuh).
#include "rows_kernel.cuh"

namespace sb {

cudaError_t rows_gathered_configure() {
    const cudaError_t e = rows_set_all<false, kGathered>();
    return e != cudaSuccess ? e : rows_set_all<true, kGathered>();
}

cudaError_t rows_gathered_launch(const RowsArgs& g, RowsTileShape t, int sm_count, int* d_error, cudaStream_t stream) {
    return g.fp8 ? rows_pick<true, kGathered>(g, t, sm_count, d_error, stream) : rows_pick<false, kGathered>(g, t, sm_count, d_error, stream);
}

}  // namespace sb
