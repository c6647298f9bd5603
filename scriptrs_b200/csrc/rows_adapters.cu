// Products with low-rank adapters (rows_kernel.cuh).
#include "rows_kernel.cuh"

namespace sb {

cudaError_t rows_adapters_configure() { return rows_set_all<false, kAdapters>(); }

cudaError_t rows_adapters_launch(const RowsArgs& g, RowsTileShape t, int sm_count, int* d_error, cudaStream_t stream) {
    return rows_pick<false, kAdapters>(g, t, sm_count, d_error, stream);
}

}  // namespace sb
