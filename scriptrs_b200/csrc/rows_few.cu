// Products of at most 32 rows: groups of rows, picked by an index or not, and rows with low-rank adapters (rows_kernel.cuh).
#include "rows_kernel.cuh"

namespace sb {

cudaError_t rows_few_configure() {
    cudaError_t e = rows_set_all<false, kFewGathered>();
    if (e == cudaSuccess) e = rows_set_all<true, kFewGathered>();
    return e != cudaSuccess ? e : rows_set_all<false, kFewAdapters>();
}

bool rows_few(const RowsArgs& g) { return g.M <= kFewRows; }

cudaError_t rows_few_launch(const RowsArgs& g, RowsTileShape t, int sm_count, int* d_error, cudaStream_t stream) {
    if (g.row_adapter) return rows_pick<false, kFewAdapters>(g, t, sm_count, d_error, stream);
    return g.fp8 ? rows_pick<true, kFewGathered>(g, t, sm_count, d_error, stream) : rows_pick<false, kFewGathered>(g, t, sm_count, d_error, stream);
}

}  // namespace sb
