// Products whose weights a row chooses: grouped products (rows.cu), the adapters' down-projection (adapter_down.cu), and
// the router with the weighted sum of the experts' rows (route.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "rows_tile.h"

namespace sb {

struct RowsArgs {
    const void* a;            // [a_rows x K], pitch lda elements, bf16 (e4m3 when fp8)
    const int32_t* rows;      // [M] the row of `a` behind each output row, or null: row i behind output row i
    const void* w;            // [n_groups x N x K], same type
    const float* bias;        // [n_groups x N] or null
    const float* row_scale;   // fp8: [a_rows] or null
    const float* col_scale;   // fp8: [n_groups x N] or null
    const int32_t* offsets;   // [n_groups + 1]; null: one group of M rows
    void* out;                // [M x N], pitch ldo elements
    int64_t a_rows, lda, ldo;
    int M, N, K, n_groups;
    int act, out_mode;
    float alpha;
    bool fp8;
    // low-rank addition (one group, bf16): low[i] U_a^T for the adapter a of row i
    const int32_t* row_adapter;  // [M], ids outside [0, n_adapters): none; null: no adapters
    const void* up;              // [n_adapters x N x rank] bf16
    const float* low;            // [M x rank] f32, scaled; written by the kernel ahead in the stream
    int n_adapters, rank;
};

cudaError_t rows_configure(const char** why);
// cudaErrorInvalidValue: a tensor map was refused (alignment or size).
cudaError_t rows_launch(const RowsArgs& g, int sm_count, int* d_error, cudaStream_t stream);
// 2-D row-major tensor; boxes of 128 bytes x box_rows, 128-byte swizzle.
bool rows_map(CUtensorMap* map, const void* ptr, int64_t rows, int64_t cols, int64_t pitch, bool fp8, int box_rows);
// The result's map: boxes of 32 rows x row_bytes (64 or 128, swizzled over as many).
bool rows_out_map(CUtensorMap* map, void* ptr, int64_t rows, int64_t cols, int64_t pitch, bool f32, int row_bytes);
// The forms of the kernel (rows_grouped.cu, rows_gathered.cu, rows_adapters.cu, rows_few.cu).
cudaError_t rows_few_configure();
bool rows_few(const RowsArgs& g);
cudaError_t rows_few_launch(const RowsArgs& g, RowsTileShape t, int sm_count, int* d_error, cudaStream_t stream);
cudaError_t rows_grouped_configure();
cudaError_t rows_gathered_configure();
cudaError_t rows_adapters_configure();
cudaError_t rows_grouped_launch(const RowsArgs& g, RowsTileShape t, int sm_count, int* d_error, cudaStream_t stream);
cudaError_t rows_gathered_launch(const RowsArgs& g, RowsTileShape t, int sm_count, int* d_error, cudaStream_t stream);
cudaError_t rows_adapters_launch(const RowsArgs& g, RowsTileShape t, int sm_count, int* d_error, cudaStream_t stream);

struct AdapterDownArgs {
    const void* a;    // [M x K] bf16, pitch lda
    const void* down; // [n_adapters x rank x K] bf16
    const float* scale;  // [n_adapters] or null
    const int32_t* row_adapter;
    float* low;          // [M x rank]
    int64_t lda;
    int M, K, rank, n_adapters;
};
cudaError_t adapter_down_configure();
cudaError_t adapter_down_launch(const AdapterDownArgs& g, int sm_count, int* d_error, cudaStream_t stream);

struct RouteArgs {
    const void* logits;  // [rows x n_experts], pitch ld
    int64_t ld;
    int rows, n_experts, top_k;
    bool bf16, normalize;
    bool vec;  // rows and their parts lie on 16-byte boundaries (set by route_launch)
    int32_t *experts, *offsets, *order, *slots;
    float* weights;
    int32_t* work;
};
cudaError_t route_configure();
int64_t route_work_bytes(int64_t rows, int64_t n_experts, int64_t top_k);
cudaError_t route_launch(const RouteArgs& g, cudaStream_t stream, int64_t* launches);

struct CombineArgs {
    const void* y;  // [y_rows x cols], pitch ldy, bf16 or f32
    const int32_t* slots;
    const float* weights;  // or null: ones
    void* out;             // [rows x cols], pitch ldo
    int64_t ldy, ldo, y_rows;
    int rows, top_k, cols, out_mode;
    bool y_f32;
    float alpha;
};
cudaError_t combine_launch(const CombineArgs& g, cudaStream_t stream);

}  // namespace sb
