// extern "C" layer: products whose weights a row chooses.
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "context.h"
#include "gemm_tile.h"
#include "rows.h"

using namespace sb;

namespace {

bool off_boundary(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) != 0; }

constexpr int64_t kLimit = INT32_MAX;
constexpr int64_t kMaxRank = 128, kMaxRouteExperts = 1024, kMaxRouteTopK = 16;

bool route_sizes(int64_t rows, int64_t n_experts, int64_t top_k) {
    return rows >= 0 && n_experts > 0 && n_experts <= kMaxRouteExperts && top_k > 0 && top_k <= kMaxRouteTopK && top_k <= n_experts && rows <= kLimit / top_k;
}
bool adapter_rank(int64_t rank) { return rank > 0 && rank <= kMaxRank && rank % 8 == 0; }

// Sets up the kernels that an entry point may launch, in its first call on a context: loading them takes 12 ms in the first context of a
// process, which one that only transcribes does not pay.  The call may be one that is captured: nothing here is work on a stream, so this
// thread steps out of the capture's checks meanwhile.
template <typename Fn>
int32_t set_up(bool* ready, Fn configure) {
    if (*ready) return SB_OK;
    const char* why = nullptr;
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    SB_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
    const cudaError_t e = configure(&why);
    SB_CUDA(cudaThreadExchangeStreamCaptureMode(&mode));
    if (e != cudaSuccess) return fail(SB_CUDA_ERROR, std::string("row product set-up failed: ") + (why ? why : cudaGetErrorString(e)));
    *ready = true;
    return SB_OK;
}

// What the product entry points share.  (The context is looked at last, so that the arguments' checks need no GPU.)
int32_t check_product(const void* d_a, int64_t lda, const void* d_w, const float* d_bias, const void* d_out, int64_t ldo,
                      int64_t M, int64_t N, int64_t K, int64_t groups, bool fp8, int32_t act, int32_t out_mode) {
    if (M < 0 || N <= 0 || K <= 0 || groups <= 0 || M > kLimit - 512 || N > kLimit / 2 || K > kLimit / 2 || groups > kLimit - 512 || groups > kLimit / N)
        return fail(SB_INVALID_ARGUMENT, "bad product shape");
    // tiles of 128 rows x 32 columns are counted in 32 bits
    if ((M / 128 + 1) * (N / 32 + 1) > (int64_t)1 << 25) return fail(SB_INVALID_ARGUMENT, "the result is too large for one call");
    if (act < 0 || act > 2 || out_mode < 0 || out_mode > 2) return fail(SB_INVALID_ARGUMENT, "unknown activation or output mode");
    if (M == 0) return SB_OK;
    if (!d_a || !d_w || !d_out) return fail(SB_INVALID_ARGUMENT, "null argument");
    const int eb = fp8 ? 1 : 2;
    if (K % (16 / eb) || lda < K || (lda * eb) % 16 || lda > ((int64_t)1 << 39) || ldo < N)
        return fail(SB_INVALID_ARGUMENT, "K and the row pitches do not fit: K and lda in whole 16 bytes, lda >= K, ldo >= N");
    if (off_boundary(d_a, 16) || off_boundary(d_w, 16) || off_boundary(d_out, out_mode ? 4 : 2) || off_boundary(d_bias, 4))
        return fail(SB_INVALID_ARGUMENT, "operands lie on 16-byte boundaries, the result and the bias on those of their type");
    return SB_OK;
}

}  // namespace

extern "C" {

int64_t sb_route_topk_workspace(int64_t rows, int64_t n_experts, int64_t top_k) {
    if (rows == 0 || !route_sizes(rows, n_experts, top_k)) return 0;
    return std::max<int64_t>(route_work_bytes(rows, n_experts, top_k), 16);
}

int64_t sb_adapter_gemm_workspace(int64_t M, int64_t rank) {
    if (M <= 0 || M > kLimit - 512 || !adapter_rank(rank)) return 0;
    return M * rank * 4;  // the rows' products with the adapters' first matrices, f32
}

int32_t sb_route_topk(sb_ctx* c, const void* d_logits, int32_t logits_bf16, int64_t ld, int64_t rows, int64_t n_experts, int64_t top_k,
                      int32_t normalize, int32_t* d_experts, float* d_weights, int32_t* d_offsets, int32_t* d_order, int32_t* d_slots,
                      void* d_work, int64_t work_bytes) {
    if (!route_sizes(rows, n_experts, top_k) || ld < n_experts) return fail(SB_INVALID_ARGUMENT, "bad router shape");
    if (!d_offsets || off_boundary(d_offsets, 4)) return fail(SB_INVALID_ARGUMENT, "the offsets are null or misaligned");
    if (rows > 0) {
        if (!d_logits || !d_experts || !d_weights || !d_order || !d_slots) return fail(SB_INVALID_ARGUMENT, "null argument");
        if (off_boundary(d_logits, logits_bf16 ? 2 : 4) || off_boundary(d_experts, 4) || off_boundary(d_weights, 4) || off_boundary(d_order, 4) ||
            off_boundary(d_slots, 4) || off_boundary(d_work, 16))
            return fail(SB_INVALID_ARGUMENT, "arrays lie on the boundaries of their types, the workspace on a 16-byte one");
        const int64_t need = sb_route_topk_workspace(rows, n_experts, top_k);
        if (work_bytes < need || !d_work) return fail(SB_BUFFER_TOO_SMALL, "workspace of " + std::to_string(need) + " bytes needed");
    }
    if (!c) return fail(SB_INVALID_ARGUMENT, "ctx is null");
    SB_CUDA(cudaSetDevice(c->device));
    const int32_t st = set_up(&c->route_ready, [](const char**) { return route_configure(); });
    if (st != SB_OK) return st;
    RouteArgs g{};
    g.logits = d_logits; g.ld = ld; g.rows = (int)rows; g.n_experts = (int)n_experts; g.top_k = (int)top_k;
    g.bf16 = logits_bf16 != 0; g.normalize = normalize != 0;
    g.experts = d_experts; g.weights = d_weights; g.offsets = d_offsets; g.order = d_order; g.slots = d_slots;
    g.work = static_cast<int32_t*>(d_work);
    c->prof.begin("route", c->stream);
    const cudaError_t e = route_launch(g, c->stream, &c->launches);
    c->prof.end(c->stream);
    SB_CUDA(e);
    return SB_OK;
}

int32_t sb_grouped_gemm(sb_ctx* c, const void* d_a, int64_t lda, int64_t a_rows, const int32_t* d_rows, const void* d_w, const float* d_bias,
                        const float* d_row_scale, const float* d_col_scale, const int32_t* d_offsets, int64_t n_groups, void* d_out,
                        int64_t ldo, int64_t M, int64_t N, int64_t K, int32_t fp8, int32_t act, int32_t out_mode, float alpha) {
    int32_t st = check_product(d_a, lda, d_w, d_bias, d_out, ldo, M, N, K, n_groups, fp8 != 0, act, out_mode);
    if (st != SB_OK) return st;
    if (M > 0 && !d_offsets) return fail(SB_INVALID_ARGUMENT, "the offsets are null");
    if (off_boundary(d_offsets, 4) || off_boundary(d_rows, 4) || off_boundary(d_row_scale, 4) || off_boundary(d_col_scale, 4))
        return fail(SB_INVALID_ARGUMENT, "offsets, row indices and scales lie on 4-byte boundaries");
    if (M > 0 && (a_rows <= 0 || a_rows > kLimit || (!d_rows && a_rows < M))) return fail(SB_INVALID_ARGUMENT, "too few rows in A");
    if (!fp8 && (d_row_scale || d_col_scale)) return fail(SB_INVALID_ARGUMENT, "scales belong to e4m3 operands");
    if (!c) return fail(SB_INVALID_ARGUMENT, "ctx is null");
    if (M == 0) return SB_OK;
    SB_CUDA(cudaSetDevice(c->device));
    st = set_up(&c->rows_ready, rows_configure);
    if (st != SB_OK) return st;
    RowsArgs g{};
    g.a = d_a; g.rows = d_rows; g.w = d_w; g.bias = d_bias; g.row_scale = d_row_scale; g.col_scale = d_col_scale; g.offsets = d_offsets;
    g.out = d_out; g.a_rows = a_rows; g.lda = lda; g.ldo = ldo; g.M = (int)M; g.N = (int)N; g.K = (int)K; g.n_groups = (int)n_groups;
    g.act = act; g.out_mode = out_mode; g.alpha = alpha; g.fp8 = fp8 != 0;
    c->prof.begin("grouped_gemm", c->stream);
    const cudaError_t e = rows_launch(g, c->sm_count, c->d_error, c->stream);
    c->prof.end(c->stream);
    if (e == cudaErrorInvalidValue) return fail(SB_INVALID_ARGUMENT, "product shape or alignment not supported");
    SB_CUDA(e);
    c->launches += 1;
    return SB_OK;
}

int32_t sb_combine_rows(sb_ctx* c, const void* d_y, int32_t y_f32, int64_t ldy, int64_t y_rows, const int32_t* d_slots, const float* d_weights,
                        void* d_out, int64_t ldo, int64_t rows, int64_t top_k, int64_t cols, int32_t out_mode, float alpha) {
    // (columns and a row's results are counted in 32 bits, past the last by up to a warp's pieces)
    if (rows < 0 || rows > kLimit || top_k <= 0 || top_k > kLimit / 2 || cols <= 0 || cols > kLimit / 2 || y_rows < 0 || y_rows > kLimit || ldy < cols ||
        ldo < cols || out_mode < 0 || out_mode > 2)
        return fail(SB_INVALID_ARGUMENT, "bad shape or output mode");
    if (rows > 0 && ((!d_y && y_rows > 0) || !d_slots || !d_out)) return fail(SB_INVALID_ARGUMENT, "null argument");
    if (off_boundary(d_y, y_f32 ? 4 : 2) || off_boundary(d_out, out_mode ? 4 : 2) || off_boundary(d_slots, 4) || off_boundary(d_weights, 4))
        return fail(SB_INVALID_ARGUMENT, "arrays lie on the boundaries of their types");
    if (!c) return fail(SB_INVALID_ARGUMENT, "ctx is null");
    if (rows == 0) return SB_OK;
    SB_CUDA(cudaSetDevice(c->device));
    CombineArgs g{};
    g.y = d_y; g.slots = d_slots; g.weights = d_weights; g.out = d_out; g.ldy = ldy; g.ldo = ldo; g.y_rows = y_rows;
    g.rows = (int)rows; g.top_k = (int)top_k; g.cols = (int)cols; g.out_mode = out_mode; g.y_f32 = y_f32 != 0; g.alpha = alpha;
    c->prof.begin("combine_rows", c->stream);
    const cudaError_t e = combine_launch(g, c->stream);
    c->prof.end(c->stream);
    SB_CUDA(e);
    c->launches += 1;
    return SB_OK;
}

int32_t sb_adapter_gemm(sb_ctx* c, const void* d_a, int64_t lda, const void* d_w, const float* d_bias, const void* d_down, const void* d_up,
                        const float* d_scale, const int32_t* d_row_adapter, int64_t n_adapters, int64_t rank, void* d_out, int64_t ldo,
                        int64_t M, int64_t N, int64_t K, int32_t act, int32_t out_mode, float alpha, void* d_work, int64_t work_bytes) {
    int32_t st = check_product(d_a, lda, d_w, d_bias, d_out, ldo, M, N, K, 1, false, act, out_mode);
    if (st != SB_OK) return st;
    if (n_adapters <= 0 || n_adapters > kLimit / std::max(N, kMaxRank) || !adapter_rank(rank))
        return fail(SB_INVALID_ARGUMENT, "adapters: at least one, rank a multiple of 8 up to 128");
    if (M > 0 && (!d_down || !d_up || !d_row_adapter)) return fail(SB_INVALID_ARGUMENT, "null argument");
    if (off_boundary(d_down, 16) || off_boundary(d_up, 16) || off_boundary(d_work, 16) || off_boundary(d_scale, 4) || off_boundary(d_row_adapter, 4))
        return fail(SB_INVALID_ARGUMENT, "adapters and workspace lie on 16-byte boundaries, ids and scales on 4-byte ones");
    const int64_t need = sb_adapter_gemm_workspace(M, rank);
    if (M > 0 && (work_bytes < need || !d_work)) return fail(SB_BUFFER_TOO_SMALL, "workspace of " + std::to_string(need) + " bytes needed");
    if (!c) return fail(SB_INVALID_ARGUMENT, "ctx is null");
    if (M == 0) return SB_OK;
    SB_CUDA(cudaSetDevice(c->device));
    st = set_up(&c->rows_ready, rows_configure);
    if (st != SB_OK) return st;
    float* low = static_cast<float*>(d_work);
    RowsArgs g{};
    g.a = d_a; g.w = d_w; g.bias = d_bias; g.out = d_out; g.a_rows = M; g.lda = lda; g.ldo = ldo; g.M = (int)M; g.N = (int)N; g.K = (int)K;
    g.n_groups = 1; g.act = act; g.out_mode = out_mode; g.alpha = alpha;
    g.row_adapter = d_row_adapter; g.up = d_up; g.low = low; g.n_adapters = (int)n_adapters; g.rank = (int)rank;
    AdapterDownArgs d{};
    d.a = d_a; d.down = d_down; d.scale = d_scale; d.row_adapter = d_row_adapter; d.low = low; d.lda = lda;
    d.M = (int)M; d.K = (int)K; d.rank = (int)rank; d.n_adapters = (int)n_adapters;
    c->prof.begin("adapter_down", c->stream);
    cudaError_t e = adapter_down_launch(d, c->sm_count, c->d_error, c->stream);
    c->prof.end(c->stream);
    if (e == cudaErrorInvalidValue) return fail(SB_INVALID_ARGUMENT, "adapter shape or alignment not supported");
    SB_CUDA(e);
    c->prof.begin("adapter_gemm", c->stream);
    e = rows_launch(g, c->sm_count, c->d_error, c->stream);
    c->prof.end(c->stream);
    if (e == cudaErrorInvalidValue) return fail(SB_INVALID_ARGUMENT, "product shape or alignment not supported");
    SB_CUDA(e);
    c->launches += 2;
    return SB_OK;
}

}  // extern "C"
