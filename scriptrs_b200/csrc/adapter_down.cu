// Down-projection of the low-rank adapters: low[i] = scale_a (x[i] D_a^T) for the adapter a of row i, kept in 32 bits, and for
// every 128 rows the list of the adapters among them in the order of their first rows (the tiles of rows.cu go by it).
//
// Bound by reading the rows once (2 K bytes each against K * rank products), so the products run on mma.sync m16n8k16 with
// operands straight from global memory: a block takes 16 rows x COLS columns, its eight warps every eighth 32 columns of K, the
// partial sums meet in shared memory in the order of the warps.  Rows of several adapters in a block are products of their own,
// of which each row takes its adapter's (selected, not masked by zeros: nothing of one adapter reaches another's rows).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "launch.cuh"
#include "rows.h"

namespace sb {

namespace {

constexpr int kDownWarps = 8;

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// NT tiles of 8 columns per block.
template <int NT>
__global__ void __launch_bounds__(kDownWarps * 32) adapter_down_kernel(const AdapterDownArgs p) {
    constexpr int kCols = NT * 8;
    __shared__ float part[kDownWarps][16][kCols];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row0 = blockIdx.x * 16, col0 = blockIdx.y * kCols;
    pdl_wait();
    pdl_trigger();  // what runs beside this block may rely on all that came before it, but not on `low` and the lists

    const int my_row = row0 + (lane & 15);
    int id = my_row < p.M ? __ldg(p.row_adapter + my_row) : -1;
    if ((unsigned)id >= (unsigned)p.n_adapters) id = -1;

    if (blockIdx.y == 0 && (blockIdx.x & 7) == 0 && warp == kDownWarps - 1) {
        int ids[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = row0 + 4 * lane + j;
            ids[j] = r < p.M ? __ldg(p.row_adapter + r) : -1;
            if ((unsigned)ids[j] >= (unsigned)p.n_adapters) ids[j] = -1;
        }
        int32_t* list = p.lists + (int64_t)(blockIdx.x >> 3) * kAdapterListInts;
        int count = 0;
        while (true) {
            int first = -1;
#pragma unroll
            for (int j = 3; j >= 0; --j)
                if (ids[j] >= 0) first = ids[j];
            const uint32_t have = __ballot_sync(0xffffffffu, first >= 0);
            if (!have) break;
            const int cur = __shfl_sync(0xffffffffu, first, __ffs(have) - 1);
            if (lane == 0) list[4 + count] = cur;
            ++count;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (ids[j] == cur) ids[j] = -1;
        }
        if (lane == 0) list[0] = count;
    }

    const int g = lane >> 2, q = lane & 3;  // fragment row / column group
    const __nv_bfloat16* a = static_cast<const __nv_bfloat16*>(p.a);
    const __nv_bfloat16* down = static_cast<const __nv_bfloat16*>(p.down);
    const int id_lo = __shfl_sync(0xffffffffu, id, g), id_hi = __shfl_sync(0xffffffffu, id, g + 8);
    float sum[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[n][i] = 0.0f;

    uint32_t left = __ballot_sync(0xffffffffu, id >= 0) & 0xffffu;
    while (left) {
        const int cur = __shfl_sync(0xffffffffu, id, __ffs(left) - 1);
        left &= ~__ballot_sync(0xffffffffu, id == cur);
        float acc[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[n][i] = 0.0f;
        const __nv_bfloat16* d = down + (int64_t)cur * p.rank * p.K;
        // 32 columns of K: a lane's 16 bytes are the fragments of two products, the same permutation of K on both sides
#pragma unroll 2
        for (int k = warp * 32; k < p.K; k += kDownWarps * 32) {
            const int kk = k + 8 * q;
            const bool in = kk < p.K;
            uint4 xl = make_uint4(0, 0, 0, 0), xh = xl;
            if (in && row0 + g < p.M) xl = __ldg(reinterpret_cast<const uint4*>(a + (int64_t)(row0 + g) * p.lda + kk));
            if (in && row0 + g + 8 < p.M) xh = __ldg(reinterpret_cast<const uint4*>(a + (int64_t)(row0 + g + 8) * p.lda + kk));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int col = col0 + 8 * n + g;
                uint4 w = make_uint4(0, 0, 0, 0);
                if (in && col < p.rank) w = __ldg(reinterpret_cast<const uint4*>(d + (int64_t)col * p.K + kk));
                mma_bf16(acc[n], xl.x, xh.x, xl.y, xh.y, w.x, w.y);
                mma_bf16(acc[n], xl.z, xh.z, xl.w, xh.w, w.z, w.w);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (id_lo == cur) { sum[n][0] = acc[n][0]; sum[n][1] = acc[n][1]; }
            if (id_hi == cur) { sum[n][2] = acc[n][2]; sum[n][3] = acc[n][3]; }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        *reinterpret_cast<float2*>(&part[warp][g][8 * n + 2 * q]) = make_float2(sum[n][0], sum[n][1]);
        *reinterpret_cast<float2*>(&part[warp][g + 8][8 * n + 2 * q]) = make_float2(sum[n][2], sum[n][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * kCols; i += kDownWarps * 32) {
        const int r = i / kCols, c = i % kCols, row = row0 + r;
        if (row >= p.M || col0 + c >= p.rank) continue;
        const int who = __ldg(p.row_adapter + row);
        float s = 0.0f;
        if ((unsigned)who < (unsigned)p.n_adapters) {
#pragma unroll
            for (int w = 0; w < kDownWarps; ++w) s += part[w][r][c];
            if (p.scale) s *= __ldg(p.scale + who);
        }
        p.low[(int64_t)row * p.rank + col0 + c] = s;
    }
}

}  // namespace

cudaError_t adapter_down_launch(const AdapterDownArgs& g, int sm_count, cudaStream_t stream) {
    if (g.M <= 0) return cudaSuccess;
    const int blocks = (g.M + 15) / 16;
    // few rows: the columns are spread over blocks too
    const int nt = blocks >= sm_count ? (g.rank > 32 ? 8 : (g.rank > 16 ? 4 : 2)) : (g.rank > 8 ? 2 : 1);
    const dim3 grid(blocks, (g.rank + nt * 8 - 1) / (nt * 8));
    switch (nt) {
        case 1: return launch_pdl(adapter_down_kernel<1>, grid, kDownWarps * 32, 0, stream, 1, g);
        case 2: return launch_pdl(adapter_down_kernel<2>, grid, kDownWarps * 32, 0, stream, 1, g);
        case 4: return launch_pdl(adapter_down_kernel<4>, grid, kDownWarps * 32, 0, stream, 1, g);
        default: return launch_pdl(adapter_down_kernel<8>, grid, kDownWarps * 32, 0, stream, 1, g);
    }
}

}  // namespace sb
