// Down-projection of the low-rank adapters: low[i] = scale_a (x[i] D_a^T) for the adapter a of row i, kept in 32 bits, and for
// the rows of every tile of the product the list of the adapters among them, in the order of their first rows.
//
// Bound by reading the rows once (2 K bytes each against K * rank products), so the products run on mma.sync m16n8k16 with
// operands straight from global memory.  A warp takes 16 rows x COLS columns and every KW-th 32 columns of K; the partial sums
// meet in shared memory in a fixed order.  KW = 8 (16 rows a block) spreads few rows over many SMs, KW = 2 (64 rows a block)
// reads an adapter's matrix from L1 for four row tiles.  Rows of several adapters in a tile are products of their own, of which
// each row takes its adapter's (selected, not masked by zeros: nothing of one adapter reaches another's rows).  Where nearly
// every row has its own adapter (live streams), 16 such products would run one after the other; there a row is a chain of dot
// products over the lanes instead.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "launch.cuh"
#include "rows.h"

namespace sb {

namespace {

constexpr int kDownWarps = 8;
constexpr int kMaxProducts = 3;  // adapters in 16 rows above which the rows are taken one by one

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float s) {
    s = fmaf(__uint_as_float(a << 16), __uint_as_float(b << 16), s);
    return fmaf(__uint_as_float(a & 0xffff0000u), __uint_as_float(b & 0xffff0000u), s);
}

// NT tiles of 8 columns per block; KW warps share the K of 16 rows.
template <int NT, int KW>
__global__ void __launch_bounds__(kDownWarps * 32) adapter_down_kernel(const AdapterDownArgs p) {
    constexpr int kCols = NT * 8, kRows = 16 * (kDownWarps / KW);
    __shared__ float part[KW][kRows][kCols];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int block0 = blockIdx.x * kRows, col0 = blockIdx.y * kCols;
    pdl_wait();
    pdl_trigger();  // what runs beside this block may rely on all that came before it, but not on `low` and the lists

    if (blockIdx.y == 0 && block0 % p.list_rows == 0 && warp == kDownWarps - 1) {
        int ids[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = block0 + 8 * lane + j;
            ids[j] = 8 * lane + j < p.list_rows && r < p.M ? __ldg(p.row_adapter + r) : -1;
            if ((unsigned)ids[j] >= (unsigned)p.n_adapters) ids[j] = -1;
        }
        int32_t* list = p.lists + (int64_t)(block0 / p.list_rows) * kAdapterListInts;
        int count = 0;
        while (true) {
            int first = -1;
#pragma unroll
            for (int j = 7; j >= 0; --j)
                if (ids[j] >= 0) first = ids[j];
            const uint32_t have = __ballot_sync(0xffffffffu, first >= 0);
            if (!have) break;
            const int cur = __shfl_sync(0xffffffffu, first, __ffs(have) - 1);
            if (lane == 0) list[4 + count] = cur;
            ++count;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (ids[j] == cur) ids[j] = -1;
        }
        if (lane == 0) list[0] = count;
    }

    const int kw = warp % KW, tile_row = warp / KW * 16, row0 = block0 + tile_row;
    const int my_row = row0 + (lane & 15);
    int id = my_row < p.M ? __ldg(p.row_adapter + my_row) : -1;
    if ((unsigned)id >= (unsigned)p.n_adapters) id = -1;
    const __nv_bfloat16* a = static_cast<const __nv_bfloat16*>(p.a);
    const __nv_bfloat16* down = static_cast<const __nv_bfloat16*>(p.down);
    uint32_t left = __ballot_sync(0xffffffffu, id >= 0) & 0xffffu;
    int products = 0;
    for (uint32_t l = left; l && products <= kMaxProducts; ++products) {
        const int cur = __shfl_sync(0xffffffffu, id, __ffs(l) - 1);
        l &= ~__ballot_sync(0xffffffffu, id == cur);
    }

    if (products <= kMaxProducts) {
        const int g = lane >> 2, q = lane & 3;  // fragment row / column group
        const int id_lo = __shfl_sync(0xffffffffu, id, g), id_hi = __shfl_sync(0xffffffffu, id, g + 8);
        float sum[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[n][i] = 0.0f;
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
#pragma unroll(NT >= 8 ? 2 : 4)
            for (int k = kw * 32; k < p.K; k += KW * 32) {
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
            *reinterpret_cast<float2*>(&part[kw][tile_row + g][8 * n + 2 * q]) = make_float2(sum[n][0], sum[n][1]);
            *reinterpret_cast<float2*>(&part[kw][tile_row + g + 8][8 * n + 2 * q]) = make_float2(sum[n][2], sum[n][3]);
        }
    } else {
        // rows kw, kw + KW, ... of the tile, eight columns at a time, K over the lanes
        for (int r = 0; r < 16; ++r) {
            const int cur = __shfl_sync(0xffffffffu, id, r);
            const bool mine = r % KW == kw && cur >= 0;
            for (int c = 0; c < kCols; c += 8) {
                float acc[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
                if (mine) {
                    const __nv_bfloat16* x = a + (int64_t)(row0 + r) * p.lda;
                    const __nv_bfloat16* d = down + ((int64_t)cur * p.rank + col0 + c) * p.K;
#pragma unroll 2
                    for (int k = lane * 8; k < p.K; k += 256) {
                        const uint4 xv = __ldg(reinterpret_cast<const uint4*>(x + k));
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            if (col0 + c + j >= p.rank) break;
                            const uint4 w = __ldg(reinterpret_cast<const uint4*>(d + (int64_t)j * p.K + k));
                            acc[j] = dot2(xv.w, w.w, dot2(xv.z, w.z, dot2(xv.y, w.y, dot2(xv.x, w.x, acc[j]))));
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int s = 16; s; s >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], s);
                }
                if (lane < 8) {
                    float v = acc[0];
#pragma unroll
                    for (int j = 1; j < 8; ++j)
                        if (lane == j) v = acc[j];
                    part[kw][tile_row + r][c + lane] = v;
                }
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kRows * kCols; i += kDownWarps * 32) {
        const int r = i / kCols, c = i % kCols, row = block0 + r;
        if (row >= p.M || col0 + c >= p.rank) continue;
        const int who = __ldg(p.row_adapter + row);
        float s = 0.0f;
        if ((unsigned)who < (unsigned)p.n_adapters) {
#pragma unroll
            for (int w = 0; w < KW; ++w) s += part[w][r][c];
            if (p.scale) s *= __ldg(p.scale + who);
        }
        p.low[(int64_t)row * p.rank + col0 + c] = s;
    }
}

template <int NT, int KW>
cudaError_t down_t(const AdapterDownArgs& g, cudaStream_t stream) {
    const int rows = 16 * (kDownWarps / KW);
    const dim3 grid((g.M + rows - 1) / rows, (g.rank + NT * 8 - 1) / (NT * 8));
    return launch_pdl(adapter_down_kernel<NT, KW>, grid, kDownWarps * 32, 0, stream, 1, g);
}

}  // namespace

cudaError_t adapter_down_launch(const AdapterDownArgs& g, int sm_count, cudaStream_t stream) {
    if (g.M <= 0) return cudaSuccess;
    // 64 rows a block once those give every SM two blocks; else 16, and few rows spread their columns over blocks too
    if (g.M >= 128 * sm_count) return g.rank > 32 ? down_t<8, 2>(g, stream) : (g.rank > 16 ? down_t<4, 2>(g, stream) : down_t<2, 2>(g, stream));
    if (g.M >= 16 * sm_count) return g.rank > 32 ? down_t<8, 8>(g, stream) : (g.rank > 16 ? down_t<4, 8>(g, stream) : down_t<2, 8>(g, stream));
    return down_t<1, 8>(g, stream);
}

}  // namespace sb
