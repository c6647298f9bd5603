// Down-projection of the low-rank adapters: low[i] = scale_a (x[i] D_a^T) for the adapter a of row i, kept in 32 bits.
//
// Bound by reading the rows once (2 K bytes each against K * rank products).  Three kernels:
//   - many rows: 128 rows a CTA on tcgen05, rows and adapters through a TMA ring; a pass over K for every few adapters among the
//     rows, whose matrices lie side by side as one operand; each row takes its own adapter's columns of the accumulator (selected,
//     not masked by zeros: nothing of one adapter reaches another's rows).
//   - very few rows: a warp per row and eight columns, K over the lanes.
//   - between them: 16 rows a block on mma.sync m16n8k16 with operands straight from global memory, K over the warps, the columns over
//     blocks; a row takes its adapter's product (selected, not masked by zeros).
//     Where more than six adapters meet in the 16 rows, a row is a chain of dot products over the lanes of a warp instead.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "adapter_ids.cuh"
#include "launch.cuh"
#include "rows.h"
#include "tc_ptx.cuh"

namespace sb {

namespace {

constexpr int kDownWarps = 8;
constexpr int kDotsMost = 4096;  // rows x rank up to which every row reads its adapter for itself (8 MB from L2 at K = 1024)
constexpr int kMaxProducts = 6;  // adapters in 16 rows above which the rows are taken one by one: at 2048 rows of 1024 a product
                                 // costs 1.1 us at rank 16 and 4 us at rank 64, the rows one by one 7 and 28

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

// Eight columns of a row's product, K over the lanes, AHEAD steps of 256 columns asked for at once; lane j < 8 returns column j.
template <int AHEAD>
__device__ __forceinline__ float row_dots(const __nv_bfloat16* x, const __nv_bfloat16* d, int K, int cols, int lane) {
    float acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
    for (int k0 = lane * 8; k0 < K; k0 += 256 * AHEAD) {
        uint4 xv[AHEAD], w[AHEAD][8];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int k = k0 + 256 * u;
            xv[u] = make_uint4(0, 0, 0, 0);
            if (k < K) xv[u] = __ldg(reinterpret_cast<const uint4*>(x + k));
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                w[u][j] = make_uint4(0, 0, 0, 0);
                if (k < K && j < cols) w[u][j] = __ldg(reinterpret_cast<const uint4*>(d + (int64_t)j * K + k));
            }
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                acc[j] = dot2(xv[u].w, w[u][j].w, dot2(xv[u].z, w[u][j].z, dot2(xv[u].y, w[u][j].y, dot2(xv[u].x, w[u][j].x, acc[j]))));
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int s = 16; s; s >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], s);
    float v = acc[0];
#pragma unroll
    for (int j = 1; j < 8; ++j)
        if (lane == j) v = acc[j];
    return v;
}

// Very few rows: a warp per row and eight columns.
__global__ void __launch_bounds__(kDownWarps * 32, 1) adapter_down_dots_kernel(const AdapterDownArgs p, int groups) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    const int64_t item = (int64_t)blockIdx.x * kDownWarps + warp;
    const int row = (int)(item / groups), c = (int)(item % groups) * 8;
    if (row >= p.M) return;
    const int id = __ldg(p.row_adapter + row);
    float v = 0.0f;
    if ((unsigned)id < (unsigned)p.n_adapters) {
        v = row_dots<4>(static_cast<const __nv_bfloat16*>(p.a) + (int64_t)row * p.lda,
                        static_cast<const __nv_bfloat16*>(p.down) + ((int64_t)id * p.rank + c) * p.K, p.K, 8, lane);
        if (p.scale) v *= __ldg(p.scale + id);
    }
    if (lane < 8) p.low[(int64_t)row * p.rank + c + lane] = v;
}

// NT tiles of 8 columns of 16 rows per block; the warps share K.
template <int NT>
__global__ void __launch_bounds__(kDownWarps * 32, 1) adapter_down_kernel(const AdapterDownArgs p) {
    constexpr int kCols = NT * 8, kRows = 16;
    __shared__ float part[kDownWarps][kRows][kCols];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row0 = blockIdx.x * kRows, col0 = blockIdx.y * kCols;
    pdl_wait();
    pdl_trigger();  // what runs beside this block may rely on all that came before it, but not on `low`

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
            // 32 columns of K: a lane's 16 bytes are the fragments of two products, the same permutation of K on both sides; four
            // steps' rows are asked for at once
            for (int k0 = warp * 32; k0 < p.K; k0 += 4 * kDownWarps * 32) {
                uint4 xl[4], xh[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int kk = k0 + u * kDownWarps * 32 + 8 * q;
                    xl[u] = xh[u] = make_uint4(0, 0, 0, 0);
                    if (kk < p.K && row0 + g < p.M) xl[u] = __ldg(reinterpret_cast<const uint4*>(a + (int64_t)(row0 + g) * p.lda + kk));
                    if (kk < p.K && row0 + g + 8 < p.M) xh[u] = __ldg(reinterpret_cast<const uint4*>(a + (int64_t)(row0 + g + 8) * p.lda + kk));
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int kk = k0 + u * kDownWarps * 32 + 8 * q;
                    uint4 w[NT];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const int col = col0 + 8 * n + g;
                        w[n] = make_uint4(0, 0, 0, 0);
                        if (kk < p.K && col < p.rank) w[n] = __ldg(reinterpret_cast<const uint4*>(d + (int64_t)col * p.K + kk));
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma_bf16(acc[n], xl[u].x, xh[u].x, xl[u].y, xh[u].y, w[n].x, w[n].y);
                        mma_bf16(acc[n], xl[u].z, xh[u].z, xl[u].w, xh[u].w, w[n].z, w[n].w);
                    }
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
    } else {
        // every eighth row a warp, eight columns at a time
        for (int r = 0; r < 16; ++r) {
            const int cur = __shfl_sync(0xffffffffu, id, r);
            const bool mine = r % kDownWarps == warp && cur >= 0;
            for (int c = 0; c < kCols; c += 8) {
                const int cols = min(p.rank - col0 - c, 8);
                float v = 0.0f;
                if (mine && cols > 0) v = row_dots<4>(a + (int64_t)(row0 + r) * p.lda, down + ((int64_t)cur * p.rank + col0 + c) * p.K, p.K, cols, lane);
                if (lane < 8) part[warp][r][c + lane] = v;
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kRows * kCols; i += kDownWarps * 32) {
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

// ---------------------------------------------------------------------------------------------- many rows: tcgen05
constexpr int kTcRows = 128, kTcThreads = 192;
constexpr int tc_cols(int rank) { return rank <= 16 ? 16 : (rank <= 32 ? 32 : (rank <= 64 ? 64 : 128)); }
template <int RN>
struct DownTc {
    static constexpr int kAtOnce = RN == 16 ? 4 : (RN == 128 ? 1 : 2);  // adapters of a pass
    static constexpr int kCols = kAtOnce * RN;                          // their columns of the accumulator
    static constexpr uint32_t kTmemCols = 2 * kCols;  // two accumulators by turns, for a pass over K each
    static constexpr int kABytes = kTcRows * 128, kOneBytes = RN * 128, kBBytes = kAtOnce * kOneBytes, kStageBytes = kABytes + kBBytes;
    static constexpr int kStages = std::min(224 * 1024 / kStageBytes, 8);
    static constexpr int kSmemBytes = kStages * kStageBytes + 256 + 1024;
};

// One CTA per SM, tiles of 128 rows by turns.  Warp 0 loads, warp 1 issues the MMAs, warps 2 to 5 read the results, a row per thread.
template <int RN>
__global__ void __launch_bounds__(kTcThreads) adapter_down_tc_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_d,
                                                                     const AdapterDownArgs p, int* __restrict__ error) {
    using namespace ptx;
    using C = DownTc<RN>;
    constexpr int S = C::kStages;
    extern __shared__ unsigned char smem_dyn[];
    const uint32_t base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
    unsigned char* base_ptr = smem_dyn + (base - smem_u32(smem_dyn));
    const uint32_t a_base = base, b_base = base + S * C::kABytes, bar_base = base + S * C::kStageBytes;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (S + s); };
    auto done_bar = [&](int a) { return bar_base + 8u * (2 * S + a); };
    auto free_bar = [&](int a) { return bar_base + 8u * (2 * S + 2 + a); };
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base_ptr + S * C::kStageBytes + 8 * (2 * S + 4));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = warp_index(), lane = threadIdx.x & 31;
    const int k_tiles = (p.K + 63) / 64, tiles = (p.M + kTcRows - 1) / kTcRows;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(done_bar(a), 1);
            mbar_init(free_bar(a), 4);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_trigger();
    AdapterIds<kTcRows> ids;  // of a tile; every warp goes through them by itself

    if (warp == 0) {
        int stage = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
            for (ids.load(p.row_adapter, p.n_adapters, t * kTcRows, p.M, lane); ok;) {
                int id[C::kAtOnce], n = 0;
#pragma unroll
                for (int e = 0; e < C::kAtOnce; ++e) {
                    id[e] = ids.next();
                    n += id[e] >= 0;
                }
                if (n == 0) break;
                bool failed = false;
                if (elect_one()) {
                    int s = stage;
                    uint32_t sp = ph;
                    for (int kt = 0; kt < k_tiles; ++kt) {
                        if (!mbar_wait(empty_bar(s), sp ^ 1, abort_flag)) { failed = true; break; }
                        mbar_expect_tx(full_bar(s), C::kABytes + n * C::kOneBytes);
                        tma_load_2d(a_base + s * C::kABytes, &tma_a, full_bar(s), kt * 64, t * kTcRows);
#pragma unroll
                        for (int e = 0; e < C::kAtOnce; ++e)
                            if (e < n) tma_load_2d(b_base + s * C::kBBytes + e * C::kOneBytes, &tma_d, full_bar(s), kt * 64, id[e] * p.rank);
                        if (++s == S) { s = 0; sp ^= 1; }
                    }
                }
                ok = !__any_sync(0xffffffffu, failed);
                stage += k_tiles;
                ph ^= (uint32_t)(stage / S) & 1u;
                stage %= S;
            }
        }
        if (!ok) {
            const long long t0 = clock64();
            while (clock64() - t0 < 2000000) {}
        }
    } else if (warp == 1) {
        int stage = 0;
        uint32_t ph = 0;
        bool ok = true;
        int pass = 0;
        for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
            for (ids.load(p.row_adapter, p.n_adapters, t * kTcRows, p.M, lane); ok; ++pass) {
                int n = 0;
#pragma unroll
                for (int e = 0; e < C::kAtOnce; ++e) n += ids.next() >= 0;
                if (n == 0) break;
                // fp32 accumulate, bf16 operands, both K-major, M = 128, N = the columns of this pass's adapters
                const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n * RN >> 3) << 17) | ((uint32_t)(kTcRows >> 4) << 24);
                const int acc = pass & 1;
                bool failed = false;
                if (elect_one()) {
                    int s = stage;
                    uint32_t sp = ph;
                    if (!mbar_wait(free_bar(acc), ((pass >> 1) & 1) ^ 1, abort_flag)) failed = true;
                    tc_fence_after();
                    for (int kt = 0; kt < k_tiles && !failed; ++kt) {
                        if (!mbar_wait(full_bar(s), sp, abort_flag)) { failed = true; break; }
                        tc_fence_after();
                        const uint64_t adesc = make_smem_desc(a_base + s * C::kABytes), bdesc = make_smem_desc(b_base + s * C::kBBytes);
#pragma unroll
                        for (int i = 0; i < 4; ++i) tc_mma<false>(tmem + acc * C::kCols, adesc + 2 * i, bdesc + 2 * i, idesc, (kt | i) ? 1u : 0u);
                        tc_commit(empty_bar(s));
                        if (++s == S) { s = 0; sp ^= 1; }
                    }
                    if (!failed) tc_commit(done_bar(acc));
                }
                ok = !__any_sync(0xffffffffu, failed);
                stage += k_tiles;
                ph ^= (uint32_t)(stage / S) & 1u;
                stage %= S;
            }
        }
    } else {
        const int quad = warp & 3;
        bool ok = true;
        int pass = 0;
        for (int t = blockIdx.x; ok && t < tiles; t += gridDim.x) {
            const int row = t * kTcRows + 32 * quad + lane;
            const int id = row < p.M ? __ldg(p.row_adapter + row) : -1;
            const bool has = (unsigned)id < (unsigned)p.n_adapters;
            const float f = has ? (p.scale ? __ldg(p.scale + id) : 1.0f) : 0.0f;
            float4* out = reinterpret_cast<float4*>(p.low + (int64_t)row * p.rank);
            if (row < p.M && !has)
                for (int c = 0; c < p.rank; c += 4) out[c / 4] = make_float4(0.f, 0.f, 0.f, 0.f);
            for (ids.load(p.row_adapter, p.n_adapters, t * kTcRows, p.M, lane); ok; ++pass) {
                int n = 0, mine = -1;  // place of this row's adapter in the pass
#pragma unroll
                for (int e = 0; e < C::kAtOnce; ++e) {
                    const int next = ids.next();
                    n += next >= 0;
                    if (has && next == id) mine = e;
                }
                if (n == 0) break;
                const int acc = pass & 1;
                ok = __all_sync(0xffffffffu, mbar_wait(done_bar(acc), (pass >> 1) & 1, abort_flag));
                if (!ok) break;
                tc_fence_after();
                for (int e = 0; e < n; ++e) {
                    if (!__any_sync(0xffffffffu, mine == e)) continue;
                    for (int c = 0; c < p.rank; c += 16) {
                        uint32_t v[16];
                        tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + acc * C::kCols + e * RN + c, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (mine == e && c + 4 * i < p.rank)
                                out[c / 4 + i] = make_float4(f * __uint_as_float(v[4 * i]), f * __uint_as_float(v[4 * i + 1]),
                                                             f * __uint_as_float(v[4 * i + 2]), f * __uint_as_float(v[4 * i + 3]));
                        __syncwarp();
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(free_bar(acc));
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::kTmemCols);
    }
    if (threadIdx.x == 0 && *abort_flag) atomicExch(error, 1);
}

template <int RN>
cudaError_t down_tc_t(const AdapterDownArgs& g, int sm_count, int* d_error, cudaStream_t stream) {
    alignas(64) CUtensorMap ma, md;
    if (!rows_map(&ma, g.a, g.M, g.K, g.lda, false, kTcRows) || !rows_map(&md, g.down, (int64_t)g.n_adapters * g.rank, g.K, g.K, false, RN))
        return cudaErrorInvalidValue;
    const int blocks = std::min((g.M + kTcRows - 1) / kTcRows, sm_count);
    return launch_pdl(adapter_down_tc_kernel<RN>, dim3(blocks), kTcThreads, DownTc<RN>::kSmemBytes, stream, 1, ma, md, g, d_error);
}

template <int NT>
cudaError_t down_t(const AdapterDownArgs& g, cudaStream_t stream) {
    const dim3 grid((g.M + 15) / 16, (g.rank + NT * 8 - 1) / (NT * 8));
    return launch_pdl(adapter_down_kernel<NT>, grid, kDownWarps * 32, 0, stream, 1, g);
}

}  // namespace

cudaError_t adapter_down_configure() {
    cudaError_t e = cudaSuccess;
    auto set = [&](auto kernel, int bytes) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    };
    set(adapter_down_tc_kernel<16>, DownTc<16>::kSmemBytes);
    set(adapter_down_tc_kernel<32>, DownTc<32>::kSmemBytes);
    set(adapter_down_tc_kernel<64>, DownTc<64>::kSmemBytes);
    set(adapter_down_tc_kernel<128>, DownTc<128>::kSmemBytes);
    return e;
}

cudaError_t adapter_down_launch(const AdapterDownArgs& g, int sm_count, int* d_error, cudaStream_t stream) {
    if (g.M <= 0) return cudaSuccess;
    if (g.M >= 16 * sm_count) {
        switch (tc_cols(g.rank)) {
            case 16: return down_tc_t<16>(g, sm_count, d_error, stream);
            case 32: return down_tc_t<32>(g, sm_count, d_error, stream);
            case 64: return down_tc_t<64>(g, sm_count, d_error, stream);
            default: return down_tc_t<128>(g, sm_count, d_error, stream);
        }
    }
    if ((int64_t)g.M * g.rank <= kDotsMost) {
        const int groups = g.rank / 8;
        const int blocks = (g.M * groups + kDownWarps - 1) / kDownWarps;
        return launch_pdl(adapter_down_dots_kernel, dim3(blocks), kDownWarps * 32, 0, stream, 1, g, groups);
    }
    // the columns are spread over blocks too, as far as that fills the SMs
    const int blocks = (g.M + 15) / 16;
    return blocks * 4 >= sm_count ? down_t<2>(g, stream) : down_t<1>(g, stream);
}

}  // namespace sb
