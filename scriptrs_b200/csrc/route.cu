// The router's choice and the way back: the best experts of every row with their weights, the order that puts rows of one
// expert side by side, and the weighted sum of a row's results.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include <algorithm>

#include "gemm_tile.h"
#include "launch.cuh"
#include "rows.h"

namespace sb {

namespace {

constexpr int kRouteWarps = 8;
constexpr int kRouteRows = 128;  // per block of the choice and of the placement
constexpr int kMaxExperts = 1024, kMaxTopK = 16;

// Order-preserving image of a float; 0 for what is never chosen (-inf, NaN).  +inf counts as the largest finite value, -0 as 0.
__device__ __forceinline__ uint32_t route_key(float x) {
    if (!(x > -INFINITY)) return 0u;
    const uint32_t u = __float_as_uint(fminf(x, FLT_MAX) + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float route_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// A warp per row, the row's experts in registers (PER a lane, expert = 32 i + lane).  Each of the k rounds takes the largest
// key and, among equal ones, the lowest expert.
template <int PER, typename T>
__device__ __forceinline__ void route_row(const RouteArgs& p, int row, int lane, int32_t* chosen) {
    const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.ld;
    uint32_t key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = 32 * i + lane;
        float v = -INFINITY;
        if (e < p.n_experts) {
            if constexpr (sizeof(T) == 2) v = __bfloat162float(x[e]);
            else v = x[e];
        }
        key[i] = route_key(v);
    }
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) most = max(most, key[i]);
    most = __reduce_max_sync(0xffffffffu, most);
    const float top = most ? route_value(most) : 0.0f;
    float total = 0.0f;
    if (!p.normalize) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (key[i]) total += expf(route_value(key[i]) - top);
#pragma unroll
        for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    }
    float mine = 0.0f;  // lane j: the j-th choice
    int who = -1;
    for (int j = 0; j < p.top_k; ++j) {
        uint32_t best = 0;
        int at = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (key[i] > best) { best = key[i]; at = 32 * i + lane; }
        const uint32_t all = __reduce_max_sync(0xffffffffu, best);
        if (!all) break;
        const int e = (int)__reduce_min_sync(0xffffffffu, best == all ? (uint32_t)at : 0xffffffffu);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (32 * i + lane == e) key[i] = 0;
        const float w = expf(route_value(all) - top);
        if (p.normalize) total += w;
        if (lane == j) { mine = w; who = e; }
    }
    if (lane < p.top_k) {
        p.experts[(int64_t)row * p.top_k + lane] = who;
        p.weights[(int64_t)row * p.top_k + lane] = who >= 0 ? mine / total : 0.0f;
        chosen[lane] = who;
    }
}

// The choice, and how often each expert was chosen in this block's rows: counts[block][expert].
template <int PER, typename T>
__global__ void __launch_bounds__(kRouteWarps * 32) route_choose_kernel(const RouteArgs p) {
    __shared__ int32_t chosen[kRouteRows * kMaxTopK];
    __shared__ int32_t count[kMaxExperts];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row0 = blockIdx.x * kRouteRows, rows = min(kRouteRows, p.rows - row0);
    for (int e = threadIdx.x; e < p.n_experts; e += blockDim.x) count[e] = 0;
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    for (int r = warp; r < rows; r += kRouteWarps) route_row<PER, T>(p, row0 + r, lane, chosen + r * p.top_k);
    __syncthreads();
    for (int i = threadIdx.x; i < rows * p.top_k; i += blockDim.x)
        if (chosen[i] >= 0) atomicAdd(&count[chosen[i]], 1);
    __syncthreads();
    for (int e = threadIdx.x; e < p.n_experts; e += blockDim.x) p.work[(int64_t)blockIdx.x * p.n_experts + e] = count[e];
}

// counts[block][expert] -> the place of the block's first row of that expert; offsets.
__global__ void __launch_bounds__(1024) route_scan_kernel(const RouteArgs p, int blocks) {
    __shared__ int32_t warp_sum[32];
    const int e = threadIdx.x, warp = e >> 5, lane = e & 31;
    pdl_wait();
    pdl_trigger();
    int total = 0;
    if (e < p.n_experts) {
#pragma unroll 8
        for (int b = 0; b < blocks; ++b) total += p.work[(int64_t)b * p.n_experts + e];
    }
    int upto = total;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += v;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    if (warp == 0) {
        int s = lane < (int)(blockDim.x >> 5) ? warp_sum[lane] : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, s, d);
            if (lane >= d) s += v;
        }
        warp_sum[lane] = s;
    }
    __syncthreads();
    if (warp) upto += warp_sum[warp - 1];
    if (e < p.n_experts) {
        int at = upto - total;
        p.offsets[e] = at;
        if (e == p.n_experts - 1) p.offsets[p.n_experts] = upto;
        for (int b = 0; b < blocks; ++b) {
            int32_t* c = p.work + (int64_t)b * p.n_experts + e;
            const int n = *c;
            *c = at;
            at += n;
        }
    }
}

// Rows of a block to their places, in order: one warp, 32 choices at a time, equal experts ranked by their lanes.
__global__ void __launch_bounds__(256) route_place_kernel(const RouteArgs p) {
    __shared__ int32_t next[kMaxExperts];
    const int lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    for (int e = threadIdx.x; e < p.n_experts; e += blockDim.x) next[e] = p.work[(int64_t)blockIdx.x * p.n_experts + e];
    const int used = p.offsets[p.n_experts];
    const int64_t first = (int64_t)blockIdx.x * kRouteRows * p.top_k;
    const int64_t end = min(first + (int64_t)kRouteRows * p.top_k, (int64_t)p.rows * p.top_k);
    for (int64_t i = first + threadIdx.x; i < end; i += blockDim.x)
        if (i >= used) p.order[i] = -1;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    for (int64_t i0 = first; i0 < end; i0 += 32) {
        const int64_t i = i0 + lane;
        const int e = i < end ? p.experts[i] : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        int at = -1;
        if (e >= 0) at = next[e] + __popc(same & ((1u << lane) - 1u));
        __syncwarp();
        if (e >= 0 && (same >> lane) == 1u) next[e] = at + 1;  // the last of its kind
        __syncwarp();
        if (i < end) p.slots[i] = at;
        if (at >= 0) p.order[at] = (int)(i / p.top_k);
    }
}

template <typename T>
cudaError_t route_choose(const RouteArgs& g, int blocks, cudaStream_t st) {
    const int per = (g.n_experts + 31) / 32;
    const int threads = kRouteWarps * 32;
    if (per <= 1) return launch_pdl(route_choose_kernel<1, T>, dim3(blocks), threads, 0, st, 1, g);
    if (per <= 2) return launch_pdl(route_choose_kernel<2, T>, dim3(blocks), threads, 0, st, 1, g);
    if (per <= 4) return launch_pdl(route_choose_kernel<4, T>, dim3(blocks), threads, 0, st, 1, g);
    if (per <= 8) return launch_pdl(route_choose_kernel<8, T>, dim3(blocks), threads, 0, st, 1, g);
    return launch_pdl(route_choose_kernel<32, T>, dim3(blocks), threads, 0, st, 1, g);
}

// out[row] (+)= alpha sum_j weights[row][j] y[slots[row][j]], in 32 bits in the order of j, rounded once.  A thread takes eight
// columns where rows lie on 16-byte boundaries, else one.
template <typename Y, int PER>
__global__ void __launch_bounds__(256) combine_kernel(const CombineArgs p) {
    pdl_wait();
    pdl_trigger();
    const int groups = (p.cols + PER - 1) / PER;
    const int64_t total = (int64_t)p.rows * groups;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int row = (int)(i / groups), col = (int)(i % groups) * PER;
        float sum[PER];
#pragma unroll
        for (int c = 0; c < PER; ++c) sum[c] = 0.0f;
        for (int j = 0; j < p.top_k; ++j) {
            const int at = __ldg(p.slots + (int64_t)row * p.top_k + j);
            if ((unsigned)at >= (unsigned long long)p.y_rows) continue;
            const float w = p.weights ? __ldg(p.weights + (int64_t)row * p.top_k + j) : 1.0f;
            const Y* y = static_cast<const Y*>(p.y) + (int64_t)at * p.ldy + col;
            if constexpr (PER == 8 && sizeof(Y) == 2) {
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(y));
                const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    sum[2 * c] = fmaf(w, __uint_as_float(u[c] << 16), sum[2 * c]);
                    sum[2 * c + 1] = fmaf(w, __uint_as_float(u[c] & 0xffff0000u), sum[2 * c + 1]);
                }
            } else if constexpr (PER == 8) {
#pragma unroll
                for (int c = 0; c < 8; c += 4) {
                    const float4 v = __ldg(reinterpret_cast<const float4*>(y + c));
                    sum[c] = fmaf(w, v.x, sum[c]); sum[c + 1] = fmaf(w, v.y, sum[c + 1]);
                    sum[c + 2] = fmaf(w, v.z, sum[c + 2]); sum[c + 3] = fmaf(w, v.w, sum[c + 3]);
                }
            } else {
                sum[0] = fmaf(w, (float)y[0], sum[0]);
            }
        }
        if (p.out_mode == kOutBf16) {
            __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + (int64_t)row * p.ldo + col;
            if constexpr (PER == 8) {
                uint32_t u[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    __nv_bfloat162 b = __floats2bfloat162_rn(p.alpha * sum[2 * c], p.alpha * sum[2 * c + 1]);
                    u[c] = *reinterpret_cast<uint32_t*>(&b);
                }
                *reinterpret_cast<uint4*>(out) = make_uint4(u[0], u[1], u[2], u[3]);
            } else {
                *out = __float2bfloat16_rn(p.alpha * sum[0]);
            }
        } else {
            float* out = static_cast<float*>(p.out) + (int64_t)row * p.ldo + col;
#pragma unroll
            for (int c = 0; c < PER; c += 4) {
                if constexpr (PER == 8) {
                    float4 v = make_float4(p.alpha * sum[c], p.alpha * sum[c + 1], p.alpha * sum[c + 2], p.alpha * sum[c + 3]);
                    if (p.out_mode == kOutResidual) {
                        const float4 o = *reinterpret_cast<const float4*>(out + c);
                        v = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
                    }
                    *reinterpret_cast<float4*>(out + c) = v;
                } else {
                    *out = (p.out_mode == kOutResidual ? *out : 0.0f) + p.alpha * sum[0];
                }
            }
        }
    }
}

}  // namespace

int64_t route_work_bytes(int64_t rows, int64_t n_experts, int64_t) {
    return (rows + kRouteRows - 1) / kRouteRows * n_experts * (int64_t)sizeof(int32_t);
}

cudaError_t route_launch(const RouteArgs& g, cudaStream_t stream, int64_t* launches) {
    if (g.rows <= 0) return cudaMemsetAsync(g.offsets, 0, sizeof(int32_t) * (g.n_experts + 1), stream);
    const int blocks = (g.rows + kRouteRows - 1) / kRouteRows;
    cudaError_t e = g.bf16 ? route_choose<__nv_bfloat16>(g, blocks, stream) : route_choose<float>(g, blocks, stream);
    if (e != cudaSuccess) return e;
    e = launch_pdl(route_scan_kernel, dim3(1), (g.n_experts + 31) / 32 * 32, 0, stream, 1, g, blocks);
    if (e != cudaSuccess) return e;
    *launches += 3;
    return launch_pdl(route_place_kernel, dim3(blocks), 256, 0, stream, 1, g);
}

cudaError_t combine_launch(const CombineArgs& g, cudaStream_t stream) {
    if (g.rows <= 0) return cudaSuccess;
    const int ye = g.y_f32 ? 4 : 2, oe = g.out_mode == kOutBf16 ? 2 : 4;
    const bool vec = g.cols % 8 == 0 && !((reinterpret_cast<uintptr_t>(g.y) | reinterpret_cast<uintptr_t>(g.out)) & 15) &&
                     !((g.ldy * ye) & 15) && !((g.ldo * oe) & 15);
    const int64_t threads = (int64_t)g.rows * (vec ? g.cols / 8 : g.cols);
    const dim3 grid((unsigned)std::min<int64_t>((threads + 255) / 256, 1 << 20));
    if (vec) return g.y_f32 ? launch_pdl(combine_kernel<float, 8>, grid, 256, 0, stream, 1, g)
                            : launch_pdl(combine_kernel<__nv_bfloat16, 8>, grid, 256, 0, stream, 1, g);
    return g.y_f32 ? launch_pdl(combine_kernel<float, 1>, grid, 256, 0, stream, 1, g)
                   : launch_pdl(combine_kernel<__nv_bfloat16, 1>, grid, 256, 0, stream, 1, g);
}

}  // namespace sb
