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
#include "tc_ptx.cuh"

namespace sb {

namespace {

constexpr int kRouteThreads = 1024, kRouteWarps = kRouteThreads / 32;
constexpr int kRouteRows = 512;     // most rows of a block
constexpr int kRouteOneBlock = 128; // rows up to which one block does everything
constexpr int kRouteSums = 256;     // blocks up to which each sums the counts of those before it by itself
constexpr int kMaxExperts = 1024, kMaxTopK = 16;

// Rows per block: as many blocks as there are SMs to fill with a pass of 64 rows or more.
int route_block_rows(int64_t rows) {
    if (rows <= kRouteOneBlock) return kRouteOneBlock;
    return (int)std::min<int64_t>(kRouteRows, (rows + 147) / 148 <= 64 ? 64 : ((rows + 147) / 148 + 63) / 64 * 64);
}
int64_t route_blocks(int64_t rows) { return (rows + route_block_rows(rows) - 1) / route_block_rows(rows); }

// What a logit counts as: NaN as -inf, which is never chosen, +inf as the largest finite value of its type.
template <typename T>
__device__ __forceinline__ float route_logit(float x) {
    return fminf(fmaxf(x, -INFINITY), sizeof(T) == 2 ? __uint_as_float(0x7f7f0000u) : FLT_MAX);
}
// Order-preserving image of a float (-0 as 0); below kRouteNone: -inf.
constexpr uint32_t kRouteNone = 0x00800000u;
__device__ __forceinline__ uint32_t route_key(float x) {
    const int s = __float_as_int(x + 0.0f);
    return (uint32_t)(s ^ ((s >> 31) | (int)0x80000000));
}
__device__ __forceinline__ float route_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// exp(x) for x <= 0: the argument's rounding is 2^-24 of it, the function's error 2^-22, and what counts lies near 0.
__device__ __forceinline__ float route_exp(float x) { return ptx::ex2_approx(x * 1.44269504f); }

// LANES lanes take a row, PER neighbouring experts each, in registers.  A round finds the largest key below the one before as the
// maximum of key - previous in unsigned arithmetic: what lies below wraps round to the top, nearest first.
//   bf16: a key is 16 bits, the expert (counted down) takes the other 16: keys differ and a round yields one choice.
//   f32:  a round yields a value; the experts that have it follow in ascending order.
// `live`: the row exists (its lanes take part in the shuffles either way).
template <int LANES, int PER, typename T>
__device__ __forceinline__ void route_row(const RouteArgs& p, int row, bool live, int lane, int16_t* chosen) {
    constexpr bool kPacked = sizeof(T) == 2;
    const int l = lane % LANES;
    uint32_t key[PER];
    float total = 0.0f, top;
    uint32_t first;
    // the largest of key - below (mod 2^32) over the row
    auto most = [&](uint32_t below) {
        uint32_t m = key[0] - below;
#pragma unroll
        for (int i = 1; i < PER; ++i) m = __viaddmax_u32(key[i], 0u - below, m);
#pragma unroll
        for (int d = LANES / 2; d; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
        return m;
    };
    // a packed key's lower half stands for the zeros of a bf16 value, inverted where it is negative
    auto value = [](uint32_t k) {
        if (kPacked) k = (k & 0xffff0000u) | ((k & 0x80000000u) ? 0u : 0xffffu);
        return route_value(k);
    };
    {
        float f[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) f[i] = -INFINITY;
        const T* x = static_cast<const T*>(p.logits) + (int64_t)row * p.ld;
        constexpr int kVec = 16 / (int)sizeof(T);
        if (PER % kVec == 0 && p.vec) {
#pragma unroll
            for (int i = 0; i < PER; i += kVec) {
                if (!live || l * PER + i >= p.n_experts) continue;
                const uint4 v = __ldg(reinterpret_cast<const uint4*>(x + l * PER + i));
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < kVec; ++j) {
                    if constexpr (kPacked) f[(i + j) % PER] = __uint_as_float(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
                    else f[(i + j) % PER] = __uint_as_float(w[j]);
                }
            }
        } else if (live) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (l * PER + i < p.n_experts) f[i] = (float)x[l * PER + i];
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            f[i] = route_logit<T>(f[i]);
            key[i] = route_key(f[i]);
            if (kPacked) key[i] = (key[i] & 0xffff0000u) | (0xffffu - (uint32_t)(l * PER + i));
        }
        first = most(0u);
        top = first >= kRouteNone ? value(first) : 0.0f;
        if (!p.normalize) {
#pragma unroll
            for (int i = 0; i < PER; ++i) total += route_exp(f[i] - top);
#pragma unroll
            for (int d = LANES / 2; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
        }
    }
    constexpr int kKeep = (kMaxTopK + LANES - 1) / LANES;  // lane l keeps the choices l, l + LANES, ...
    float mine[kKeep];
    int who[kKeep];
#pragma unroll
    for (int i = 0; i < kKeep; ++i) { mine[i] = 0.0f; who[i] = -1; }
    auto keep = [&](int j, float w, int e) {
        if (p.normalize) total += w;
#pragma unroll
        for (int i = 0; i < kKeep; ++i)
            if (l + i * LANES == j) { mine[i] = w; who[i] = e; }
    };
    uint32_t best = first;
    if constexpr (kPacked) {
        for (int j = 0; j < p.top_k; ++j) {
            if (best >= kRouteNone) keep(j, route_exp(value(best) - top), (int)(0xffffu - (best & 0xffffu)));
            const uint32_t next = most(best) + best;  // shuffles: by every lane, its row over or not
            best = best >= kRouteNone ? next : 0u;
        }
    } else {
        const int group0 = lane / LANES * LANES;
        int j = 0;
        while (__any_sync(0xffffffffu, best >= kRouteNone && j < p.top_k)) {
            uint32_t has = 0;  // this lane's experts with that value
#pragma unroll
            for (int i = 0; i < PER; ++i) has |= key[i] == best ? 1u << i : 0u;
            if (best < kRouteNone) has = 0;
            const float w = best >= kRouteNone ? route_exp(value(best) - top) : 0.0f;
            while (true) {
                const uint32_t lanes = (__ballot_sync(0xffffffffu, has != 0) >> group0) & (LANES == 32 ? 0xffffffffu : (1u << LANES) - 1u);
                const bool go = lanes && j < p.top_k;
                if (!__any_sync(0xffffffffu, go)) break;
                const int from = group0 + (lanes ? __ffs(lanes) - 1 : 0);
                const int at = __shfl_sync(0xffffffffu, l * PER + __ffs(has) - 1, from);
                if (go) {
                    keep(j, w, at);
                    ++j;
                    if (lane == from) has &= has - 1;
                }
            }
            const uint32_t next = most(best) + best;
            best = best >= kRouteNone ? next : 0u;
        }
    }
    if (!live) return;
    const int64_t out = (int64_t)row * p.top_k;
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
        const int j = l + i * LANES;
        if (j >= p.top_k) break;
        p.experts[out + j] = who[i];
        p.weights[out + j] = who[i] >= 0 ? __fdividef(mine[i], total) : 0.0f;  // 1 <= total <= 1024
        chosen[j] = (int16_t)who[i];
    }
}

// Exclusive sums over the block's threads (thread = expert); *all: the sum of all.
__device__ __forceinline__ int block_before(int n, int* warp_sum, int* all) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int upto = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += v;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    int before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < kRouteWarps; ++w) {
        if (w < warp) before += warp_sum[w];
        sum += warp_sum[w];
    }
    *all = sum;
    return before + upto - n;
}

// The block's choices (in shared memory, in order) to their places.  base[e]: the first place of the block's rows of expert e.
// Each warp takes a run of them, 32 at a time: equal experts are ranked by their lanes, behind those of the chunks and warps
// before.  Called by the whole block; part: [kRouteWarps][n_experts].
__device__ __forceinline__ void route_place(const RouteArgs& p, const int16_t* chosen, const int* base, uint16_t* part, int row0, int n) {
    const int64_t first = (int64_t)row0 * p.top_k;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int run = (n + kRouteWarps * 32 - 1) / (kRouteWarps * 32) * 32, lo = min(warp * run, n), hi = min(lo + run, n);
    for (int i = threadIdx.x; i < kRouteWarps * p.n_experts; i += kRouteThreads) part[i] = 0;
    __syncthreads();
    uint16_t* count = part + warp * p.n_experts;
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const int e = i0 + lane < hi ? chosen[i0 + lane] : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        if (e >= 0 && (same >> lane) == 1u) count[e] += (uint16_t)__popc(same);  // the last of its kind
        __syncwarp();
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.n_experts; e += kRouteThreads) {
        uint32_t at = 0, c[kRouteWarps];
#pragma unroll
        for (int w = 0; w < kRouteWarps; ++w) c[w] = part[w * p.n_experts + e];
#pragma unroll
        for (int w = 0; w < kRouteWarps; ++w) {
            part[w * p.n_experts + e] = (uint16_t)at;
            at += c[w];
        }
    }
    __syncthreads();
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const int e = i0 + lane < hi ? chosen[i0 + lane] : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        int at = -1, rank = 0;
        if (e >= 0) {
            rank = count[e] + __popc(same & ((1u << lane) - 1u));
            at = base[e] + rank;
        }
        __syncwarp();
        if (e >= 0 && (same >> lane) == 1u) count[e] = (uint16_t)(rank + 1);
        __syncwarp();
        if (i0 + lane < hi) p.slots[first + i0 + lane] = at;
        if (at >= 0) p.order[at] = row0 + (int)((uint32_t)(i0 + lane) / (uint32_t)p.top_k);
    }
}

// The choice, and how often each expert was chosen by this block's rows: table[expert][block].  One block alone goes on to the
// places.
template <int LANES, int PER, typename T>
__global__ void __launch_bounds__(kRouteThreads) route_choose_kernel(const RouteArgs p, int block_rows, int blocks) {
    __shared__ int16_t chosen[kRouteRows * kMaxTopK];
    __shared__ int32_t count[kMaxExperts];
    __shared__ int warp_sum[kRouteWarps];
    extern __shared__ uint16_t part[];  // one block alone
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row0 = blockIdx.x * block_rows, rows = min(block_rows, p.rows - row0);
    for (int e = threadIdx.x; e < p.n_experts; e += kRouteThreads) count[e] = 0;
    pdl_wait();
    pdl_trigger();
    constexpr int kPer = 32 / LANES;  // rows of a warp at once
    for (int r0 = warp * kPer; r0 < rows; r0 += kRouteWarps * kPer) {
        const int r = r0 + lane / LANES;
        route_row<LANES, PER, T>(p, row0 + r, r < rows, lane, chosen + min(r, rows - 1) * p.top_k);
    }
    __syncthreads();
    const int n = rows * p.top_k;
    for (int i = threadIdx.x; i < n; i += kRouteThreads)
        if (chosen[i] >= 0) atomicAdd(&count[chosen[i]], 1);
    __syncthreads();
    if (blocks > 1) {
        for (int e = threadIdx.x; e < p.n_experts; e += kRouteThreads) p.work[(int64_t)e * (blocks + 1) + blockIdx.x] = count[e];
        return;
    }
    int used = 0;
    for (int e0 = 0; e0 < p.n_experts; e0 += kRouteThreads) {
        const int e = e0 + threadIdx.x;
        int all;
        const int at = used + block_before(e < p.n_experts ? count[e] : 0, warp_sum, &all);
        if (e < p.n_experts) {
            p.offsets[e] = at;
            count[e] = at;
        }
        used += all;
    }
    if (threadIdx.x == 0) p.offsets[p.n_experts] = used;
    for (int i = used + threadIdx.x; i < n; i += kRouteThreads) p.order[i] = -1;
    __syncthreads();
    route_place(p, chosen, count, part, 0, n);
}

// Many blocks: table[expert][block] -> the sums of the blocks before, [blocks] the sum of all; a warp per expert.
__global__ void __launch_bounds__(256) route_sums_kernel(const RouteArgs p, int blocks) {
    const int e = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    if (e >= p.n_experts) return;
    int32_t* row = p.work + (int64_t)e * (blocks + 1);
    int before = 0;
    for (int b0 = 0; b0 < blocks; b0 += 32) {
        const int n = b0 + lane < blocks ? row[b0 + lane] : 0;
        int upto = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += v;
        }
        if (b0 + lane < blocks) row[b0 + lane] = before + upto - n;
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) row[blocks] = before;
}

// The places of a block's rows: what the blocks before it hold of every expert, what all hold, then the block's own order.
__global__ void __launch_bounds__(kRouteThreads) route_place_kernel(const RouteArgs p, int block_rows, int blocks) {
    __shared__ int16_t chosen[kRouteRows * kMaxTopK];
    __shared__ int32_t base[kMaxExperts], total[kMaxExperts];
    __shared__ int warp_sum[kRouteWarps];
    extern __shared__ uint16_t part[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, block = blockIdx.x;
    const int64_t first = (int64_t)block * block_rows * p.top_k;
    const int n = (int)min((int64_t)block_rows * p.top_k, (int64_t)p.rows * p.top_k - first);
    pdl_wait();
    pdl_trigger();
    for (int i = threadIdx.x; i < n; i += kRouteThreads) chosen[i] = (int16_t)p.experts[first + i];
    if (blocks > kRouteSums) {
        for (int e = threadIdx.x; e < p.n_experts; e += kRouteThreads) {
            base[e] = p.work[(int64_t)e * (blocks + 1) + block];
            total[e] = p.work[(int64_t)e * (blocks + 1) + blocks];
        }
    } else {
        // four experts a warp at a time, all their counts asked for at once
        for (int e0 = warp * 4; e0 < p.n_experts; e0 += kRouteWarps * 4) {
            int before[4] = {0, 0, 0, 0}, all[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < kRouteSums / 32; ++i) {
                const int b = i * 32 + lane;
                if (i * 32 >= blocks) break;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int c = b < blocks && e0 + j < p.n_experts ? p.work[(int64_t)(e0 + j) * (blocks + 1) + b] : 0;
                    all[j] += c;
                    if (b < block) before[j] += c;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int x = __reduce_add_sync(0xffffffffu, before[j]), y = __reduce_add_sync(0xffffffffu, all[j]);
                if (lane == 0 && e0 + j < p.n_experts) { base[e0 + j] = x; total[e0 + j] = y; }
            }
        }
    }
    __syncthreads();
    int used = 0;
    for (int e0 = 0; e0 < p.n_experts; e0 += kRouteThreads) {
        const int e = e0 + threadIdx.x;
        int all;
        const int at = used + block_before(e < p.n_experts ? total[e] : 0, warp_sum, &all);
        if (e < p.n_experts) {
            base[e] += at;
            if (block == 0) p.offsets[e] = at;
        }
        used += all;
    }
    if (block == 0 && threadIdx.x == 0) p.offsets[p.n_experts] = used;
    for (int64_t i = max(first, (int64_t)used) + threadIdx.x; i < first + n; i += kRouteThreads) p.order[i] = -1;
    __syncthreads();
    route_place(p, chosen, base, part, block * block_rows, n);
}

// fn(kernel) for the form of the choice that a number of experts takes
template <typename T, typename Fn>
cudaError_t route_form(int n_experts, Fn fn) {
    if (n_experts <= 32) return fn(route_choose_kernel<4, 8, T>);
    if (n_experts <= 64) return fn(route_choose_kernel<8, 8, T>);
    if (n_experts <= 128) return fn(route_choose_kernel<8, 16, T>);
    if (n_experts <= 256) return fn(route_choose_kernel<16, 16, T>);
    return fn(route_choose_kernel<32, 32, T>);
}
size_t route_part_bytes(int n_experts) { return (size_t)kRouteWarps * n_experts * sizeof(uint16_t); }

// out[row] (+)= alpha sum_j weights[row][j] y[slots[row][j]], in 32 bits in the order of j, rounded once.  A thread takes eight
// columns where rows lie on 16-byte boundaries, else one; four results' pieces are asked for at once.
template <typename Y, int PER>
__global__ void __launch_bounds__(256) combine_kernel(const CombineArgs p) {
    pdl_wait();
    pdl_trigger();
    constexpr int kAhead = 4, kWords = PER * (int)sizeof(Y) / 16 > 0 ? PER * (int)sizeof(Y) / 16 : 1;
    const int groups = (p.cols + PER - 1) / PER;
    const int64_t total = (int64_t)p.rows * groups;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int row = (int)(i / groups), col = (int)(i % groups) * PER;
        float sum[PER];
#pragma unroll
        for (int c = 0; c < PER; ++c) sum[c] = 0.0f;
        for (int j0 = 0; j0 < p.top_k; j0 += kAhead) {
            int at[kAhead];
            float w[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int64_t k = (int64_t)row * p.top_k + j0 + j;
                at[j] = j0 + j < p.top_k ? __ldg(p.slots + k) : -1;
                if ((unsigned)at[j] >= (unsigned long long)p.y_rows) at[j] = -1;
                w[j] = at[j] >= 0 ? (p.weights ? __ldg(p.weights + k) : 1.0f) : 0.0f;
            }
            if constexpr (PER == 8) {
                uint4 v[kAhead][kWords];
#pragma unroll
                for (int j = 0; j < kAhead; ++j)
#pragma unroll
                    for (int q = 0; q < kWords; ++q) {
                        v[j][q] = make_uint4(0, 0, 0, 0);
                        if (at[j] >= 0) v[j][q] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const Y*>(p.y) + (int64_t)at[j] * p.ldy + col) + q);
                    }
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    if (at[j] < 0) continue;
                    if constexpr (sizeof(Y) == 2) {
                        const uint32_t u[4] = {v[j][0].x, v[j][0].y, v[j][0].z, v[j][0].w};
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            sum[2 * c] = fmaf(w[j], __uint_as_float(u[c] << 16), sum[2 * c]);
                            sum[2 * c + 1] = fmaf(w[j], __uint_as_float(u[c] & 0xffff0000u), sum[2 * c + 1]);
                        }
                    } else {
#pragma unroll
                        for (int q = 0; q < kWords; ++q) {
                            const uint32_t u[4] = {v[j][q].x, v[j][q].y, v[j][q].z, v[j][q].w};
#pragma unroll
                            for (int c = 0; c < 4; ++c) sum[4 * q + c] = fmaf(w[j], __uint_as_float(u[c]), sum[4 * q + c]);
                        }
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < kAhead; ++j)
                    if (at[j] >= 0) sum[0] = fmaf(w[j], (float)static_cast<const Y*>(p.y)[(int64_t)at[j] * p.ldy + col], sum[0]);
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
    const int64_t blocks = route_blocks(rows);
    return blocks > 1 ? n_experts * (blocks + 1) * (int64_t)sizeof(int32_t) : 0;
}

cudaError_t route_configure() {
    const int most = (int)route_part_bytes(kMaxExperts);
    cudaError_t e = cudaFuncSetAttribute(route_place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    auto set = [&](auto kernel) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most); };
    for (int n : {32, 64, 128, 256, 1024}) {
        if (e == cudaSuccess) e = route_form<float>(n, set);
        if (e == cudaSuccess) e = route_form<__nv_bfloat16>(n, set);
    }
    return e;
}

cudaError_t route_launch(const RouteArgs& args, cudaStream_t stream, int64_t* launches) {
    if (args.rows <= 0) return cudaMemsetAsync(args.offsets, 0, sizeof(int32_t) * (args.n_experts + 1), stream);
    RouteArgs g = args;
    const int eb = g.bf16 ? 2 : 4;
    g.vec = !(reinterpret_cast<uintptr_t>(g.logits) & 15) && !((g.ld * eb) & 15) && !((g.n_experts * eb) & 15);
    const int block_rows = route_block_rows(g.rows), blocks = (int)route_blocks(g.rows);
    auto choose = [&](auto kernel) {
        return launch_pdl(kernel, dim3(blocks), kRouteThreads, blocks == 1 ? route_part_bytes(g.n_experts) : 0, stream, 1, g, block_rows, blocks);
    };
    cudaError_t e = g.bf16 ? route_form<__nv_bfloat16>(g.n_experts, choose) : route_form<float>(g.n_experts, choose);
    *launches += 1;
    if (e != cudaSuccess || blocks == 1) return e;
    if (blocks > kRouteSums) {
        e = launch_pdl(route_sums_kernel, dim3((g.n_experts + 7) / 8), 256, 0, stream, 1, g, blocks);
        *launches += 1;
        if (e != cudaSuccess) return e;
    }
    *launches += 1;
    return launch_pdl(route_place_kernel, dim3(blocks), kRouteThreads, route_part_bytes(g.n_experts), stream, 1, g, block_rows, blocks);
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
