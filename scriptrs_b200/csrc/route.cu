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
constexpr int kCombineFew = 148 * 8;  // pieces of 32 lanes up to which each gets a warp: eight warps an SM

// Rows per block: as many blocks as there are SMs to fill with a pass of 64 rows or more.
int route_block_rows(int64_t rows) {
    if (rows <= kRouteOneBlock) return kRouteOneBlock;
    return (int)std::min<int64_t>(kRouteRows, (rows + 147) / 148 <= 64 ? 64 : ((rows + 147) / 148 + 63) / 64 * 64);
}
int64_t route_blocks(int64_t rows) { return (rows + route_block_rows(rows) - 1) / route_block_rows(rows); }

// What a logit counts as: NaN as -inf, which is never chosen, +inf as the largest finite value of its type.
__device__ __forceinline__ float route_logit(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }
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

// the largest of key - below (mod 2^32) over the row
template <int LANES, int PER>
__device__ __forceinline__ uint32_t route_most(const uint32_t (&key)[PER], uint32_t below) {
    uint32_t m = key[0] - below;
#pragma unroll
    for (int i = 1; i < PER; ++i) m = __viaddmax_u32(key[i], 0u - below, m);
#pragma unroll
    for (int d = LANES / 2; d; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
    return m;
}
template <int LANES>
__device__ __forceinline__ float route_sum(float v) {
#pragma unroll
    for (int d = LANES / 2; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}

// LANES lanes take a row, PER neighbouring experts each, in registers.  A round finds the largest key below the one before as the
// maximum of key - previous in unsigned arithmetic: what lies below wraps round to the top, nearest first.
//   bf16: a key is 16 bits, the expert (counted down) takes the other 16: keys differ and a round yields one choice.
//   f32:  a round yields a value; the experts that have it follow in ascending order.
// `live`: the row exists (its lanes take part in the shuffles either way).
// Bound by issue slots, so for bf16 the keys are made two at a time, NaN and +inf are looked at only where a row's largest key says that
// there are some, and a choice is turned back into its value once, by the lane that keeps it (52360 rows of 128, 4 each: 15 -> 11 us).
template <int LANES, int PER>
__device__ __forceinline__ void route_row(const RouteArgs& p, int row, bool live, int lane, int16_t* chosen, const __nv_bfloat16* logits) {
    const int l = lane % LANES;
    uint32_t w[PER / 2], key[PER];
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) w[i] = 0xff80ff80u;  // -inf
    const unsigned short* x = reinterpret_cast<const unsigned short*>(logits) + (int64_t)row * p.ld + l * PER;
    const int mine = p.n_experts - l * PER;  // experts from this lane's first on
    if (p.vec) {
#pragma unroll
        for (int i = 0; i < PER; i += 8) {
            if (!live || i >= mine) continue;
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(x + i));
            w[i / 2] = v.x; w[i / 2 + 1] = v.y; w[i / 2 + 2] = v.z; w[i / 2 + 3] = v.w;
        }
    } else if (live) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (i < mine) w[i / 2] = i % 2 ? (w[i / 2] & 0xffffu) | ((uint32_t)__ldg(x + i) << 16) : (w[i / 2] & 0xffff0000u) | __ldg(x + i);
    }
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) {
        // -0 as 0; then a negative value's bits are inverted, the others' sign set
        asm("{\n\t.reg .b32 z, n;\n\tmov.b32 z, 0;\n\tadd.rn.bf16x2 %0, %0, z;\n\tprmt.b32 n, %0, z, 0xBB99;\n\tor.b32 n, n, 0x80008000;\n\txor.b32 %1, %0, n;\n\t}"
            : "+r"(w[i]), "=r"(key[2 * i]));
        key[2 * i + 1] = (key[2 * i] & 0xffff0000u) | (0xffffu - (uint32_t)(l * PER + 2 * i + 1));
        key[2 * i] = (key[2 * i] << 16) | (0xffffu - (uint32_t)(l * PER + 2 * i));
    }
    uint32_t first = route_most<LANES>(key, 0u);
    if (__any_sync(0xffffffffu, first >= 0xff800000u)) {  // +inf (counts as the largest finite value) or, above it, NaN (as -inf)
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (key[i] < 0xff800000u) continue;
            const bool nan = key[i] >= 0xff810000u;
            key[i] = (key[i] & 0xffffu) | (nan ? 0u : 0xff7f0000u);
            const uint32_t as = nan ? 0xff80u : 0x7f7fu;
            w[i / 2] = i % 2 ? (w[i / 2] & 0xffffu) | (as << 16) : (w[i / 2] & 0xffff0000u) | as;
        }
        first = route_most<LANES>(key, 0u);
    }
    // a key's lower half stands for the zeros of a bf16 value, inverted where it is negative
    auto value = [](uint32_t k) { return route_value((k & 0xffff0000u) | ((k & 0x80000000u) ? 0u : 0xffffu)); };
    const float top = first >= kRouteNone ? value(first) : 0.0f;
    float total = 0.0f;
    if (!p.normalize) {
#pragma unroll
        for (int i = 0; i < PER / 2; ++i)
            total += route_exp(__uint_as_float(w[i] << 16) - top) + route_exp(__uint_as_float(w[i] & 0xffff0000u) - top);
        total = route_sum<LANES>(total);
    }
    constexpr int kKeep = (kMaxTopK + LANES - 1) / LANES;  // lane l keeps the choices l, l + LANES, ...
    uint32_t kept[kKeep];
#pragma unroll
    for (int i = 0; i < kKeep; ++i) kept[i] = 0u;
    uint32_t best = first;
    for (int j = 0;; ++j) {
#pragma unroll
        for (int i = 0; i < kKeep; ++i)
            if (l + i * LANES == j) kept[i] = best;
        if (j + 1 == p.top_k) break;
        const uint32_t next = route_most<LANES>(key, best) + best;  // shuffles: by every lane, its row over or not
        best = best >= kRouteNone ? next : 0u;
    }
    float weight[kKeep];
#pragma unroll
    for (int i = 0; i < kKeep; ++i) weight[i] = kept[i] >= kRouteNone ? route_exp(value(kept[i]) - top) : 0.0f;
    if (p.normalize) {
#pragma unroll
        for (int i = 0; i < kKeep; ++i) total += weight[i];
        total = route_sum<LANES>(total);
    }
    if (!live) return;
    const int64_t out = (int64_t)row * p.top_k;
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
        const int j = l + i * LANES;
        if (j >= p.top_k) break;
        const int who = kept[i] >= kRouteNone ? (int)(0xffffu - (kept[i] & 0xffffu)) : -1;
        p.experts[out + j] = who;
        p.weights[out + j] = who >= 0 ? __fdividef(weight[i], total) : 0.0f;  // 1 <= total <= 1024
        chosen[j] = (int16_t)who;
    }
}

template <int LANES, int PER>
__device__ __forceinline__ void route_row(const RouteArgs& p, int row, bool live, int lane, int16_t* chosen, const float* logits) {
    const int l = lane % LANES;
    uint32_t key[PER];
    float total = 0.0f, top;
    uint32_t first;
    {
        float f[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) f[i] = -INFINITY;
        const float* x = logits + (int64_t)row * p.ld;
        if (PER % 4 == 0 && p.vec) {
#pragma unroll
            for (int i = 0; i < PER; i += 4) {
                if (!live || l * PER + i >= p.n_experts) continue;
                const float4 v = __ldg(reinterpret_cast<const float4*>(x + l * PER + i));
                f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
            }
        } else if (live) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (l * PER + i < p.n_experts) f[i] = x[l * PER + i];
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            f[i] = route_logit(f[i]);
            key[i] = route_key(f[i]);
        }
        first = route_most<LANES>(key, 0u);
        top = first >= kRouteNone ? route_value(first) : 0.0f;
        if (!p.normalize) {
#pragma unroll
            for (int i = 0; i < PER; ++i) total += route_exp(f[i] - top);
            total = route_sum<LANES>(total);
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
    const int group0 = lane / LANES * LANES;
    int j = 0;
    while (__any_sync(0xffffffffu, best >= kRouteNone && j < p.top_k)) {
        uint32_t has = 0;  // this lane's experts with that value
#pragma unroll
        for (int i = 0; i < PER; ++i) has |= key[i] == best ? 1u << i : 0u;
        if (best < kRouteNone) has = 0;
        const float w = best >= kRouteNone ? route_exp(route_value(best) - top) : 0.0f;
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
        const uint32_t next = route_most<LANES>(key, best) + best;
        best = best >= kRouteNone ? next : 0u;
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
        route_row<LANES, PER>(p, row0 + r, r < rows, lane, chosen + min(r, rows - 1) * p.top_k, static_cast<const T*>(p.logits));
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

// PER neighbouring values, at an address on a boundary of all of them (at most 16 bytes).
template <typename T, int PER>
struct Piece {
    static constexpr int kBytes = PER * (int)sizeof(T), kWords = kBytes >= 4 ? kBytes / 4 : 1;
    uint32_t w[kWords];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0u;
    }
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kBytes >= 16) {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) {
                const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p) + i / 4);
                w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
            }
        } else if constexpr (kBytes == 8) {
            const uint2 v = __ldcs(reinterpret_cast<const uint2*>(p));
            w[0] = v.x; w[1] = v.y;
        } else if constexpr (kBytes == 4) {
            w[0] = __ldcs(reinterpret_cast<const unsigned int*>(p));
        } else {
            w[0] = __ldcs(reinterpret_cast<const unsigned short*>(p));
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else return __uint_as_float(i % 2 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
    __device__ __forceinline__ void set(int i, float v) {
        if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v);
        else {
            const uint32_t h = __bfloat16_as_ushort(__float2bfloat16_rn(v));
            w[i / 2] = i % 2 ? (w[i / 2] & 0xffffu) | (h << 16) : h;
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kBytes >= 16) {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) reinterpret_cast<uint4*>(p)[i / 4] = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        } else if constexpr (kBytes == 8) {
            *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
        } else if constexpr (kBytes == 4) {
            *reinterpret_cast<uint32_t*>(p) = w[0];
        } else {
            *reinterpret_cast<unsigned short*>(p) = (unsigned short)w[0];
        }
    }
};

// out[row] (+)= alpha sum_j weights[row][j] y[slots[row][j]], in 32 bits in the order of j, rounded once.  A warp takes U pieces a lane
// of a row, a piece as many columns as the rows' boundaries allow, so that slots and weights are read once for all of them, and asks
// for the pieces of four results at once: bound by the bytes in flight.
// With one or two results a row it asks for no more than those (registers for four leave too few warps: 60 against 44 us at 52360 x
// 1024, one result); a few rows are spread over as many warps as they give (U = 1).
template <typename Y, typename O, int PER, int kAhead, int U>
__global__ void __launch_bounds__(256) combine_kernel(const CombineArgs p, int chunks) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t total = (int64_t)p.rows * chunks;
    for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < total; i += (int64_t)gridDim.x * 8) {
        // (a 64-bit division only where the work does not fit 32 bits)
        const int row = total <= 0xffffffffLL ? (int)((uint32_t)i / (uint32_t)chunks) : (int)(i / chunks);
        const int col0 = ((int)(i - (int64_t)row * chunks) * U * 32 + lane) * PER;
        const int64_t k0 = (int64_t)row * p.top_k;
        float sum[U][PER];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < PER; ++c) sum[u][c] = 0.0f;
        for (int j0 = 0; j0 < p.top_k; j0 += kAhead) {
            int at[kAhead];
            float w[kAhead];
            Piece<Y, PER> v[kAhead][U];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                at[j] = j0 + j < p.top_k ? __ldg(p.slots + k0 + j0 + j) : -1;
                w[j] = j0 + j < p.top_k && p.weights ? __ldg(p.weights + k0 + j0 + j) : 1.0f;
                if ((unsigned)at[j] >= (unsigned long long)p.y_rows) at[j] = -1;
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (at[j] < 0) continue;
                const Y* y = static_cast<const Y*>(p.y) + (int64_t)at[j] * p.ldy;
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (col0 + u * 32 * PER < p.cols) v[j][u].load(y + col0 + u * 32 * PER);
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (at[j] < 0) continue;  // (a weight of zero would not do: 0 * inf)
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int c = 0; c < PER; ++c) sum[u][c] = fmaf(w[j], v[j][u].get(c), sum[u][c]);
            }
        }
        O* out = static_cast<O*>(p.out) + (int64_t)row * p.ldo;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int col = col0 + u * 32 * PER;
            if (col >= p.cols) continue;
            Piece<O, PER> r;
            r.zero();
            if (sizeof(O) == 4 && p.out_mode == kOutResidual) r.load(out + col);
#pragma unroll
            for (int c = 0; c < PER; ++c) {
                float v = p.alpha * sum[u][c];
                if (sizeof(O) == 4 && p.out_mode == kOutResidual) v += r.get(c);
                r.set(c, v);
            }
            r.store(out + col);
        }
    }
}

template <typename Y, typename O, int PER>
cudaError_t combine_per(const CombineArgs& g, cudaStream_t stream) {
    constexpr int kWide = PER == 8 ? 4 : 8;  // pieces a lane: 2 KB of a bf16 row a warp, less of rows on narrower boundaries
    auto go = [&](auto kernel, int pieces) {
        const int wide = 32 * PER * pieces, chunks = (g.cols + wide - 1) / wide;
        const dim3 grid((unsigned)std::min<int64_t>(((int64_t)g.rows * chunks + 7) / 8, 1 << 20));
        return launch_pdl(kernel, grid, 256, 0, stream, 1, g, chunks);
    };
    if ((int64_t)g.rows * ((g.cols + 32 * PER - 1) / (32 * PER)) <= kCombineFew) return go(combine_kernel<Y, O, PER, 4, 1>, 1);
    if (g.top_k == 1) return go(combine_kernel<Y, O, PER, 1, kWide>, kWide);
    if (g.top_k == 2) return go(combine_kernel<Y, O, PER, 2, kWide>, kWide);
    return go(combine_kernel<Y, O, PER, 4, kWide>, kWide);
}

template <typename Y, typename O>
cudaError_t combine_t(const CombineArgs& g, cudaStream_t stream) {
    // boundaries that every row of both sides has, in values: a piece of PER lies on min(PER values, 16 bytes)
    auto fits = [&](int per) {
        const int yb = std::min<int>(per * sizeof(Y), 16), ob = std::min<int>(per * sizeof(O), 16);
        return g.cols % per == 0 && !(reinterpret_cast<uintptr_t>(g.y) % yb) && !(reinterpret_cast<uintptr_t>(g.out) % ob) &&
               !((g.ldy * (int)sizeof(Y)) % yb) && !((g.ldo * (int)sizeof(O)) % ob);
    };
    const int per = fits(8) ? 8 : (fits(4) ? 4 : (fits(2) ? 2 : 1));
    switch (per) {
        case 8: return combine_per<Y, O, 8>(g, stream);
        case 4: return combine_per<Y, O, 4>(g, stream);
        case 2: return combine_per<Y, O, 2>(g, stream);
        default: return combine_per<Y, O, 1>(g, stream);
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
    if (g.out_mode == kOutBf16) return g.y_f32 ? combine_t<float, __nv_bfloat16>(g, stream) : combine_t<__nv_bfloat16, __nv_bfloat16>(g, stream);
    return g.y_f32 ? combine_t<float, float>(g, stream) : combine_t<__nv_bfloat16, float>(g, stream);
}

}  // namespace sb
