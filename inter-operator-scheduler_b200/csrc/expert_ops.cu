// The bandwidth-bound operators of an expert layer: the router with its plan, the 8-bit row quantiser and the
// gate-weighted sum of expert rows.  Their counterparts among the convolution network's operators are in
// bandwidth_ops.cu; the products are in expert_mm.cu.
#include "expert_ops.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

namespace ios {
namespace {

// ---- element access ----------------------------------------------------------------------------
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// ---- router ------------------------------------------------------------------------------------

// A logit as an unsigned key whose order is the logits' order; 0 for a logit that may not be chosen (NaN, -inf).
// Both zeros get one key, so that they tie.
__device__ __forceinline__ uint32_t logit_key(float v) {
    if (!(v > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}

// exp(v - top), with +inf logits sharing the weight among themselves instead of producing NaN
__device__ __forceinline__ float softmax_term(float v, float top) { return v == top ? 1.0f : expf(v - top); }

constexpr int kRouteThreads = 512;
constexpr int kRouteWarps = kRouteThreads / 32;

// The k best experts of tokens [first, last): one warp per token, logit e in register e / 32 of lane e % 32.
// Each pick takes two warp reductions (largest key, then its lowest index) and drops the winner.
template <class T, int PER>
__device__ __forceinline__ void pick_experts(const RouteParams &p, int first, int last) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int t = first + warp; t < last; t += kRouteWarps) {
        const T *row = static_cast<const T *>(p.logits) + (long long)t * p.stride;
        uint32_t key[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = i * 32 + lane;
            key[i] = e < p.experts ? logit_key(to_float(row[e])) : 0u;
        }
        uint32_t mine = 0;
        int mine_at = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (key[i] > mine) { mine = key[i]; mine_at = i; }
        const uint32_t top = __reduce_max_sync(0xffffffffu, mine);
        const float top_logit = key_logit(top);
        float sum = 0.0f;
        if (!p.renormalize && top != 0) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (key[i]) sum += softmax_term(key_logit(key[i]), top_logit);
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        }
        int my_expert = -1;          // lane j keeps pick j
        float my_weight = 0.0f;
        for (int j = 0; j < p.k; ++j) {
            const uint32_t best = __reduce_max_sync(0xffffffffu, mine);
            if (best == 0) break;                                                // no expert left: the rest stays -1
            const uint32_t at = __reduce_min_sync(0xffffffffu, mine == best ? uint32_t(mine_at * 32 + lane) : 0xffffffffu);
            if (lane == j) {
                my_expert = int(at);
                my_weight = softmax_term(key_logit(best), top_logit);
            }
            if (lane == int(at & 31u)) {
                mine = 0;
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    if (i == int(at >> 5)) key[i] = 0;
                    if (key[i] > mine) { mine = key[i]; mine_at = i; }
                }
            }
        }
        if (p.renormalize) {
            sum = my_weight;
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        }
        if (lane < p.k) {
            p.chosen[(long long)t * p.k + lane] = my_expert;
            p.gates[(long long)t * p.k + lane] = my_expert >= 0 ? my_weight / sum : 0.0f;
        }
    }
}

// Exclusive prefix sums of count[0 .. n) (n <= 2 * kRouteThreads) in place; returns the total.  All threads call it.
__device__ int exclusive_scan(int *count, int n) {
    __shared__ int warp_total[kRouteWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, e = 2 * threadIdx.x;
    const int a = e < n ? count[e] : 0, b = e + 1 < n ? count[e + 1] : 0;
    int run = a + b;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, run, s);
        if (lane >= s) run += v;
    }
    if (lane == 31) warp_total[warp] = run;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kRouteWarps; ++w) {
        if (w < warp) before += warp_total[w];
        total += warp_total[w];
    }
    const int start = before + run - a - b;
    __syncthreads();
    if (e < n) count[e] = start;
    if (e + 1 < n) count[e + 1] = start + a;
    __syncthreads();
    return total;
}

// Picks the experts of one range of tokens and counts its pairs by expert.  The order of the plan is the order of
// the pairs (token, then pick) within each expert: every warp ranks a contiguous run of pairs, 32 at a time by
// matching equal experts across its lanes, so nothing depends on timing.
// kSingle: the grid is one block and the plan is finished here; otherwise slots[] holds ranks inside the block and
// route_place_kernel adds what lies before it.
template <class T, int PER, bool kSingle>
__global__ void __launch_bounds__(kRouteThreads) route_pick_kernel(const RouteParams p, int per_block) {
    extern __shared__ int counts[];                    // [kRouteWarps][experts], then [experts]
    const int first = blockIdx.x * per_block, last = min(p.tokens, first + per_block);
    for (int i = threadIdx.x; i < kRouteWarps * p.experts; i += kRouteThreads) counts[i] = 0;
    pick_experts<T, PER>(p, first, last);
    __syncthreads();

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long pair0 = (long long)first * p.k;
    const int pairs = (last - first) * p.k;
    const int run = (pairs + kRouteWarps * 32 - 1) / (kRouteWarps * 32) * 32;          // pairs per warp
    const int begin = min(pairs, warp * run), end = min(pairs, begin + run);
    int *mine = counts + warp * p.experts;
    for (int i = begin + lane; i - lane < end; i += 32) {
        const int e = i < end ? p.chosen[pair0 + i] : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        const int before = __popc(same & ((1u << lane) - 1u));
        int base = 0;
        if (e >= 0) base = mine[e];
        __syncwarp();
        if (e >= 0 && before == 0) mine[e] = base + __popc(same);
        __syncwarp();
        if (i < end) p.slots[pair0 + i] = e >= 0 ? base + before : -1;
    }
    __syncthreads();
    // counts per warp -> what lies before each warp; totals of the block behind them
    int *totals = counts + kRouteWarps * p.experts;
    for (int e = threadIdx.x; e < p.experts; e += kRouteThreads) {
        int sum = 0;
        for (int w = 0; w < kRouteWarps; ++w) {
            const int c = counts[w * p.experts + e];
            counts[w * p.experts + e] = sum;
            sum += c;
        }
        totals[e] = sum;
        if (!kSingle) p.block_counts[(long long)blockIdx.x * p.experts + e] = sum;
    }
    __syncthreads();
    int used = 0;
    if (kSingle) {
        used = exclusive_scan(totals, p.experts);
        for (int e = threadIdx.x; e < p.experts; e += kRouteThreads) p.offsets[e] = totals[e];
        if (threadIdx.x == 0) p.offsets[p.experts] = used;
    }
    for (int i = begin + lane; i < end; i += 32) {
        const int e = p.chosen[pair0 + i];
        if (e < 0) continue;
        const int slot = p.slots[pair0 + i] + mine[e] + (kSingle ? totals[e] : 0);
        p.slots[pair0 + i] = slot;
        if (kSingle) p.rows[slot] = first + i / p.k;
    }
    if (kSingle)
        for (int i = used + int(threadIdx.x); i < pairs; i += kRouteThreads) p.rows[i] = -1;
}

// Second pass of a plan over many blocks: block b adds, per expert, the expert's start and the pairs of blocks < b.
__global__ void __launch_bounds__(kRouteThreads) route_place_kernel(const RouteParams p, int per_block, int blocks) {
    extern __shared__ int counts[];                    // [experts] starts, then [experts] pairs in earlier blocks
    int *start = counts, *earlier = counts + p.experts;
    for (int e = threadIdx.x; e < p.experts; e += kRouteThreads) {
        int sum = 0, before = 0;
        for (int b = 0; b < blocks; ++b) {
            if (b == int(blockIdx.x)) before = sum;
            sum += p.block_counts[(long long)b * p.experts + e];
        }
        start[e] = sum;
        earlier[e] = before;
    }
    __syncthreads();
    const int used = exclusive_scan(start, p.experts);
    if (blockIdx.x == 0) {
        for (int e = threadIdx.x; e < p.experts; e += kRouteThreads) p.offsets[e] = start[e];
        if (threadIdx.x == 0) p.offsets[p.experts] = used;
    }
    const int first = blockIdx.x * per_block, last = min(p.tokens, first + per_block);
    const long long pair0 = (long long)first * p.k;
    const int pairs = (last - first) * p.k;
    for (int i = threadIdx.x; i < pairs; i += kRouteThreads) {
        const int e = p.chosen[pair0 + i];
        if (e < 0) continue;
        const int slot = p.slots[pair0 + i] + start[e] + earlier[e];
        p.slots[pair0 + i] = slot;
        p.rows[slot] = first + i / p.k;
    }
    const long long all = (long long)p.tokens * p.k;
    for (long long i = used + (long long)blockIdx.x * kRouteThreads + threadIdx.x; i < all; i += (long long)blocks * kRouteThreads)
        p.rows[i] = -1;
}

// Tokens one block plans: a small call is one block and one launch; beyond that at most 128 blocks, because every
// block of the second pass reads the counts of all of them.
constexpr int kRouteSingleTokens = 256;
int route_per_block(int tokens) { return tokens <= kRouteSingleTokens ? tokens : std::max(32, (tokens + 127) / 128); }
int route_blocks(int tokens) { return (tokens + route_per_block(tokens) - 1) / route_per_block(tokens); }

template <class T, int PER>
cudaError_t route_run(const RouteParams &p, cudaStream_t stream) {
    const int per_block = route_per_block(p.tokens), blocks = route_blocks(p.tokens);
    const size_t smem = size_t(kRouteWarps + 1) * p.experts * sizeof(int);
    const void *fn = blocks == 1 ? reinterpret_cast<const void *>(route_pick_kernel<T, PER, true>)
                                 : reinterpret_cast<const void *>(route_pick_kernel<T, PER, false>);
    if (smem > 48 * 1024) {
        cudaError_t err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
        if (err != cudaSuccess) return err;
    }
    if (blocks == 1) {
        route_pick_kernel<T, PER, true><<<1, kRouteThreads, smem, stream>>>(p, per_block);
        return cudaGetLastError();
    }
    route_pick_kernel<T, PER, false><<<blocks, kRouteThreads, smem, stream>>>(p, per_block);
    route_place_kernel<<<blocks, kRouteThreads, 2 * p.experts * sizeof(int), stream>>>(p, per_block, blocks);
    return cudaGetLastError();
}

template <class T>
cudaError_t route_typed(const RouteParams &p, cudaStream_t stream) {
    if (p.experts <= 32) return route_run<T, 1>(p, stream);
    if (p.experts <= 64) return route_run<T, 2>(p, stream);
    if (p.experts <= 128) return route_run<T, 4>(p, stream);
    if (p.experts <= 256) return route_run<T, 8>(p, stream);
    if (p.experts <= 512) return route_run<T, 16>(p, stream);
    return route_run<T, 32>(p, stream);
}

// ---- row quantiser -----------------------------------------------------------------------------

// The whole number nearest to 127 x / largest (halves to even), from the float product x * inverse and, where that
// falls next to a half, from the exact comparison of 127 |x| with (n + 1/2) largest: both are at most 33 bits long,
// so their difference in double precision is exact.  NaN gives 0, an infinity +-127.
__device__ __forceinline__ int quantize_one(float x, float inverse, float largest, float lift) {
    if (!(fabsf(x) <= 3.402823466e38f)) return isnan(x) ? 0 : (x > 0 ? 127 : -127);
    const float t = fabsf(x * lift) * inverse;
    const float n = floorf(t);
    int q;
    if (fabsf(t - n - 0.5f) < 1e-3f) {
        const double d = 127.0 * double(fabsf(x)) - (double(n) + 0.5) * double(largest);
        q = int(n) + (d > 0.0 || (d == 0.0 && (int(n) & 1)) ? 1 : 0);
    } else {
        q = int(rintf(t));
    }
    q = min(q, 127);
    return x < 0 ? -q : q;
}

// One row per block.  The row is read twice: the second pass finds it in L1.
template <class T>
__global__ void __launch_bounds__(256) quantize_kernel(const QuantizeParams p) {
    __shared__ float warp_max[8];
    for (long long r = blockIdx.x; r < p.total; r += gridDim.x) {
        long long src = p.rows ? p.rows[r] : r;
        const bool live = src >= 0 && src < p.x_rows;
        const T *x = static_cast<const T *>(p.x) + (live ? src : 0) * p.x_stride;
        float largest = 0.0f;
        if (live)
            for (int c = threadIdx.x; c < p.inner; c += blockDim.x) {
                const float v = fabsf(to_float(x[c]));
                if (v <= 3.402823466e38f) largest = fmaxf(largest, v);
            }
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, s));
        if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = largest;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w) largest = fmaxf(largest, warp_max[w]);
        __syncthreads();
        if (threadIdx.x == 0) p.scale[r] = largest / 127.0f;
        // rows of tiny values are lifted by 2^64, so that 127 / largest stays finite
        const float lift = largest < 1e-30f ? 18446744073709551616.0f : 1.0f;
        const float inverse = largest > 0.0f ? 127.0f / (largest * lift) : 0.0f;
        signed char *q = p.q + r * p.q_stride;
        for (int c = threadIdx.x; c < p.inner; c += blockDim.x)
            q[c] = live ? (signed char)quantize_one(to_float(x[c]), inverse, largest, lift) : 0;
    }
}

// ---- weighted sum of expert rows ----------------------------------------------------------------

template <class T, class O>
__global__ void __launch_bounds__(256) combine_kernel(const CombineParams p) {
    for (long long t = blockIdx.x; t < p.tokens; t += gridDim.x) {
        const float *gates = p.gates + t * p.k;
        const int *slots = p.slots + t * p.k;
        O *out = static_cast<O *>(p.out) + t * p.out_stride;
        for (int c = threadIdx.x; c < p.channels; c += blockDim.x) {
            float sum = 0.0f;
            for (int j = 0; j < p.k; ++j) {
                const int s = slots[j];
                if (s >= 0 && s < p.y_rows) sum += gates[j] * to_float(static_cast<const T *>(p.y)[(long long)s * p.y_stride + c]);
            }
            out[c] = from_float<O>(sum);
        }
    }
}

template <class T>
void combine_typed(const CombineParams &p, unsigned blocks, cudaStream_t stream) {
    if (p.out_type == Elem::F32) combine_kernel<T, float><<<blocks, 256, 0, stream>>>(p);
    else if (p.out_type == Elem::F16) combine_kernel<T, __half><<<blocks, 256, 0, stream>>>(p);
    else combine_kernel<T, __nv_bfloat16><<<blocks, 256, 0, stream>>>(p);
}

}  // namespace

size_t route_workspace_bytes(int tokens, int experts) {
    const int blocks = route_blocks(tokens);
    return blocks == 1 ? 0 : size_t(blocks) * experts * sizeof(int);
}

cudaError_t launch_route(const RouteParams &p, cudaStream_t stream) {
    if (p.type == Elem::F32) return route_typed<float>(p, stream);
    if (p.type == Elem::F16) return route_typed<__half>(p, stream);
    return route_typed<__nv_bfloat16>(p, stream);
}

cudaError_t launch_quantize(const QuantizeParams &p, cudaStream_t stream) {
    const unsigned blocks = unsigned(std::min<long long>(p.total, INT_MAX));
    if (p.type == Elem::F32) quantize_kernel<float><<<blocks, 256, 0, stream>>>(p);
    else if (p.type == Elem::F16) quantize_kernel<__half><<<blocks, 256, 0, stream>>>(p);
    else quantize_kernel<__nv_bfloat16><<<blocks, 256, 0, stream>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_combine(const CombineParams &p, cudaStream_t stream) {
    const unsigned blocks = unsigned(std::min<long long>(p.tokens, INT_MAX));
    if (p.type == Elem::F32) combine_typed<float>(p, blocks, stream);
    else if (p.type == Elem::F16) combine_typed<__half>(p, blocks, stream);
    else combine_typed<__nv_bfloat16>(p, blocks, stream);
    return cudaGetLastError();
}

}  // namespace ios
