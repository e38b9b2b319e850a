// The bandwidth-bound operators of an expert layer: the router with its plan, the 8-bit row quantiser and the
// gate-weighted sum of expert rows.  Their counterparts among the convolution network's operators are in
// bandwidth_ops.cu; the products are in expert_mm.cu.
#include "expert_ops.h"
#include "kernels.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

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

// V elements that are moved by one access
template <class T, int V>
struct alignas(V * sizeof(T)) Vector {
    T v[V];
};
template <class O, int V>
__device__ __forceinline__ void store_vector(O *p, const float (&v)[V]) {
    constexpr int kBytes = V * int(sizeof(O)), kPiece = kBytes < 16 ? kBytes : 16, kPer = kPiece / int(sizeof(O));
    alignas(16) O out[V];
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = from_float<O>(v[i]);
#pragma unroll
    for (int i = 0; i < V; i += kPer) {
        if (kPiece == 16) *reinterpret_cast<uint4 *>(p + i) = *reinterpret_cast<const uint4 *>(out + i);
        else if (kPiece == 8) *reinterpret_cast<uint2 *>(p + i) = *reinterpret_cast<const uint2 *>(out + i);
        else p[i] = out[i];
    }
}

// Launches with programmatic dependency: the kernels wait for their predecessors by themselves (grid_dependency_entry),
// so a block's start-up overlaps the end of the kernel before.
template <class... Params, class... Args>
cudaError_t launch(void (*kernel)(Params...), dim3 grid, int block, size_t smem, cudaStream_t stream, const Args &...args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(unsigned(block));
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, Params(args)...);
}
template <class... Params, class... Args>
cudaError_t launch(void (*kernel)(Params...), long long blocks, int block, size_t smem, cudaStream_t stream, const Args &...args) {
    return launch(kernel, dim3(unsigned(blocks)), block, smem, stream, args...);
}

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
// The same in 16 bits
__device__ __forceinline__ uint32_t ordered16(uint32_t b, bool able) {
    if (b == 0x8000u) b = 0;
    return !able ? 0u : (b & 0x8000u) ? (~b & 0xFFFFu) : (b | 0x8000u);
}
__device__ __forceinline__ uint32_t unordered16(uint32_t key) { return (key & 0x8000u) ? (key & 0x7FFFu) : (~key & 0xFFFFu); }

// What the picks compare: for 16-bit logits the key above the complement of the expert's index, so that one reduction finds
// the largest logit and the lowest index that has it; for float32 the key alone.
template <class T> struct Rank;
template <> struct Rank<float> {
    static constexpr bool kWithIndex = false;
    static __device__ __forceinline__ uint32_t of(float v, int) { return logit_key(v); }
    static __device__ __forceinline__ float logit(uint32_t rank) { return key_logit(rank); }
};
template <> struct Rank<__half> {
    static constexpr bool kWithIndex = true;
    static __device__ __forceinline__ uint32_t of(__half v, int e) {
        const uint32_t key = ordered16(__half_as_ushort(v), __half2float(v) > -INFINITY);
        return key ? key << 16 | (0xFFFFu - uint32_t(e)) : 0u;
    }
    static __device__ __forceinline__ float logit(uint32_t rank) { return __half2float(__ushort_as_half(uint16_t(unordered16(rank >> 16)))); }
};
template <> struct Rank<__nv_bfloat16> {
    static constexpr bool kWithIndex = true;
    static __device__ __forceinline__ uint32_t of(__nv_bfloat16 v, int e) {
        const uint32_t key = ordered16(__bfloat16_as_ushort(v), __bfloat162float(v) > -INFINITY);
        return key ? key << 16 | (0xFFFFu - uint32_t(e)) : 0u;
    }
    static __device__ __forceinline__ float logit(uint32_t rank) { return __uint_as_float(unordered16(rank >> 16) << 16); }
};

// exp(v - top), with +inf logits sharing the weight among themselves instead of producing NaN
__device__ __forceinline__ float softmax_term(float v, float top) { return v == top ? 1.0f : expf(v - top); }

// 32 warps, a token each at a time; a call of up to 8 tokens takes 8 warps, whose barriers cost less (4 tokens, 64 experts, k = 8: 3.1 us
// for 4.4; 32 tokens with 8 warps: 6.4 for 5.5)
constexpr int kRouteThreads = 1024;
constexpr int kRoutePairs = 8192;         // pairs that a block plans in shared memory
constexpr int kRouteDirectBlocks = 128;   // blocks whose counts each block of the second pass sums for itself

// The k best experts of tokens [first, last): one warp per token, logit e in register e / 32 of lane e % 32; the next
// token's logits are on their way meanwhile.  Each pick takes one or two warp reductions and drops the winner.
template <class T, int PER>
__device__ __forceinline__ void pick_experts(const RouteParams &p, int first, int last, int *chosen) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    T ahead[PER];
    const auto ask = [&](int t) {
        const T *row = static_cast<const T *>(p.logits) + (long long)t * p.stride;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (i * 32 + lane < p.experts) ahead[i] = row[i * 32 + lane];
    };
    if (first + warp < last) ask(first + warp);
    for (int t = first + warp; t < last; t += warps) {
        uint32_t rank[PER], mine = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            rank[i] = i * 32 + lane < p.experts ? Rank<T>::of(ahead[i], i * 32 + lane) : 0u;
            mine = max(mine, rank[i]);
        }
        if (t + warps < last) ask(t + warps);
        const uint32_t top = __reduce_max_sync(0xffffffffu, mine);
        const float top_logit = Rank<T>::logit(top);
        float sum = 0.0f;
        if (!p.renormalize && top != 0) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (rank[i]) sum += softmax_term(Rank<T>::logit(rank[i]), top_logit);
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        }
        int my_expert = -1;          // lane j keeps pick j
        uint32_t my_rank = 0;
        for (int j = 0; j < p.k; ++j) {
            const uint32_t best = j == 0 ? top : __reduce_max_sync(0xffffffffu, mine);
            if (best == 0) break;                                                // no expert left: the rest stays -1
            uint32_t at;
            if (Rank<T>::kWithIndex) {
                at = 0xFFFFu - (best & 0xFFFFu);
            } else {
                uint32_t lowest = 0xffffffffu;
#pragma unroll
                for (int i = PER - 1; i >= 0; --i)
                    if (rank[i] == best) lowest = uint32_t(i * 32 + lane);
                at = __reduce_min_sync(0xffffffffu, lowest);
            }
            if (lane == j) {
                my_expert = int(at);
                my_rank = best;
            }
            mine = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (i * 32 + lane == int(at)) rank[i] = 0;
                mine = max(mine, rank[i]);
            }
        }
        const float weight = my_expert >= 0 ? softmax_term(Rank<T>::logit(my_rank), top_logit) : 0.0f;
        if (p.renormalize) {
            sum = weight;
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        }
        if (lane < p.k) {
            p.chosen[(long long)t * p.k + lane] = my_expert;
            p.gates[(long long)t * p.k + lane] = my_expert >= 0 ? weight / sum : 0.0f;
            chosen[(t - first) * p.k + lane] = my_expert;
        }
    }
}

// Exclusive prefix sums of count[0 .. n) in place; returns the total.  All threads call it.
__device__ int exclusive_scan(int *count, int n) {
    __shared__ int warp_total[kRouteThreads / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int per = (n + int(blockDim.x) - 1) / int(blockDim.x), begin = min(int(threadIdx.x) * per, n), end = min(begin + per, n);
    int sum = 0;
    for (int e = begin; e < end; ++e) sum += count[e];
    int run = sum;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, run, s);
        if (lane >= s) run += v;
    }
    if (lane == 31) warp_total[warp] = run;
    __syncthreads();
    int start = run - sum, total = 0;
    for (int w = 0; w < warps; ++w) {
        if (w < warp) start += warp_total[w];
        total += warp_total[w];
    }
    for (int e = begin; e < end; ++e) {
        const int c = count[e];
        count[e] = start;
        start += c;
    }
    __syncthreads();
    return total;
}

// Picks the experts of one range of tokens and counts its pairs by expert.  The order of the plan is the order of
// the pairs (token, then pick) within each expert: every warp ranks a contiguous run of pairs, 32 at a time by
// matching equal experts across its lanes, so nothing depends on timing.
// kSingle: the grid is one block and the plan is finished here; otherwise slots[] holds ranks inside the block and
// route_place_kernel adds what lies before it.
// (16384 tokens, 128 experts, k = 8, bfloat16: 16 us from cold caches, bound by instructions, not by the 4 MB read: 490 a token, most
// of them the picks' comparing and selecting; instructions issue in 65 % of the cycles and the ALU is busy in 67 %.  The second pass
// takes 9.5 us, waiting for loads: the counts of all blocks, then what the first pass left of each pair.)
template <class T, int PER, bool kSingle>
__global__ void __launch_bounds__(kRouteThreads) route_pick_kernel(const RouteParams p, int per_block) {
    extern __shared__ int shared[];                    // [warps][experts] counts, [experts] totals, then chosen and rank of the pairs
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int first = blockIdx.x * per_block, last = min(p.tokens, first + per_block);
    const int pairs = (last - first) * p.k;
    int *counts = shared, *totals = counts + warps * p.experts, *chosen = totals + p.experts, *rank = chosen + per_block * p.k;
    for (int i = threadIdx.x; i < warps * p.experts; i += blockDim.x) counts[i] = 0;
    grid_dependency_entry();
    pick_experts<T, PER>(p, first, last, chosen);
    __syncthreads();

    const long long pair0 = (long long)first * p.k;
    const int run = (pairs + warps * 32 - 1) / (warps * 32) * 32;                      // pairs per warp
    const int begin = min(pairs, warp * run), end = min(pairs, begin + run);
    int *mine = counts + warp * p.experts;
    for (int i = begin + lane; i - lane < end; i += 32) {
        const int e = i < end ? chosen[i] : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, e);
        const int before = __popc(same & ((1u << lane) - 1u));
        int base = 0;
        if (e >= 0) base = mine[e];
        __syncwarp();
        if (e >= 0 && before == 0) mine[e] = base + __popc(same);
        __syncwarp();
        if (i < end) rank[i] = base + before;
    }
    __syncthreads();
    // counts per warp -> what lies before each warp; totals of the block behind them
    for (int e = threadIdx.x; e < p.experts; e += blockDim.x) {
        int sum = 0;
        for (int w = 0; w < warps; ++w) {
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
        for (int e = threadIdx.x; e < p.experts; e += blockDim.x) p.offsets[e] = totals[e];
        if (threadIdx.x == 0) p.offsets[p.experts] = used;
    }
    for (int i = begin + lane; i < end; i += 32) {
        const int e = chosen[i];
        const int slot = e < 0 ? -1 : rank[i] + mine[e] + (kSingle ? totals[e] : 0);
        p.slots[pair0 + i] = slot;
        if (kSingle && e >= 0) p.rows[slot] = first + i / p.k;
    }
    if (kSingle)
        for (int i = used + int(threadIdx.x); i < pairs; i += blockDim.x) p.rows[i] = -1;
}

// Very long calls: the counts of every expert become, in place, the pairs of earlier blocks, its total stands behind them.  A lane per
// expert, a warp per range of blocks.  (Blocks of the second pass that each read all counts would read blocks^2 x experts.)
__global__ void __launch_bounds__(kRouteThreads) route_scan_kernel(const RouteParams p, int blocks) {
    constexpr int kRanges = kRouteThreads / 32;
    __shared__ int sums[kRanges][32];
    const int lane = threadIdx.x & 31, range = threadIdx.x >> 5, e = int(blockIdx.x) * 32 + lane;
    grid_dependency_entry();
    const int b0 = int((long long)blocks * range / kRanges), b1 = int((long long)blocks * (range + 1) / kRanges);
    int *counts = p.block_counts + e;
    int sum = 0;
    if (e < p.experts) {
#pragma unroll 8
        for (int b = b0; b < b1; ++b) sum += counts[(long long)b * p.experts];
    }
    sums[range][lane] = sum;
    __syncthreads();
    if (e >= p.experts) return;
    int run = 0;
    for (int r = 0; r < range; ++r) run += sums[r][lane];
#pragma unroll 8
    for (int b = b0; b < b1; ++b) {
        const int c = counts[(long long)b * p.experts];
        counts[(long long)b * p.experts] = run;
        run += c;
    }
    if (range == kRanges - 1) counts[(long long)blocks * p.experts] = run;
}

// Second pass of a plan over many blocks: block b adds, per expert, the expert's start and the pairs of blocks < b.
// Every block sums the counts of all blocks; the threads share that by expert and by range of blocks.  Beyond
// kRouteDirectBlocks, route_scan_kernel has summed them.
__global__ void __launch_bounds__(kRouteThreads) route_place_kernel(const RouteParams p, int per_block, int blocks) {
    extern __shared__ int shared[];                    // [experts] starts, [experts] pairs in earlier blocks
    int *start = shared, *earlier = shared + p.experts;
    for (int e = threadIdx.x; e < 2 * p.experts; e += blockDim.x) shared[e] = 0;
    grid_dependency_entry();
    __syncthreads();
    const int ranges = max(1, int(blockDim.x) / p.experts);        // threads per expert
    const int e = int(threadIdx.x) % p.experts, range = int(threadIdx.x) / p.experts;
    if (blocks > kRouteDirectBlocks) {
        for (int i = threadIdx.x; i < p.experts; i += blockDim.x) {
            start[i] = p.block_counts[(long long)blocks * p.experts + i];
            earlier[i] = p.block_counts[(long long)blockIdx.x * p.experts + i];
        }
    } else if (range < ranges) {
        const int b0 = blocks * range / ranges, b1 = blocks * (range + 1) / ranges;
        int sum = 0, before = 0;
#pragma unroll 8
        for (int b = b0; b < b1; ++b) {
            const int c = p.block_counts[(long long)b * p.experts + e];
            sum += c;
            if (b < int(blockIdx.x)) before += c;
        }
        atomicAdd(&start[e], sum);                      // whole numbers: the order does not matter
        atomicAdd(&earlier[e], before);
    }
    __syncthreads();
    const int used = exclusive_scan(start, p.experts);
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i < p.experts; i += blockDim.x) p.offsets[i] = start[i];
        if (threadIdx.x == 0) p.offsets[p.experts] = used;
    }
    const int first = blockIdx.x * per_block, last = min(p.tokens, first + per_block);
    const long long pair0 = (long long)first * p.k;
    const int pairs = (last - first) * p.k;
    for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
        const int expert = p.chosen[pair0 + i];
        if (expert < 0) continue;
        const int slot = p.slots[pair0 + i] + start[expert] + earlier[expert];
        p.slots[pair0 + i] = slot;
        p.rows[slot] = first + i / p.k;
    }
    const long long all = (long long)p.tokens * p.k;
    for (long long i = used + (long long)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (long long)blocks * blockDim.x)
        p.rows[i] = -1;
}

// Tokens one block plans: a small call is one block and one launch; beyond that at most kRouteDirectBlocks blocks, because every
// block of the second pass reads the counts of all of them, until kRoutePairs fill a block; then as many blocks as there are such.
// (One block, k = 8: 64 tokens of 64 experts take 7.5 us, as in two launches; 128 tokens 12.0 for 7.7, yet a call outside a graph 14.4
// for 16.3, because the host's part of a launch is longer; 128 tokens of 256 experts 20.9 for 10.1, a call 21.0 for 16.3; 200 tokens
// of 64 experts would take 17.5 for 7.9.)
constexpr int kRouteSingleTokens = 128;
int route_per_block(int tokens, int k) {
    if (tokens <= kRouteSingleTokens) return tokens;
    return std::min(std::max(32, (tokens + kRouteDirectBlocks - 1) / kRouteDirectBlocks), kRoutePairs / k);
}
int route_blocks(int tokens, int k) { return (tokens + route_per_block(tokens, k) - 1) / route_per_block(tokens, k); }

// The largest dynamic shared memory that a router kernel is launched with: kMaxExperts experts, kRoutePairs pairs (a single block:
// 128 tokens of kMaxChosen, half of that).  The limit is set to this, once per kernel and device and never to a call's own size:
// it belongs to the kernel, and another host thread may launch that between this thread's setting and its launch.
constexpr size_t kRouteSmem = (size_t(kRouteThreads / 32 + 1) * kMaxExperts + 2 * size_t(kRoutePairs)) * sizeof(int);
static_assert(kRouteSingleTokens * kMaxChosen <= kRoutePairs && 32 * kMaxChosen <= kRoutePairs && kRouteSmem + 1024 <= 227 * 1024, "fits an SM");
template <class T, int PER, bool kSingle>
cudaError_t allow_route_smem() {
    static std::atomic<uint64_t> prepared{0};                // devices (of the first 64) that know
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return err;
    const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
    if (prepared.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    err = cudaFuncSetAttribute(route_pick_kernel<T, PER, kSingle>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kRouteSmem));
    if (err == cudaSuccess) prepared.fetch_or(bit, std::memory_order_relaxed);
    return err;
}

template <class T, int PER>
cudaError_t route_run(const RouteParams &p, cudaStream_t stream) {
    const int per_block = route_per_block(p.tokens, p.k), blocks = route_blocks(p.tokens, p.k);
    const int threads = p.tokens <= 8 ? 256 : kRouteThreads;
    const size_t smem = (size_t(threads / 32 + 1) * p.experts + 2 * size_t(per_block) * p.k) * sizeof(int);
    const auto pick = blocks == 1 ? route_pick_kernel<T, PER, true> : route_pick_kernel<T, PER, false>;
    cudaError_t err = blocks == 1 ? allow_route_smem<T, PER, true>() : allow_route_smem<T, PER, false>();
    if (err != cudaSuccess) return err;
    err = launch(pick, blocks, threads, smem, stream, p, per_block);
    if (err == cudaSuccess && blocks > kRouteDirectBlocks)
        err = launch(route_scan_kernel, (p.experts + 31) / 32, kRouteThreads, 0, stream, p, blocks);
    if (err == cudaSuccess && blocks > 1)
        err = launch(route_place_kernel, blocks, kRouteThreads, 2 * size_t(p.experts) * sizeof(int), stream, p, per_block, blocks);
    return err;
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

// What a row is scaled by, a power of two, before its quotients are worked out: rows of tiny values are lifted, so that
// 127 / largest stays finite, and rows of huge ones lowered, so that 254 times an element does.  (An element that the lowering
// makes subnormal is below 2^-160 of the largest: it becomes 0 either way.)
__device__ __forceinline__ float row_lift(float largest) {
    return largest < 1e-30f ? 18446744073709551616.0f : largest > 1e30f ? 1.0f / 18446744073709551616.0f : 1.0f;      // 2^64, 2^-64
}

// The whole number nearest to 127 x / largest (halves to even), from the float product x * inverse and, where that
// falls next to a half, from the exact comparison of 127 |x| with (n + 1/2) largest.  For 16-bit x both sides have at most 19
// bits, and lifted as above they stay inside float32's range: its fused difference has the right sign; for float32 they have 33
// and the difference is exact in double precision.  (Exact halves
// are common: in bfloat16 one element in a thousand is half of its row's largest, which gives 63.5.)  NaN gives 0, an
// infinity +-127.
template <class T>
__device__ __forceinline__ int quantize_one(float x, float inverse, float largest, float lift) {
    if (!(fabsf(x) <= 3.402823466e38f)) return isnan(x) ? 0 : (x > 0 ? 127 : -127);
    const float t = fabsf(x * lift) * inverse;
    const float n = floorf(t);
    int q = int(rintf(t));
    if (fabsf(t - n - 0.5f) < 1e-3f) {
        bool above, equal;
        if (sizeof(T) == 2) {
            const float d = fmaf(-(2.0f * n + 1.0f), largest * lift, 254.0f * fabsf(x * lift));
            above = d > 0.0f;
            equal = d == 0.0f;
        } else {
            const double d = 127.0 * double(fabsf(x)) - (double(n) + 0.5) * double(largest);
            above = d > 0.0;
            equal = d == 0.0;
        }
        q = int(n) + (above || (equal && (int(n) & 1)) ? 1 : 0);
    }
    q = min(q, 127);
    return x < 0 ? -q : q;
}

// Eight elements as they lie in memory, and their magnitudes as whole numbers: in each of the three types the order of the
// bits without the sign is the order of the magnitudes, infinities and NaN on top.
template <class T> struct Eight;
template <> struct Eight<float> {
    uint32_t w[8];
    static constexpr uint32_t kInfinite = 0x7F800000u;
    __device__ __forceinline__ void load(const float *p) {
        const uint4 a = *reinterpret_cast<const uint4 *>(p), b = *reinterpret_cast<const uint4 *>(p + 4);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 0;
    }
    __device__ __forceinline__ float at(int i) const { return __uint_as_float(w[i]); }
    __device__ __forceinline__ void raise(uint32_t &most) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) most = max(most, w[i] & 0x7FFFFFFFu);
    }
    static __device__ __forceinline__ uint32_t key(uint32_t most) { return most; }
    static __device__ __forceinline__ float magnitude(uint32_t key) { return __uint_as_float(key); }
};
struct EightHalves {
    uint32_t w[4];
    __device__ __forceinline__ void load(const void *p) {
        const uint4 a = *static_cast<const uint4 *>(p);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
    }
    __device__ __forceinline__ void clear() { w[0] = w[1] = w[2] = w[3] = 0; }
    __device__ __forceinline__ void raise(uint32_t &most) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) most = __vmaxu2(most, w[i] & 0x7FFF7FFFu);
    }
    static __device__ __forceinline__ uint32_t key(uint32_t most) { return max(most & 0xFFFFu, most >> 16); }
};
template <> struct Eight<__half> : EightHalves {
    static constexpr uint32_t kInfinite = 0x7C00u;
    __device__ __forceinline__ float at(int i) const { return __half2float(__ushort_as_half(uint16_t(w[i >> 1] >> (16 * (i & 1))))); }
    static __device__ __forceinline__ float magnitude(uint32_t key) { return __half2float(__ushort_as_half(uint16_t(key))); }
};
template <> struct Eight<__nv_bfloat16> : EightHalves {
    static constexpr uint32_t kInfinite = 0x7F80u;
    __device__ __forceinline__ float at(int i) const { return __uint_as_float((i & 1) ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16); }
    static __device__ __forceinline__ float magnitude(uint32_t key) { return __uint_as_float(key << 16); }
};

// Rows whose vectors of eight elements stay in the registers of a group of G threads, V per thread: read once.  Adding
// 1.5 * 2^23 leaves the quotient's nearest whole number in the low bits of the sum; elements next to a half, and all of a row
// that holds an infinity or NaN, take the exact form instead.  (8192 rows of 4096 bfloat16, 100 MB: 28 us, 3.6 TB/s; float32, 168 MB:
// 5.1 TB/s -- bound by 14 instructions per element.  Blocks that stay and fetch the next row ahead took 38 us: fewer of them fit.)
template <class T, int G, int V>
__global__ void __launch_bounds__(G < 256 ? 256 : G) quantize_rows_kernel(const QuantizeParams p) {
    constexpr int kBlock = G < 256 ? 256 : G;
    constexpr float kMagic = 12582912.0f;
    __shared__ uint32_t warp_key[kBlock / 32];
    const int member = threadIdx.x % G, warp0 = threadIdx.x / G * (G / 32);
    const long long r = (long long)blockIdx.x * (kBlock / G) + threadIdx.x / G;
    grid_dependency_entry();
    const long long src = r >= p.total ? -1 : p.rows ? p.rows[r] : r;
    const bool live = src >= 0 && src < p.x_rows;
    const T *x = static_cast<const T *>(p.x) + (live ? src : 0) * p.x_stride;
    Eight<T> v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = (i * G + member) * 8;
        if (live && c < p.inner) v[i].load(x + c);
        else v[i].clear();
    }
    const auto most_of_row = [&](uint32_t key) {
        key = __reduce_max_sync(0xffffffffu, key);
        if (G > 32) {
            if ((threadIdx.x & 31) == 0) warp_key[threadIdx.x >> 5] = key;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < G / 32; ++w) key = max(key, warp_key[warp0 + w]);
        }
        return key;
    };
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i].raise(most);
    uint32_t key = most_of_row(Eight<T>::key(most));
    const bool odd = key >= Eight<T>::kInfinite;
    if (G > 32 ? __syncthreads_or(odd) : odd) {              // the largest finite magnitude of such a row
        float largest = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float a = fabsf(v[i].at(j));
                if (a <= 3.402823466e38f) largest = fmaxf(largest, a);
            }
        const uint32_t finite = most_of_row(__float_as_uint(largest));
        if (odd) key = finite;
    }
    if (r >= p.total) return;
    const float largest = odd ? __uint_as_float(key) : Eight<T>::magnitude(key);
    if (member == 0) p.scale[r] = largest / 127.0f;
    const float lift = row_lift(largest);
    const float inverse = largest > 0.0f ? 127.0f / (largest * lift) : 0.0f;
    signed char *q = p.q + r * p.q_stride;
    // (the quotient is off by less than 127 * 2^-23; rows that need the exact form throughout get it: NaN compares as near, too)
    const float near = odd || lift != 1.0f ? -1.0f : 0.49998f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = (i * G + member) * 8;
        if (c >= p.inner) continue;
        uint32_t n[8];
        float off[8], most_off = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float sum = fmaf(v[i].at(j), inverse, kMagic);
            n[j] = __float_as_uint(sum);
            off[j] = fabsf(fmaf(v[i].at(j), inverse, kMagic - sum));
            most_off = fmaxf(most_off, off[j]);
        }
        if (!(most_off <= near)) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!(off[j] <= near)) n[j] = uint32_t(quantize_one<T>(v[i].at(j), inverse, largest, lift));
        }
        uint2 packed;
        packed.x = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
        packed.y = __byte_perm(__byte_perm(n[4], n[5], 0x0040), __byte_perm(n[6], n[7], 0x0040), 0x5410);
        *reinterpret_cast<uint2 *>(q + c) = packed;
    }
}

// Rows of any length, alignment and stride: a row per block, read twice, element by element.  (8192 rows of 4095 bfloat16: 53 us, of
// 20000: 234; float32 55 and 332.  Bound by instructions, as above, and by loads of one element.)
template <class T>
__global__ void __launch_bounds__(256) quantize_any_kernel(const QuantizeParams p) {
    __shared__ float warp_max[8];
    const long long r = blockIdx.x;
    grid_dependency_entry();
    const long long src = p.rows ? p.rows[r] : r;
    const bool live = src >= 0 && src < p.x_rows;
    const T *x = static_cast<const T *>(p.x) + (live ? src : 0) * p.x_stride;
    float largest = 0.0f;
    if (live)
        for (int c = threadIdx.x; c < p.inner; c += 256) {
            const float v = fabsf(to_float(x[c]));
            if (v <= 3.402823466e38f) largest = fmaxf(largest, v);
        }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, s));
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = largest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) largest = fmaxf(largest, warp_max[w]);
    if (threadIdx.x == 0) p.scale[r] = largest / 127.0f;
    const float lift = row_lift(largest);
    const float inverse = largest > 0.0f ? 127.0f / (largest * lift) : 0.0f;
    signed char *q = p.q + r * p.q_stride;
    for (int c = threadIdx.x; c < p.inner; c += 256)
        q[c] = live ? (signed char)quantize_one<T>(to_float(x[c]), inverse, largest, lift) : 0;
}

template <class T>
cudaError_t quantize_typed(const QuantizeParams &p, cudaStream_t stream) {
    const bool vectors = reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.x_stride * int(sizeof(T)) % 16 == 0 && p.inner % 8 == 0 &&
                         reinterpret_cast<uintptr_t>(p.q) % 8 == 0 && p.q_stride % 8 == 0;
    const int pieces = p.inner / 8;
    const auto go = [&](auto kernel, int block, long long rows) {
        return launch(kernel, (p.total + rows - 1) / rows, block, 0, stream, p);
    };
    // a warp per row up to 1024 elements, four warps up to 4096, sixteen up to 16384
    if (!vectors || pieces > 512 * 4) return go(quantize_any_kernel<T>, 256, 1);
    if (pieces <= 32) return go(quantize_rows_kernel<T, 32, 1>, 256, 8);
    if (pieces <= 64) return go(quantize_rows_kernel<T, 32, 2>, 256, 8);
    if (pieces <= 128) return go(quantize_rows_kernel<T, 32, 4>, 256, 8);
    if (pieces <= 256) return go(quantize_rows_kernel<T, 128, 2>, 256, 2);
    if (pieces <= 512) return go(quantize_rows_kernel<T, 128, 4>, 256, 2);
    if (pieces <= 1024) return go(quantize_rows_kernel<T, 512, 2>, 512, 1);
    return go(quantize_rows_kernel<T, 512, 4>, 512, 1);
}

// ---- weighted sum of expert rows ----------------------------------------------------------------

// V consecutive channels of a token per thread, 16 bytes of the rows at a time (or one element: V = 1); eight rows are
// asked for before the first is added.  (8192 tokens x 8 rows of 2048 halves: 303 MB in 50 us, 6.0 TB/s, bound by memory.)
template <class T, class O, int V>
__global__ void __launch_bounds__(256) combine_kernel(const CombineParams p, int across) {
    const int lane = threadIdx.x % across;
    const long long t = (long long)blockIdx.x * (256 / across) + threadIdx.x / across;
    const int c = (int(blockIdx.y) * across + lane) * V;
    grid_dependency_entry();
    if (t >= p.tokens || c >= p.channels) return;
    const float *gates = p.gates + t * p.k;
    const int *slots = p.slots + t * p.k;
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.0f;
    // (every load is made, from row 0 where a slot names none: under a branch they would wait for one another)
    for (int j0 = 0; j0 < p.k && p.y_rows > 0; j0 += 8) {
        Vector<T, V> part[8];
        float gate[8];
        bool live[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int s = j0 + j < p.k ? slots[j0 + j] : -1;
            live[j] = s >= 0 && s < p.y_rows;
            gate[j] = live[j] ? gates[j0 + j] : 0.0f;
            part[j] = *reinterpret_cast<const Vector<T, V> *>(static_cast<const T *>(p.y) + (live[j] ? (long long)s * p.y_stride : 0) + c);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (live[j]) {
#pragma unroll
                for (int i = 0; i < V; ++i) sum[i] += gate[j] * to_float(part[j].v[i]);
            }
    }
    store_vector(static_cast<O *>(p.out) + t * p.out_stride + c, sum);
}

template <class T, class O>
cudaError_t combine_run(const CombineParams &p, cudaStream_t stream) {
    constexpr int kWide = 16 / int(sizeof(T));
    const bool vectors = reinterpret_cast<uintptr_t>(p.y) % 16 == 0 && p.y_stride % kWide == 0 && p.channels % kWide == 0 &&
                         reinterpret_cast<uintptr_t>(p.out) % 16 == 0 && p.out_stride * int(sizeof(O)) % 16 == 0;
    const int pieces = vectors ? p.channels / kWide : p.channels;
    int across = 8;                                    // threads of a block along the channels
    while (across < 256 && across < pieces) across *= 2;
    const dim3 grid(unsigned((p.tokens + 256 / across - 1) / (256 / across)), unsigned((pieces + across - 1) / across));
    return vectors ? launch(combine_kernel<T, O, kWide>, grid, 256, 0, stream, p, across)
                   : launch(combine_kernel<T, O, 1>, grid, 256, 0, stream, p, across);
}

template <class T>
cudaError_t combine_typed(const CombineParams &p, cudaStream_t stream) {
    if (p.out_type == Elem::F32) return combine_run<T, float>(p, stream);
    if (p.out_type == Elem::F16) return combine_run<T, __half>(p, stream);
    return combine_run<T, __nv_bfloat16>(p, stream);
}

}  // namespace

size_t route_workspace_bytes(int tokens, int experts, int k) {
    const int blocks = route_blocks(tokens, k);
    return blocks == 1 ? 0 : size_t(blocks + (blocks > kRouteDirectBlocks ? 1 : 0)) * experts * sizeof(int);
}

cudaError_t launch_route(const RouteParams &p, cudaStream_t stream) {
    if (p.type == Elem::F32) return route_typed<float>(p, stream);
    if (p.type == Elem::F16) return route_typed<__half>(p, stream);
    return route_typed<__nv_bfloat16>(p, stream);
}

cudaError_t launch_quantize(const QuantizeParams &p, cudaStream_t stream) {
    if (p.type == Elem::F32) return quantize_typed<float>(p, stream);
    if (p.type == Elem::F16) return quantize_typed<__half>(p, stream);
    return quantize_typed<__nv_bfloat16>(p, stream);
}

cudaError_t launch_combine(const CombineParams &p, cudaStream_t stream) {
    if (p.type == Elem::F32) return combine_typed<float>(p, stream);
    if (p.type == Elem::F16) return combine_typed<__half>(p, stream);
    return combine_typed<__nv_bfloat16>(p, stream);
}

}  // namespace ios
