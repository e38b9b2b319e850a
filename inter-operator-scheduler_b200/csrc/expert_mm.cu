// Matrix products over ragged groups of rows on the 5th-generation tensor cores (sm_100a):
//
//     y[r, n] = act(row_scale[src] channel_scale[g, n] sum_k x[src, k] w[g, n, k] + bias[g, n]),   r in group g
//
// * The weights' channels are the 128 rows of a tcgen05.mma (TMEM lanes), a group's rows are its columns: N may be any
//   multiple of 16 up to 256, so a group of one row costs a 16-column instruction instead of a 128-row one, and a
//   group's end needs no masked store -- the epilogue writes whole columns, one row of y each.  K advances one 128-byte
//   swizzle row per step (64 elements of 16 bits, 128 of 8 bits, 32 of float32).
// * The group sizes are only known on the device.  Every CTA works out the same list of tiles from the offsets (one
//   scan) and resident CTAs walk it; a group's rows are dealt evenly to its tiles.
// * Few rows: bound by the weights, which are read once (4 tokens x 8 of 64 experts, gated, 2048 -> 1280, bfloat16: 273 MB
//   in 46 us, 5.9 TB/s of the 6.5 that a copy reaches; what is left is four rounds of tiles where 3.5 would do).
// * Many rows: bound by the tensor cores and the power they draw.  Pairs of CTAs (cta_group::2) share the rows of a tile of
//   256 channels x 256 rows, which halves the loads of x and doubles the K steps in flight: 32768 rows in four groups, 2048 ->
//   1280, bfloat16: 1500 TFLOP/s after 1200 with one CTA per tile; 8192 x 4096 x 8192 in 8 bits: 3300 TOP/s.
// * Products too small to fill the GPU split K over a thread-block cluster: the CTAs deal the tile's columns among
//   themselves, push their partial sums into the shared memory of the CTA that finishes a column, and that CTA adds them
//   in rank order.  No workspace, no counters, the same bits every time.
// * Operands arrive by TMA where their rows start on 16-byte boundaries.  Rows gathered by index then come four at a time
//   (tile::gather4).  Such a load keeps a warp for some 130 cycles, so eight warps share them (4096 tokens x 8 of 64 experts, gated:
//   405 us with four warps, 305 with eight, 348 with sixteen, which leave the epilogue too few registers; now 287, and 264 from
//   rows that lie sorted).  Gathering by cp.async took 737 us: its fence between the copies and the tensor core waits for every copy under way.
// * Anything else goes through registers of sixteen loader warps, word by word, shifted into place: 4096 x 8 rows of 2047
//   bfloat16 at 135 TFLOP/s.
// * float32: three products a_hi b_hi + a_hi b_lo + a_lo b_hi of TF32 numbers; the operands are split in shared memory, after
//   they have landed (or by the loader warps): 16384 rows, 2048 -> 1024, at 130 TFLOP/s, bound by three stages being loaded,
//   split and multiplied in turn.  The tensor core truncates where it adds, which costs 1e-6 of a sum over 128 elements; so the
//   sums of every K step, 32 elements, are added up in tensor memory, rounded to nearest, and no slower.  Off by, relative to a
//   result of normal numbers: 0.9e-7 at 8 elements, 2.4e-7 from 32 on, 3.2e-7 at 32768 (a float32 product on the CUDA cores, 256 rows:
//   0.5e-7 at 8, 1e-7 at 32, 2e-7 at 128, 8e-7 at 2048).
// * 16-bit operands: the sums of a tile's K range stay in one accumulator of 32 bits, whose additions truncate.  That costs 2e-6 of the
//   result at 1408 elements, 4e-6 at 2048 where a few channels are ten times the others, and grows with the length (a library product: 2e-6
//   at 2048, 9e-6 at 8192).  Far below half a step of a 16-bit result, of which it moves 2 in a thousand to the neighbour;
//   visible in float32 results.  Adding up step by step as above would need a third accumulator, which 256-column tiles leave no room for.
// * gated: 16 rows of the gate half and the 16 rows of the same channels of the other half alternate in the tile (one box of
//   a five-dimensional view), so that a lane and the lane 16 further on hold the two factors of one result.
// * Loads and tensor-core instructions are issued from warp-uniform code by a predicated lane.  Issued from a branch that one
//   lane takes, each cost some 100 cycles, and 8192 x 4096 x 8192 in 8 bits took 300 us instead of 165.
//
// Warp roles: 0 = weight loads, 1 = MMA issuer, 2 = tensor memory, 3 = row loads, 4..11 (4..7) = epilogue, then
// gathering, loader or splitting warps.  Every wait on an mbarrier is bounded, and every warp reaches the barriers that it shares with
// others (the epilogue's once per tile, the last one) whether or not it gave up.  A time-out is counted in a word of the device,
// loads in flight are waited for, tensor memory is freed and the kernel returns.
#include "expert_ops.h"
#include "kernels.h"
#include "tc_device.h"

#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <climits>

namespace ios {
namespace {

enum Kind { kF16 = 0, kI8 = 1, kX3 = 2 };       // instruction: 16-bit floats, 8-bit integers, three TF32 products
enum Loads { kTma = 0, kGather = 1, kRegs = 2 };  // operands by TMA / rows gathered by TMA, four at a time / all through registers

constexpr int kGatherWarps = 8, kLoaderWarps = 16;
constexpr int kLoaderRows = 128 / kLoaderWarps; // rows of each operand that a loader warp moves
constexpr int kBoxRows = 64;                    // rows of x per TMA load, in wide tiles
constexpr int kNarrowCols = 32;                 // tiles up to here gather a step's rows with one warp
constexpr int kMaxThreads = 768;
constexpr int kSplitWarps = 8;                  // float32 by TMA: warps that split the operands where they have landed
// Two epilogue warps per lane quarter share a tile's columns; one beside gathering, loading or splitting warps, which need
// the registers.
__host__ __device__ constexpr int epilogue_warps(int kind, int loads) { return loads == kTma && kind != kX3 ? 8 : 4; }
__host__ __device__ constexpr int threads_of(int kind, int loads) {
    return 32 * (4 + epilogue_warps(kind, loads) + (loads == kTma ? 0 : loads == kGather ? kGatherWarps : kLoaderWarps) +
                 (kind == kX3 && loads != kRegs ? kSplitWarps : 0));
}
constexpr int kLoaderCols = 128;                // widest tile of the loader warps (their registers hold a step)
constexpr int kTurnCols = 16;                   // columns an epilogue warp turns round at a time: few, because a small
                                                // product runs this code once, and cold code costs more than it does
constexpr int kTurnBytes = kTurnCols * 32 * 4;  // ... in this much shared memory
constexpr int kListed = 96;                     // tiles of a CTA that are found when it starts
constexpr int kChunkSteps = 1;                  // float32: K steps per partial sum
constexpr int kMaxStages = 12;
constexpr int kMaxGroupTiles = INT_MAX / kMaxExperts - 1;    // tiles of a group: their sum over all groups fits an int
constexpr int kBarBytes = 3 * kMaxStages * 8 + 48;    // mbarriers: three per stage, six more
constexpr size_t kSmemLimit = 227 * 1024, kStaticBytes = 4608;    // ... of which the kernel's static arrays may take

// Waits that ran out since the library was loaded, by the code of the waiting role (see time_out); read by expert_mm_status and never
// cleared: what one reader has seen is news to the next.
constexpr int kWaitCodes = 8;
__device__ unsigned g_expert_timeouts[kWaitCodes];

struct MmGeom {
    int tn;             // columns a tile may have
    int n_tiles;        // channel tiles of a group
    int tile_channels;  // output channels per channel tile: 128 per CTA, gated 64
    int grain;          // columns of a tile come in multiples of this: 16, pairs 32
    int k_steps;
    int cluster;        // CTAs that share a tile's K range
    int stages;
    int box_rows;       // rows per TMA box of x
    int one_box;        // 1: (gated) the tile's alternating rows are one box of a five-dimensional view
    int tmem_cols;
    uint32_t format;    // operand format field of the instruction descriptor
    int esize;
    uint32_t wait_ns;   // what a wait may take
    int recv_off, turn_off, table_off, bar_off;   // byte offsets in shared memory
};

// The same value in every lane, and known to the compiler as such: what depends on it may live in uniform registers, where
// the tensor core's and the TMA unit's operands have to be.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

struct Tile {
    int group, row0, valid, cols, channel0;
};

// Columns per tile of a group: its rows dealt evenly to the fewest tiles.
__device__ __forceinline__ int even_cols(int count, const MmGeom &t) {
    const int tiles = (count + t.tn - 1) / t.tn;
    return ((count + tiles - 1) / tiles + t.grain - 1) & -t.grain;
}

// The list of tiles: bound[g] = first row of group g, first[g] = tiles before group g.  Offsets come from the device:
// whatever they hold, a group stays inside [0, total].  All threads call it; a barrier has to follow.
struct Table {
    int4 *listed;             // the CTA's first kListed tiles: (row0, channel0, group, valid)
    int *bound, *first;       // groups + 1 each; all in shared memory
};
__device__ __forceinline__ int tiles_of(int count, const MmGeom &t) {
    if (count <= 0) return 0;
    const int cols = even_cols(count, t);
    return int(min((long long)((count + cols - 1) / cols) * t.n_tiles, (long long)kMaxGroupTiles));
}
__device__ void build_table(const GroupedParams &p, const MmGeom &t, const Table &table, int threads) {
    if (p.groups == 1) {
        if (threadIdx.x == 0) {
            const int begin = p.offsets ? min(max(p.offsets[0], 0), p.total) : 0;
            const int end = p.offsets ? min(max(p.offsets[1], begin), p.total) : p.total;
            table.bound[0] = begin;
            table.bound[1] = end;
            table.first[0] = 0;
            table.first[1] = tiles_of(end - begin, t);
        }
        return;
    }
    __shared__ int warp_total[kMaxThreads / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int g = threadIdx.x; g <= p.groups; g += threads) table.bound[g] = min(max(p.offsets[g], 0), p.total);
    __syncthreads();
    const int per = (p.groups + threads - 1) / threads, g0 = min(int(threadIdx.x) * per, p.groups), g1 = min(g0 + per, p.groups);
    int sum = 0;
    for (int g = g0; g < g1; ++g) {
        const int n = tiles_of(table.bound[g + 1] - table.bound[g], t);
        table.first[g] = n;
        sum += n;
    }
    int run = sum;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, run, s);
        if (lane >= s) run += v;
    }
    if (lane == 31) warp_total[warp] = run;
    __syncthreads();
    int start = run - sum;
    for (int w = 0; w < warp; ++w) start += warp_total[w];
    for (int g = g0; g < g1; ++g) {
        const int n = table.first[g];
        table.first[g] = start;
        start += n;
    }
    if (g0 < p.groups && g1 == p.groups) table.first[p.groups] = start;
}

// Tiles of a group: up to 8 column tiles side by side, then the next channels, so that neighbours in the list share
// weights and rows in L2.
__device__ int4 find_tile(const MmGeom &t, const Table &table, int groups, int index, int cta_channel) {
    int lo = 0, hi = groups;                      // table.first[lo] <= index < table.first[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (table.first[mid] <= index) lo = mid;
        else hi = mid;
    }
    const int begin = table.bound[lo], count = table.bound[lo + 1] - begin;
    const int cols = even_cols(count, t);
    const int col_tiles = (count + cols - 1) / cols;
    const int at = index - table.first[lo];
    const int band = at / (8 * t.n_tiles);
    const int wide = min(8, col_tiles - band * 8);
    const int inside = at - band * 8 * t.n_tiles;
    const int col0 = (band * 8 + inside % wide) * cols;
    return make_int4(begin + col0, inside / wide * t.tile_channels + cta_channel, lo, min(cols, count - col0));
}
// The CTA's n-th tile, number `index` of all.  Every role asks for it, whole warps at a time; finding a tile takes 1400
// cycles, so the first are found by a thread each when the kernel starts.
__device__ __forceinline__ Tile tile_of(const GroupedParams &p, const MmGeom &t, const Table &table, int n, int index, int cta_channel) {
    const int4 found = n < kListed ? table.listed[n] : find_tile(t, table, p.groups, index, cta_channel);
    Tile tile;
    tile.row0 = uniform(found.x);
    tile.channel0 = uniform(found.y);
    tile.group = uniform(found.z);
    tile.valid = uniform(found.w);
    tile.cols = (tile.valid + t.grain - 1) & -t.grain;
    return tile;
}

// Row of the weights (inside its group) that tile row r holds
template <bool GATED>
__device__ __forceinline__ int weight_row(const GroupedParams &p, const Tile &tile, int r) {
    if (!GATED) return tile.channel0 + r;
    return ((r >> 4) & 1) * p.channels + tile.channel0 + (r >> 5) * 16 + (r & 15);
}

// Loads into shared memory, counted on `bar` -- with PAIR that may be the other CTA's.  Like umma below they are called by
// a whole warp with equal arguments and issued by one lane: from a branch that only one lane takes, every operand has to
// be moved to a uniform register on the spot, which costs some 100 cycles per load.
#define IOS_TMA(RANK, MODE, COORDS, ...)                                                                       \
    do {                                                                                                       \
        if (PAIR)                                                                                              \
            asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t"                                       \
                         "@q cp.async.bulk.tensor." RANK ".cta_group::2.shared::cluster.global" MODE             \
                         ".mbarrier::complete_tx::bytes [%1], [%2, {" COORDS "}], [%3];\n\t}"                    \
                         ::"r"(elected), "r"(dst), "l"(tmap), "r"(bar), __VA_ARGS__ : "memory");                \
        else                                                                                                   \
            asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t"                                       \
                         "@q cp.async.bulk.tensor." RANK ".shared::cluster.global" MODE                          \
                         ".mbarrier::complete_tx::bytes [%1], [%2, {" COORDS "}], [%3];\n\t}"                    \
                         ::"r"(elected), "r"(dst), "l"(tmap), "r"(bar), __VA_ARGS__ : "memory");                \
    } while (0)
template <bool PAIR>
__device__ __forceinline__ void load_2d(uint32_t elected, uint32_t dst, const void *tmap, uint32_t bar, int c0, int c1) {
    IOS_TMA("2d", "", "%4, %5", "r"(c0), "r"(c1));
}
template <bool PAIR>
__device__ __forceinline__ void load_3d(uint32_t elected, uint32_t dst, const void *tmap, uint32_t bar, int c0, int c1, int c2) {
    IOS_TMA("3d", "", "%4, %5, %6", "r"(c0), "r"(c1), "r"(c2));
}
template <bool PAIR>
__device__ __forceinline__ void load_5d(uint32_t elected, uint32_t dst, const void *tmap, uint32_t bar, int c0, int c3, int c4) {
    IOS_TMA("5d", "", "%4, %7, %7, %5, %6", "r"(c0), "r"(c3), "r"(c4), "r"(0));
}
// four rows of a matrix, any four, behind one another
template <bool PAIR>
__device__ __forceinline__ void load_rows4(uint32_t elected, uint32_t dst, const void *tmap, uint32_t bar, int c0, int4 rows) {
    IOS_TMA("2d", ".tile::gather4", "%4, %5, %6, %7, %8", "r"(c0), "r"(rows.x), "r"(rows.y), "r"(rows.z), "r"(rows.w));
}
#undef IOS_TMA
// one arrival and `bytes` to come
__device__ __forceinline__ void expect(uint32_t elected, uint32_t bar, uint32_t bytes) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t"
                 "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%1], %2;\n\t}" ::"r"(elected), "r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t elect() {
    uint32_t elected;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.b32 %0, 1, 0, q;\n\t}" : "=r"(elected));
    return elected;
}
// Low word of a K-major operand's descriptor (128-byte swizzle); the high word is the same for all.
__device__ __forceinline__ uint32_t desc_low(uint32_t addr) { return ((addr & 0x3FFFF) >> 4) | (1u << 16); }
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
// D += A B for one K block of 32 bytes, by one CTA or by a pair (whose halves of A, B and D lie at the same addresses).
// The whole warp calls it with equal arguments, which then live in uniform registers, and one lane issues.
#define IOS_UMMA(GROUP, KIND_NAME)                                                                             \
    asm volatile(                                                                                              \
        "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"                                                         \
        "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"                                                     \
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"                                                   \
        "@q tcgen05.mma.cta_group::" GROUP ".kind::" KIND_NAME " [%0], a, b, %3, p;\n\t}"                       \
        ::"r"(tmem_d), "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(kDescHigh), "r"(elected)       \
        : "memory")
template <int KIND, bool PAIR>
__device__ __forceinline__ void umma(uint32_t elected, uint32_t tmem_d, uint32_t a_low, uint32_t b_low, uint32_t idesc, uint32_t accumulate) {
    if (KIND == kF16) {
        if (PAIR) IOS_UMMA("2", "f16");
        else IOS_UMMA("1", "f16");
    } else if (KIND == kI8) {
        if (PAIR) IOS_UMMA("2", "i8");
        else IOS_UMMA("1", "i8");
    } else {
        IOS_UMMA("1", "tf32");
    }
}
#undef IOS_UMMA
// arrives at `bar` (of both CTAs of a pair) once the instructions issued so far have finished
template <bool PAIR>
__device__ __forceinline__ void commit(uint32_t elected, uint32_t bar) {
    if (PAIR)
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t"
                     "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%1], %2;\n\t}"
                     ::"r"(elected), "r"(bar), "h"(uint16_t(3))
                     : "memory");
    else
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t"
                     "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}"
                     ::"r"(elected), "r"(bar)
                     : "memory");
}
// Bounded wait, for a barrier that (CLUSTER) other CTAs of the cluster may arrive at.  The clock runs on while the GPU does other
// work, so what counts is the barrier's state some time after it has run out.
template <bool CLUSTER>
__device__ __forceinline__ bool passed(uint32_t bar, uint32_t parity) {
    if (!CLUSTER) return mbar_try_wait(bar, parity);
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
template <bool CLUSTER>
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, uint32_t wait_ns) {
    uint32_t start = 0, late = 0;
    for (uint32_t spin = 1;; ++spin) {
        if (passed<CLUSTER>(bar, parity)) return true;
        if ((spin & 63u) != 0) continue;
        if (late) return false;
        uint32_t now;
        asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(now));
        if (spin == 64u) start = now;
        else late = now - start > wait_ns;
    }
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void store_cluster(uint32_t dst, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(v) : "memory");
}
// Records a wait that ran out.  The loads that this CTA has under way land within microseconds; those counted in another
// CTA's barriers cannot be waited for from here, so a millisecond is let pass.
__device__ __noinline__ void time_out(int code) {
    atomicAdd(&g_expert_timeouts[code], 1u);
    const uint64_t t0 = global_ns();
    while (global_ns() - t0 < 1000000) __nanosleep(1000);
}

// ---- loader warps: aligned words of rows that start anywhere --------------------------------------
// The word at byte `off` of a row, where it may lie partly or wholly outside: elements outside are zeros and are not read.
__device__ __noinline__ uint32_t load_edge(const uint8_t *row, long long off, long long row_bytes, int esize) {
    uint32_t out = 0;
    if (off >= 0 && off + 4 <= row_bytes) return __ldg(reinterpret_cast<const uint32_t *>(row + off));
    if (esize == 4) return 0u;
    for (int b = 0; b < 4; b += esize) {
        if (off + b < 0 || off + b >= row_bytes) continue;
        const uint32_t v = esize == 1 ? uint32_t(row[off + b]) : uint32_t(*reinterpret_cast<const uint16_t *>(row + off + b));
        out |= v << (8 * b);
    }
    return out;
}

// x = hi + lo + (at most 2^-22 |x|, or 2^-137 where lo is subnormal) for the tensor core, which drops the low 13 bits of an operand: hi is rounded to the
// bits it keeps, lo is what is missing plus half a step of its own.  (Whole-number arithmetic: cvt.rna.tf32 runs at an eighth of
// its rate.)  Values that would round to infinity are cut instead; an infinity's lo is NaN.
__device__ __forceinline__ void split_tf32(uint32_t x, uint32_t *hi, uint32_t *lo) {
    const uint32_t h = ((x & 0x7FFFFFFFu) >= 0x7F7FF000u ? x : x + 0x1000u) & 0xFFFFE000u;
    *hi = h;
    *lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(h)) + 0x1000u;
}

// sigmoid(v) = (v < 0 ? e : 1) / (1 + e) with e = exp(-|v|): exp(-v) passes float32 from v = -88 on, where the result is still one.
__device__ __noinline__ float act_far(float v, int act) {
    if (act == 3) return tanhf(v);
    const float e = expf(-fabsf(v));
    return (act == 4 ? (v < 0.0f ? v * e : v) : (v < 0.0f ? e : 1.0f)) / (1.0f + e);
}
// the activation of N values; one branch for all of them.  Results that are rounded to 16 bits take the fast exponential, which is off
// by 2 + 1.2 |v| steps of 2^-23: 1.5e-5 of the result at the most, a thirtieth of half a float16 step, where silu is all but zero, and
// 1e-6 around v = 5.  (32768 rows, 256 -> 2048, bfloat16: 91 us; with the exact exponential 104 in place, 264 called.)
template <int N>
__device__ __forceinline__ void activate(float *v, int act, bool fast) {
    if (act == 0) return;
    if (act == 1) {
#pragma unroll
        for (int c = 0; c < N; ++c) v[c] = fmaxf(v[c], 0.0f);
    } else if (act == 4 && fast) {
#pragma unroll
        for (int c = 0; c < N; ++c) {
            const float e = __expf(-fabsf(v[c]));
            v[c] = __fdividef(v[c] < 0.0f ? v[c] * e : v[c], 1.0f + e);
        }
    } else {
#pragma unroll
        for (int c = 0; c < N; ++c) v[c] = act_far(v[c], act);
    }
}

// What an epilogue warp needs to write the results of its lanes' channels.
struct Out {
    uint8_t *turn;              // shared memory of this warp, kTurnBytes
    uint8_t *first;             // &y[tile.row0][first channel of this warp]
    long long row_bytes;
    int rows, channels;         // valid rows of the tile, valid channels of this warp
    int vectors;                // rows may be written 16 bytes at a time
};
// Rows c0 .. c0 + 15 of the results, from [column][WIDTH channels] in shared memory: whole segments of rows, 32 to 128 bytes.
template <class T, int WIDTH>
__device__ __forceinline__ void write_rows(const Out &o, int c0, int lane) {
    constexpr int kPieces = WIDTH * int(sizeof(T)) / 16;              // 16-byte pieces of a row
    const int count = min(kTurnCols, o.rows - c0);
    if (o.vectors) {
        const int row = lane / kPieces;
        uint8_t *to = o.first + (c0 + row) * o.row_bytes + (lane % kPieces) * 16;
#pragma unroll
        for (int q = 0; q < kTurnCols * kPieces / 32; ++q) {
            if (row + q * (32 / kPieces) < count) *reinterpret_cast<uint4 *>(to) = reinterpret_cast<const uint4 *>(o.turn)[q * 32 + lane];
            to += (32 / kPieces) * o.row_bytes;
        }
    } else {
        for (int i = lane; i < count * WIDTH; i += 32)
            if (i % WIDTH < o.channels)
                reinterpret_cast<T *>(o.first + (c0 + i / WIDTH) * o.row_bytes)[i % WIDTH] = reinterpret_cast<const T *>(o.turn)[i];
    }
}
// v[c] (gated: v[c / 2], the lanes' halves holding alternate columns) are the results of columns c0 .. c0 + 15 of this
// lane's channel.  The warp turns them round in shared memory.
template <bool GATED>
__device__ __forceinline__ void write_columns(const Out &o, Elem type, const float *v, int c0, int lane) {
    constexpr int kWidth = GATED ? 16 : 32;                           // channels of the warp
    const int at = GATED ? (lane >> 4) * 16 + (lane & 15) : lane;
    if (!GATED && type != Elem::F32 && o.vectors) {
        // two columns to a word, [column pair][channel]; lane l takes eight channels of pair l / 4 apart again
        uint32_t *turn = reinterpret_cast<uint32_t *>(o.turn);
        if (type == Elem::BF16) {
#pragma unroll
            for (int c = 0; c < kTurnCols; c += 2) {
                const __nv_bfloat162 two = __floats2bfloat162_rn(v[c], v[c + 1]);
                turn[c * 16 + lane] = *reinterpret_cast<const uint32_t *>(&two);
            }
        } else {
#pragma unroll
            for (int c = 0; c < kTurnCols; c += 2) {
                const __half2 two = __floats2half2_rn(v[c], v[c + 1]);
                turn[c * 16 + lane] = *reinterpret_cast<const uint32_t *>(&two);
            }
        }
        __syncwarp();
        const uint4 a = reinterpret_cast<const uint4 *>(turn)[lane * 2], b = reinterpret_cast<const uint4 *>(turn)[lane * 2 + 1];
        const int row = c0 + (lane >> 2) * 2;
        uint8_t *to = o.first + row * o.row_bytes + (lane & 3) * 16;
        if (row < o.rows)
            *reinterpret_cast<uint4 *>(to) = make_uint4(__byte_perm(a.x, a.y, 0x5410), __byte_perm(a.z, a.w, 0x5410),
                                                        __byte_perm(b.x, b.y, 0x5410), __byte_perm(b.z, b.w, 0x5410));
        if (row + 1 < o.rows)
            *reinterpret_cast<uint4 *>(to + o.row_bytes) = make_uint4(__byte_perm(a.x, a.y, 0x7632), __byte_perm(a.z, a.w, 0x7632),
                                                                      __byte_perm(b.x, b.y, 0x7632), __byte_perm(b.z, b.w, 0x7632));
        __syncwarp();
        return;
    }
    if (type == Elem::F32) {
#pragma unroll
        for (int c = 0; c < (GATED ? kTurnCols / 2 : kTurnCols); ++c) reinterpret_cast<float *>(o.turn)[c * 32 + at] = v[c];
    } else if (type == Elem::BF16) {
#pragma unroll
        for (int c = 0; c < (GATED ? kTurnCols / 2 : kTurnCols); ++c) reinterpret_cast<__nv_bfloat16 *>(o.turn)[c * 32 + at] = __float2bfloat16_rn(v[c]);
    } else {
#pragma unroll
        for (int c = 0; c < (GATED ? kTurnCols / 2 : kTurnCols); ++c) reinterpret_cast<__half *>(o.turn)[c * 32 + at] = __float2half_rn(v[c]);
    }
    __syncwarp();
    if (type == Elem::F32) write_rows<float, kWidth>(o, c0, lane);
    else write_rows<uint16_t, kWidth>(o, c0, lane);
    __syncwarp();
}

// 16 columns on their way into registers, which may be looked at after tmem_arrived
__device__ __forceinline__ void tmem_ask16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_arrived(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :: "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
          "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
        : "memory");
}

template <int KIND, int LOADS, bool PAIR, bool GATED>
__global__ void __launch_bounds__(threads_of(KIND, LOADS), 1)
expert_mm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const GroupedParams p,
                 const MmGeom t) {
    constexpr int kPlanes = KIND == kX3 ? 2 : 1;
    constexpr int kEpilogueWarps = epilogue_warps(KIND, LOADS), kLoadWarp0 = 4 + kEpilogueWarps;
    constexpr bool kSplit = KIND == kX3 && LOADS != kRegs;
    constexpr int kSplitWarp0 = kLoadWarp0 + (LOADS == kGather ? kGatherWarps : 0);
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(16) float row_scale_s[2][256];
    __shared__ uint32_t live_s[2][8];                            // one bit per column: its row exists
    __shared__ uint32_t tmem_slot;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *generic = smem_raw + (base - smem_u32(smem_raw));
    const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const uint32_t b_bytes = uint32_t(PAIR ? t.tn / 2 : t.tn) * kRowBytes;
    const uint32_t stage_bytes = kPlanes * (kATileBytes + b_bytes);
    const uint32_t full0 = base + t.bar_off, empty0 = full0 + 8u * t.stages;
    const uint32_t acc_full0 = empty0 + 8u * t.stages, acc_empty0 = acc_full0 + 16u;
    const uint32_t recv_full = acc_empty0 + 16u, recv_free = recv_full + 8u, ready0 = recv_free + 8u;
    int *const bounds = reinterpret_cast<int *>(generic + t.table_off + kListed * sizeof(int4));
    const Table table = {reinterpret_cast<int4 *>(generic + t.table_off), bounds, bounds + p.groups + 1};

    if (LOADS != kRegs && threadIdx.x == 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < t.stages; ++s) {
            mbar_init(full0 + 8u * s, LOADS == kRegs ? kLoaderWarps : 1);
            mbar_init(empty0 + 8u * s, 1);
            mbar_init(ready0 + 8u * s, kSplitWarps);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(acc_full0 + 8u * a, 1);
            mbar_init(acc_empty0 + 8u * a, (PAIR ? 2 : 1) * kEpilogueWarps);
        }
        mbar_init(recv_full, uint32_t(kEpilogueWarps * t.cluster));
        mbar_init(recv_free, uint32_t(kEpilogueWarps * t.cluster));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 2) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(t.tmem_cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            tmem_alloc(smem_u32(&tmem_slot), uint32_t(t.tmem_cols));
            tmem_relinquish();
        }
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    build_table(p, t, table, threads_of(KIND, LOADS));
    __syncthreads();
    const int rank = PAIR || t.cluster > 1 ? uniform(int(cluster_cta_rank())) : 0;
    const int sharing = PAIR ? 2 : t.cluster;                    // CTAs of a tile
    const int tile0 = int(blockIdx.x) / sharing, tile_step = int(gridDim.x) / sharing;
    const int k_begin = PAIR ? 0 : t.k_steps * rank / t.cluster, k_end = PAIR ? t.k_steps : t.k_steps * (rank + 1) / t.cluster;
    const int cta_channel = PAIR ? rank * (t.tile_channels / 2) : 0;
    const int total_tiles = uniform(table.first[p.groups]);
    if (threadIdx.x < kListed && int(threadIdx.x) * tile_step < total_tiles - tile0)
        table.listed[threadIdx.x] = find_tile(t, table, p.groups, tile0 + int(threadIdx.x) * tile_step, cta_channel);
    tc_fence_before();
    __syncthreads();
    if (PAIR || t.cluster > 1) cluster_sync_all();
    tc_fence_after();
    // (only now: a successor that were to share this SM must find the tensor memory taken, not take it)
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t tmem = uint32_t(uniform(int(tmem_slot)));
    // a pair's loads are counted in the CTA of rank 0, whose MMA issuer works for both
    const uint32_t full_at = PAIR ? cluster_map(full0, 0) : full0;
    const int k_elems = kRowBytes / t.esize;

    // Bytes that the rows of one K step bring into the CTA that holds columns from `col0` on.  Every warp that brings rows
    // brings some, also where the tile needs none: otherwise the ring of stages could run on without it, and a wait by
    // parity does not notice two rounds.
    const auto row_bytes_of = [&](const Tile &tile, int col0) {
        const int unit = LOADS == kGather ? 4 : t.box_rows, least = LOADS == kGather && t.tn > kNarrowCols ? 4 * kGatherWarps : 1;
        const int rows = max(least, min(PAIR ? tile.cols / 2 : tile.cols, tile.valid - col0));
        return uint32_t((rows + unit - 1) / unit * unit) * kRowBytes;
    };
    if (LOADS != kRegs && warp == 0) {
        // ---------------- weights; arms the stage's barrier for the rows as well ----------------
        const uint32_t elected = elect();
        int s = 0;
        uint32_t phase = 1;
        int armed = 0;
        bool ok = true;
        for (int i = tile0, n = 0; i < total_tiles && ok; i += tile_step, ++n) {
            const Tile tile = tile_of(p, t, table, n, i, cta_channel);
            const uint32_t bytes = (PAIR ? 2 : 1) * kATileBytes + row_bytes_of(tile, 0) + (PAIR ? row_bytes_of(tile, tile.cols / 2) : 0);
            for (int k = k_begin; k < k_end; ++k) {
                ok = __all_sync(0xffffffffu, wait<false>(empty0 + 8u * s, phase, t.wait_ns) ? 1 : 0) != 0;
                if (!ok) break;
                const uint32_t dst = base + uint32_t(s) * stage_bytes, bar = full_at + 8u * s;
                if (!PAIR || rank == 0) expect(elected, full0 + 8u * s, bytes);
                if (!GATED) {
                    load_3d<PAIR>(elected, dst, &map_w, bar, k * k_elems, tile.channel0, tile.group);
                } else if (t.one_box) {
                    load_5d<PAIR>(elected, dst, &map_w, bar, k * k_elems, tile.channel0 / 16, tile.group);
                } else {
#pragma unroll
                    for (int b = 0; b < 8; ++b)
                        load_3d<PAIR>(elected, dst + uint32_t(b) * 16u * kRowBytes, &map_w, bar, k * k_elems, weight_row<GATED>(p, tile, b * 16), tile.group);
                }
                ++armed;
                if (++s == t.stages) { s = 0; phase ^= 1u; }
            }
        }
        if (!ok) {
            if (lane == 0) time_out(1);
            for (int j = armed - 1, left = t.stages; j >= 0 && left > 0 && (!PAIR || rank == 0); --j, --left)
                mbar_wait(full0 + 8u * (j % t.stages), uint32_t((j / t.stages) & 1), nullptr);
        }
    } else if (LOADS == kTma && warp == 3) {
        // ---------------- rows ----------------
        const uint32_t elected = elect();
        int s = 0;
        uint32_t phase = 1;
        bool ok = true;
        for (int i = tile0, n = 0; i < total_tiles && ok; i += tile_step, ++n) {
            const Tile tile = tile_of(p, t, table, n, i, cta_channel);
            const int col0 = PAIR ? rank * (tile.cols / 2) : 0;              // a pair's CTAs hold half of the columns each
            const int loads = int(row_bytes_of(tile, col0)) / (t.box_rows * kRowBytes);
            for (int k = k_begin; k < k_end; ++k) {
                ok = __all_sync(0xffffffffu, wait<false>(empty0 + 8u * s, phase, t.wait_ns) ? 1 : 0) != 0;
                if (!ok) break;
                const uint32_t dst = base + uint32_t(s) * stage_bytes + kPlanes * kATileBytes, bar = full_at + 8u * s;
                for (int b = 0; b < loads; ++b)
                    load_2d<PAIR>(elected, dst + uint32_t(b * t.box_rows) * kRowBytes, &map_x, bar, k * k_elems, tile.row0 + col0 + b * t.box_rows);
                if (++s == t.stages) { s = 0; phase ^= 1u; }
            }
        }
        if (!ok && lane == 0) time_out(2);
    } else if (LOADS == kGather && warp >= kLoadWarp0 && warp < kLoadWarp0 + kGatherWarps) {
        // ---------------- gathered rows, in groups of four: a group per lane ----------------
        // Wide tiles: the groups of every step are dealt to all warps.  Narrow tiles, a few groups per step: every warp loads
        // all groups of its turn's steps -- and there are no more turns than stages, or a warp's wait by parity could take the
        // stage's last round but one for its last.
        const int part = warp - kLoadWarp0;
        const bool narrow = t.tn <= kNarrowCols;
        const int turns = t.stages >= kGatherWarps ? kGatherWarps : kGatherWarps / 2;
        const int group = narrow ? lane : lane * kGatherWarps + part;
        int s = 0, step = 0;
        uint32_t phase = 1;
        bool ok = true;
        for (int i = tile0, n = 0; i < total_tiles && ok; i += tile_step, ++n) {
            const Tile tile = tile_of(p, t, table, n, i, cta_channel);
            const int col0 = PAIR ? rank * (tile.cols / 2) : 0;
            const bool loads = group < int(row_bytes_of(tile, col0)) / (4 * kRowBytes);
            int at[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int r = p.rows[tile.row0 + min(col0 + group * 4 + q, tile.valid - 1)];
                at[q] = r >= 0 && r < p.x_rows ? r : 0;               // the epilogue makes zeros of a row that is none
            }
            const int4 src = make_int4(at[0], at[1], at[2], at[3]);
            for (int k = k_begin; k < k_end; ++k, ++step) {
                if (!narrow || (step & (turns - 1)) == part) {
                    ok = __all_sync(0xffffffffu, wait<false>(empty0 + 8u * s, phase, t.wait_ns) ? 1 : 0) != 0;
                    if (!ok) break;
                    if (loads)
                        load_rows4<PAIR>(1u, base + uint32_t(s) * stage_bytes + kPlanes * kATileBytes + uint32_t(group) * 4u * kRowBytes, &map_x,
                                         full_at + 8u * s, k * k_elems, src);
                    __syncwarp();
                }
                if (++s == t.stages) { s = 0; phase ^= 1u; }
            }
        }
        if (!ok && lane == 0) time_out(3);
    } else if (LOADS == kRegs && warp >= kLoadWarp0) {
        // ---------------- loader warps ----------------
        // Each warp moves 8 rows of the weights and 8 of x: lane l the word at 4 l of a row's 128 bytes.  A row that starts off
        // a word boundary takes the 33 words around them, shifted into place between neighbouring lanes; the last words of the
        // 16 rows are loaded together, lane r that of row r.  The next step is asked for before this one is stored.  Where the
        // rows start stands in shared memory, so that nothing but loads is left to do for a row (16 instructions and a branch
        // per row took 130 cycles).  Rows that are not there repeat some row that is: their results are not stored, or made
        // zeros by the epilogue.
        __shared__ unsigned long long src_s[kLoaderWarps][2 * kLoaderRows];
        constexpr int kR = kLoaderRows;
        const int part = warp - kLoadWarp0;
        const unsigned long long *src = src_s[part];
        const long long row_bytes = (long long)p.inner * t.esize;
        int s = 0;
        uint32_t phase = 1;
        bool ok = true;
        for (int i = tile0, n = 0; i < total_tiles && ok; i += tile_step, ++n) {
            const Tile tile = tile_of(p, t, table, n, i, cta_channel);
            const bool with_x = part * kR < tile.cols;
            unsigned long long own;                          // lane r: where row r of the warp's 16 starts
            {
                const int r = min(weight_row<GATED>(p, tile, part * kR + (lane & (kR - 1))), (GATED ? 2 * p.channels : p.channels) - 1);
                own = reinterpret_cast<unsigned long long>(p.w) + (tile.group * p.w_group_stride + r * p.w_stride) * t.esize;
                if (lane >= kR && p.x_rows > 0) {
                    const int c = tile.row0 + min(part * kR + (lane & (kR - 1)), tile.valid - 1), at = p.rows ? p.rows[c] : c;
                    own = reinterpret_cast<unsigned long long>(p.x) + (at >= 0 && at < p.x_rows ? at : 0) * p.x_stride * t.esize;
                }
            }
            __syncwarp();
            if (lane < 2 * kR) src_s[part][lane] = own;
            __syncwarp();
            const uint32_t own_skew = uint32_t(own) & 3u;
            const bool skewed = __any_sync(0xffffffffu, own_skew != 0);
            // Steps whose words are whole words of their rows (or, without skew, of the zeros behind them).
            const auto plain = [&](int k) {
                return (!skewed && (row_bytes & 3) == 0) || ((k > 0 || !skewed) && (k + 1LL) * kRowBytes + 4 <= row_bytes);
            };
            const auto fetch = [&](uint32_t *v, uint32_t &last, int k) {
                const long long byte0 = (long long)k * kRowBytes;
                const bool inside = byte0 + 4 * lane + 4 <= row_bytes;
#pragma unroll
                for (int r = 0; r < kR; ++r)
                    v[r] = inside ? __ldg(reinterpret_cast<const uint32_t *>((src[r] & ~3ull) + byte0 + 4 * lane)) : 0u;
                if (with_x) {
#pragma unroll
                    for (int r = kR; r < 2 * kR; ++r)
                        v[r] = inside ? __ldg(reinterpret_cast<const uint32_t *>((src[r] & ~3ull) + byte0 + 4 * lane)) : 0u;
                }
                if (skewed) last = own_skew ? __ldg(reinterpret_cast<const uint32_t *>((own & ~3ull) + byte0 + kRowBytes)) : 0u;
            };
            uint32_t now[2 * kR], next[2 * kR], now_last = 0, next_last = 0;
#pragma unroll
            for (int r = 0; r < 2 * kR; ++r) now[r] = next[r] = 0;
            if (plain(k_begin)) fetch(now, now_last, k_begin);
            for (int k = k_begin; k < k_end; ++k) {
                if (k + 1 < k_end && plain(k + 1)) fetch(next, next_last, k + 1);
                ok = __all_sync(0xffffffffu, wait<false>(empty0 + 8u * s, phase, t.wait_ns) ? 1 : 0) != 0;
                if (!ok) break;
                uint8_t *stage = generic + size_t(s) * stage_bytes + part * kR * kRowBytes + (lane & 3) * 4;
                const auto store = [&](int r, uint32_t word) {
                    uint8_t *dst = stage + (r < kR ? 0 : kPlanes * kATileBytes) + sw128_offset(r & (kR - 1), lane >> 2);
                    if (KIND != kX3) {
                        *reinterpret_cast<uint32_t *>(dst) = word;
                    } else {
                        uint32_t hi, lo;
                        split_tf32(word, &hi, &lo);
                        *reinterpret_cast<uint32_t *>(dst) = hi;
                        *reinterpret_cast<uint32_t *>(dst + (r < kR ? uint32_t(kATileBytes) : b_bytes)) = lo;
                    }
                };
                const auto shifted = [&](int r, uint32_t word, uint32_t last) {
                    const uint32_t beside = __shfl_down_sync(0xffffffffu, word, 1);
                    return __funnelshift_r(word, lane == 31 ? last : beside, 8 * (uint32_t(src[r]) & 3u));
                };
                if (!plain(k)) {
                    const long long byte0 = (long long)k * kRowBytes;
#pragma unroll 1
                    for (int r = 0; r < (with_x ? 2 * kR : kR); ++r) {
                        const uint8_t *row = reinterpret_cast<const uint8_t *>(src[r]);
                        const int skew = int(src[r] & 3ull);
                        const uint32_t word = load_edge(row, byte0 + 4 * lane - skew, row_bytes, t.esize);
                        const uint32_t last = lane == 31 && skew ? load_edge(row, byte0 + kRowBytes - skew, row_bytes, t.esize) : 0u;
                        store(r, shifted(r, word, last));
                    }
                } else if (!skewed) {
#pragma unroll
                    for (int r = 0; r < kR; ++r) store(r, now[r]);
                    if (with_x) {
#pragma unroll
                        for (int r = kR; r < 2 * kR; ++r) store(r, now[r]);
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < kR; ++r) store(r, shifted(r, now[r], __shfl_sync(0xffffffffu, now_last, r)));
                    if (with_x) {
#pragma unroll
                        for (int r = kR; r < 2 * kR; ++r) store(r, shifted(r, now[r], __shfl_sync(0xffffffffu, now_last, r)));
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(full0 + 8u * s);
                if (++s == t.stages) { s = 0; phase ^= 1u; }
#pragma unroll
                for (int r = 0; r < 2 * kR; ++r) now[r] = next[r];
                now_last = next_last;
            }
        }
        if (!ok && lane == 0) time_out(6);
    } else if (kSplit && warp >= kSplitWarp0) {
        // ---------------- landed float32 operands into two TF32 numbers each, the larger in place ----------------
        const int tid = int(threadIdx.x) - 32 * kSplitWarp0;
        int s = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int i = tile0, n = 0; i < total_tiles && ok; i += tile_step, ++n) {
            const Tile tile = tile_of(p, t, table, n, i, cta_channel);
            for (int k = k_begin; k < k_end; ++k) {
                ok = __all_sync(0xffffffffu, wait<false>(full0 + 8u * s, phase, t.wait_ns) ? 1 : 0) != 0;
                if (!ok) break;
                uint8_t *stage = generic + size_t(s) * stage_bytes;
                const auto split = [&](uint8_t *at, uint32_t apart) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(at);
                    uint4 hi, lo;
                    split_tf32(x.x, &hi.x, &lo.x);
                    split_tf32(x.y, &hi.y, &lo.y);
                    split_tf32(x.z, &hi.z, &lo.z);
                    split_tf32(x.w, &hi.w, &lo.w);
                    *reinterpret_cast<uint4 *>(at) = hi;
                    *reinterpret_cast<uint4 *>(at + apart) = lo;
                };
                constexpr int kThreads = 32 * kSplitWarps;
#pragma unroll
                for (int q = 0; q < kATileBytes / 16 / kThreads; ++q) split(stage + (q * kThreads + tid) * 16, kATileBytes);
#pragma unroll 4
                for (int v = tid; v < tile.cols * (kRowBytes / 16); v += kThreads) split(stage + 2 * kATileBytes + v * 16, b_bytes);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(ready0 + 8u * s);
                if (++s == t.stages) { s = 0; phase ^= 1u; }
            }
        }
        if (!ok && lane == 0) time_out(7);
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        if (!PAIR || rank == 0) {
            const uint32_t elected = elect();
            int s = 0;
            uint32_t phase = 0;
            int turn = 0;                                       // accumulator hand-overs so far
            bool ok = true;
            const uint32_t a_low0 = desc_low(base), stage_low = stage_bytes >> 4, b_low0 = kPlanes * kATileBytes >> 4;
            for (int i = tile0, n = 0; i < total_tiles && ok; i += tile_step, ++n) {
                const Tile tile = tile_of(p, t, table, n, i, cta_channel);
                // sums in float32 / int32 (bit 4 / 5), operand formats, both K-major, N and M
                const uint32_t idesc = (KIND == kI8 ? 2u << 4 : 1u << 4) | (t.format << 7) | (t.format << 10) |
                                       (uint32_t(tile.cols >> 3) << 17) | (uint32_t((PAIR ? 2 : 1) * kTileM >> 4) << 24);
                for (int k = k_begin; k < k_end;) {
                    const int stop = KIND == kX3 ? min(k + kChunkSteps, k_end) : k_end;
                    const uint32_t a = uint32_t(turn) & 1u, d = tmem + a * uint32_t(t.tn);
                    ok = __all_sync(0xffffffffu, wait<PAIR>(acc_empty0 + 8u * a, ((uint32_t(turn) >> 1) & 1u) ^ 1u, t.wait_ns) ? 1 : 0) != 0;
                    uint32_t acc = 0;
                    for (; ok && k < stop; ++k) {
                        ok = __all_sync(0xffffffffu, wait<PAIR>((kSplit ? ready0 : full0) + 8u * s, phase, t.wait_ns) ? 1 : 0) != 0;
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t a_low = a_low0 + uint32_t(s) * stage_low, b_low = a_low + b_low0;
#pragma unroll
                        for (uint32_t q = 0; q < 8; q += 2) {
                            if (KIND != kX3) {
                                umma<KIND, PAIR>(elected, d, a_low + q, b_low + q, idesc, acc);
                            } else {
                                const uint32_t a_rest = a_low + (kATileBytes >> 4), b_rest = b_low + (b_bytes >> 4);
                                umma<KIND, PAIR>(elected, d, a_rest + q, b_low + q, idesc, acc);
                                umma<KIND, PAIR>(elected, d, a_low + q, b_rest + q, idesc, 1u);
                                umma<KIND, PAIR>(elected, d, a_low + q, b_low + q, idesc, 1u);
                            }
                            acc = 1;
                        }
                        commit<PAIR>(elected, empty0 + 8u * s);
                        if (++s == t.stages) { s = 0; phase ^= 1u; }
                    }
                    if (!ok) break;
                    commit<PAIR>(elected, acc_full0 + 8u * a);
                    ++turn;
                }
            }
            if (!ok && lane == 0) time_out(4);
        }
    } else if (warp >= 4 && warp < kLoadWarp0) {
        // ---------------- epilogue ----------------
        // warps 4 + q and 8 + q read lanes 32 q .. 32 q + 31 of tensor memory and alternate in the columns
        constexpr int kShare = kEpilogueWarps / 4;
        const int quad = warp & 3, share = (warp >> 2) - 1, tid = int(threadIdx.x) - 128, lane_row = quad * 32 + lane;
        const uint32_t lane_tmem = tmem + (uint32_t(quad * 32) << 16);
        const uint32_t recv = base + t.recv_off;
        float *recv_generic = reinterpret_cast<float *>(generic + t.recv_off);
        const int out_size = elem_size(p.out_type);
        constexpr int kWidth = GATED ? 16 : 32;                       // channels of a warp
        const int half = GATED ? lane >> 4 : 0;
        Out o;
        o.turn = generic + t.turn_off + (warp - 4) * kTurnBytes;
        o.row_bytes = p.y_stride * out_size;
        int turn = 0, round = 0;
        bool ok = true;
#pragma unroll 1
        for (int i = tile0, n = 0; i < total_tiles && ok; i += tile_step, ++n, ++round) {
            const Tile tile = tile_of(p, t, table, n, i, cta_channel);
            const int warp_channel = tile.channel0 + quad * kWidth;
            const int channel = warp_channel + lane % kWidth;
            const long long per_channel = (long long)tile.group * (GATED ? 2 : 1) * p.channels + (long long)half * p.channels + channel;
            const float channel_scale = p.channel_scale && channel < p.channels ? p.channel_scale[per_channel] : 1.0f;
            const float bias = p.bias && channel < p.channels ? p.bias[per_channel] : 0.0f;
            o.first = static_cast<uint8_t *>(p.y) + (tile.row0 * p.y_stride + warp_channel) * out_size;
            o.rows = tile.valid;
            o.channels = max(0, min(kWidth, p.channels - warp_channel));
            o.vectors = ((reinterpret_cast<uintptr_t>(o.first) | uintptr_t(o.row_bytes)) & 15) == 0 && o.channels == kWidth;
            const float *row_scale = row_scale_s[round & 1];
            const uint32_t *live = live_s[round & 1];
            if (p.row_scale || (LOADS != kTma && p.rows)) {
                for (int c = tid; c < max(t.tn, 32); c += 32 * kEpilogueWarps) {              // whole warps
                    const int src = c >= tile.valid ? 0 : p.rows ? p.rows[tile.row0 + c] : tile.row0 + c;
                    const bool known = src >= 0 && src < p.x_rows;
                    row_scale_s[round & 1][c] = p.row_scale && known ? p.row_scale[src] : 1.0f;
                    const uint32_t mask = __ballot_sync(0xffffffffu, known);
                    if (lane == 0) live_s[round & 1][c >> 5] = mask;
                }
                asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpilogueWarps) : "memory");
            }
            // ---- the sums of this CTA's K range ----
            uint32_t sums = lane_tmem + (uint32_t(turn) & 1u) * uint32_t(t.tn), held = acc_empty0 + 8u * (uint32_t(turn) & 1u);
            if (KIND != kX3) {
                ok = wait<PAIR>(acc_full0 + 8u * (uint32_t(turn) & 1u), (uint32_t(turn) >> 1) & 1u, t.wait_ns);
                ++turn;
            } else {
                // added up in tensor memory behind the two accumulators
                sums = lane_tmem + 2u * uint32_t(t.tn);
                for (int k = k_begin; k < k_end && ok; k += kChunkSteps, ++turn) {
                    const uint32_t a = uint32_t(turn) & 1u;
                    ok = __all_sync(0xffffffffu, wait<PAIR>(acc_full0 + 8u * a, (uint32_t(turn) >> 1) & 1u, t.wait_ns) ? 1 : 0) != 0;
                    if (!ok) break;
                    tc_fence_after();
                    for (int c0 = share * 16; c0 < tile.cols; c0 += kShare * 16) {
                        float v[16], sum[16];
                        tmem_ld16(lane_tmem + a * uint32_t(t.tn) + c0, v);
                        if (k != k_begin) {
                            tmem_ld16(sums + c0, sum);
#pragma unroll
                            for (int c = 0; c < 16; ++c) v[c] += sum[c];
                        }
                        tmem_st16(sums + c0, v);
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(acc_empty0 + 8u * a);          // (no pairs)
                }
            }
            if (ok && t.cluster > 1 && round > 0) ok = wait<true>(recv_free, uint32_t(round - 1) & 1u, t.wait_ns);
            ok = __all_sync(0xffffffffu, ok ? 1 : 0) != 0;
            if (!ok) break;
            tc_fence_after();
            const auto release = [&]() {                              // the accumulator may be written again
                if (KIND == kX3) return;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (PAIR) mbar_arrive_cluster(cluster_map(held, 0));
                    else mbar_arrive(held);
                }
            };
            int from = share * kTurnCols, step = kShare * kTurnCols;
            const int per = tile.cols / t.cluster;                    // columns that each CTA finishes
            if (t.cluster > 1) {
                for (int c0 = share * 16; c0 < tile.cols; c0 += kShare * 16) {
                    float v[16];
                    tmem_ld16(sums + c0, v);
                    int d = c0 / per, at = c0 - d * per;
#pragma unroll
                    for (int c = 0; c < 16; ++c) {
                        store_cluster(cluster_map(recv + uint32_t((rank * per + at) * kTileM + lane_row) * 4u, uint32_t(d)), v[c]);
                        if (++at == per) { at = 0; ++d; }
                    }
                }
                release();
                __syncwarp();
                if (lane < t.cluster) mbar_arrive_cluster(cluster_map(recv_full, uint32_t(lane)));
                ok = __all_sync(0xffffffffu, wait<true>(recv_full, uint32_t(round) & 1u, t.wait_ns) ? 1 : 0) != 0;
                if (!ok) break;
                // pairs of columns: a gated result takes two lanes' columns at once
                const int mine = kShare == 1 ? per : (per / 2 + 1) / 2 * 2;          // columns of the first warp of a quarter
                from = rank * per + share * mine;
                step = kTurnCols;
                o.rows = min(tile.valid, rank * per + (share == 0 ? mine : per));
            }
            // ---- scales, bias, activation, store: 16 columns at a time (those behind the last are not used) ----
            uint32_t ahead[kTurnCols];
            if (t.cluster == 1 && from < o.rows) tmem_ask16(sums + from, ahead);
#pragma unroll 1
            for (int c0 = from; c0 < o.rows; c0 += step) {
                float v[kTurnCols];
                if (t.cluster == 1) {
                    tmem_arrived(ahead);
#pragma unroll
                    for (int c = 0; c < kTurnCols; ++c) v[c] = __uint_as_float(ahead[c]);
                    if (c0 + step < o.rows) tmem_ask16(sums + c0 + step, ahead);
                    else release();
                } else {
                    // the partial sums of all ranks, in rank order
                    const float *part = recv_generic + (c0 - rank * per) * kTileM + lane_row;
                    const int count = o.rows - c0;
#pragma unroll
                    for (int c = 0; c < kTurnCols; ++c) v[c] = c < count ? part[c * kTileM] : 0.0f;
#pragma unroll 1
                    for (int q = 1; q < t.cluster; ++q) {
                        part += per * kTileM;
#pragma unroll
                        for (int c = 0; c < kTurnCols; ++c) {
                            const float more = c < count ? part[c * kTileM] : 0.0f;
                            v[c] = KIND == kI8 ? __int_as_float(__float_as_int(v[c]) + __float_as_int(more)) : v[c] + more;
                        }
                    }
                }
                if (o.channels == 0) continue;
                if (KIND == kI8) {
#pragma unroll
                    for (int c = 0; c < kTurnCols; ++c) v[c] = float(__float_as_int(v[c]));
                }
                if (LOADS != kTma && p.rows) {                        // a row that is none was loaded as some other one
                    const uint32_t mask = __funnelshift_r(live[c0 >> 5], live[min(c0 >> 5, 6) + 1], c0);
                    if ((mask & 0xffffu) != 0xffffu) {
#pragma unroll
                        for (int c = 0; c < kTurnCols; ++c)
                            if (!((mask >> c) & 1u)) v[c] = 0.0f;
                    }
                }
                if (p.row_scale) {
                    if (t.cluster == 1) {
#pragma unroll
                        for (int c = 0; c < kTurnCols; c += 4) {
                            const float4 f = *reinterpret_cast<const float4 *>(row_scale + c0 + c);
                            v[c] *= f.x; v[c + 1] *= f.y; v[c + 2] *= f.z; v[c + 3] *= f.w;
                        }
                    } else {                                          // a rank's columns start at any even one
#pragma unroll
                        for (int c = 0; c < kTurnCols; ++c) v[c] *= row_scale[c0 + c];
                    }
                }
#pragma unroll
                for (int c = 0; c < kTurnCols; ++c) v[c] = v[c] * channel_scale + bias;
                if (!GATED) {
                    activate<kTurnCols>(v, p.act, p.out_type != Elem::F32);
                } else {
                    // the lower half of the warp finishes the even columns, the upper half the odd ones
                    float up[kTurnCols / 2];
#pragma unroll
                    for (int c = 0; c < kTurnCols / 2; ++c) {
                        const float other = __shfl_xor_sync(0xffffffffu, half ? v[2 * c] : v[2 * c + 1], 16);
                        up[c] = half ? v[2 * c + 1] : other;
                        v[c] = half ? other : v[2 * c];
                    }
                    activate<kTurnCols / 2>(v, p.act, p.out_type != Elem::F32);
#pragma unroll
                    for (int c = 0; c < kTurnCols / 2; ++c) v[c] *= up[c];
                }
                write_columns<GATED>(o, p.out_type, v, c0, lane);
            }
            if (t.cluster == 1) {
                if (from >= o.rows) release();
            } else {
                __syncwarp();
                if (lane < t.cluster) mbar_arrive_cluster(cluster_map(recv_free, uint32_t(lane)));
            }
        }
        if (!ok) {
            if (lane == 0) time_out(5);
            __syncwarp();
            // the rest may still be at work: their barrier needs this warp in every tile to come
            if (p.row_scale || (LOADS != kTma && p.rows))
                for (int i = tile0 + (round + 1) * tile_step; i < total_tiles; i += tile_step)
                    asm volatile("bar.sync 1, %0;" ::"n"(32 * kEpilogueWarps) : "memory");
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    // nobody may still push into, load into or multiply from the shared memory of a CTA that has gone
    if (PAIR || t.cluster > 1) cluster_sync_all();
    if (warp == 2) {
        tc_fence_after();
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(t.tmem_cols) : "memory");
        else tmem_dealloc(tmem, uint32_t(t.tmem_cols));
    }
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                  const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_fn() {
    static const EncodeTiledFn fn = [] {
        void *sym = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            sym = nullptr;
        return reinterpret_cast<EncodeTiledFn>(sym);
    }();
    return fn;
}

bool encode(CUtensorMap *map, Elem type, const void *base, int rank, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box) {
    const CUtensorMapDataType types[] = {CU_TENSOR_MAP_DATA_TYPE_FLOAT32, CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                                         CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, CU_TENSOR_MAP_DATA_TYPE_UINT8};
    const cuuint32_t steps[5] = {1, 1, 1, 1, 1};
    return encode_fn()(map, types[int(type)], cuuint32_t(rank), const_cast<void *>(base), dims, strides, box, steps,
                       CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The weights: boxes of one swizzle row x 128 rows of a group; gated: (element, channel of 16, half, block of 16 channels, group)
// in boxes of 16 x 2 x 4 channels, or 16 rows at a time where the channels do not come in sixteens.
bool encode_weights(CUtensorMap *map, const GroupedParams &p, const MmGeom &t) {
    const cuuint64_t row = cuuint64_t(p.w_stride) * t.esize, wide = cuuint64_t(p.gated ? 2 : 1) * p.channels;
    const cuuint64_t group = p.groups == 1 ? 16 : cuuint64_t(p.w_group_stride) * t.esize;      // (one group: no stride needed)
    const cuuint32_t elems = cuuint32_t(kRowBytes / t.esize);
    if (t.one_box) {
        const cuuint64_t dims[5] = {cuuint64_t(p.inner), 16, 2, cuuint64_t(p.channels / 16), cuuint64_t(p.groups)};
        const cuuint64_t strides[4] = {row, row * p.channels, row * 16, group};
        const cuuint32_t box[5] = {elems, 16, 2, 4, 1};
        return encode(map, p.type, p.w, 5, dims, strides, box);
    }
    const cuuint64_t dims[3] = {cuuint64_t(p.inner), wide, cuuint64_t(p.groups)};
    const cuuint64_t strides[2] = {row, group};
    const cuuint32_t box[3] = {elems, cuuint32_t(p.gated ? 16 : kTileM), 1};
    return encode(map, p.type, p.w, 3, dims, strides, box);
}

// The rows: boxes of box_rows of them, or single ones to gather.
bool encode_rows(CUtensorMap *map, const GroupedParams &p, const MmGeom &t) {
    const cuuint64_t dims[2] = {cuuint64_t(p.inner), cuuint64_t(p.x_rows)};
    const cuuint64_t strides[1] = {cuuint64_t(p.x_stride) * t.esize};
    const cuuint32_t box[2] = {cuuint32_t(kRowBytes / t.esize), cuuint32_t(p.rows ? 1 : t.box_rows)};
    return encode(map, p.type, p.x, 2, dims, strides, box);
}

// May TMA read rows of this stride?  (16-byte aligned rows that do not overlap, strides below 2^40 bytes)
bool tma_rows(const void *base, long long stride, int inner, int esize) {
    const long long bytes = stride * esize;
    return reinterpret_cast<uintptr_t>(base) % 16 == 0 && bytes % 16 == 0 && stride >= inner && bytes < (1LL << 40);
}

int ceil_div(long long a, long long b) { return int((a + b - 1) / b); }

bool tma_able(const GroupedParams &p) {
    const int esize = elem_size(p.type);
    const long long wide = p.gated ? 2 * p.channels : p.channels, group_bytes = p.w_group_stride * esize;
    return p.x_rows > 0 && tma_rows(p.x, p.x_stride, p.inner, esize) && tma_rows(p.w, p.w_stride, p.inner, esize) &&
           (p.groups == 1 || (group_bytes % 16 == 0 && p.w_group_stride >= wide * p.w_stride && group_bytes < (1LL << 40)));
}

// Columns of a tile: the smallest power of two that holds an average group, so that most groups read their weights once.
int columns_for(const GroupedParams &p, int most) {
    const int average = ceil_div(p.total, std::min(p.groups, p.total));
    int tn = 16;
    while (tn < average && tn < most) tn *= 2;
    return tn;
}

std::atomic<uint32_t> g_wait_us{0};                           // testing aid: what a wait may take; 0: the default

// Chooses the tiling; touches no device.  Returns the CTAs to launch.
int choose(const GroupedParams &p, int sm_count, bool tma, MmGeom *t, bool *pair) {
    const int esize = elem_size(p.type);
    t->esize = esize;
    const uint32_t wait_us = g_wait_us.load(std::memory_order_relaxed);
    t->wait_ns = wait_us ? wait_us * 1000u : uint32_t(kWaitBudgetNs);
    t->format = p.type == Elem::BF16 ? 1u : p.type == Elem::F16 ? 0u : p.type == Elem::S8 ? 1u : 2u;
    t->tile_channels = p.gated ? kTileM / 2 : kTileM;
    t->n_tiles = ceil_div(p.channels, t->tile_channels);
    t->k_steps = ceil_div((long long)p.inner * esize, kRowBytes);
    const int busy = std::min(p.groups, p.total);
    t->tn = columns_for(p, tma && p.type != Elem::F32 ? 256 : kLoaderCols);
    auto tiles = [&]() { return (long long)t->n_tiles * std::max<long long>(busy, ceil_div(p.total, t->tn)); };
    // ... or half of that where twice the tiles still run at once (200 rows, 4096 -> 2048 in 8 bits: 20.5 us instead of 24.6)
    if (tiles() * 2 <= sm_count && t->tn > 128) t->tn = 128;
    // K split: as long as it fills SMs that would idle and leaves every CTA two K steps (one row, 4096 -> 1024 in 8 bits, eight
    // CTAs to a tile: 14.4 us instead of 16.4; where only two fit, 4096 -> 8192, 18.5 either way)
    t->cluster = 1;
    while (t->cluster < 8 && t->tn <= 128 && tiles() * t->cluster * 2 <= sm_count && t->k_steps >= 4 * t->cluster) t->cluster *= 2;
    // Pairs of CTAs share the rows of a tile of 256 channels: half of the loads of x per SM, and with them more K steps in
    // flight (32768 rows in four groups, 2048 -> 1280, bfloat16: 113 us instead of 129; 1024 rows, 4096 -> 8192 in 8 bits: 43 instead
    // of 45; level where there are few tiles)
    *pair = tma && t->tn == 256;
    t->grain = *pair ? 32 : 16;
    if (*pair) {
        t->tile_channels *= 2;
        t->n_tiles = ceil_div(p.channels, t->tile_channels);
    }
    // (eight boxes of 16 rows instead: 272 us for 266, 4096 tokens x 8 of 64 experts)
    t->one_box = p.gated && p.channels % 16 == 0;
    t->box_rows = std::min(*pair ? t->tn / 2 : t->tn, kBoxRows);
    t->tmem_cols = std::max(32, (p.type == Elem::F32 ? 4 : 2) * t->tn);      // two accumulators; float32: and their sum (a power of two)
    const int planes = p.type == Elem::F32 ? 2 : 1;
    const size_t stage = size_t(planes) * (kATileBytes + (*pair ? t->tn / 2 : t->tn) * kRowBytes);
    const size_t recv = t->cluster > 1 ? size_t(t->tn) * kTileM * sizeof(float) : 0;
    const size_t table = kListed * sizeof(int4) + (2 * size_t(p.groups + 1) * sizeof(int) + 15) / 16 * 16;
    const size_t turn = 8 * kTurnBytes;
    // The stages take what is left: no second CTA with tensor memory of this kernel fits beside one, and what a CTA leaves of its SM (27 KB,
    // float32 43 KB and 8 thousand registers) is too little for a CTA of another kernel's cluster.  So no two clusters can hold one SM's tensor
    // memory each and wait for the other's.
    const size_t fixed = 1024 + recv + turn + table + kBarBytes + kStaticBytes;
    t->stages = int(std::min<size_t>(kMaxStages, (kSmemLimit - fixed) / stage));
    static_assert((kSmemLimit - 1024 - kNarrowCols * kTileM * 4 - 8 * kTurnBytes - kListed * 16 - 2 * (kMaxExperts + 4) * 4 - kBarBytes - kStaticBytes) /
                  (2 * (kATileBytes + kNarrowCols * kRowBytes)) >= kGatherWarps / 2, "narrow tiles gather in that many turns");
    t->recv_off = int(t->stages * stage);
    t->turn_off = int(t->recv_off + recv);
    t->table_off = int(t->turn_off + turn);
    t->bar_off = int(t->table_off + table);
    const long long most = (long long)t->n_tiles * (p.total / t->tn + busy);         // no distribution needs more
    const int sharing = *pair ? 2 : t->cluster;
    return int(std::min<long long>(sm_count / sharing, most)) * sharing;
}

template <int KIND, int LOADS, bool PAIR, bool GATED>
cudaError_t run(const GroupedParams &p, const MmGeom &t, int ctas, const CUtensorMap &map_w, const CUtensorMap &map_x, cudaStream_t stream) {
    const auto kernel = expert_mm_kernel<KIND, LOADS, PAIR, GATED>;
    static std::atomic<uint64_t> prepared{0};                // devices (of the first 64) that know the kernel's shared memory
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return err;
    const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
    if (!(prepared.load(std::memory_order_relaxed) & bit)) {
        err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmemLimit - kStaticBytes));
        if (err != cudaSuccess) return err;
        prepared.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(unsigned(ctas));
    config.blockDim = dim3(threads_of(KIND, LOADS));
    config.dynamicSmemBytes = size_t(t.bar_off + kBarBytes + 1024);
    config.stream = stream;
    cudaLaunchAttribute attributes[2] = {};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // the set-up overlaps the end of the kernel before
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = unsigned(PAIR ? 2 : t.cluster);
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, kernel, map_w, map_x, p, t);
}

// SMs of the current device, asked once per device
cudaError_t sm_count_of_current(int *count) {
    static std::atomic<int> known[64];
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return err;
    *count = device < 64 ? known[device].load(std::memory_order_relaxed) : 0;
    if (*count > 0) return cudaSuccess;
    err = cudaDeviceGetAttribute(count, cudaDevAttrMultiProcessorCount, device);
    if (err == cudaSuccess && device < 64) known[device].store(*count, std::memory_order_relaxed);
    return err;
}

}  // namespace

void set_product_wait(int us) { g_wait_us.store(uint32_t(us), std::memory_order_relaxed); }

bool grouped_too_large(const GroupedParams &p) {
    return p.total > 0 && (long long)ceil_div(p.total, columns_for(p, kLoaderCols)) * ceil_div(p.channels, kTileM / 2) > kMaxGroupTiles;
}

cudaError_t launch_grouped(const GroupedParams &given, cudaStream_t stream) {
    int sm_count = 0;
    cudaError_t err = sm_count_of_current(&sm_count);
    if (err != cudaSuccess) return err;
    GroupedParams p = given;
    const int wide = p.gated ? 2 * p.channels : p.channels;
    // a stride that separates nothing may hold anything
    const int apart = (p.inner + 15) / 16 * 16;
    if (p.x_rows <= 1) p.x_stride = apart;
    if (wide == 1) p.w_stride = apart;
    MmGeom t = {};
    bool pair = false;
    bool tma = tma_able(p) && encode_fn();
    int ctas = choose(p, sm_count, tma, &t, &pair);
    alignas(64) CUtensorMap map_w = {}, map_x = {};
    if (tma) {
        if (!encode_weights(&map_w, p, t) || !encode_rows(&map_x, p, t)) {
            tma = false;                             // a shape that no tensor map describes
            ctas = choose(p, sm_count, tma, &t, &pair);
        }
    }
#define IOS_RUN(KIND, LOADS, PAIR)                                                                     \
    return p.gated ? run<KIND, LOADS, PAIR, true>(p, t, ctas, map_w, map_x, stream)                      \
                   : run<KIND, LOADS, PAIR, false>(p, t, ctas, map_w, map_x, stream)
    if (p.type == Elem::F32) {
        if (!tma) IOS_RUN(kX3, kRegs, false);
        if (p.rows) IOS_RUN(kX3, kGather, false);
        IOS_RUN(kX3, kTma, false);
    }
    if (p.type == Elem::S8) {
        if (!tma) IOS_RUN(kI8, kRegs, false);
        if (pair && p.rows) IOS_RUN(kI8, kGather, true);
        if (pair) IOS_RUN(kI8, kTma, true);
        if (p.rows) IOS_RUN(kI8, kGather, false);
        IOS_RUN(kI8, kTma, false);
    }
    if (!tma) IOS_RUN(kF16, kRegs, false);
    if (pair && p.rows) IOS_RUN(kF16, kGather, true);
    if (pair) IOS_RUN(kF16, kTma, true);
    if (p.rows) IOS_RUN(kF16, kGather, false);
    IOS_RUN(kF16, kTma, false);
#undef IOS_RUN
}

cudaError_t expert_mm_status(int device, cudaStream_t stream, int *code) {
    static thread_local unsigned seen[kMaxStatusDevices][kWaitCodes] = {};     // by this host thread
    unsigned now[kWaitCodes];
    cudaError_t err = cudaMemcpyFromSymbolAsync(now, g_expert_timeouts, sizeof now, 0, cudaMemcpyDeviceToHost, stream);
    if (err == cudaSuccess) err = cudaStreamSynchronize(stream);
    if (err != cudaSuccess) return err;
    *code = 0;
    for (int c = kWaitCodes - 1; c > 0; --c) {
        if (now[c] != seen[device][c]) *code = c;
        seen[device][c] = now[c];
    }
    return cudaSuccess;
}

}  // namespace ios
