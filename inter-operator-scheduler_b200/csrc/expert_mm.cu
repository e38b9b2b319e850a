// Matrix products over ragged groups of rows: y[r, :] = act(x[src(r), :] w[g]^T ...) for the rows r of group g.
//
// A 64 x 64 output tile per block, operands staged in shared memory, float (8-bit: int) sums in registers.  The group
// sizes are only known on the device, so the grid covers the most tiles any distribution of the rows can need and
// every block finds its own tile from the offsets.
#include "expert_ops.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ios {
namespace {

constexpr int kTile = 64, kStep = 16, kThreads = 256;

template <class T> struct Arith { using Sum = float; };
template <> struct Arith<signed char> { using Sum = int; };
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ int widen(signed char v) { return v; }

__device__ __forceinline__ float apply_act(float v, int act) {
    switch (act) {
        case 1: return fmaxf(v, 0.0f);
        case 2: return 1.0f / (1.0f + __expf(-v));
        case 3: return tanhf(v);
        case 4: return v / (1.0f + __expf(-v));
        default: return v;
    }
}

// offsets come from the device: whatever they hold, a group stays inside [0, total]
__device__ __forceinline__ void group_rows(const GroupedParams &p, int g, int *begin, int *end) {
    if (!p.offsets) { *begin = 0; *end = p.total; return; }
    *begin = min(max(p.offsets[g], 0), p.total);
    *end = min(max(p.offsets[g + 1], *begin), p.total);
}

template <class T>
__global__ void __launch_bounds__(kThreads) grouped_kernel(const GroupedParams p) {
    using Sum = typename Arith<T>::Sum;
    __shared__ Sum xs[kStep][kTile + 4], ws[2][kStep][kTile + 4];
    int tile = blockIdx.x, g = 0, begin = 0, end = 0;
    for (;; ++g) {
        if (g == p.groups) return;
        group_rows(p, g, &begin, &end);
        const int tiles = (end - begin + kTile - 1) / kTile;
        if (tile < tiles) break;
        tile -= tiles;
    }
    const int row0 = begin + tile * kTile, n0 = blockIdx.y * kTile;
    const int halves = p.gated ? 2 : 1;
    const T *w = static_cast<const T *>(p.w) + (long long)g * p.w_group_stride;
    const int tr = threadIdx.x / 16 * 4, tc = threadIdx.x % 16 * 4;
    Sum acc[2][4][4] = {};
    for (int k0 = 0; k0 < p.inner; k0 += kStep) {
        for (int i = threadIdx.x; i < kTile * kStep; i += kThreads) {
            const int r = i / kStep, k = i % kStep;
            Sum v = 0;
            if (row0 + r < end && k0 + k < p.inner) {
                const long long src = p.rows ? p.rows[row0 + r] : row0 + r;
                if (src >= 0 && src < p.x_rows) v = widen(static_cast<const T *>(p.x)[src * p.x_stride + k0 + k]);
            }
            xs[k][r] = v;
            for (int h = 0; h < halves; ++h) {
                Sum u = 0;
                if (n0 + r < p.channels && k0 + k < p.inner)
                    u = widen(w[((long long)h * p.channels + n0 + r) * p.w_stride + k0 + k]);
                ws[h][k][r] = u;
            }
        }
        __syncthreads();
        for (int k = 0; k < kStep; ++k)
            for (int h = 0; h < halves; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[h][i][j] += xs[k][tr + i] * ws[h][k][tc + j];
        __syncthreads();
    }
    const int per_group = halves * p.channels;
    for (int i = 0; i < 4; ++i) {
        const int r = row0 + tr + i;
        if (r >= end) continue;
        const long long src = p.rows ? p.rows[r] : r;
        const float rs = p.row_scale && src >= 0 && src < p.x_rows ? p.row_scale[src] : 1.0f;
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + tc + j;
            if (n >= p.channels) continue;
            float v[2] = {0.0f, 1.0f};
            for (int h = 0; h < halves; ++h) {
                const long long at = (long long)g * per_group + h * p.channels + n;
                v[h] = float(acc[h][i][j]) * rs;
                if (p.channel_scale) v[h] *= p.channel_scale[at];
                if (p.bias) v[h] += p.bias[at];
            }
            const float out = apply_act(v[0], p.act) * v[1];
            const long long at = (long long)r * p.y_stride + n;
            if (p.out_type == Elem::F32) static_cast<float *>(p.y)[at] = out;
            else if (p.out_type == Elem::F16) static_cast<__half *>(p.y)[at] = __float2half_rn(out);
            else static_cast<__nv_bfloat16 *>(p.y)[at] = __float2bfloat16_rn(out);
        }
    }
}

}  // namespace

cudaError_t launch_grouped(const GroupedParams &p, cudaStream_t stream) {
    const long long tiles = (p.total + kTile - 1) / kTile + (p.offsets ? p.groups : 0);
    const dim3 grid(unsigned(tiles), unsigned((p.channels + kTile - 1) / kTile));
    switch (p.type) {
        case Elem::F32: grouped_kernel<float><<<grid, kThreads, 0, stream>>>(p); break;
        case Elem::F16: grouped_kernel<__half><<<grid, kThreads, 0, stream>>>(p); break;
        case Elem::BF16: grouped_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p); break;
        case Elem::S8: grouped_kernel<signed char><<<grid, kThreads, 0, stream>>>(p); break;
    }
    return cudaGetLastError();
}

}  // namespace ios
