// Operators of a mixture-of-experts layer on device tensors: parameter blocks and host launchers.
//
// They work on plain row-major matrices that the caller owns (device pointers, a row stride in elements, unit column
// stride) instead of a plan's NHWC arena: a matrix row is a token's vector, the same thing as an NHWC pixel.
#pragma once
#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>

namespace ios {

// element types at this boundary; the values are those of IOS_F32 .. IOS_S8 in ios_runtime.h
enum class Elem : int { F32 = 0, F16 = 1, BF16 = 2, S8 = 3 };
__host__ __device__ constexpr int elem_size(Elem t) { return t == Elem::F32 ? 4 : t == Elem::S8 ? 1 : 2; }

constexpr int kMaxExperts = 1024;    // experts of a router / groups of a ragged product
constexpr int kMaxChosen = 32;       // experts per token

struct RouteParams {
    const void *logits;
    Elem type;
    int tokens, experts, k;
    long long stride;       // elements between the logits of consecutive tokens
    int renormalize;        // 1: the gates of a token sum to one; 0: softmax over all its experts
    int *chosen;            // [tokens][k]
    float *gates;           // [tokens][k]
    int *offsets;           // [experts + 1]
    int *rows;              // [tokens * k]
    int *slots;             // [tokens][k]
    int *block_counts;      // workspace, [blocks][experts], long calls: and their sums; unused when one block does everything
};
size_t route_workspace_bytes(int tokens, int experts, int k);
cudaError_t launch_route(const RouteParams &p, cudaStream_t stream);

struct QuantizeParams {
    const void *x;
    Elem type;
    long long x_rows, x_stride;
    int inner;
    const int *rows;        // source row of every output row, or null: row i of x
    long long total;        // output rows
    signed char *q;
    long long q_stride;
    float *scale;           // [total]
};
cudaError_t launch_quantize(const QuantizeParams &p, cudaStream_t stream);

struct CombineParams {
    const void *y;
    Elem type;
    long long y_rows, y_stride;
    const float *gates;     // [tokens][k]
    const int *slots;       // [tokens][k], outside [0, y_rows): no row
    long long tokens;
    int k, channels;
    void *out;
    Elem out_type;
    long long out_stride;
};
cudaError_t launch_combine(const CombineParams &p, cudaStream_t stream);

// y[r, n] = act(row_scale * channel_scale[g, n] * sum_k x[src(r), k] w[g, n, k] + bias[g, n]) for the rows r of group g;
// gated: w, channel_scale and bias have 2 * channels rows per group, y = act(first half) * second half.
struct GroupedParams {
    const void *x, *w;
    Elem type;
    long long x_rows, x_stride;
    long long w_stride, w_group_stride;
    int groups, channels, inner;
    const int *offsets;          // [groups + 1] on the device, or null: one group of all rows
    const int *rows;             // source row of every output row, or null: row r of x
    int total;                   // rows of y that offsets may name
    const float *row_scale;      // [x_rows] or null
    const float *channel_scale;  // [groups][channels or 2 * channels] or null
    const float *bias;           // likewise or null
    int act;                     // 0 identity, 1 relu, 2 sigmoid, 3 tanh, 4 silu
    int gated;
    void *y;
    Elem out_type;
    long long y_stride;
};
cudaError_t launch_grouped(const GroupedParams &p, cudaStream_t stream);
// more tiles than the kernel's table counts
bool grouped_too_large(const GroupedParams &p);
// Testing aid: what a wait inside a product may take, in microseconds (at most 2 seconds); 0: the default, 2 seconds.
void set_product_wait(int us);
// Waits for the stream; *code: a wait that ran out in a product on the current device, `device`, since this host thread's last call
// (its first: since the library was loaded), 0 for none.
constexpr int kMaxStatusDevices = 64;
cudaError_t expert_mm_status(int device, cudaStream_t stream, int *code);

}  // namespace ios
