// C entry points of the operators on device tensors (the expert layer and its 8-bit products).
//
// Every call checks its arguments, switches to the device that owns its output for the duration of the call, enqueues
// its kernels on the caller's stream and returns without waiting.  Nothing is allocated and nothing is kept between
// calls, so calls may overlap on any streams and may be captured into graphs.
#include <cuda_runtime.h>

#include <cstdarg>
#include <climits>
#include <cstdio>

#include "../../include/ios_runtime.h"
#include "expert_ops.h"

namespace ios {
void record_error(const char *message);

namespace {

int fail(int status, const char *format, ...) {
    char text[240];
    va_list args;
    va_start(args, format);
    std::vsnprintf(text, sizeof text, format, args);
    va_end(args);
    record_error(text);
    return status;
}

constexpr int kMaxRows = 1 << 30;       // row numbers and what is added to them stay inside an int
// Elements of a 16-bit product.  Its sums are waited for once, at the end of the rows: that many at odd addresses take 0.7 s of the 2
// that a wait may take, four times as many ran out of time (float32 waits at every step, 8-bit rows are shorter).
constexpr int kMaxInner16 = 1 << 25;

bool float_type(int t) { return t == IOS_F32 || t == IOS_F16 || t == IOS_BF16; }

// Makes the device that owns `out` current until the end of the call.
class DeviceScope {
public:
    ~DeviceScope() {
        if (previous_ >= 0) cudaSetDevice(previous_);
    }
    int enter(const void *out) {
        int current = 0;
        if (cudaError_t err = cudaGetDevice(&current)) return cuda("cudaGetDevice", err);
        if (int status = locate(out, "the output", &device_)) return status;
        if (device_ != current) {
            if (cudaError_t err = cudaSetDevice(device_)) return cuda("cudaSetDevice", err);
            previous_ = current;
        }
        return IOS_OK;
    }
    // `memory` must live on the same device (NULL passes: an optional argument)
    int same(const void *memory, const char *what) const {
        int device = 0;
        if (!memory) return IOS_OK;
        if (int status = locate(memory, what, &device)) return status;
        if (device != device_) return fail(IOS_ERR_ARGUMENT, "%s is on device %d, the output on device %d", what, device, device_);
        return IOS_OK;
    }
    static int cuda(const char *what, cudaError_t err) {
        cudaGetLastError();
        return fail(IOS_ERR_CUDA, "%s failed: %s", what, cudaGetErrorString(err));
    }

private:
    static int locate(const void *memory, const char *what, int *device) {
        cudaPointerAttributes attributes;
        if (cudaError_t err = cudaPointerGetAttributes(&attributes, memory)) return cuda("cudaPointerGetAttributes", err);
        if (attributes.type != cudaMemoryTypeDevice && attributes.type != cudaMemoryTypeManaged)
            return fail(IOS_ERR_ARGUMENT, "%s is not in device memory", what);
        *device = attributes.device;
        return IOS_OK;
    }
    int device_ = 0, previous_ = -1;
};

int finish(const char *what, cudaError_t err) {
    if (err != cudaSuccess) return DeviceScope::cuda(what, err);
    record_error("");
    return IOS_OK;
}

int check_grouped(const GroupedParams &p, const char *what) {
    if (p.act < 0 || p.act > 4) return fail(IOS_ERR_ARGUMENT, "%s: act must be 0..4", what);
    if (p.channels <= 0 || p.inner <= 0 || p.total < 0 || p.x_rows < 0)
        return fail(IOS_ERR_ARGUMENT, "%s: channels and inner must be positive, row counts not negative", what);
    if (p.channels > INT_MAX / 4) return fail(IOS_ERR_LIMIT, "%s: too many channels", what);
    if (p.groups <= 0 || p.groups > kMaxExperts) return fail(IOS_ERR_LIMIT, "%s: 1..%d groups, not %d", what, kMaxExperts, p.groups);
    if (p.x_stride < 0 || p.w_stride < 0 || p.w_group_stride < 0) return fail(IOS_ERR_ARGUMENT, "%s: negative stride", what);
    if (p.y_stride < p.channels) return fail(IOS_ERR_ARGUMENT, "%s: rows of y overlap (stride %lld, %d channels)", what, p.y_stride, p.channels);
    if (p.type == Elem::S8 && p.inner >= 131072)
        return fail(IOS_ERR_LIMIT, "%s: 8-bit products of 131072 or more elements can pass the 32 bits of their sum", what);
    if (elem_size(p.type) == 2 && p.inner > kMaxInner16) return fail(IOS_ERR_LIMIT, "%s: 16-bit products of more than 2^25 elements take too long for one wait", what);
    if (p.total > kMaxRows || grouped_too_large(p)) return fail(IOS_ERR_LIMIT, "%s: %d rows of %d channels are too many for one call", what, p.total, p.channels);
    if (!p.rows && p.x_rows < p.total) return fail(IOS_ERR_ARGUMENT, "%s: x has %lld rows, y %d", what, p.x_rows, p.total);
    return IOS_OK;
}

int check_route_limits(int tokens, int experts, int k) {
    if (experts > kMaxExperts || k > kMaxChosen)
        return fail(IOS_ERR_LIMIT, "route_experts: at most %d experts and %d of them per token", kMaxExperts, kMaxChosen);
    if ((long long)tokens * k > kMaxRows) return fail(IOS_ERR_LIMIT, "route_experts: more than 2^30 pairs");
    return IOS_OK;
}

int run_grouped(const GroupedParams &p, const char *what, void *stream) {
    if (int status = check_grouped(p, what)) return status;
    if (p.total == 0) {
        record_error("");
        return IOS_OK;
    }
    if ((!p.x && p.x_rows > 0) || !p.w || !p.y) return fail(IOS_ERR_ARGUMENT, "%s: x, w and y must not be NULL", what);
    DeviceScope scope;
    if (int status = scope.enter(p.y)) return status;
    if (int status = scope.same(p.x, "x")) return status;
    if (int status = scope.same(p.w, "w")) return status;
    if (int status = scope.same(p.offsets, "offsets")) return status;
    if (int status = scope.same(p.rows, "rows")) return status;
    if (int status = scope.same(p.row_scale, "row_scale")) return status;
    if (int status = scope.same(p.channel_scale, "channel_scale")) return status;
    if (int status = scope.same(p.bias, "bias")) return status;
    return finish(what, launch_grouped(p, static_cast<cudaStream_t>(stream)));
}

}  // namespace
}  // namespace ios

using namespace ios;

extern "C" int ios_route_experts_workspace(int tokens, int experts, int k, size_t *bytes) {
    if (!bytes || tokens < 0 || experts <= 0 || k <= 0 || k > experts)
        return fail(IOS_ERR_ARGUMENT, "route_experts_workspace: bytes must not be NULL, tokens >= 0 and 1 <= k <= experts are needed");
    if (int status = check_route_limits(tokens, experts, k)) return status;
    *bytes = tokens == 0 ? 0 : route_workspace_bytes(tokens, experts, k);
    record_error("");
    return IOS_OK;
}

extern "C" int ios_route_experts(const void *logits, int type, int tokens, int experts, long long stride, int k,
                                 int renormalize, int *chosen, float *gates, int *offsets, int *rows, int *slots,
                                 void *workspace, size_t workspace_bytes, void *cuda_stream) {
    if (!float_type(type)) return fail(IOS_ERR_ARGUMENT, "route_experts: logits must be float32, float16 or bfloat16");
    if (tokens < 0 || experts <= 0 || k <= 0 || k > experts || stride < 0)
        return fail(IOS_ERR_ARGUMENT, "route_experts: tokens >= 0, 1 <= k <= experts and stride >= 0 are needed");
    if (int status = check_route_limits(tokens, experts, k)) return status;
    if (!offsets || (tokens > 0 && (!logits || !chosen || !gates || !rows || !slots)))
        return fail(IOS_ERR_ARGUMENT, "route_experts: logits and the outputs must not be NULL");
    const size_t need = tokens == 0 ? 0 : route_workspace_bytes(tokens, experts, k);
    if (workspace_bytes < need || (need > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 3))))
        return fail(IOS_ERR_ARGUMENT, "route_experts: needs %zu bytes of 4-byte aligned workspace", need);
    DeviceScope scope;
    if (int status = scope.enter(offsets)) return status;
    if (tokens == 0)
        return finish("route_experts", cudaMemsetAsync(offsets, 0, size_t(experts + 1) * sizeof(int), static_cast<cudaStream_t>(cuda_stream)));
    if (int status = scope.same(logits, "logits")) return status;
    if (int status = scope.same(chosen, "chosen")) return status;
    if (int status = scope.same(gates, "gates")) return status;
    if (int status = scope.same(rows, "rows")) return status;
    if (int status = scope.same(slots, "slots")) return status;
    if (need > 0)
        if (int status = scope.same(workspace, "the workspace")) return status;
    RouteParams p = {};
    p.logits = logits;
    p.type = Elem(type);
    p.tokens = tokens;
    p.experts = experts;
    p.k = k;
    p.stride = stride;
    p.renormalize = renormalize != 0;
    p.chosen = chosen;
    p.gates = gates;
    p.offsets = offsets;
    p.rows = rows;
    p.slots = slots;
    p.block_counts = static_cast<int *>(workspace);
    return finish("route_experts", launch_route(p, static_cast<cudaStream_t>(cuda_stream)));
}

extern "C" int ios_grouped_matmul(const void *x, int type, long long x_rows, long long x_stride, const void *w, int groups,
                                  int channels, int inner, long long w_stride, long long w_group_stride, const int *offsets,
                                  const int *rows, int total_rows, const float *row_scale, const float *channel_scale,
                                  const float *bias, int act, int gated, void *y, int y_type, long long y_stride,
                                  void *cuda_stream) {
    if ((!float_type(type) && type != IOS_S8) || !float_type(y_type))
        return fail(IOS_ERR_ARGUMENT, "grouped_matmul: x is float32, float16, bfloat16 or int8, y one of the first three");
    if (!offsets && total_rows > 0) return fail(IOS_ERR_ARGUMENT, "grouped_matmul: offsets must not be NULL");
    GroupedParams p = {};
    p.x = x;
    p.w = w;
    p.type = Elem(type);
    p.x_rows = x_rows;
    p.x_stride = x_stride;
    p.w_stride = w_stride;
    p.w_group_stride = w_group_stride;
    p.groups = groups;
    p.channels = channels;
    p.inner = inner;
    p.offsets = offsets;
    p.rows = rows;
    p.total = total_rows;
    p.row_scale = row_scale;
    p.channel_scale = channel_scale;
    p.bias = bias;
    p.act = act;
    p.gated = gated != 0;
    p.y = y;
    p.out_type = Elem(y_type);
    p.y_stride = y_stride;
    return run_grouped(p, "grouped_matmul", cuda_stream);
}

extern "C" int ios_matmul_int8(const signed char *a, long long a_stride, const signed char *b, long long b_stride, int rows,
                               int channels, int inner, const float *row_scale, const float *channel_scale,
                               const float *bias, int act, void *y, int y_type, long long y_stride, void *cuda_stream) {
    if (!float_type(y_type)) return fail(IOS_ERR_ARGUMENT, "matmul_int8: y must be float32, float16 or bfloat16");
    GroupedParams p = {};
    p.x = a;
    p.w = b;
    p.type = Elem::S8;
    p.x_rows = rows;
    p.x_stride = a_stride;
    p.w_stride = b_stride;
    p.groups = 1;
    p.channels = channels;
    p.inner = inner;
    p.total = rows;
    p.row_scale = row_scale;
    p.channel_scale = channel_scale;
    p.bias = bias;
    p.act = act;
    p.y = y;
    p.out_type = Elem(y_type);
    p.y_stride = y_stride;
    return run_grouped(p, "matmul_int8", cuda_stream);
}

extern "C" int ios_quantize_rows(const void *x, int type, long long x_rows, long long x_stride, int inner, const int *rows,
                                 long long total_rows, signed char *q, long long q_stride, float *scale, void *cuda_stream) {
    if (!float_type(type)) return fail(IOS_ERR_ARGUMENT, "quantize_rows: x must be float32, float16 or bfloat16");
    if (inner <= 0 || x_rows < 0 || total_rows < 0 || x_stride < 0 || q_stride < inner)
        return fail(IOS_ERR_ARGUMENT, "quantize_rows: inner > 0, row counts >= 0, x_stride >= 0, q_stride >= inner are needed");
    if (total_rows > kMaxRows) return fail(IOS_ERR_LIMIT, "quantize_rows: more than 2^30 rows");
    if (!rows && x_rows < total_rows) return fail(IOS_ERR_ARGUMENT, "quantize_rows: x has %lld rows, q %lld", x_rows, total_rows);
    if (total_rows == 0) {
        record_error("");
        return IOS_OK;
    }
    if ((!x && x_rows > 0) || !q || !scale) return fail(IOS_ERR_ARGUMENT, "quantize_rows: x, q and scale must not be NULL");
    DeviceScope scope;
    if (int status = scope.enter(q)) return status;
    if (int status = scope.same(x, "x")) return status;
    if (int status = scope.same(scale, "scale")) return status;
    if (int status = scope.same(rows, "rows")) return status;
    QuantizeParams p = {};
    p.x = x;
    p.type = Elem(type);
    p.x_rows = x_rows;
    p.x_stride = x_stride;
    p.inner = inner;
    p.rows = rows;
    p.total = total_rows;
    p.q = q;
    p.q_stride = q_stride;
    p.scale = scale;
    return finish("quantize_rows", launch_quantize(p, static_cast<cudaStream_t>(cuda_stream)));
}

extern "C" int ios_combine_experts(const void *y, int type, long long y_rows, long long y_stride, const float *gates,
                                   const int *slots, long long tokens, int k, int channels, void *out, int out_type,
                                   long long out_stride, void *cuda_stream) {
    if (!float_type(type) || !float_type(out_type))
        return fail(IOS_ERR_ARGUMENT, "combine_experts: y and out must be float32, float16 or bfloat16");
    if (k <= 0 || channels <= 0 || tokens < 0 || y_rows < 0 || y_stride < 0 || out_stride < channels)
        return fail(IOS_ERR_ARGUMENT, "combine_experts: k, channels > 0, tokens, y_rows, y_stride >= 0, out_stride >= channels are needed");
    if (tokens > kMaxRows || channels > 1 << 23) return fail(IOS_ERR_LIMIT, "combine_experts: at most 2^30 tokens of 2^23 channels");
    if (tokens == 0) {
        record_error("");
        return IOS_OK;
    }
    if ((!y && y_rows > 0) || !gates || !slots || !out)
        return fail(IOS_ERR_ARGUMENT, "combine_experts: y, gates, slots and out must not be NULL");
    DeviceScope scope;
    if (int status = scope.enter(out)) return status;
    if (y_rows > 0)
        if (int status = scope.same(y, "y")) return status;
    if (int status = scope.same(gates, "gates")) return status;
    if (int status = scope.same(slots, "slots")) return status;
    CombineParams p = {};
    p.y = y;
    p.type = Elem(type);
    p.y_rows = y_rows;
    p.y_stride = y_stride;
    p.gates = gates;
    p.slots = slots;
    p.tokens = tokens;
    p.k = k;
    p.channels = channels;
    p.out = out;
    p.out_type = Elem(out_type);
    p.out_stride = out_stride;
    return finish("combine_experts", launch_combine(p, static_cast<cudaStream_t>(cuda_stream)));
}

extern "C" int ios_device_ops_status(int device, void *cuda_stream) {
    int current = 0, code = 0;
    if (device < 0 || device >= kMaxStatusDevices)
        return fail(IOS_ERR_ARGUMENT, "device_ops_status: device must be 0..%d", kMaxStatusDevices - 1);
    if (cudaError_t err = cudaGetDevice(&current)) return DeviceScope::cuda("cudaGetDevice", err);
    if (cudaError_t err = cudaSetDevice(device)) return DeviceScope::cuda("cudaSetDevice", err);
    const cudaError_t err = expert_mm_status(device, static_cast<cudaStream_t>(cuda_stream), &code);
    cudaSetDevice(current);
    if (err != cudaSuccess) return DeviceScope::cuda("reading the time-out counts", err);
    if (code != 0) return fail(IOS_ERR_TIMEOUT, "a bounded wait inside a product ran out (code %d): its output is incomplete", code);
    record_error("");
    return IOS_OK;
}
