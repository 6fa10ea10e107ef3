// norm.cu -- root-mean-square norm with the residual's addition
// (ttc_rms_norm) and its gradients (ttc_rms_norm_backward).
#include <algorithm>

#include "ffn.cuh"

namespace ttc {
namespace {

constexpr int kThreads = 256;

struct NormParams {
    long long rows;
    int cols;
    float eps;
    const void *x, *residual, *weight;
    void *y, *hidden;
    float* scales;
    long long ldx, ldr, ldy, ldh;
    int weight_f32;
};

// Sum and maximum over the block, in a fixed order, to every thread.
__device__ __forceinline__ float2 block_sum_max(float s, float m) {
    __shared__ float2 part[kThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
    if (lane == 0) part[warp] = make_float2(s, m);
    __syncthreads();
    float2 t = part[0];
    for (int w = 1; w < kThreads / 32; ++w) {
        t.x += part[w].x;
        t.y = fmaxf(t.y, part[w].y);
    }
    return t;
}

constexpr float kMinScale = 1.17549435e-38f;  // 2^-126

template <class T>
__device__ __forceinline__ float weight_at(const NormParams& p, int c) {
    return p.weight_f32 ? static_cast<const float*>(p.weight)[c] : to_f32<T>(static_cast<const T*>(p.weight)[c]);
}

// One block per row, two passes over it.
template <class T, class Y>
__global__ void __launch_bounds__(kThreads) rms_norm_kernel(const __grid_constant__ NormParams p) {
    const long long r = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + r * p.ldx;
    const T* res = p.residual ? static_cast<const T*>(p.residual) + r * p.ldr : nullptr;
    float sum = 0.0f, top = 0.0f;
    for (int c = threadIdx.x; c < p.cols; c += kThreads) {
        float h = to_f32<T>(x[c]);
        if (res) h += to_f32<T>(res[c]);
        sum += h * h;
        top = fmaxf(top, fabsf(h * weight_at<T>(p, c)));
    }
    const float2 t = block_sum_max(sum, top);
    const float rstd = rsqrtf(t.x / (float)p.cols + p.eps);
    float inv = 1.0f;
    if (sizeof(Y) == 1) {
        const float scale = fmaxf(t.y * rstd * (1.0f / 448.0f), kMinScale);
        inv = 1.0f / scale;
        if (threadIdx.x == 0) p.scales[r] = scale;
    }
    Y* y = static_cast<Y*>(p.y) + r * p.ldy;
    T* hid = p.hidden ? static_cast<T*>(p.hidden) + r * p.ldh : nullptr;
    for (int c = threadIdx.x; c < p.cols; c += kThreads) {
        float h = to_f32<T>(x[c]);
        if (res) h += to_f32<T>(res[c]);
        if (hid) hid[c] = from_f32<T>(h);
        y[c] = from_f32<Y>(h * rstd * weight_at<T>(p, c) * inv);
    }
}

struct NormBackwardParams {
    long long rows;
    int cols;
    float eps;
    const void *dy, *hidden, *weight, *dhidden;
    void* dx;
    float* partials;  // [gridDim.x, cols] sums of dy * hidden * rstd, or NULL
    long long lddy, ldh, lddh, lddx;
    int weight_f32;
};

// Block b takes rows b, b + gridDim.x, ...; a thread owns the same columns of
// every row, so its running weight gradients sit in the block's own row of
// the partials without atomics.
template <class T>
__global__ void __launch_bounds__(kThreads) rms_norm_backward_kernel(const __grid_constant__ NormBackwardParams p) {
    float* part = p.partials ? p.partials + (long long)blockIdx.x * p.cols : nullptr;
    if (part)
        for (int c = threadIdx.x; c < p.cols; c += kThreads) part[c] = 0.0f;
    auto weight = [&](int c) {
        return p.weight_f32 ? static_cast<const float*>(p.weight)[c] : to_f32<T>(static_cast<const T*>(p.weight)[c]);
    };
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* dy = static_cast<const T*>(p.dy) + r * p.lddy;
        const T* hid = static_cast<const T*>(p.hidden) + r * p.ldh;
        const T* dh = p.dhidden ? static_cast<const T*>(p.dhidden) + r * p.lddh : nullptr;
        T* dx = static_cast<T*>(p.dx) + r * p.lddx;
        float sum = 0.0f, dot = 0.0f;
        for (int c = threadIdx.x; c < p.cols; c += kThreads) {
            const float h = to_f32<T>(hid[c]);
            sum += h * h;
            dot += to_f32<T>(dy[c]) * weight(c) * h;
        }
        __shared__ float2 red[kThreads / 32];
        sum = warp_sum(sum);
        dot = warp_sum(dot);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(sum, dot);
        __syncthreads();
        sum = dot = 0.0f;
        for (int w = 0; w < kThreads / 32; ++w) {
            sum += red[w].x;
            dot += red[w].y;
        }
        const float rstd = rsqrtf(sum / (float)p.cols + p.eps);
        const float k = dot * rstd * rstd / (float)p.cols;
        for (int c = threadIdx.x; c < p.cols; c += kThreads) {
            const float h = to_f32<T>(hid[c]), g = to_f32<T>(dy[c]);
            float d = rstd * (g * weight(c) - h * k);
            if (dh) d += to_f32<T>(dh[c]);
            if (part) part[c] += g * h * rstd;
            dx[c] = from_f32<T>(d);
        }
    }
}

// out[c] = sum over b < n of partials[b][c], in order.
__global__ void __launch_bounds__(kThreads) sum_partials_kernel(const float* partials, int n, int cols, void* out,
                                                                int dtype) {
    const int c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= cols) return;
    float s = 0.0f;
    for (int b = 0; b < n; ++b) s += partials[(long long)b * cols + c];
    if (dtype == TTC_BF16)
        static_cast<__nv_bfloat16*>(out)[c] = from_f32<__nv_bfloat16>(s);
    else if (dtype == TTC_F16)
        static_cast<__half*>(out)[c] = from_f32<__half>(s);
    else
        static_cast<float*>(out)[c] = s;
}

int check_norm_types(const char* op, int dtype, int weight_dtype, long long rows, int cols, float eps) {
    if (rows < 0 || cols < 1)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: shape %lld x %d", op, rows, cols);
    if (rows > INT32_MAX)
        return set_error(TTC_ERR_UNSUPPORTED, "tt_cuda: %s: %lld rows exceed %d", op, rows, INT32_MAX);
    if (dtype != TTC_F32 && dtype != TTC_F16 && dtype != TTC_BF16)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: dtype %d is not F32, F16 or BF16", op, dtype);
    if (weight_dtype != dtype && weight_dtype != TTC_F32)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: weight_dtype %d is neither dtype (%s) nor F32", op,
                         weight_dtype, dtype_name(dtype));
    if (!(eps >= 0.0f)) return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: eps %g is not >= 0", op, eps);
    return TTC_OK;
}

int check_norm(const ttc_rms_norm_desc& d) {
    const char* op = "rms_norm";
    if (int rc = check_norm_types(op, d.dtype, d.weight_dtype, d.rows, d.cols, d.eps)) return rc;
    if (d.y_dtype != d.dtype && d.y_dtype != TTC_E4M3)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: y_dtype %d is neither dtype (%s) nor E4M3", op,
                         d.y_dtype, dtype_name(d.dtype));
    const bool any = d.rows > 0;
    if (int rc = check_tensor(op, "x", d.x, d.dtype, d.ldx, d.cols, any)) return rc;
    if (int rc = check_tensor(op, "residual", d.residual, d.dtype, d.ldr, d.cols, false)) return rc;
    if (int rc = check_tensor(op, "weight", d.weight, d.weight_dtype, d.cols, d.cols, any)) return rc;
    if (int rc = check_tensor(op, "y", d.y, d.y_dtype, d.ldy, d.cols, any)) return rc;
    if (int rc = check_tensor(op, "hidden", d.hidden, d.dtype, d.ldh, d.cols, false)) return rc;
    if (int rc = check_tensor(op, "scales", d.scales, TTC_F32, 1, 1, any && d.y_dtype == TTC_E4M3)) return rc;
    if (d.scales && d.y_dtype != TTC_E4M3)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: scales are written with y_dtype E4M3 only", op);
    return TTC_OK;
}

int check_norm_backward(const ttc_rms_norm_backward_desc& d) {
    const char* op = "rms_norm_backward";
    if (int rc = check_norm_types(op, d.dtype, d.weight_dtype, d.rows, d.cols, d.eps)) return rc;
    const bool any = d.rows > 0;
    if (int rc = check_tensor(op, "dy", d.dy, d.dtype, d.lddy, d.cols, any)) return rc;
    if (int rc = check_tensor(op, "hidden", d.hidden, d.dtype, d.ldh, d.cols, any)) return rc;
    if (int rc = check_tensor(op, "weight", d.weight, d.weight_dtype, d.cols, d.cols, any)) return rc;
    if (int rc = check_tensor(op, "dhidden", d.dhidden, d.dtype, d.lddh, d.cols, false)) return rc;
    if (int rc = check_tensor(op, "dx", d.dx, d.dtype, d.lddx, d.cols, any)) return rc;
    return check_tensor(op, "dweight", d.dweight, d.weight_dtype, d.cols, d.cols, false);
}

// Blocks of the backward kernel. Fixed by the shape alone, so that the
// workspace size needs no device and results are the same on every call.
int backward_blocks(long long rows) { return (int)std::min<long long>(rows, 148 * 4); }

size_t backward_bytes(const ttc_rms_norm_backward_desc& d) {
    return d.dweight ? align256((size_t)backward_blocks(d.rows) * d.cols * sizeof(float)) : 0;
}

template <class T>
void launch_norm(const NormParams& p, int y_dtype, cudaStream_t st) {
    if (y_dtype == TTC_E4M3)
        rms_norm_kernel<T, __nv_fp8_e4m3><<<(unsigned)p.rows, kThreads, 0, st>>>(p);
    else
        rms_norm_kernel<T, T><<<(unsigned)p.rows, kThreads, 0, st>>>(p);
}

}  // namespace

int check_workspace(const char* op, const void* ws, size_t have, size_t need) {
    if (need == 0) return TTC_OK;
    if (!ws || have < need)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: workspace of %zu bytes, %zu are needed", op,
                         ws ? have : (size_t)0, need);
    if ((uintptr_t)ws % 256)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: workspace (%p) is not 256-byte aligned", op, ws);
    return TTC_OK;
}

int launch_sum_partials(const float* partials, int n, int cols, void* out, int dtype, cudaStream_t st) {
    sum_partials_kernel<<<(cols + kThreads - 1) / kThreads, kThreads, 0, st>>>(partials, n, cols, out, dtype);
    count_launch();
    return check_cuda(cudaGetLastError(), "partial sums launch");
}

}  // namespace ttc

using namespace ttc;

extern "C" {

int ttc_rms_norm(const ttc_rms_norm_desc* desc) {
    if (!desc) return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: rms_norm: desc is NULL");
    const ttc_rms_norm_desc& d = *desc;
    if (int rc = check_norm(d)) return rc;
    TTC_REQUIRE_INIT();
    if (d.rows == 0) return TTC_OK;
    DeviceGuard guard;
    NormParams p{d.rows, d.cols,   d.eps, d.x,   d.residual, d.weight, d.y, d.hidden,
                 d.scales, d.ldx, d.ldr, d.ldy, d.ldh,      d.weight_dtype == TTC_F32};
    if (d.dtype == TTC_BF16)
        launch_norm<__nv_bfloat16>(p, d.y_dtype, rt().stream);
    else if (d.dtype == TTC_F16)
        launch_norm<__half>(p, d.y_dtype, rt().stream);
    else
        launch_norm<float>(p, d.y_dtype, rt().stream);
    count_launch();
    return check_cuda(cudaGetLastError(), "rms_norm launch");
}

int ttc_rms_norm_backward_workspace(const ttc_rms_norm_backward_desc* desc, size_t* bytes) {
    if (!desc || !bytes)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: rms_norm_backward_workspace: NULL argument");
    *bytes = 0;
    if (int rc = check_norm_backward(*desc)) return rc;
    *bytes = backward_bytes(*desc);
    return TTC_OK;
}

int ttc_rms_norm_backward(const ttc_rms_norm_backward_desc* desc) {
    if (!desc) return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: rms_norm_backward: desc is NULL");
    const ttc_rms_norm_backward_desc& d = *desc;
    if (int rc = check_norm_backward(d)) return rc;
    if (int rc = check_workspace("rms_norm_backward", d.workspace, d.workspace_bytes, backward_bytes(d))) return rc;
    TTC_REQUIRE_INIT();
    DeviceGuard guard;
    cudaStream_t st = rt().stream;
    if (d.rows == 0) {
        if (d.dweight) TTC_CUDA(cudaMemsetAsync(d.dweight, 0, (size_t)d.cols * dtype_size(d.weight_dtype), st));
        return TTC_OK;
    }
    const int blocks = backward_blocks(d.rows);
    NormBackwardParams p{d.rows, d.cols, d.eps,  d.dy,  d.hidden, d.weight, d.dhidden, d.dx,
                         d.dweight ? (float*)d.workspace : nullptr,
                         d.lddy, d.ldh,  d.lddh, d.lddx, d.weight_dtype == TTC_F32};
    if (d.dtype == TTC_BF16)
        rms_norm_backward_kernel<__nv_bfloat16><<<blocks, kThreads, 0, st>>>(p);
    else if (d.dtype == TTC_F16)
        rms_norm_backward_kernel<__half><<<blocks, kThreads, 0, st>>>(p);
    else
        rms_norm_backward_kernel<float><<<blocks, kThreads, 0, st>>>(p);
    count_launch();
    if (int rc = check_cuda(cudaGetLastError(), "rms_norm_backward launch")) return rc;
    return d.dweight ? launch_sum_partials(p.partials, blocks, d.cols, d.dweight, d.weight_dtype, st) : TTC_OK;
}

}  // extern "C"
