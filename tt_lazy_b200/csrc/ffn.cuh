// ffn.cuh -- shared parts of the feed-forward operators (norm.cu, linear.cu):
// element types, 8-element vector access, activations and their derivatives.
// The translation units that include it are compiled with multiply-add
// contraction on (their results are rounded once, to a stored type; nothing
// here is held to another implementation bit for bit).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "ttc_internal.cuh"

namespace ttc {

inline int dtype_size(int dtype) {
    return dtype == TTC_F32 ? 4 : dtype == TTC_F16 || dtype == TTC_BF16 ? 2 : dtype == TTC_E4M3 ? 1 : 0;
}
inline const char* dtype_name(int dtype) {
    return dtype == TTC_F32 ? "f32" : dtype == TTC_F16 ? "f16" : dtype == TTC_BF16 ? "bf16" : dtype == TTC_E4M3 ? "e4m3" : "?";
}

// The library launches on its own device whatever device the caller has
// current, and leaves the caller's device as it found it.
class DeviceGuard {
   public:
    DeviceGuard() {
        if (cudaGetDevice(&prev_) != cudaSuccess) prev_ = -1;
        if (prev_ != rt().device) cudaSetDevice(rt().device);
    }
    ~DeviceGuard() {
        if (prev_ >= 0 && prev_ != rt().device) cudaSetDevice(prev_);
    }

   private:
    int prev_ = -1;
};

// Checks of one tensor argument: set (or optional), aligned to its elements,
// rows that do not overlap. Status code, with the message in ttc_last_error().
inline int check_tensor(const char* op, const char* name, const void* p, int dtype, long long ld, long long width,
                        bool needed) {
    if (!p)
        return needed ? set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: %s is NULL", op, name) : TTC_OK;
    if ((uintptr_t)p % dtype_size(dtype))
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: %s (%p) is not aligned to its %d-byte elements", op,
                         name, p, dtype_size(dtype));
    if (ld < width)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: leading dimension %lld of %s is below its width %lld",
                         op, ld, name, width);
    return TTC_OK;
}

// Set-up that a kernel needs once on each device. Counts as done only where
// prepare() returned TTC_OK: after a failure the next call tries again.
class OncePerDevice {
   public:
    template <class F>
    int operator()(int device, F&& prepare) {
        if (done_[device]) return TTC_OK;
        if (int rc = prepare()) return rc;
        done_[device] = true;
        return TTC_OK;
    }

   private:
    bool done_[kMaxDevices] = {};
};

#ifdef __CUDACC__
#define TTC_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define TTC_HOST_DEVICE inline
#endif

// Copies on their way into a warp's buffers, each with an mbarrier of its own: a bit
// a buffer. One whose wait ran out stays on its way, and its barrier in the same
// phase, so that it is waited for once more before the kernel leaves.
struct CopiesInFlight {
    uint32_t phase = 0, pending = 0;
    TTC_HOST_DEVICE void sent(int buffer) { pending |= 1u << buffer; }
    TTC_HOST_DEVICE bool on_its_way(int buffer) const { return pending >> buffer & 1; }
    TTC_HOST_DEVICE uint32_t parity(int buffer) const { return phase >> buffer & 1; }
    TTC_HOST_DEVICE bool waited(int buffer, bool landed) {
        if (landed) {
            phase ^= 1u << buffer;
            pending &= ~(1u << buffer);
        }
        return landed;
    }
};

inline size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

// True when groups of 8 elements of `p` can be read with 16-byte accesses (two
// for fp32): address and row pitch on 16-byte boundaries.
inline bool vec8_ok(const void* p, int dtype, long long ld) {
    return p == nullptr || ((uintptr_t)p % 16 == 0 && (ld * dtype_size(dtype)) % 16 == 0);
}

int check_workspace(const char* op, const void* ws, size_t have, size_t need);
// out[c] = sum over b < n of partials[b][c], in a fixed order, stored as dtype.
int launch_sum_partials(const float* partials, int n, int cols, void* out, int dtype);

// ------------------------------------------------------------------ products
// One product C [M, N] = sum over `segs` segments of A_s [M, K] B_s [K, N], or
// (gated) the two products A B_0 and A B_1, with what happens to it on the way
// out. mn_major: stored with the M (A) or N (B) index contiguous.
struct Operand {
    const void* ptr;
    long long ld;
};
struct ProductEpilogue {
    void* out;
    void* out2;       // with split: the part of the output from `split` on
    long long ldo;
    int out_dtype;    // of out, bias, residual, pre
    int act;
    const void* bias;
    const void* residual;
    long long ldr;
    void* pre;        // linear: the value before the activation
    void* gate;       // gated: the two products
    void* up;
    long long ldp;    // of pre, gate and up
    const float* row_scales;
    const float* col_scales[2];
    int split_rows;   // > 0: rows from here on go to out2 ...
    int split_cols;   // (or columns, with > 0 here)
    int split_skip;   // ... after this many that go nowhere
    bool vec;         // every tensor here can be read and written 8 elements at a time
};
struct Product {
    int M, N, K;
    int dtype;  // of A and B
    int segs, gated;
    int a_mn, b_mn;
    Operand a[2], b[2];
    ProductEpilogue epi;
};
// Runs one product, or two of one 16-bit type that do not depend on one another, on
// the library stream. `scratch` (256-byte aligned) holds the padded copies of
// operands that cannot be read in place, of product_scratch() bytes.
int run_products(const Product* products, int count, void* scratch);
size_t product_scratch(const Product* products, int count);

// The attribute of a launch in clusters; returns the number of attributes (0 or 1).
inline int cluster_attribute(cudaLaunchAttribute& attr, int cluster) {
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)cluster;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    return cluster > 1;
}
// The attributes of a launch that may begin while the kernel before it in the
// stream still runs (the kernel calls grid_wait() before it touches memory), in
// clusters where `cluster` > 1.
inline int launch_attributes(cudaLaunchAttribute (&attr)[2], int cluster) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    return 1 + cluster_attribute(attr[1], cluster);
}

#ifdef __CUDACC__

// Launches a kernel that way, on the library stream.
template <class... Params, class... Args>
int launch_overlapped(void (*kernel)(Params...), dim3 grid, int block, int cluster, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)block);
    cfg.stream = rt().stream;
    cfg.attrs = attr;
    cfg.numAttrs = launch_attributes(attr, cluster);
    return check_cuda(cudaLaunchKernelEx(&cfg, kernel, args...), "kernel launch");
}

// Waits until the kernels before this one in the stream have finished and their
// writes are visible; lets the kernel after this one start to be launched.
// Kernels that begin with it read what those wrote with plain loads: the
// read-only path (__ldg) is for memory that nobody writes while a kernel runs, and
// the compiler may move its loads above the wait.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) {
    return __half2float(v);
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
    return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f32<__nv_fp8_e4m3>(__nv_fp8_e4m3 v) {
    return (float)v;
}
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __nv_fp8_e4m3 from_f32<__nv_fp8_e4m3>(float v) {
    return __nv_fp8_e4m3(v);  // nearest even, saturating at +-448, NaN stays NaN
}

// Eight 16-bit elements in four registers, as floats.
template <class T>
__device__ __forceinline__ void unpack8(const uint4& a, float (&v)[8]) {
    static_assert(sizeof(T) == 2, "16-bit elements");
    const T* e = reinterpret_cast<const T*>(&a);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(e[i]);
}

// Two values in one register, each rounded to nearest even.
template <class T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// Eight consecutive elements; n < 8 or `vec` false takes them one by one
// (elements past n read as 0 and are not stored).
template <class T>
__device__ __forceinline__ void load8(const T* p, int n, bool vec, float (&v)[8]) {
    if (vec && n >= 8) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
            unpack8<T>(*reinterpret_cast<const uint4*>(p), v);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32<T>(p[i]) : 0.0f;
    }
}
template <class T>
__device__ __forceinline__ void store8(T* p, int n, bool vec, const float (&v)[8]) {
    if (vec && n >= 8) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            static_assert(sizeof(T) == 2, "8 elements are 16 or 32 bytes");
            *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                                                      pack2<T>(v[6], v[7]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = from_f32<T>(v[i]);
    }
}

// Activations in fp32, with the hardware's approximate 2^x and 1 / x (good to
// 2^-22). Each is z times a factor s in [0, 1] and is off by at most
// 2^-21 (1 + |ln s|) of its own value: s is an exponential of a rounded argument,
// and that of -80 is known to 80 roundings. So the tails keep their leading digits
// (f16 and bf16 results are the exact ones to within half a step and 2^-15), down to
// 2^-119, below which a result may come out as 0: the approximations flush what is
// below 2^-126.
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2E = 1.4426950408889634f;
__device__ __forceinline__ float sigmoid_f32(float z) { return rcp_approx(1.0f + exp2_approx(-kLog2E * z)); }
// The normal distribution function at z, and e = e^(-z^2 / 2), which its density
// needs too. For x >= 0 the function at -x is e times a smooth decreasing factor
// (half the scaled complementary error function of x / sqrt(2)), here t P(t) with
// t = 1 / (1 + 0.305 x) and P of degree 7: fitted to that factor over 0 <= x <= 14
// (past 13.2 e is 0), minimising the greatest relative error by iterated reweighting
// (Lawson), 1e-7. Relative, since gelu's negative tail is this value itself: a form
// with a bounded absolute error (1.5e-7) was off by 5e-4 of it at -4 and 1e-2 at -8.
// Three multiply-adds more than that form, and half the instructions of erff with a
// separate exponential.
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    const float t = rcp_approx(fmaf(0.305f, fabsf(z), 1.0f));
    e = exp2_approx(-0.5f * kLog2E * z * z);
    float q = fmaf(t, 0.036699191f, -0.1529883f);
    q = fmaf(t, q, 0.18571687f);
    q = fmaf(t, q, -0.037976794f);
    q = fmaf(t, q, 0.12102166f);
    q = fmaf(t, q, 0.10342088f);
    q = fmaf(t, q, 0.1224668f);
    q = fmaf(t, q, 0.12163974f);
    q = t * q * e;
    return z < 0.0f ? q : 1.0f - q;
}
constexpr float kGeluTanhScale = 1.5957691216057308f;  // 2 sqrt(2 / pi): (1 + tanh t) / 2 = sigmoid(2 t)
__device__ __forceinline__ float activate(int act, float z) {
    switch (act) {
        case TTC_ACT_RELU: return z < 0.0f ? 0.0f : z;
        case TTC_ACT_SILU: return z * sigmoid_f32(z);
        case TTC_ACT_GELU: {
            float e;
            return z * normal_cdf(z, e);
        }
        case TTC_ACT_GELU_TANH: return z * sigmoid_f32(kGeluTanhScale * (z + 0.044715f * z * z * z));
        default: return z;
    }
}
// n values, with the choice of activation outside the loop.
template <int N>
__device__ __forceinline__ void activate_all(int act, float (&v)[N]) {
    auto all = [&](auto one) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = one(v[i]);
    };
    switch (act) {
        case TTC_ACT_RELU: all([](float z) { return activate(TTC_ACT_RELU, z); }); break;
        case TTC_ACT_SILU: all([](float z) { return activate(TTC_ACT_SILU, z); }); break;
        case TTC_ACT_GELU: all([](float z) { return activate(TTC_ACT_GELU, z); }); break;
        case TTC_ACT_GELU_TANH: all([](float z) { return activate(TTC_ACT_GELU_TANH, z); }); break;
        default: break;
    }
}
// The activation and its derivative.
__device__ __forceinline__ void activate_grad(int act, float z, float& a, float& da) {
    switch (act) {
        case TTC_ACT_RELU:
            a = z < 0.0f ? 0.0f : z;
            da = z > 0.0f ? 1.0f : 0.0f;
            break;
        case TTC_ACT_SILU: {
            const float p = sigmoid_f32(z);
            a = z * p;
            da = p + a * (1.0f - p);
            break;
        }
        case TTC_ACT_GELU: {
            float e;
            const float cdf = normal_cdf(z, e);
            a = z * cdf;
            da = fmaf(z * 0.39894228040143268f, e, cdf);
            break;
        }
        case TTC_ACT_GELU_TANH: {
            const float p = sigmoid_f32(kGeluTanhScale * (z + 0.044715f * z * z * z));
            a = z * p;
            // p (1 - p) is 0 in fp32 long before |z| = 16; past that z^2 would
            // overflow and 0 * inf make a NaN of a slope that is 0 or 1.
            const float zc = fminf(fmaxf(z, -16.0f), 16.0f);
            da = p + zc * p * (1.0f - p) * kGeluTanhScale * (1.0f + 0.134145f * zc * zc);
            break;
        }
        default:
            a = z;
            da = 1.0f;
    }
}

// The epilogue for tensors that nothing wider than an element can reach: eight
// rows (row, row + step, ...; the first `count` exist) of one column, whose scales
// and bias are given, a lane of a warp each of 32 neighbouring columns. Eight at a
// time so that the residual's loads are on their way together and a row's address
// takes one addition: 5000 x 4097 e4m3 results 179 us, 209 with a multiplication a
// row, 460 with one row after the other. Bound by the instructions of eight warps an
// SM (64 a row of 32 before the addresses were shared); the next rows' residual
// ahead of these rows' results took 189.
template <int DT>
struct Element {
    using T = typename std::conditional<DT == TTC_F32, float,
                                        typename std::conditional<DT == TTC_BF16, __nv_bfloat16, __half>::type>::type;
    static __device__ __forceinline__ float load(const void* base, long long i) {
        return to_f32<T>(static_cast<const T*>(base)[i]);
    }
    static __device__ __forceinline__ void store(void* base, long long i, float v) {
        static_cast<T*>(base)[i] = from_f32<T>(v);
    }
};
template <int DT, bool GATED>
__device__ __forceinline__ void finish_column(const ProductEpilogue& e, int row, int step, int count, int col,
                                              float (&v)[8], float (&u)[8], float s0, float s1, float bias) {
    using E = Element<DT>;
    // f(i, index): the rows' indices into a matrix of pitch ld, from one multiplication
    auto each = [&](long long ld, int first, int column, auto f) {
        long long at = first * ld + column;
        const long long down = step * ld;
#pragma unroll
        for (int i = 0; i < 8; ++i, at += down)
            if (i < count) f(i, at);
    };
    float res[8];
    if (!GATED && e.residual) each(e.ldr, row, col, [&](int i, long long at) { res[i] = E::load(e.residual, at); });
    if (e.row_scales)
        each(1, row, 0, [&](int i, long long at) {
            const float rs = e.row_scales[at];
            v[i] *= rs * s0;
            if (GATED) u[i] *= rs * s1;
        });
    if (GATED) {
        if (e.gate)
            each(e.ldp, row, col, [&](int i, long long at) {
                E::store(e.gate, at, v[i]);
                E::store(e.up, at, u[i]);
            });
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += bias;
        if (e.pre) each(e.ldp, row, col, [&](int i, long long at) { E::store(e.pre, at, v[i]); });
    }
    activate_all<8>(e.act, v);
    if (GATED) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= u[i];
    } else if (e.residual) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += res[i];
    }
    if (e.split_rows > 0) {
        each(1, row, 0, [&](int i, long long r) {
            const long long second = r - e.split_rows - e.split_skip;
            if (r < e.split_rows)
                E::store(e.out, r * e.ldo + col, v[i]);
            else if (second >= 0)
                E::store(e.out2, second * e.ldo + col, v[i]);
        });
        return;
    }
    void* out = e.out;
    if (e.split_cols > 0 && col >= e.split_cols) {
        col -= e.split_cols + e.split_skip;
        if (col < 0) return;
        out = e.out2;
    }
    each(e.ldo, row, col, [&](int i, long long at) { E::store(out, at, v[i]); });
}
__device__ __forceinline__ float bias_at(const ProductEpilogue& e, int col) {
    if (!e.bias) return 0.0f;
    return e.out_dtype == TTC_BF16  ? Element<TTC_BF16>::load(e.bias, col)
           : e.out_dtype == TTC_F16 ? Element<TTC_F16>::load(e.bias, col)
                                    : Element<TTC_F32>::load(e.bias, col);
}
#endif  // __CUDACC__

}  // namespace ttc
