// linear.cu -- the products of a feed-forward block (ttc_linear,
// ttc_gated_linear) and their gradients: argument checks, the element-wise
// half of the backward passes, and the products each call is made of (the
// products themselves: linear_tc.cu).
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "ffn.cuh"
#include "tc_util.cuh"

namespace ttc {
namespace {

// ------------------------------------------------------------------- checks
// Keeps every tile count and padded width inside 32 bits; offsets are 64-bit.
constexpr int kMaxRows = 1 << 30, kMaxWidth = 1 << 23;

int check_product(const char* op, int M, int N, int K, int dtype, int trans_w, int act, bool backward) {
    if (M < 0 || N < 1 || K < 1)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: shape M %d, N %d, K %d", op, M, N, K);
    if (M > kMaxRows || N > kMaxWidth || K > kMaxWidth)
        return set_error(TTC_ERR_UNSUPPORTED, "tt_cuda: %s: M %d, N %d, K %d exceed %d rows, width %d", op, M, N, K,
                         kMaxRows, kMaxWidth);
    if (dtype == TTC_F32)
        return set_error(TTC_ERR_UNSUPPORTED, "tt_cuda: %s takes 16-bit and 8-bit operands; ttc_gemm has fp32 products",
                         op);
    if (dtype != TTC_F16 && dtype != TTC_BF16 && (dtype != TTC_E4M3 || backward))
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: dtype %d is not F16%s", op, dtype,
                         backward ? " or BF16" : ", BF16 or E4M3");
    if (trans_w != 0 && trans_w != 1)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: trans_w %d is not 0 or 1", op, trans_w);
    if (dtype == TTC_E4M3 && !trans_w)
        return set_error(TTC_ERR_UNSUPPORTED, "tt_cuda: %s: E4M3 weights are stored [N, K] (trans_w = 1)", op);
    if (act < TTC_ACT_NONE || act > TTC_ACT_GELU_TANH)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: unknown activation %d", op, act);
    return TTC_OK;
}

int check_out_type(const char* op, int dtype, int y_dtype) {
    const bool ok = dtype == TTC_E4M3 ? y_dtype == TTC_F16 || y_dtype == TTC_BF16 || y_dtype == TTC_F32
                                      : y_dtype == dtype || y_dtype == TTC_F32;
    if (!ok)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: y_dtype %s does not go with dtype %s", op,
                         dtype_name(y_dtype), dtype_name(dtype));
    return TTC_OK;
}

int check_scales(const char* op, const char* name, const float* s, int dtype, bool any) {
    if (dtype == TTC_E4M3) return check_tensor(op, name, s, TTC_F32, 1, 1, any);
    if (s) return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: %s go with E4M3 operands only", op, name);
    return TTC_OK;
}

int check_linear(const ttc_linear_desc& d) {
    const char* op = "linear";
    if (int rc = check_product(op, d.M, d.N, d.K, d.dtype, d.trans_w, d.act, false)) return rc;
    if (int rc = check_out_type(op, d.dtype, d.y_dtype)) return rc;
    const bool any = d.M > 0;
    if (int rc = check_tensor(op, "x", d.x, d.dtype, d.ldx, d.K, any)) return rc;
    if (int rc = check_tensor(op, "w", d.w, d.dtype, d.ldw, d.trans_w ? d.K : d.N, any)) return rc;
    if (int rc = check_tensor(op, "y", d.y, d.y_dtype, d.ldy, d.N, any)) return rc;
    if (int rc = check_tensor(op, "bias", d.bias, d.y_dtype, d.N, d.N, false)) return rc;
    if (int rc = check_tensor(op, "residual", d.residual, d.y_dtype, d.ldr, d.N, false)) return rc;
    if (int rc = check_tensor(op, "pre", d.pre, d.y_dtype, d.ldp, d.N, false)) return rc;
    if (int rc = check_scales(op, "x_scales", d.x_scales, d.dtype, any)) return rc;
    return check_scales(op, "w_scales", d.w_scales, d.dtype, any);
}

int check_gated(const ttc_gated_linear_desc& d) {
    const char* op = "gated_linear";
    if (int rc = check_product(op, d.M, d.N, d.K, d.dtype, d.trans_w, d.act, false)) return rc;
    if (int rc = check_out_type(op, d.dtype, d.y_dtype)) return rc;
    const bool any = d.M > 0;
    const long long wide = d.trans_w ? d.K : d.N;
    if (int rc = check_tensor(op, "x", d.x, d.dtype, d.ldx, d.K, any)) return rc;
    if (int rc = check_tensor(op, "wg", d.wg, d.dtype, d.ldw, wide, any)) return rc;
    if (int rc = check_tensor(op, "wu", d.wu, d.dtype, d.ldw, wide, any)) return rc;
    if (int rc = check_tensor(op, "y", d.y, d.y_dtype, d.ldy, d.N, any)) return rc;
    if (!d.gate != !d.up)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: gate and up are stored both or neither", op);
    if (int rc = check_tensor(op, "gate", d.gate, d.y_dtype, d.ldp, d.N, false)) return rc;
    if (int rc = check_tensor(op, "up", d.up, d.y_dtype, d.ldp, d.N, false)) return rc;
    if (int rc = check_scales(op, "x_scales", d.x_scales, d.dtype, any)) return rc;
    if (int rc = check_scales(op, "wg_scales", d.wg_scales, d.dtype, any)) return rc;
    return check_scales(op, "wu_scales", d.wu_scales, d.dtype, any);
}

int check_linear_backward(const ttc_linear_backward_desc& d) {
    const char* op = "linear_backward";
    if (int rc = check_product(op, d.M, d.N, d.K, d.dtype, d.trans_w, d.act, true)) return rc;
    const bool any = d.M > 0;
    const long long wide = d.trans_w ? d.K : d.N;
    if (int rc = check_tensor(op, "dy", d.dy, d.dtype, d.lddy, d.N, any)) return rc;
    if (int rc = check_tensor(op, "x", d.x, d.dtype, d.ldx, d.K, any && d.dw)) return rc;
    if (int rc = check_tensor(op, "w", d.w, d.dtype, d.ldw, wide, any && d.dx)) return rc;
    if (int rc = check_tensor(op, "pre", d.pre, d.dtype, d.ldp, d.N, any && d.act != TTC_ACT_NONE)) return rc;
    if (int rc = check_tensor(op, "dx", d.dx, d.dtype, d.lddx, d.K, false)) return rc;
    if (int rc = check_tensor(op, "dw", d.dw, d.dtype, d.lddw, wide, false)) return rc;
    return check_tensor(op, "dbias", d.dbias, d.dtype, d.N, d.N, false);
}

int check_gated_backward(const ttc_gated_linear_backward_desc& d) {
    const char* op = "gated_linear_backward";
    if (int rc = check_product(op, d.M, d.N, d.K, d.dtype, d.trans_w, d.act, true)) return rc;
    const bool any = d.M > 0;
    const long long wide = d.trans_w ? d.K : d.N;
    if (!d.dwg != !d.dwu)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: dwg and dwu are computed both or neither", op);
    if (int rc = check_tensor(op, "dy", d.dy, d.dtype, d.lddy, d.N, any)) return rc;
    if (int rc = check_tensor(op, "x", d.x, d.dtype, d.ldx, d.K, any && d.dwg)) return rc;
    if (int rc = check_tensor(op, "wg", d.wg, d.dtype, d.ldw, wide, any && d.dx)) return rc;
    if (int rc = check_tensor(op, "wu", d.wu, d.dtype, d.ldw, wide, any && d.dx)) return rc;
    if (int rc = check_tensor(op, "gate", d.gate, d.dtype, d.ldp, d.N, any)) return rc;
    if (int rc = check_tensor(op, "up", d.up, d.dtype, d.ldp, d.N, any)) return rc;
    if (int rc = check_tensor(op, "dx", d.dx, d.dtype, d.lddx, d.K, false)) return rc;
    if (int rc = check_tensor(op, "dwg", d.dwg, d.dtype, d.lddw, wide, false)) return rc;
    return check_tensor(op, "dwu", d.dwu, d.dtype, d.lddw, wide, false);
}

// ---------------------------------------- element-wise half of the backward
// A block of 8 warps walks a band of rows of a 256-column stripe: a lane owns
// 8 columns, a warp one row at a time, so that a column's sum for dbias stays
// in a register. Memory bound: each value is read once and written once, 16
// bytes per lane and access, a row's loads ahead of its arithmetic, as packed
// registers. In bf16, buffers in turn so that none is still in L2: 4096 x 8192 with
// gelu and dbias 40 us (5.0 TB/s), the gated pair with silu 56 us (6.0 TB/s); 8192 x
// 16384 with gelu 145 us (5.5 TB/s), the pair of 4096 x 16384 107 us (6.3 TB/s).
// Measured where these took 39 and 51: the row ahead as floats 72 and 88, without
// it 47 and 73.
//
// What the products read of dz (dg, du) is rounded to their 16-bit type: a tensor-core
// operand has no wider form of that speed. The column sums take the values before it.
constexpr int kStripe = 256, kBandWarps = 8;
// Rows of a block: 64, more when that would make over 256 bands of partial sums,
// and fewer, down to one a warp, while that leaves SMs without two blocks: a
// warp's rows come one after the other (what this kernel adds to a call with silu,
// 64 rows and then fewer: 128 x 4096 8.4 -> 3.7 us, 2461 x 663 12.3 -> 4.3).
// Bands of up to 32 rows that are at most a cluster are `joined`: the cluster adds
// up dbias itself. (With 64 rows that costs more than a second launch: 512 x 1024
// 10.3 us, 1000 x 1000 in bands of 8 rows 5.0.)
constexpr int kClusterBands = 8, kJoinedRows = 32;
struct Bands {
    int rows, n, stripes;
    bool joined;
};
Bands bands_of(int M, int N, bool dbias) {
    Bands b;
    b.stripes = (N + kStripe - 1) / kStripe;
    auto count = [&](int rows) { return (M + rows - 1) / rows; };
    b.joined = dbias && count(kJoinedRows) <= kClusterBands;
    b.rows = b.joined ? kJoinedRows : std::max(64, count(256));
    const int most = b.joined ? kClusterBands : 256;
    while (b.rows > kBandWarps && (long long)count(b.rows) * b.stripes < 2 * 148 && count(b.rows / 2) <= most) b.rows /= 2;
    b.n = count(b.rows);
    return b;
}

struct LinearGradParams {
    int M, N, band_rows;
    const void *dy, *pre;
    long long lddy, ldp;
    void* dz;  // or NULL: only the column sums
    long long lddz;
    float* partials;  // [bands, N] column sums of dz, or NULL
    void* dbias;      // [N], or NULL: the bands of a stripe are one cluster, which adds them up itself
    bool vec_dy, vec_pre, vec_dz;
};

// ACT at compile time: as a switch in the loop it took half as long again.
template <class T, int ACT>
__global__ void __launch_bounds__(32 * kBandWarps, 4) linear_grad_kernel(const __grid_constant__ LinearGradParams p) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col = blockIdx.y * kStripe + lane * 8, n = p.N - col;
    float sum[8] = {};
    grid_wait();
    grid_trigger();
    if (n > 0) {
        const long long r1 = min((long long)p.M, (blockIdx.x + 1ll) * p.band_rows);
        // whole aligned groups: the next row is on its way while this one is computed
        const bool ahead = p.vec_dy && n >= 8 && (ACT == TTC_ACT_NONE || p.vec_pre);
        uint4 gn = {}, zn = {};
        auto fetch = [&](long long r) {
            gn = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.dy) + r * p.lddy + col);
            if (ACT != TTC_ACT_NONE)
                zn = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.pre) + r * p.ldp + col);
        };
        long long r = (long long)blockIdx.x * p.band_rows + warp;
        if (ahead && r < r1) fetch(r);
        for (; r < r1; r += kBandWarps) {
            float g[8], z[8];
            if (ahead) {
                unpack8<T>(gn, g);
                if (ACT != TTC_ACT_NONE) unpack8<T>(zn, z);
                if (r + kBandWarps < r1) fetch(r + kBandWarps);
            } else {
                load8(static_cast<const T*>(p.dy) + r * p.lddy + col, n, p.vec_dy, g);
                if (ACT != TTC_ACT_NONE) load8(static_cast<const T*>(p.pre) + r * p.ldp + col, n, p.vec_pre, z);
            }
            if (ACT != TTC_ACT_NONE) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float y, dy;
                    activate_grad(ACT, z[i], y, dy);
                    g[i] *= dy;
                }
            }
            if (p.dz) store8(static_cast<T*>(p.dz) + r * p.lddz + col, n, p.vec_dz, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += g[i];
        }
    }
    if (!p.partials && !p.dbias) return;
    __shared__ float part[kBandWarps][kStripe];
#pragma unroll
    for (int i = 0; i < 8; ++i) part[warp][lane * 8 + i] = sum[i];
    __syncthreads();
    const int c = blockIdx.y * kStripe + threadIdx.x;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kBandWarps; ++w) s += part[w][threadIdx.x];
    if (!p.dbias) {
        if (c < p.N) p.partials[(long long)blockIdx.x * p.N + c] = s;
        return;
    }
    if (gridDim.x > 1) {
        part[0][threadIdx.x] = s;  // this thread's own column
        cluster_sync();
        if (blockIdx.x == 0) {
            const uint32_t at = smem_u32(&part[0][threadIdx.x]);
            for (int b = 1; b < (int)gridDim.x; ++b) {
                float v;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr(at, b)) : "memory");
                s += v;
            }
        }
        cluster_sync();  // nobody leaves while its shared memory is still read
    }
    if (blockIdx.x == 0 && c < p.N) static_cast<T*>(p.dbias)[c] = from_f32<T>(s);
}

struct GatedGradParams {
    int M, N, band_rows;
    const void *dy, *gate, *up;
    long long lddy, ldp;
    void *dg, *du;
    long long ldd;
    bool vec_dy, vec_gate, vec_up;  // dg and du are always padded
};

template <class T, int ACT>
__global__ void __launch_bounds__(32 * kBandWarps, 4) gated_grad_kernel(const __grid_constant__ GatedGradParams p) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col = blockIdx.y * kStripe + lane * 8, n = p.N - col;
    grid_wait();
    grid_trigger();
    if (n <= 0) return;
    const long long r1 = min((long long)p.M, (blockIdx.x + 1ll) * p.band_rows);
    const bool ahead = n >= 8 && p.vec_dy && p.vec_gate && p.vec_up;
    uint4 dn = {}, gn = {}, un = {};
    auto fetch = [&](long long r) {
        dn = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.dy) + r * p.lddy + col);
        gn = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.gate) + r * p.ldp + col);
        un = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.up) + r * p.ldp + col);
    };
    long long r = (long long)blockIdx.x * p.band_rows + warp;
    if (ahead && r < r1) fetch(r);
    for (; r < r1; r += kBandWarps) {
        float d[8], g[8], u[8];
        if (ahead) {
            unpack8<T>(dn, d);
            unpack8<T>(gn, g);
            unpack8<T>(un, u);
            if (r + kBandWarps < r1) fetch(r + kBandWarps);
        } else {
            load8(static_cast<const T*>(p.dy) + r * p.lddy + col, n, p.vec_dy, d);
            load8(static_cast<const T*>(p.gate) + r * p.ldp + col, n, p.vec_gate, g);
            load8(static_cast<const T*>(p.up) + r * p.ldp + col, n, p.vec_up, u);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float y, dy;
            activate_grad(ACT, g[i], y, dy);
            g[i] = d[i] * u[i] * dy;
            u[i] = d[i] * y;
        }
        store8(static_cast<T*>(p.dg) + r * p.ldd + col, n, true, g);
        store8(static_cast<T*>(p.du) + r * p.ldd + col, n, true, u);
    }
}

// f(the activation as a compile-time constant)
template <class F>
int with_activation(int act, F&& f) {
    switch (act) {
        case TTC_ACT_RELU: return f(std::integral_constant<int, TTC_ACT_RELU>());
        case TTC_ACT_SILU: return f(std::integral_constant<int, TTC_ACT_SILU>());
        case TTC_ACT_GELU: return f(std::integral_constant<int, TTC_ACT_GELU>());
        case TTC_ACT_GELU_TANH: return f(std::integral_constant<int, TTC_ACT_GELU_TANH>());
        default: return f(std::integral_constant<int, TTC_ACT_NONE>());
    }
}

// Rows of 16-bit scratch matrices start on 16-byte boundaries.
long long padded(long long n) { return (n + 7) & ~7ll; }

// Memory carved from a call's workspace; with base NULL it only counts.
struct Carver {
    char* base;
    size_t used = 0;
    void* take(size_t bytes) {
        void* p = base ? base + used : nullptr;
        used += align256(bytes);
        return p;
    }
};

bool all_vec(const ProductEpilogue& e) {
    const int t = e.out_dtype;
    return vec8_ok(e.out, t, e.ldo) && vec8_ok(e.out2, t, e.ldo) && vec8_ok(e.bias, t, 0) &&
           vec8_ok(e.residual, t, e.ldr) && vec8_ok(e.pre, t, e.ldp) && vec8_ok(e.gate, t, e.ldp) &&
           vec8_ok(e.up, t, e.ldp) && vec8_ok(e.col_scales[0], TTC_F32, 0) && vec8_ok(e.col_scales[1], TTC_F32, 0);
}

Product linear_product(const ttc_linear_desc& d) {
    Product p;
    std::memset(&p, 0, sizeof p);
    p.M = d.M;
    p.N = d.N;
    p.K = d.K;
    p.dtype = d.dtype;
    p.segs = 1;
    p.b_mn = !d.trans_w;
    p.a[0] = {d.x, d.ldx};
    p.b[0] = {d.w, d.ldw};
    ProductEpilogue& e = p.epi;
    e.out = d.y;
    e.ldo = d.ldy;
    e.out_dtype = d.y_dtype;
    e.act = d.act;
    e.bias = d.bias;
    e.residual = d.residual;
    e.ldr = d.ldr;
    e.pre = d.pre;
    e.ldp = d.ldp;
    e.row_scales = d.x_scales;
    e.col_scales[0] = d.w_scales;
    e.vec = all_vec(e);
    return p;
}

Product gated_product(const ttc_gated_linear_desc& d) {
    Product p;
    std::memset(&p, 0, sizeof p);
    p.M = d.M;
    p.N = d.N;
    p.K = d.K;
    p.dtype = d.dtype;
    p.segs = 1;
    p.gated = 1;
    p.b_mn = !d.trans_w;
    p.a[0] = {d.x, d.ldx};
    p.b[0] = {d.wg, d.ldw};
    p.b[1] = {d.wu, d.ldw};
    ProductEpilogue& e = p.epi;
    e.out = d.y;
    e.ldo = d.ldy;
    e.out_dtype = d.y_dtype;
    e.act = d.act;
    e.gate = d.gate;
    e.up = d.up;
    e.ldp = d.ldp;
    e.row_scales = d.x_scales;
    e.col_scales[0] = d.wg_scales;
    e.col_scales[1] = d.wu_scales;
    e.vec = all_vec(e);
    return p;
}

// A gradient's product: no scales, no activation.
Product grad_product(int M, int N, int K, int dtype, Operand a, bool a_mn, Operand b, bool b_mn, void* out,
                     long long ldo) {
    Product p;
    std::memset(&p, 0, sizeof p);
    p.M = M;
    p.N = N;
    p.K = K;
    p.dtype = dtype;
    p.segs = 1;
    p.a_mn = a_mn;
    p.b_mn = b_mn;
    p.a[0] = a;
    p.b[0] = b;
    p.epi.out = out;
    p.epi.ldo = ldo;
    p.epi.out_dtype = dtype;
    p.epi.vec = all_vec(p.epi);
    return p;
}

// A gradient matrix [rows, cols] of no rows of input.
int zero_matrix(void* p, long long ld, long long rows, long long cols, int dtype) {
    TTC_CUDA(cudaMemset2DAsync(p, (size_t)ld * dtype_size(dtype), 0, (size_t)cols * dtype_size(dtype), (size_t)rows,
                               rt().stream));
    return TTC_OK;
}

// Both backward calls are planned once, with ws NULL to count the workspace
// and with the workspace to run.
int plan_linear_backward(const ttc_linear_backward_desc& d, void* ws, size_t* bytes, bool run) {
    Carver c{(char*)ws};
    const bool dz_needed = d.act != TTC_ACT_NONE && (d.dx || d.dw);
    const long long lddz = padded(d.N);
    const int es = dtype_size(d.dtype);
    Operand dz{d.dy, d.lddy};
    LinearGradParams g;
    std::memset(&g, 0, sizeof g);
    if (dz_needed) {
        g.dz = c.take((size_t)d.M * lddz * es);
        dz = {g.dz, lddz};
    }
    const Bands b = bands_of(d.M, d.N, d.dbias != nullptr);
    if (d.dbias) g.partials = (float*)c.take((size_t)b.n * d.N * sizeof(float));
    void* scratch = c.base ? c.base + c.used : nullptr;
    // dx [M, K] = dz [M, N] W^T: the sum runs over N, which is contiguous in a
    // weight stored [K, N] and strided in one stored [N, K].
    Product products[2];
    int count = 0;
    if (d.dx)
        products[count++] = grad_product(d.M, d.K, d.N, d.dtype, dz, false, {d.w, d.ldw}, d.trans_w, d.dx, d.lddx);
    // dw [K, N] = x^T dz, or [N, K] = dz^T x; the sum runs over the rows.
    if (d.dw)
        products[count++] = d.trans_w
                                ? grad_product(d.N, d.K, d.M, d.dtype, dz, true, {d.x, d.ldx}, true, d.dw, d.lddw)
                                : grad_product(d.K, d.N, d.M, d.dtype, {d.x, d.ldx}, true, dz, true, d.dw, d.lddw);
    if (bytes) *bytes = c.used + product_scratch(products, count);
    if (!run) return TTC_OK;
    if (dz_needed || d.dbias) {
        g.M = d.M;
        g.N = d.N;
        g.band_rows = b.rows;
        g.dy = d.dy;
        g.pre = d.pre;
        g.lddy = d.lddy;
        g.ldp = d.ldp;
        g.lddz = lddz;
        g.vec_dy = vec8_ok(d.dy, d.dtype, d.lddy);
        g.vec_pre = vec8_ok(d.pre, d.dtype, d.ldp);
        g.vec_dz = true;
        if (b.joined) {
            g.dbias = d.dbias;
            g.partials = nullptr;
        }
        const dim3 grid((unsigned)b.n, (unsigned)b.stripes);
        count_launch();
        if (int rc = with_activation(d.act, [&](auto act) {
                return launch_overlapped(d.dtype == TTC_BF16 ? linear_grad_kernel<__nv_bfloat16, act()>
                                                             : linear_grad_kernel<__half, act()>,
                                         grid, 32 * kBandWarps, b.joined ? b.n : 1, g);
            }))
            return rc;
        if (d.dbias && !b.joined)
            if (int rc = launch_sum_partials(g.partials, b.n, d.N, d.dbias, d.dtype)) return rc;
    }
    return run_products(products, count, scratch);
}

int plan_gated_backward(const ttc_gated_linear_backward_desc& d, void* ws, size_t* bytes, bool run) {
    if (!d.dx && !d.dwg) {
        if (bytes) *bytes = 0;
        return TTC_OK;
    }
    Carver c{(char*)ws};
    // [dg | du], each padded to whole 16-byte groups, side by side in one
    // matrix: the weight gradients are one product over both.
    const long long np = padded(d.N), ldd = 2 * np;
    const int es = dtype_size(d.dtype);
    char* dgu = (char*)c.take((size_t)d.M * ldd * es);
    void* scratch = c.base ? c.base + c.used : nullptr;
    const Operand dg{dgu, ldd}, du{dgu ? dgu + np * es : nullptr, ldd};
    // dx [M, K] = dg Wg^T + du Wu^T: one accumulation over both weights.
    Product products[2];
    int count = 0;
    if (d.dx) {
        Product& px = products[count++];
        px = grad_product(d.M, d.K, d.N, d.dtype, dg, false, {d.wg, d.ldw}, d.trans_w, d.dx, d.lddx);
        px.segs = 2;
        px.a[1] = du;
        px.b[1] = {d.wu, d.ldw};
    }
    const int both = (int)(np + d.N);
    Product pw;
    if (d.trans_w) {  // [dwg; dwu] = [dg | du]^T x, one block of rows for each
        pw = grad_product(both, d.K, d.M, d.dtype, dg, true, {d.x, d.ldx}, true, d.dwg, d.lddw);
        pw.epi.split_rows = d.N;
    } else {  // [dwg | dwu] = x^T [dg | du]
        pw = grad_product(d.K, both, d.M, d.dtype, {d.x, d.ldx}, true, dg, true, d.dwg, d.lddw);
        pw.epi.split_cols = d.N;
    }
    pw.epi.split_skip = (int)(np - d.N);
    pw.epi.out2 = d.dwu;
    pw.epi.vec = all_vec(pw.epi);
    if (d.dwg) products[count++] = pw;
    if (bytes) *bytes = c.used + product_scratch(products, count);
    if (!run) return TTC_OK;
    GatedGradParams g;
    std::memset(&g, 0, sizeof g);
    g.M = d.M;
    g.N = d.N;
    const Bands b = bands_of(d.M, d.N, false);
    g.band_rows = b.rows;
    g.dy = d.dy;
    g.gate = d.gate;
    g.up = d.up;
    g.lddy = d.lddy;
    g.ldp = d.ldp;
    g.dg = const_cast<void*>(dg.ptr);
    g.du = const_cast<void*>(du.ptr);
    g.ldd = ldd;
    g.vec_dy = vec8_ok(d.dy, d.dtype, d.lddy);
    g.vec_gate = vec8_ok(d.gate, d.dtype, d.ldp);
    g.vec_up = vec8_ok(d.up, d.dtype, d.ldp);
    const dim3 grid((unsigned)b.n, (unsigned)b.stripes);
    count_launch();
    if (int rc = with_activation(d.act, [&](auto act) {
            return launch_overlapped(
                d.dtype == TTC_BF16 ? gated_grad_kernel<__nv_bfloat16, act()> : gated_grad_kernel<__half, act()>, grid,
                32 * kBandWarps, 1, g);
        }))
        return rc;
    return run_products(products, count, scratch);
}

}  // namespace
}  // namespace ttc

using namespace ttc;

extern "C" {

int ttc_linear_workspace(const ttc_linear_desc* desc, size_t* bytes) {
    if (!desc || !bytes) return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: linear_workspace: NULL argument");
    *bytes = 0;
    if (int rc = check_linear(*desc)) return rc;
    const Product p = linear_product(*desc);
    *bytes = product_scratch(&p, 1);
    return TTC_OK;
}

int ttc_linear(const ttc_linear_desc* desc) {
    if (!desc) return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: linear: desc is NULL");
    if (int rc = check_linear(*desc)) return rc;
    const Product p = linear_product(*desc);
    if (int rc = check_workspace("linear", desc->workspace, desc->workspace_bytes, product_scratch(&p, 1))) return rc;
    TTC_REQUIRE_INIT();
    if (desc->M == 0) return TTC_OK;
    DeviceGuard guard;
    return run_products(&p, 1, desc->workspace);
}

int ttc_gated_linear_workspace(const ttc_gated_linear_desc* desc, size_t* bytes) {
    if (!desc || !bytes) return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: gated_linear_workspace: NULL argument");
    *bytes = 0;
    if (int rc = check_gated(*desc)) return rc;
    const Product p = gated_product(*desc);
    *bytes = product_scratch(&p, 1);
    return TTC_OK;
}

int ttc_gated_linear(const ttc_gated_linear_desc* desc) {
    if (!desc) return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: gated_linear: desc is NULL");
    if (int rc = check_gated(*desc)) return rc;
    const Product p = gated_product(*desc);
    if (int rc = check_workspace("gated_linear", desc->workspace, desc->workspace_bytes, product_scratch(&p, 1))) return rc;
    TTC_REQUIRE_INIT();
    if (desc->M == 0) return TTC_OK;
    DeviceGuard guard;
    return run_products(&p, 1, desc->workspace);
}

int ttc_linear_backward_workspace(const ttc_linear_backward_desc* desc, size_t* bytes) {
    if (!desc || !bytes)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: linear_backward_workspace: NULL argument");
    *bytes = 0;
    if (int rc = check_linear_backward(*desc)) return rc;
    return desc->M ? plan_linear_backward(*desc, nullptr, bytes, false) : TTC_OK;
}

int ttc_linear_backward(const ttc_linear_backward_desc* desc) {
    if (!desc) return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: linear_backward: desc is NULL");
    const ttc_linear_backward_desc& d = *desc;
    size_t need = 0;
    if (int rc = ttc_linear_backward_workspace(&d, &need)) return rc;
    if (int rc = check_workspace("linear_backward", d.workspace, d.workspace_bytes, need)) return rc;
    TTC_REQUIRE_INIT();
    DeviceGuard guard;
    if (d.M == 0) {
        if (d.dw)
            if (int rc = zero_matrix(d.dw, d.lddw, d.trans_w ? d.N : d.K, d.trans_w ? d.K : d.N, d.dtype)) return rc;
        return d.dbias ? zero_matrix(d.dbias, d.N, 1, d.N, d.dtype) : TTC_OK;
    }
    return plan_linear_backward(d, d.workspace, nullptr, true);
}

int ttc_gated_linear_backward_workspace(const ttc_gated_linear_backward_desc* desc, size_t* bytes) {
    if (!desc || !bytes)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: gated_linear_backward_workspace: NULL argument");
    *bytes = 0;
    if (int rc = check_gated_backward(*desc)) return rc;
    return desc->M ? plan_gated_backward(*desc, nullptr, bytes, false) : TTC_OK;
}

int ttc_gated_linear_backward(const ttc_gated_linear_backward_desc* desc) {
    if (!desc) return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: gated_linear_backward: desc is NULL");
    const ttc_gated_linear_backward_desc& d = *desc;
    size_t need = 0;
    if (int rc = ttc_gated_linear_backward_workspace(&d, &need)) return rc;
    if (int rc = check_workspace("gated_linear_backward", d.workspace, d.workspace_bytes, need)) return rc;
    TTC_REQUIRE_INIT();
    DeviceGuard guard;
    if (d.M == 0) {
        for (void* w : {d.dwg, d.dwu})
            if (w)
                if (int rc = zero_matrix(w, d.lddw, d.trans_w ? d.N : d.K, d.trans_w ? d.K : d.N, d.dtype)) return rc;
        return TTC_OK;
    }
    return plan_gated_backward(d, d.workspace, nullptr, true);
}

}  // extern "C"
