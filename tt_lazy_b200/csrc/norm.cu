// norm.cu -- root-mean-square norm with the residual's addition
// (ttc_rms_norm) and its gradients (ttc_rms_norm_backward).
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "ffn.cuh"
#include "tc_util.cuh"

namespace ttc {
namespace {

// Both kernels hold a row in registers: it is read once, its sums go over the
// row's threads, and the results are written from the registers. The next
// row's loads are issued before this row's reduction, so memory is busy while
// the threads wait for their sums.
//
// A thread holds C chunks of 16 bytes of a row. Rows of up to 128 chunks
// belong to one warp; longer ones to a block of up to 256 threads with two
// chunks each, and above 512 chunks to the 2, 4 or 8 blocks of a cluster that
// exchange their sums through distributed shared memory.
//
// A chunk is one 16-byte access where every tensor's rows are 16-byte aligned
// and whole chunks long (VEC), else its elements lie 32 apart, so that a warp
// still touches consecutive elements.
template <class T>
constexpr int kPer = 16 / (int)sizeof(T);  // elements of a chunk

// Thread t of the row's tpr threads.
struct Lane {
    int t, tpr;
};
template <class T, bool VEC>
__device__ __forceinline__ int column(int c, int i, Lane l) {
    return VEC ? (c * l.tpr + l.t) * kPer<T> + i : (c * l.tpr + (l.t & ~31)) * kPer<T> + i * 32 + (l.t & 31);
}

// A chunk's elements in the four registers that they fill, whichever way they came.
template <class T>
__device__ __forceinline__ void unpack(const uint4& u, float (&v)[kPer<T>]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            v[i] = __uint_as_float(w[i]);
        } else {
            const T *lo = reinterpret_cast<const T*>(&w[i]);
            v[2 * i] = to_f32<T>(lo[0]);
            v[2 * i + 1] = to_f32<T>(lo[1]);
        }
    }
}

template <class T, bool VEC, int C>
__device__ __forceinline__ void load_row(const T* row, int cols, Lane l, uint4 (&r)[C]) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if constexpr (VEC) {
            const int k = column<T, VEC>(c, 0, l);
            r[c] = k < cols ? *reinterpret_cast<const uint4*>(row + k) : make_uint4(0, 0, 0, 0);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = 0;
#pragma unroll
                for (int e = 0; e < kPer<T> / 4; ++e) {
                    const int k = column<T, VEC>(c, i * (kPer<T> / 4) + e, l);
                    if constexpr (sizeof(T) == 4) {
                        if (k < cols) w[i] = __float_as_uint(row[k]);
                    } else {
                        if (k < cols) w[i] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[k] << (16 * e);
                    }
                }
            }
            r[c] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// T is the type whose chunks the row is divided into, Y the type stored.
template <class T, class Y, bool VEC, int C>
__device__ __forceinline__ void store_row(Y* row, int cols, Lane l, const float (&v)[C][kPer<T>]) {
    struct alignas(sizeof(Y) * kPer<T>) Out {
        Y e[kPer<T>];
    };
#pragma unroll
    for (int c = 0; c < C; ++c) {
        if constexpr (VEC) {
            Out o;
#pragma unroll
            for (int i = 0; i < kPer<T>; ++i) o.e[i] = from_f32<Y>(v[c][i]);
            if (column<T, VEC>(c, 0, l) < cols)
                *reinterpret_cast<Out*>(row + column<T, VEC>(c, 0, l)) = o;
        } else {
#pragma unroll
            for (int i = 0; i < kPer<T>; ++i) {
                const int k = column<T, VEC>(c, i, l);
                if (k < cols) row[k] = from_f32<Y>(v[c][i]);
            }
        }
    }
}

template <class T>
__device__ __forceinline__ float weight_at(const void* weight, bool f32, int c) {
    return f32 ? static_cast<const float*>(weight)[c] : to_f32<T>(static_cast<const T*>(weight)[c]);
}
template <class T, bool VEC, int C>
__device__ __forceinline__ void load_weight(const void* weight, bool f32, int cols, Lane l, float (&w)[C][kPer<T>]) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < kPer<T>; ++i) {
            const int k = column<T, VEC>(c, i, l);
            w[c][i] = k >= cols ? 0.0f : weight_at<T>(weight, f32, k);
        }
}

// The larger, or NaN where either is: a row's e4m3 scale has to show that the row
// holds one.
__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

// Reduces a and b over a row's threads, in a fixed order; MAX: b is a maximum.
// ONE: the row is one warp's. Else `slots` is one of two buffers that the rows
// use in turn, so that one barrier a row is enough; in a cluster of more than
// one block every warp writes its pair into the buffer of each block.
constexpr int kSlots = 64;  // 8 blocks of 8 warps
constexpr int kMaxStages = 8;
template <bool ONE, bool MAX>
__device__ __forceinline__ void reduce_row(float& a, float& b, float2* slots, int blocks) {
    auto warp = [&] {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            const float x = __shfl_xor_sync(0xffffffffu, b, o);
            b = MAX ? max_nan(b, x) : b + x;
        }
    };
    warp();
    if constexpr (!ONE) {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
        if (blocks == 1) {
            if (lane == 0) slots[w] = make_float2(a, b);
            __syncthreads();
            a = slots[0].x;
            b = slots[0].y;
            for (int i = 1; i < warps; ++i) {
                const float2 s = slots[i];
                a += s.x;
                b = MAX ? max_nan(b, s.y) : b + s.y;
            }
        } else {
            if (lane < blocks)
                asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(
                                 cluster_addr(smem_u32(slots + cluster_rank() * warps + w), lane)),
                             "f"(a), "f"(b)
                             : "memory");
            __syncwarp();
            cluster_sync();
            const int n = warps * blocks;
            const float2 s = lane < n ? slots[lane] : make_float2(0.0f, 0.0f);
            const float2 s2 = lane + 32 < n ? slots[lane + 32] : make_float2(0.0f, 0.0f);
            a = s.x + s2.x;
            b = MAX ? max_nan(s.y, s2.y) : s.y + s2.y;
            warp();
        }
    }
}

constexpr float kMinScale = 1.17549435e-38f;  // 2^-126

// Squares of finite values can leave fp32: |h| from 2^64, and below 2^-63 where eps
// does not cover them. The sums of such a row, infinite or next to nothing, are
// taken again with the row times this power of two, exactly; 1 for any other row.
// With it the squares of 2^30 values of 2^128 add up to
// 2^126, and values of which the sum of squares was below 2^-90 to at most 2^110.
// F16 rows cannot get there.
template <class T>
__device__ __forceinline__ float range_factor(float sum, float eps) {
    if (std::is_same<T, __half>::value) return 1.0f;
    if (sum > 3.402823466e38f) return 8.271806126e-25f;                                // 2^-80
    return sum < 8.077935669e-28f && eps < 7.888609052e-31f ? 1.267650600e30f : 1.0f;  // 2^-90, 2^-100, 2^100
}

struct NormParams {
    long long rows;
    int cols;
    float eps;
    const void *x, *residual, *weight;
    void *y, *hidden;
    float* scales;
    long long ldx, ldr, ldy, ldh;
    int weight_f32;
    int cluster;  // blocks of a row
};

// Which row a thread starts at, how far it is to its next one, and its place in a row.
struct RowPlace {
    Lane lane;
    long long row, step;
};
template <bool ONE>
__device__ __forceinline__ RowPlace row_place(int cluster) {
    if (ONE) {
        const long long rows = blockDim.x / 32;
        return {{(int)threadIdx.x % 32, 32}, blockIdx.x * rows + threadIdx.x / 32, gridDim.x * rows};
    }
    const int rank = cluster > 1 ? (int)cluster_rank() : 0;
    if (cluster > 1) cluster_sync();  // every block of the row is there before one writes into another
    return {{rank * (int)blockDim.x + (int)threadIdx.x, cluster * (int)blockDim.x},
            (long long)(blockIdx.x / cluster), (long long)(gridDim.x / cluster)};
}

constexpr int kWarpRows = 4;  // rows of a block whose rows are one warp's
constexpr int kMaxBlock = 256;

template <class T, class Y, bool VEC, bool ONE, int C>
__global__ void __launch_bounds__(ONE ? 32 * kWarpRows : kMaxBlock) rms_norm_kernel(const __grid_constant__ NormParams p) {
    __shared__ float2 slots[2][kSlots];
    const RowPlace at = row_place<ONE>(p.cluster);
    const Lane l = at.lane;
    float w[C][kPer<T>];
    load_weight<T, VEC, C>(p.weight, p.weight_f32, p.cols, l, w);
    const T *x = static_cast<const T*>(p.x), *res = static_cast<const T*>(p.residual);
    const long long step = at.step;
    long long r = at.row;
    uint4 xs[C], rs[C];
    auto fetch = [&](long long row) {
        if (row >= p.rows) return;
        load_row<T, VEC, C>(x + row * p.ldx, p.cols, l, xs);
        if (res) load_row<T, VEC, C>(res + row * p.ldr, p.cols, l, rs);
    };
    fetch(r);
    for (int parity = 0; r < p.rows; r += step, parity ^= 1) {
        float h[C][kPer<T>], sum = 0.0f, top = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            unpack<T>(xs[c], h[c]);
            if (res) {
                float v[kPer<T>];
                unpack<T>(rs[c], v);
#pragma unroll
                for (int i = 0; i < kPer<T>; ++i) h[c][i] += v[i];
            }
#pragma unroll
            for (int i = 0; i < kPer<T>; ++i) {
                sum += h[c][i] * h[c][i];
                if (sizeof(Y) == 1) top = max_nan(top, fabsf(h[c][i] * w[c][i]));
            }
        }
        fetch(r + step);
        reduce_row<ONE, true>(sum, top, slots[parity], p.cluster);
        // All of the row is in registers now: x, residual, hidden and y may be the same memory.
        if (p.hidden) store_row<T, T, VEC, C>(static_cast<T*>(p.hidden) + r * p.ldh, p.cols, l, h);
        float eps = p.eps;
        if (const float f = range_factor<T>(sum, eps); f != 1.0f) {  // the same for all of the row's threads
            eps = eps * f * f;
            sum = top = 0.0f;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < kPer<T>; ++i) {
                    h[c][i] *= f;
                    sum += h[c][i] * h[c][i];
                    if (sizeof(Y) == 1) top = max_nan(top, fabsf(h[c][i] * w[c][i]));
                }
            parity ^= 1;
            reduce_row<ONE, true>(sum, top, slots[parity], p.cluster);
        }
        const float k = rsqrtf(sum / (float)p.cols + eps);
        float inv = 1.0f;
        if (sizeof(Y) == 1) {
            const float scale = max_nan(top * k * (1.0f / 448.0f), kMinScale);
            inv = 1.0f / scale;
            if (l.t == 0) p.scales[r] = scale;
        }
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < kPer<T>; ++i) h[c][i] = h[c][i] * k * w[c][i] * inv;
        store_row<T, Y, VEC, C>(static_cast<Y*>(p.y) + r * p.ldy, p.cols, l, h);
    }
}

// What a row's gradients need, from its sums of the row times f (range_factor):
// rstd, and k with hidden rstd^2 mean(dy weight hidden) = hidden k.
__device__ __forceinline__ void gradient_scalars(float sum, float dot, float eps, int cols, float f, float& rstd, float& k) {
    const float scaled = rsqrtf(sum / (float)cols + eps * f * f);
    rstd = scaled * f;
    k = dot * scaled * scaled / (float)cols * f;
}

struct NormBackwardParams {
    long long rows;
    int cols;
    float eps;
    const void *dy, *hidden, *weight, *dhidden;
    void* dx;
    float* partials;  // [blocks or clusters, cols] sums of dy * hidden * rstd, or NULL
    long long lddy, ldh, lddh, lddx;
    int weight_f32, weight_vec;  // weight_vec: of dtype, 16-byte aligned
    int cluster;
};

// The sums of a row times f = range_factor, and then its results, an element at a
// time. The kernels leave the loop over the usual rows for such a row, so that it
// takes no registers from them: nothing to 3 % (gradients of 16384 x 4096 in bf16 93.5
// -> 95.1 us, of 8192 x 8192 109.5 -> 112.8, of 4096 x 16384 125.6 -> 130.4; with
// the second sums inside the loop 70 bytes of it spilled). All of the row is read
// before the reduction between the two, each thread's results where it alone reads.
template <class T>
__device__ __forceinline__ void far_sums(const T* dy, const T* hidden, const void* weight, int weight_f32, int cols, Lane l,
                                         float f, float& sum, float& dot) {
    sum = dot = 0.0f;
#pragma unroll 1
    for (int c = l.t; c < cols; c += l.tpr) {
        const float h = to_f32<T>(hidden[c]) * f;
        sum += h * h;
        dot += to_f32<T>(dy[c]) * weight_at<T>(weight, weight_f32, c) * h;
    }
}

template <class T>
__device__ __forceinline__ void far_element(const T* hidden, const T* dy, const T* dhidden, T* dx, float w, float rstd, float k,
                                            float& dw) {
    const float h = to_f32<T>(*hidden), g = to_f32<T>(*dy);
    float d = rstd * (g * w - h * k);
    if (dhidden) d += to_f32<T>(*dhidden);
    dw += g * (h * rstd);
    *dx = from_f32<T>(d);
}

// The weight's gradient stays in registers over all of a block's rows and goes
// out once as the block's row of the partials; no atomics.
// Registers for 512 threads an SM (one row a warp: 512, 256 with four chunks).
template <class T, bool VEC, bool ONE, int C>
__global__ void __launch_bounds__(ONE ? 32 * kWarpRows : kMaxBlock, ONE ? (C == 4 ? 2 : 4) : 2)
    rms_norm_backward_kernel(const __grid_constant__ NormBackwardParams p) {
    __shared__ float2 slots[2][kSlots];
    const RowPlace at = row_place<ONE>(p.cluster);
    const Lane l = at.lane;
    float w[C][kPer<T>], dw[C][kPer<T>] = {};
    load_weight<T, VEC, C>(p.weight, p.weight_f32, p.cols, l, w);
    const T *dy = static_cast<const T*>(p.dy), *hid = static_cast<const T*>(p.hidden);
    const T* dh = static_cast<const T*>(p.dhidden);
    const long long step = at.step;
    long long r = at.row;
    uint4 gs[C], hs[C], ds[C];
    auto fetch = [&](long long row) {
        if (row >= p.rows) return;
        load_row<T, VEC, C>(dy + row * p.lddy, p.cols, l, gs);
        load_row<T, VEC, C>(hid + row * p.ldh, p.cols, l, hs);
        if (dh) load_row<T, VEC, C>(dh + row * p.lddh, p.cols, l, ds);
    };
    fetch(r);
    for (int parity = 0; r < p.rows;) {
        // The usual rows, up to one that needs a range_factor.
        float f = 1.0f, sum, dot;
        for (; r < p.rows; r += step, parity ^= 1) {
            sum = dot = 0.0f;
            uint4 g[C], h[C], d[C];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                g[c] = gs[c];
                h[c] = hs[c];
                if (dh) d[c] = ds[c];
                float hv[kPer<T>], gv[kPer<T>];
                unpack<T>(h[c], hv);
                unpack<T>(g[c], gv);
#pragma unroll
                for (int i = 0; i < kPer<T>; ++i) {
                    sum += hv[i] * hv[i];
                    dot += gv[i] * w[c][i] * hv[i];
                }
            }
            fetch(r + step);
            reduce_row<ONE, false>(sum, dot, slots[parity], p.cluster);
            f = range_factor<T>(sum, p.eps);  // the same for all of the row's threads
            if (f != 1.0f) break;
            float rstd, k;
            gradient_scalars(sum, dot, p.eps, p.cols, 1.0f, rstd, k);
            float out[C][kPer<T>];
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float hv[kPer<T>], gv[kPer<T>];
                unpack<T>(h[c], hv);
                unpack<T>(g[c], gv);
#pragma unroll
                for (int i = 0; i < kPer<T>; ++i) {
                    out[c][i] = rstd * (gv[i] * w[c][i] - hv[i] * k);
                    dw[c][i] += gv[i] * hv[i] * rstd;
                }
                if (dh) {
                    unpack<T>(d[c], gv);
#pragma unroll
                    for (int i = 0; i < kPer<T>; ++i) out[c][i] += gv[i];
                }
            }
            store_row<T, T, VEC, C>(static_cast<T*>(p.dx) + r * p.lddx, p.cols, l, out);
        }
        if (f == 1.0f) break;
        // That row, once more from memory.
        far_sums<T>(dy + r * p.lddy, hid + r * p.ldh, p.weight, p.weight_f32, p.cols, l, f, sum, dot);
        parity ^= 1;
        reduce_row<ONE, false>(sum, dot, slots[parity], p.cluster);
        float rstd, k;
        gradient_scalars(sum, dot, p.eps, p.cols, f, rstd, k);
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < kPer<T>; ++i)
                if (const int col = column<T, VEC>(c, i, l); col < p.cols)
                    far_element(hid + r * p.ldh + col, dy + r * p.lddy + col, dh ? dh + r * p.lddh + col : nullptr,
                                static_cast<T*>(p.dx) + r * p.lddx + col, w[c][i], rstd, k, dw[c][i]);
        r += step;
        parity ^= 1;
        fetch(r);
    }
    if (!p.partials) return;
    float* part = p.partials + (long long)(blockIdx.x / p.cluster) * p.cols;
    if constexpr (!ONE) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < kPer<T>; ++i) {
                const int col = column<T, VEC>(c, i, l);
                if (col < p.cols) part[col] = dw[c][i];
            }
    } else {  // the block's warps side by side, added in order
        __shared__ float rows[kWarpRows][32 * C * kPer<T>];
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < kPer<T>; ++i) rows[threadIdx.x / 32][column<T, VEC>(c, i, l)] = dw[c][i];
        __syncthreads();
        for (int col = threadIdx.x; col < p.cols; col += 32 * kWarpRows) {
            float s = rows[0][col];
#pragma unroll
            for (int k = 1; k < kWarpRows; ++k) s += rows[k][col];
            part[col] = s;
        }
    }
}

// Longer aligned rows (more than 128 chunks, up to 2048): a ring in shared memory
// that bulk copies keep full, so that several rows are on their way without
// registers for them. Between two barriers a thread adds up its share of the next
// row and finishes its share of this one, whose sums the last barrier completed:
// two independent strands of work, one barrier a row.
struct RingParams {
    NormBackwardParams p;
    int stages, row_bytes;
    int* status;
    long long wait_limit;
    int stall;  // failure-detection test: no loads at all
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

template <class T, int C, int MAX>
__global__ void __launch_bounds__(MAX, 512 / MAX) rms_norm_backward_ring_kernel(const __grid_constant__ RingParams q) {
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ float2 slots[3][MAX / 32];  // two that rows use in turn, one for sums taken again
    __shared__ alignas(8) uint64_t bars[kMaxStages];
    const NormBackwardParams& p = q.p;
    const int t = threadIdx.x, threads = blockDim.x, n = p.cols / kPer<T>;  // chunks of a row
    const int stage_bytes = (p.dhidden ? 3 : 2) * q.row_bytes;
    const uint32_t base = smem_u32(ring);
    const int mine = (int)((p.rows - blockIdx.x + gridDim.x - 1) / gridDim.x);  // rows of this block
    auto issue = [&](int i, int s) {  // one thread
        const long long r = blockIdx.x + (long long)i * gridDim.x;
        const uint32_t bar = smem_u32(&bars[s]), dst = base + s * stage_bytes;
        mbar_arrive_expect_tx(bar, stage_bytes);
        bulk_load(dst, static_cast<const T*>(p.dy) + r * p.lddy, q.row_bytes, bar);
        bulk_load(dst + q.row_bytes, static_cast<const T*>(p.hidden) + r * p.ldh, q.row_bytes, bar);
        if (p.dhidden) bulk_load(dst + 2 * q.row_bytes, static_cast<const T*>(p.dhidden) + r * p.lddh, q.row_bytes, bar);
    };
    if (t == 0) {
        for (int s = 0; s < q.stages; ++s) mbar_init(smem_u32(&bars[s]), 1);
        mbar_fence_init();
    }
    __syncthreads();
    int issued = 0;  // rows that thread 0 has sent for
    if (t == 0 && !q.stall)
        for (; issued < q.stages && issued < mine; ++issued) issue(issued, issued);
    uint4 w[C];
    float dw[C][kPer<T>] = {};
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int k = c * threads + t;
        w[c] = p.weight_vec && k < n ? __ldg(static_cast<const uint4*>(p.weight) + k) : make_uint4(0, 0, 0, 0);
    }
    auto weight = [&](int c, float (&v)[kPer<T>]) {
        if (p.weight_vec) {
            unpack<T>(w[c], v);
            return;
        }
#pragma unroll
        for (int i = 0; i < kPer<T>; ++i) {
            const int k = (c * threads + t) * kPer<T> + i;
            v[i] = k >= p.cols    ? 0.0f
                   : p.weight_f32 ? __ldg(static_cast<const float*>(p.weight) + k)
                                  : to_f32<T>(static_cast<const T*>(p.weight)[k]);
        }
    };
    auto chunk = [&](int s, int stream, int c, float (&v)[kPer<T>]) {
        const int k = c * threads + t;
        unpack<T>(k < n ? *reinterpret_cast<const uint4*>(ring + s * stage_bytes + stream * q.row_bytes + k * 16)
                        : make_uint4(0, 0, 0, 0),
                  v);
    };
    bool failed = false;
    int next = 0;  // the stage of the next row to add up, and its parity
    uint32_t parity = 0;
    auto put_sums = [&](float sum, float dot, int to) {
        sum = warp_sum(sum);
        dot = warp_sum(dot);
        if ((t & 31) == 0) slots[to][t >> 5] = make_float2(sum, dot);
    };
    auto add_up = [&](int to) {
        if (!failed) failed = !mbar_wait(smem_u32(&bars[next]), parity, q.wait_limit);
        float sum = 0.0f, dot = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float g[kPer<T>], h[kPer<T>], wv[kPer<T>];
            chunk(next, 0, c, g);
            chunk(next, 1, c, h);
            weight(c, wv);
#pragma unroll
            for (int k = 0; k < kPer<T>; ++k) {
                sum += h[k] * h[k];
                dot += g[k] * wv[k] * h[k];
            }
        }
        put_sums(sum, dot, to);
        if (++next == q.stages) {
            next = 0;
            parity ^= 1;
        }
    };
    auto totals = [&](int from) {
        float2 total = slots[from][0];
        for (int k = 1; k < threads / 32; ++k) {
            total.x += slots[from][k].x;
            total.y += slots[from][k].y;
        }
        return total;
    };
    add_up(0);
    __syncthreads();
    int s = 0;  // this row's stage
    auto end_row = [&](int i) {
        __syncthreads();
        // After a wait that ran out the stage may still be filled, so nothing more is
        // sent for: its barrier must not be armed again, nor its buffer written.
        if (t == 0 && !failed && i + q.stages < mine) {
            issue(i + q.stages, s);
            ++issued;
        }
        if (++s == q.stages) s = 0;
    };
    for (int i = 0; i < mine; ++i) {
        // The usual rows, up to one that needs a range_factor.
        float f = 1.0f;
        for (; i < mine; ++i) {
            const long long r = blockIdx.x + (long long)i * gridDim.x;
            const float2 total = totals(i & 1);
            if (i + 1 < mine) add_up((i + 1) & 1);
            f = range_factor<T>(total.x, p.eps);  // the same for all threads
            if (f != 1.0f) break;
            float rstd, k2;
            gradient_scalars(total.x, total.y, p.eps, p.cols, 1.0f, rstd, k2);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float g[kPer<T>], h[kPer<T>], wv[kPer<T>], out[1][kPer<T>];
                chunk(s, 0, c, g);
                chunk(s, 1, c, h);
                weight(c, wv);
#pragma unroll
                for (int k = 0; k < kPer<T>; ++k) {
                    out[0][k] = rstd * (g[k] * wv[k] - h[k] * k2);
                    dw[c][k] += g[k] * h[k] * rstd;
                }
                if (p.dhidden) {
                    chunk(s, 2, c, g);
#pragma unroll
                    for (int k = 0; k < kPer<T>; ++k) out[0][k] += g[k];
                }
                store_row<T, T, true, 1>(static_cast<T*>(p.dx) + r * p.lddx, p.cols, Lane{c * threads + t, 0}, out);
            }
            end_row(i);
        }
        if (f == 1.0f) break;
        // That row, still in its stage.
        const T* dy = reinterpret_cast<const T*>(ring + s * stage_bytes);
        float2 a;
        far_sums<T>(dy, dy + p.cols, p.weight, p.weight_f32, p.cols, Lane{t, threads}, f, a.x, a.y);
        put_sums(a.x, a.y, 2);
        __syncthreads();  // these slots are not written again before the barrier at the end of the row
        a = totals(2);
        float rstd, k2;
        gradient_scalars(a.x, a.y, p.eps, p.cols, f, rstd, k2);
        T* dx = static_cast<T*>(p.dx) + (blockIdx.x + (long long)i * gridDim.x) * p.lddx;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int k = 0; k < kPer<T>; ++k)
                if (const int col = (c * threads + t) * kPer<T> + k; col < p.cols)
                    far_element(dy + p.cols + col, dy + col, p.dhidden ? dy + 2 * p.cols + col : nullptr, dx + col,
                                weight_at<T>(p.weight, p.weight_f32, col), rstd, k2, dw[c][k]);
        end_row(i);
    }
    if (failed) *(volatile int*)q.status = 1;
    if (t == 0 && failed)  // never leave with copies in flight: the last rows that were sent for
        for (int i = max(0, issued - q.stages); i < issued; ++i)
            mbar_wait(smem_u32(&bars[i % q.stages]), (uint32_t)(i / q.stages) & 1, q.wait_limit);
    if (!p.partials) return;
    float* part = p.partials + (long long)blockIdx.x * p.cols;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int k = (c * threads + t) * kPer<T>;
        if (k < p.cols) {
#pragma unroll
            for (int i = 0; i < kPer<T>; i += 4)
                *reinterpret_cast<float4*>(part + k + i) = make_float4(dw[c][i], dw[c][i + 1], dw[c][i + 2], dw[c][i + 3]);
        }
    }
}

// Rows that do not fit in registers: one block a row, two passes over it (the
// second finds it in L2).
constexpr int kWide = 1024;

template <class T, class Y>
__global__ void __launch_bounds__(kWide) rms_norm_wide_kernel(const __grid_constant__ NormParams p) {
    __shared__ float2 slots[2][kSlots];
    auto weight = [&](int c) { return weight_at<T>(p.weight, p.weight_f32, c); };
    int parity = 0;
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x, parity ^= 1) {
        const T* x = static_cast<const T*>(p.x) + r * p.ldx;
        const T* res = p.residual ? static_cast<const T*>(p.residual) + r * p.ldr : nullptr;
        float sum = 0.0f, top = 0.0f;
#pragma unroll 4
        for (int c = threadIdx.x; c < p.cols; c += kWide) {
            float h = to_f32<T>(x[c]);
            if (res) h += to_f32<T>(res[c]);
            sum += h * h;
            if (sizeof(Y) == 1) top = max_nan(top, fabsf(h * weight(c)));
        }
        reduce_row<false, true>(sum, top, slots[parity], 1);
        Y* y = static_cast<Y*>(p.y) + r * p.ldy;
        T* hid = p.hidden ? static_cast<T*>(p.hidden) + r * p.ldh : nullptr;
        auto quantise = [&](float k) {  // 1 / scale
            if (sizeof(Y) != 1) return 1.0f;
            const float scale = max_nan(top * k * (1.0f / 448.0f), kMinScale);
            if (threadIdx.x == 0) p.scales[r] = scale;
            return 1.0f / scale;
        };
        if (const float f = range_factor<T>(sum, p.eps); f != 1.0f) {  // the same for all threads
            auto row = [&](int c) { return res ? to_f32<T>(x[c]) + to_f32<T>(res[c]) : to_f32<T>(x[c]); };
            sum = top = 0.0f;
#pragma unroll 1
            for (int c = threadIdx.x; c < p.cols; c += kWide) {
                const float h = row(c) * f;
                sum += h * h;
                if (sizeof(Y) == 1) top = max_nan(top, fabsf(h * weight(c)));
            }
            parity ^= 1;
            reduce_row<false, true>(sum, top, slots[parity], 1);
            const float k = rsqrtf(sum / (float)p.cols + p.eps * f * f), inv = quantise(k);
#pragma unroll 1
            for (int c = threadIdx.x; c < p.cols; c += kWide) {
                const float h = row(c);
                if (hid) hid[c] = from_f32<T>(h);
                y[c] = from_f32<Y>(h * f * k * weight(c) * inv);
            }
            continue;
        }
        const float k = rsqrtf(sum / (float)p.cols + p.eps), inv = quantise(k);
#pragma unroll 4
        for (int c = threadIdx.x; c < p.cols; c += kWide) {  // an element is read before it may be written over
            float h = to_f32<T>(x[c]);
            if (res) h += to_f32<T>(res[c]);
            if (hid) hid[c] = from_f32<T>(h);
            y[c] = from_f32<Y>(h * k * weight(c) * inv);
        }
    }
}

template <class T>
__global__ void __launch_bounds__(kWide, 1) rms_norm_backward_wide_kernel(const __grid_constant__ NormBackwardParams p) {
    __shared__ float2 slots[2][kSlots];
    float* part = p.partials ? p.partials + (long long)blockIdx.x * p.cols : nullptr;
    if (part)
        for (int c = threadIdx.x; c < p.cols; c += kWide) part[c] = 0.0f;  // a thread owns its columns throughout
    auto weight = [&](int c) { return weight_at<T>(p.weight, p.weight_f32, c); };
    int parity = 0;
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x, parity ^= 1) {
        const T* dy = static_cast<const T*>(p.dy) + r * p.lddy;
        const T* hid = static_cast<const T*>(p.hidden) + r * p.ldh;
        const T* dh = p.dhidden ? static_cast<const T*>(p.dhidden) + r * p.lddh : nullptr;
        T* dx = static_cast<T*>(p.dx) + r * p.lddx;
        float sum = 0.0f, dot = 0.0f;
#pragma unroll 4
        for (int c = threadIdx.x; c < p.cols; c += kWide) {
            const float h = to_f32<T>(hid[c]);
            sum += h * h;
            dot += to_f32<T>(dy[c]) * weight(c) * h;
        }
        reduce_row<false, false>(sum, dot, slots[parity], 1);
        float rstd, k;
        if (const float f = range_factor<T>(sum, p.eps); f != 1.0f) {  // the same for all threads
            far_sums<T>(dy, hid, p.weight, p.weight_f32, p.cols, Lane{(int)threadIdx.x, kWide}, f, sum, dot);
            parity ^= 1;
            reduce_row<false, false>(sum, dot, slots[parity], 1);
            gradient_scalars(sum, dot, p.eps, p.cols, f, rstd, k);
            float none = 0.0f;
#pragma unroll 1
            for (int c = threadIdx.x; c < p.cols; c += kWide)
                far_element(hid + c, dy + c, dh ? dh + c : nullptr, dx + c, weight(c), rstd, k, part ? part[c] : none);
            continue;
        }
        gradient_scalars(sum, dot, p.eps, p.cols, 1.0f, rstd, k);
#pragma unroll 4
        for (int c = threadIdx.x; c < p.cols; c += kWide) {
            const float h = to_f32<T>(hid[c]), g = to_f32<T>(dy[c]);
            float d = rstd * (g * weight(c) - h * k);
            if (dh) d += to_f32<T>(dh[c]);
            if (part) part[c] += g * h * rstd;
            dx[c] = from_f32<T>(d);
        }
    }
}

// out[c] = sum over b < n of partials[b][c]: 32 columns a block, 32 threads a
// column that each add every 32nd partial, then the 32 in order.
__global__ void __launch_bounds__(1024) sum_partials_kernel(const float* partials, int n, int cols, void* out,
                                                            int dtype) {
    __shared__ float part[32][33];
    const int lane = threadIdx.x & 31, g = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float s = 0.0f;
    grid_wait();
    grid_trigger();
    if (c < cols) {
#pragma unroll 8
        for (int b = g; b < n; b += 32) s += partials[(long long)b * cols + c];
    }
    part[g][lane] = s;
    __syncthreads();
    if (g != 0 || c >= cols) return;
    s = 0.0f;
#pragma unroll
    for (int k = 0; k < 32; ++k) s += part[k][lane];
    if (dtype == TTC_BF16)
        static_cast<__nv_bfloat16*>(out)[c] = from_f32<__nv_bfloat16>(s);
    else if (dtype == TTC_F16)
        static_cast<__half*>(out)[c] = from_f32<__half>(s);
    else
        static_cast<float*>(out)[c] = s;
}

constexpr int kMaxCols = 1 << 30;

int check_norm_types(const char* op, int dtype, int weight_dtype, long long rows, int cols, float eps) {
    if (rows < 0 || cols < 1)
        return set_error(TTC_ERR_INVALID_ARGUMENT, "tt_cuda: %s: shape %lld x %d", op, rows, cols);
    if (rows > INT32_MAX)
        return set_error(TTC_ERR_UNSUPPORTED, "tt_cuda: %s: %lld rows exceed %d", op, rows, INT32_MAX);
    if (cols > kMaxCols)  // column indices that step past the end of a row stay inside 32 bits
        return set_error(TTC_ERR_UNSUPPORTED, "tt_cuda: %s: %d columns exceed %d", op, cols, kMaxCols);
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

// How a row is divided: threads of a block, blocks of a cluster and chunks a
// thread; one: a warp has the row; block 0: the row does not fit.
constexpr int kRingBytes = 200 * 1024;
struct RowShape {
    int block, cluster, chunks, one;
};
RowShape row_shape(int cols, int dtype) {
    const long long n = ((long long)cols * dtype_size(dtype) + 15) / 16;
    if (n <= 128) return {32 * kWarpRows, 1, n <= 32 ? 1 : n <= 64 ? 2 : 4, 1};
    for (int cluster = 1; cluster <= 8; cluster *= 2)
        if (n <= 2ll * kMaxBlock * cluster) return {(int)((n + 64 * cluster - 1) / (64 * cluster)) * 32, cluster, 2, 0};
    return {0, 1, 0, 0};
}

// Clusters (of one block mostly) of the backward kernel at most: what 148 SMs
// hold at 512 threads each, from the shape alone, so that the workspace size
// needs no device.
int backward_clusters(long long rows, const RowShape& s) {
    if (s.block == 0) return (int)std::min<long long>(rows, 148 * 2);
    if (s.one) return (int)std::min<long long>((rows + kWarpRows - 1) / kWarpRows, 148 * (s.chunks == 4 ? 2 : 4));
    return (int)std::min<long long>(rows, 148 * std::max(6, 512 / (s.block * s.cluster)));  // 6: the ring kernel's
}

size_t backward_bytes(const ttc_rms_norm_backward_desc& d) {
    const int n = backward_clusters(d.rows, row_shape(d.cols, d.dtype));
    return d.dweight ? align256((size_t)n * d.cols * sizeof(float)) : 0;
}

// Launches `clusters` clusters, or as many as the GPU holds at once: a few more
// than that would take a second round as long as the first. Not under the tail of
// the kernel before: blocks that came while that one still holds part of an SM
// would end up unevenly spread, and these grids count on an even share (43 -> 47
// us for 8192 rows of 4096).
template <class Params>
int launch_rows(void (*kernel)(const Params), const Params& p, const RowShape& s, long long clusters,
                int* launched = nullptr) {
    struct Seen {
        const void* kernel;
        int device, block, cluster, most;
    };
    static Seen seen[64] = {};  // one launch shape an entry; a full table starts over
    static int used = 0;
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof cfg);
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3((unsigned)(clusters * s.cluster), 1, 1);
    cfg.blockDim = dim3((unsigned)s.block, 1, 1);
    cfg.stream = rt().stream;
    cfg.attrs = attr;
    cfg.numAttrs = cluster_attribute(attr[0], s.cluster);
    int most = 0;
    for (int i = 0; i < used && !most; ++i)
        if (seen[i].kernel == (const void*)kernel && seen[i].device == rt().device && seen[i].block == s.block &&
            seen[i].cluster == s.cluster)
            most = seen[i].most;
    if (!most) {
        if (s.cluster > 1) {
            TTC_CUDA(cudaOccupancyMaxActiveClusters(&most, kernel, &cfg));
        } else {
            TTC_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&most, kernel, s.block, 0));
            most *= rt().sm_count;
        }
        if (most < 1) return set_error(TTC_ERR_CUDA, "tt_cuda: rms_norm: a block of %d threads does not fit", s.block);
        if (used == 64) used = 0;
        seen[used++] = {(const void*)kernel, rt().device, s.block, s.cluster, most};
    }
    clusters = std::min<long long>(clusters, most);
    if (launched) *launched = (int)clusters;
    cfg.gridDim.x = (unsigned)(clusters * s.cluster);
    TTC_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return TTC_OK;
}

template <class T, class Y, bool VEC>
int launch_norm(const NormParams& p, const RowShape& s) {
    if (s.block == 0) {
        const long long n = std::min<long long>(p.rows, 2ll * rt().sm_count);
        rms_norm_wide_kernel<T, Y><<<(unsigned)n, kWide, 0, rt().stream>>>(p);
        return check_cuda(cudaGetLastError(), "rms_norm launch");
    }
    if (s.one) {
        const long long n = (p.rows + kWarpRows - 1) / kWarpRows;
        return launch_rows(s.chunks == 1   ? rms_norm_kernel<T, Y, VEC, true, 1>
                           : s.chunks == 2 ? rms_norm_kernel<T, Y, VEC, true, 2>
                                           : rms_norm_kernel<T, Y, VEC, true, 4>,
                           p, s, n);
    }
    // 768 threads an SM rather than the 1024 that fit: 88 us against 97 for 16384 rows of 4096 in bf16
    const long long n = s.cluster > 1 ? p.rows : std::min<long long>(p.rows, 768ll * rt().sm_count / s.block);
    return launch_rows(rms_norm_kernel<T, Y, VEC, false, 2>, p, s, n);
}

template <class T>
int launch_norm_type(const NormParams& p, int y_dtype, const RowShape& s, bool vec) {
    if (y_dtype == TTC_E4M3)
        return vec ? launch_norm<T, __nv_fp8_e4m3, true>(p, s) : launch_norm<T, __nv_fp8_e4m3, false>(p, s);
    return vec ? launch_norm<T, T, true>(p, s) : launch_norm<T, T, false>(p, s);
}

// The ring kernel's shape for the aligned rows that it is faster on; threads 0:
// another kernel takes them. As many blocks an SM as have registers (96 a thread)
// and a ring of three rows each. In us, register kernel / this one, both before they
// looked for rows that leave fp32's range: 16384 x 4096 bf16 94 / 103, 8192 x 8192
// bf16 133 / 108 (now 113), 4096 x 16384 bf16 143 / 125 (now 130), 16384 x 2048 f32
// 92 / 84 (85), 8192 x 8192 f32 231 / 187 (194). 16-bit rows up to 512 chunks have
// twice the arithmetic a byte and more rows on an SM with the register kernel.
struct RingShape {
    int threads, chunks, stages, per_sm;
};
RingShape ring_shape(int cols, int dtype, bool dhidden) {
    const int es = dtype_size(dtype), n = cols / (16 / es);
    const int stage = cols * es * (dhidden ? 3 : 2);
    if (n <= (es == 4 ? 256 : 512) || n > 2048 || cols % (16 / es) || 2 * stage > kRingBytes) return {0, 0, 0, 0};
    const int chunks = n <= 1024 ? 2 : 4, threads = (n + 32 * chunks - 1) / (32 * chunks) * 32;
    int per_sm = std::max(1, std::min(6, 65536 / 96 / threads));
    while (per_sm > 1 && 3 * stage > kRingBytes / per_sm) --per_sm;
    return {threads, chunks, std::min(kMaxStages, kRingBytes / per_sm / stage), per_sm};
}

template <class T>
int launch_ring(const NormBackwardParams& p, const RingShape& s, int& blocks) {
    RingParams q;
    q.p = p;
    q.stages = s.stages;
    q.row_bytes = p.cols * (int)sizeof(T);
    q.stall = stall_test("norm") ? 1 : 0;
    q.wait_limit = q.stall ? kStallTestLimitCycles : kWaitLimitCycles;
    if (int rc = device_status_ptr(&q.status)) return rc;
    const int smem = s.stages * q.row_bytes * (p.dhidden ? 3 : 2);
    auto kernel = s.threads <= 256 ? rms_norm_backward_ring_kernel<T, 2, 256>
                  : s.chunks == 2  ? rms_norm_backward_ring_kernel<T, 2, 512>
                                   : rms_norm_backward_ring_kernel<T, 4, 512>;
    static OncePerDevice once[3];  // one for each of the kernels
    if (int rc = once[s.threads <= 256 ? 0 : s.chunks / 2](rt().device, [&]() -> int {
            TTC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes));
            return TTC_OK;
        }))
        return rc;
    blocks = (int)std::min<long long>(p.rows, (long long)s.per_sm * std::min(rt().sm_count, 148));
    kernel<<<(unsigned)blocks, s.threads, smem, rt().stream>>>(q);
    return check_cuda(cudaGetLastError(), "rms_norm_backward launch");
}

template <class T, bool VEC>
int launch_norm_backward(const NormBackwardParams& p, const RowShape& s, int& clusters) {
    if (VEC) {
        const RingShape ring = ring_shape(p.cols, sizeof(T) == 4 ? TTC_F32 : TTC_BF16, p.dhidden != nullptr);
        if (ring.threads) return launch_ring<T>(p, ring, clusters);
    }
    if (s.block == 0) {
        rms_norm_backward_wide_kernel<T><<<clusters, kWide, 0, rt().stream>>>(p);
        return check_cuda(cudaGetLastError(), "rms_norm_backward launch");
    }
    return launch_rows(!s.one          ? rms_norm_backward_kernel<T, VEC, false, 2>
                       : s.chunks == 1 ? rms_norm_backward_kernel<T, VEC, true, 1>
                       : s.chunks == 2 ? rms_norm_backward_kernel<T, VEC, true, 2>
                                       : rms_norm_backward_kernel<T, VEC, true, 4>,
                       p, s, clusters, &clusters);
}

// Rows of `p` start on boundaries of a whole chunk's elements.
bool rows_aligned(const void* p, int elem_bytes, int per_chunk, long long ld) {
    return !p || ((uintptr_t)p % (elem_bytes * per_chunk) == 0 && ld % per_chunk == 0);
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

int launch_sum_partials(const float* partials, int n, int cols, void* out, int dtype) {
    count_launch();
    const dim3 grid((unsigned)((cols + 31) / 32));
    return launch_overlapped(sum_partials_kernel, grid, 1024, 1, partials, n, cols, out, dtype);
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
    const RowShape s = row_shape(d.cols, d.dtype);
    const NormParams p{d.rows,   d.cols, d.eps, d.x,   d.residual, d.weight,                  d.y,      d.hidden,
                       d.scales, d.ldx,  d.ldr, d.ldy, d.ldh,      d.weight_dtype == TTC_F32, s.cluster};
    const int es = dtype_size(d.dtype), per = 16 / es;
    const bool vec = d.cols % per == 0 && rows_aligned(d.x, es, per, d.ldx) && rows_aligned(d.residual, es, per, d.ldr) &&
                     rows_aligned(d.y, dtype_size(d.y_dtype), per, d.ldy) && rows_aligned(d.hidden, es, per, d.ldh);
    if (int rc = d.dtype == TTC_BF16  ? launch_norm_type<__nv_bfloat16>(p, d.y_dtype, s, vec)
                 : d.dtype == TTC_F16 ? launch_norm_type<__half>(p, d.y_dtype, s, vec)
                                      : launch_norm_type<float>(p, d.y_dtype, s, vec))
        return rc;
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
    const RowShape s = row_shape(d.cols, d.dtype);
    int clusters = backward_clusters(d.rows, s);
    const NormBackwardParams p{d.rows, d.cols, d.eps, d.dy, d.hidden, d.weight, d.dhidden, d.dx,
                               d.dweight ? (float*)d.workspace : nullptr,
                               d.lddy, d.ldh, d.lddh, d.lddx, d.weight_dtype == TTC_F32,
                               d.weight_dtype == d.dtype && (uintptr_t)d.weight % 16 == 0, s.cluster};
    const int es = dtype_size(d.dtype), per = 16 / es;
    const bool vec = d.cols % per == 0 && rows_aligned(d.dy, es, per, d.lddy) && rows_aligned(d.hidden, es, per, d.ldh) &&
                     rows_aligned(d.dhidden, es, per, d.lddh) && rows_aligned(d.dx, es, per, d.lddx);
    auto launch = [&](auto type) {
        using T = decltype(type);
        return vec ? launch_norm_backward<T, true>(p, s, clusters) : launch_norm_backward<T, false>(p, s, clusters);
    };
    if (int rc = d.dtype == TTC_BF16  ? launch(__nv_bfloat16())
                 : d.dtype == TTC_F16 ? launch(__half())
                                      : launch(0.0f))
        return rc;
    count_launch();
    if (int rc = check_cuda(cudaGetLastError(), "rms_norm_backward launch")) return rc;
    return d.dweight ? launch_sum_partials(p.partials, clusters, d.cols, d.dweight, d.weight_dtype) : TTC_OK;
}

}  // extern "C"
