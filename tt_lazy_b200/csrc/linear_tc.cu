// linear_tc.cu -- the matrix products of ttc_linear, ttc_gated_linear and their
// gradients on the 5th-generation tensor cores: tcgen05.mma kind::f16 (F16 and
// BF16 operands) or kind::f8f6f4 (E4M3), fp32 accumulators in tensor memory,
// operands staged by TMA, the epilogue on the way out.
//
// Two kernels:
//   pair_kernel   large products: persistent CTA pairs (cta_group::2), one
//                 256 x 256 tile a pair, operands in a ring of 5 stages.
//   tile_kernel   few rows of x (single tokens, small batches): one 128-wide
//                 tile of the weight's output columns against up to 256 rows,
//                 the weight as the 128-row operand of the instruction, the
//                 sum over K split over the CTAs of a cluster and joined
//                 through distributed shared memory.
//
// Both stage 128 bytes of K a row (64 16-bit or 128 8-bit elements), in the
// 128-byte swizzle, four instructions a stage. An operand whose rows are
// contiguous along K comes as one box; one that is contiguous along M or N (a
// transposed 16-bit operand) as boxes of 64 columns x 64 k-rows.
//
// The gated product is one kernel: the tile's columns are half gate and half
// up columns of the same outputs, so both accumulators of an output are in the
// same tile and the activation and the product happen in the epilogue. A
// product over two segments (dx = dg Wg^T + du Wu^T) runs the k-blocks of the
// second pair of operands after the first's into the same accumulator.
//
// Every wait is bounded, as in the TF32 kernels: an expired one is recorded in
// the status word, the other roles run out too, and the kernel frees what it
// holds and returns. No TMA load is multicast.
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "ffn.cuh"
#include "tc_util.cuh"

namespace ttc {
namespace {

// Warp 0: TMA, warp 1: MMA, warps 2-9: epilogue, two for each quarter of the
// tensor-memory lanes (one each left its scheduler waiting on itself: the
// epilogue of a 256 x 256 tile took 35 us; four each of the pair kernel have 96
// registers and half the columns a step: 37 -> 39 us for 4864 x 4096 x 1024, 58 ->
// 50 with silu, bias and residual).
constexpr int kEpilogueWarps = 8;
constexpr int kThreads = 32 * (2 + kEpilogueWarps);
constexpr int kRow = 128;      // bytes of K a stage holds of each row
constexpr int kBox = 64 * kRow;  // an MN-major box: 64 k-rows of 64 16-bit columns

struct alignas(64) ProductParams {
    CUtensorMap a[2], b[2];
    CUtensorMap out, out2, aside, residual;  // pair_kernel's tensors; out2: or up; aside: pre or gate
    Product p;
    int kb_seg, kb_total;  // k-blocks of one segment, of all segments
    int m_tiles, n_tiles;
    int tok, stages, splits;  // tile_kernel: rows of x a tile, ring stages, CTAs that share a tile
    unsigned idesc;
    int* status;
    long long wait_limit;
    int stall;
};

// The products of one tile_kernel launch. Of two, the second's blocks start at
// `second`; each has blocks in whole clusters, the last of which may have no tile.
template <int N>
struct ProductSet {
    ProductParams q[N];
    unsigned second;
};

template <int GROUP, bool F8>
__device__ __forceinline__ void mma(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                    uint32_t accumulate) {
#define TTC_MMA(GROUP_TEXT, KIND_TEXT)                                                                          \
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma." GROUP_TEXT "." KIND_TEXT         \
                 " [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),                                                  \
                 "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)                                            \
                 : "memory")
    if constexpr (GROUP == 2 && F8)
        TTC_MMA("cta_group::2", "kind::f8f6f4");
    else if constexpr (GROUP == 2)
        TTC_MMA("cta_group::2", "kind::f16");
    else if constexpr (F8)
        TTC_MMA("cta_group::1", "kind::f8f6f4");
    else
        TTC_MMA("cta_group::1", "kind::f16");
#undef TTC_MMA
}

__device__ __forceinline__ void tc_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// How the four instructions of a stage walk an operand's tile. K-major: groups
// of 8 rows every 1024 bytes, each instruction 32 bytes further along the row.
// MN-major: boxes of 64 columns (leading offset kBox), groups of 8 k-rows every
// 1024 bytes, each instruction 16 k-rows = 2048 bytes further.
struct Walk {
    uint32_t lbo, step;
};
__device__ __forceinline__ Walk walk_of(int mn) { return mn ? Walk{kBox, 2048} : Walk{16, 32}; }
__device__ __forceinline__ uint64_t walk_desc(uint32_t base, const Walk& w, int i) {
    return make_desc(base + i * w.step, w.lbo, 1024, kLayoutSW128);
}

// `rows` rows (an operand's M or N index, from row0) of k-block kb.
__device__ __forceinline__ void load_rows(uint32_t dst, const CUtensorMap* map, uint32_t bar, int mn, int kb, int bk,
                                          int row0, int rows) {
    if (!mn) {
        tma_load_2d(dst, map, bar, kb * bk, row0);
    } else {
        for (int j = 0; j < rows; j += 64) tma_load_2d(dst + j * kRow, map, bar, row0 + j, kb * bk);
    }
}

// ---------------------------------------------------------------- pair kernel
// TMA stores from a warp's own shared memory, tracked per issuing thread.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"((uint64_t)map),
                 "r"(src), "r"(c0), "r"(c1)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int PENDING>
__device__ __forceinline__ void tma_store_wait_read() {
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(PENDING) : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Sixteen bytes of DT from floats, and back.
template <int DT>
constexpr int kPer16 = DT == TTC_F32 ? 4 : 8;
template <int DT>
__device__ __forceinline__ uint4 pack16(const float* v) {
    if constexpr (DT == TTC_F32)
        return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    else if constexpr (DT == TTC_BF16)
        return make_uint4(pack2<__nv_bfloat16>(v[0], v[1]), pack2<__nv_bfloat16>(v[2], v[3]),
                          pack2<__nv_bfloat16>(v[4], v[5]), pack2<__nv_bfloat16>(v[6], v[7]));
    else
        return make_uint4(pack2<__half>(v[0], v[1]), pack2<__half>(v[2], v[3]), pack2<__half>(v[4], v[5]),
                          pack2<__half>(v[6], v[7]));
}
template <int DT>
__device__ __forceinline__ void add16(const uint4& a, float* v) {
    if constexpr (DT == TTC_F32) {
        v[0] += __uint_as_float(a.x), v[1] += __uint_as_float(a.y), v[2] += __uint_as_float(a.z);
        v[3] += __uint_as_float(a.w);
    } else {
        float t[8];
        if constexpr (DT == TTC_BF16)
            unpack8<__nv_bfloat16>(a, t);
        else
            unpack8<__half>(a, t);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += t[i];
    }
}

constexpr int kHalf = 128 * kRow;       // one CTA's rows of A, or of B: 16 KB
constexpr int kStageBytes = 2 * kHalf;  // 32 KB
constexpr int kStages = 5;
constexpr int kBuffer = 32 * kRow;      // an epilogue warp's 32 rows of 128 bytes; it has two
constexpr int kPairSmem = kStages * kStageBytes + kEpilogueWarps * 2 * kBuffer + 1024 + 512;
static_assert(kPairSmem <= 232448, "pair kernel: shared memory");
constexpr int kGroupM = 8;  // pair tiles of M that are walked together, so that their operands stay in L2

__device__ __forceinline__ void pair_coords(int tile, int m_tiles, int n_tiles, int& mt, int& nt) {
    const int per_group = kGroupM * n_tiles;
    const int group = tile / per_group, first = group * kGroupM;
    const int rows = min(kGroupM, m_tiles - first), local = tile - group * per_group;
    mt = first + local % rows;
    nt = local / rows;
}

// The epilogue warps' part; true when a wait ran out.
template <int DT, bool GATED>
__device__ __forceinline__ bool pair_epilogue(const ProductParams& q, uint8_t* staging, uint32_t tmem_base,
                                              uint32_t bar0, uint32_t rank) {
    constexpr int W = kRow / (DT == TTC_F32 ? 4 : 2);  // columns of a chunk
    constexpr int G = kPer16<DT>;                      // columns of 16 bytes
    const Product& p = q.p;
    const ProductEpilogue& e = p.epi;
    const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) - 2;
    const int quarter = (w + 2) & 3, which = w >> 2;  // quarter of the tensor-memory lanes; which of its two warps
    uint8_t* const mine = staging + w * 2 * kBuffer;
    const uint32_t mine_addr = smem_u32(mine), res_bar = bar0 + 8u * (2 * kStages + 4 + 2 * w);
    const int tile_cols = GATED ? 128 : 256, chunks = tile_cols / W;
    const int num_tiles = q.m_tiles * q.n_tiles, nclusters = gridDim.x >> 1;
    CopiesInFlight residuals;
    int seq = 0;             // chunks sent so far: the next one goes through buffer seq & 1
    auto slot = [&](int buffer, int i) -> uint4& {  // 16-byte group i of this lane's row
        return *reinterpret_cast<uint4*>(mine + buffer * kBuffer + lane * kRow + ((i ^ (lane & 7)) << 4));
    };
    // TMA writes the chunk of columns from `first` on: aligned tensors, one output
    // tensor, no per-column operand and no 16-byte group that ends inside it (a
    // store that is clipped inside a group writes the whole group).
    auto by_tma = [&](int row0, int first) {
        if (!e.vec || (first + W > p.N && (e.bias || e.row_scales || p.N % G))) return false;
        if (e.split_rows > 0) return row0 + 32 <= e.split_rows || row0 >= e.split_rows + e.split_skip;
        if (e.split_cols > 0) return first + W <= e.split_cols || first >= e.split_cols + e.split_skip;
        return true;
    };
    auto fetch_residual = [&](int buffer, int row0, int first) {
        residuals.sent(buffer);
        if (lane == 0) {
            mbar_arrive_expect_tx(res_bar + 8u * buffer, kBuffer);
            tma_load_2d(mine_addr + buffer * kBuffer, &q.residual, res_bar + 8u * buffer, first, row0);
        }
    };
    auto await_residual = [&](int buffer) {
        return residuals.waited(buffer, __all_sync(0xffffffffu, mbar_wait(res_bar + 8u * buffer, residuals.parity(buffer),
                                                                          q.wait_limit)));
    };
    // Never leave with copies in flight.
    auto leave = [&](bool failed) {
        for (int k = 0; k < 2; ++k)
            if (residuals.on_its_way(k)) await_residual(k);
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        return failed;
    };
    const bool early = e.residual && !e.pre;  // two chunks' residuals before the tile is ready

    int t = 0;
    for (int tile = blockIdx.x >> 1; tile < num_tiles; tile += nclusters, ++t) {
        int mt, nt;
        pair_coords(tile, q.m_tiles, q.n_tiles, mt, nt);
        const int b = t & 1;
        const int row0 = mt * 256 + (int)rank * 128 + quarter * 32, row = row0 + lane;
        const int col0 = nt * tile_cols;
        if (early && row0 < p.M) {
            if (lane == 0) tma_store_wait_read<0>();
            __syncwarp();
            for (int k = 0; k < 2; ++k) {
                const int first = col0 + (which + 2 * k) * W;
                if (first < p.N && by_tma(row0, first)) fetch_residual((seq + k) & 1, row0, first);
            }
        }
        if (!__all_sync(0xffffffffu, mbar_wait(bar0 + 8u * (2 * kStages + b), (t >> 1) & 1, q.wait_limit)))
            return leave(true);
        tc_fence_after();
        const uint32_t acc = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(b * 256);
        const float row_scale = e.row_scales && row < p.M ? e.row_scales[row] : 1.0f;
        auto columns32 = [&](int c, float (&v)[32]) {
            uint32_t r[32];
            tc_ld_32x32b_x32(acc + c, r);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        };
        auto scale32 = [&](const float* scales, int col, float (&v)[32]) {
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                const float4 s = *reinterpret_cast<const float4*>(scales + col + i);
                v[i] *= row_scale * s.x;
                v[i + 1] *= row_scale * s.y;
                v[i + 2] *= row_scale * s.z;
                v[i + 3] *= row_scale * s.w;
            }
        };
        // the value of 32 columns before the activation
        auto linear32 = [&](int c, float (&v)[32]) {
            columns32(c, v);
            if (e.row_scales) scale32(e.col_scales[0], col0 + c, v);
            if (e.bias) {
                const uint4* bias = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(e.bias) +
                                                                   (long long)(col0 + c) * (16 / G));
#pragma unroll
                for (int i = 0; i < 32 / G; ++i) add16<DT>(bias[i], v + i * G);
            }
        };
        auto put32 = [&](int buffer, int h, const float (&v)[32]) {
#pragma unroll
            for (int i = 0; i < 32 / G; ++i) slot(buffer, h * (32 / G) + i) = pack16<DT>(v + i * G);
        };
        auto free_buffer = [&] {  // the store before the last one has read its buffer, which is the next one's
            if (lane == 0) tma_store_wait_read<1>();
            __syncwarp();
        };
        auto send = [&](const CUtensorMap* map, int c, int r) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) tma_store_2d(map, mine_addr + (seq & 1) * kBuffer, c, r);
            ++seq;
        };
        auto release = [&] {  // the accumulator is read: the MMA warp may start the tile after next
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(cluster_addr(bar0 + 8u * (2 * kStages + 2 + b), 0));
        };
        for (int c = which; c < chunks; c += 2) {
            const int first = col0 + c * W;
            const bool last = c + 2 >= chunks;
            if (row0 >= p.M || first >= p.N) {
                if (last) release();
                continue;
            }
            if (by_tma(row0, first)) {
                if constexpr (GATED) {
                    if (e.gate) {
                        for (int k = 0; k < 2; ++k) {
                            free_buffer();
#pragma unroll
                            for (int h = 0; h < W / 32; ++h) {
                                float v[32];
                                columns32(k * 128 + c * W + h * 32, v);
                                if (e.row_scales) scale32(e.col_scales[k], first + h * 32, v);
                                put32(seq & 1, h, v);
                            }
                            send(k == 0 ? &q.aside : &q.out2, first, row0);
                        }
                    }
                    free_buffer();
#pragma unroll
                    for (int h = 0; h < W / 32; ++h) {
                        float v[32], u[32];
                        columns32(c * W + h * 32, v);
                        columns32(128 + c * W + h * 32, u);
                        if (last && h == W / 32 - 1) release();
                        if (e.row_scales) {
                            scale32(e.col_scales[0], first + h * 32, v);
                            scale32(e.col_scales[1], first + h * 32, u);
                        }
                        activate_all<32>(e.act, v);
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] *= u[i];
                        put32(seq & 1, h, v);
                    }
                    send(&q.out, first, row0);
                    continue;
                }
                if (e.pre) {
                    free_buffer();
#pragma unroll
                    for (int h = 0; h < W / 32; ++h) {
                        float v[32];
                        linear32(c * W + h * 32, v);
                        put32(seq & 1, h, v);
                    }
                    send(&q.aside, first, row0);
                }
                const int buffer = seq & 1;
                if (e.residual) {
                    if (!early || c >= 4) {  // not asked for above
                        if (lane == 0) tma_store_wait_read<0>();
                        __syncwarp();
                        fetch_residual(buffer, row0, first);
                    }
                    if (!await_residual(buffer)) return leave(true);
                } else {
                    free_buffer();
                }
#pragma unroll
                for (int h = 0; h < W / 32; ++h) {
                    float v[32];
                    linear32(c * W + h * 32, v);
                    if (last && h == W / 32 - 1) release();
                    activate_all<32>(e.act, v);
                    if (e.residual) {
#pragma unroll
                        for (int i = 0; i < 32 / G; ++i) add16<DT>(slot(buffer, h * (32 / G) + i), v + i * G);
                    }
                    put32(buffer, h, v);
                }
                if (e.split_rows > 0 && row0 >= e.split_rows)
                    send(&q.out2, first, row0 - e.split_rows - e.split_skip);
                else if (e.split_cols > 0 && first >= e.split_cols)
                    send(&q.out2, first - e.split_cols - e.split_skip, row0);
                else
                    send(&q.out, first, row0);
                continue;
            }
            // Element by element: 32 columns at a time (gated: of both products), as
            // fp32 rows of 128 bytes (the products side by side in the two buffers), read
            // back a row at a time with a column a lane.
            if (lane == 0) tma_store_wait_read<0>();
            __syncwarp();
            for (int h = 0; h < W / 32; ++h) {
                const int col = first + h * 32 + lane;
                for (int k = 0; k < (GATED ? 2 : 1); ++k) {
                    float v[32];
                    columns32(k * 128 + c * W + h * 32, v);
#pragma unroll
                    for (int i = 0; i < 8; ++i) slot(k, i) = pack16<TTC_F32>(v + 4 * i);
                }
                if (last && h == W / 32 - 1) release();
                __syncwarp();
                auto at = [&](int k, int r) {
                    return *reinterpret_cast<const float*>(mine + k * kBuffer + r * kRow +
                                                           (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
                };
                if (col < p.N) {
                    const float s0 = e.row_scales ? e.col_scales[0][col] : 1.0f;
                    const float s1 = e.row_scales && GATED ? e.col_scales[1][col] : 1.0f;
                    const float bias = bias_at(e, col);
                    const int rows = min(32, p.M - row0);
#pragma unroll 1
                    for (int r = 0; r < rows; r += 8) {
                        float v[8], u[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            v[i] = at(0, r + i);
                            if (GATED) u[i] = at(1, r + i);
                        }
                        if (GATED)
                            finish_column<DT, true>(e, row0 + r, 1, rows - r, col, v, u, s0, s1, 0.0f);
                        else
                            finish_column<DT, false>(e, row0 + r, 1, rows - r, col, v, u, s0, 1.0f, bias);
                    }
                }
                fence_async_smem();  // TMA may write the buffers next
                __syncwarp();
            }
        }
    }
    return leave(false);
}

// CTA r of a pair holds rows 128 r .. of the A tile and columns 128 r .. of the
// B tile (gated: the gate columns for r = 0, the up columns for r = 1) and gets
// its 128 rows x 256 columns of the result in its own tensor memory, two
// accumulators deep, so that the epilogue of one tile runs under the next.
//
// Epilogue: tensor memory hands each lane one row. A warp takes chunks of 128
// bytes of output (64 columns, 32 of fp32) through its two buffers in shared
// memory, in the 128-byte swizzle, and TMA carries them: the residual into the
// buffer before the tile is ready, the result out of it. Rows and columns past
// the end are clipped there. (Writing the rows with the warps' own 16-byte
// stores instead cost 15 of the 39 us of 1024 x 16384 x 512, and the address
// arithmetic 7 more.) Chunks that TMA cannot write (unaligned tensors, the
// seam of a split output, the last columns of a biased or scaled one or of a
// width that is no multiple of 16 bytes) go element by element, a column a lane.
template <bool F8, bool GATED, int DT>
__global__ void __launch_bounds__(kThreads, 1) pair_kernel(const __grid_constant__ ProductParams q) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* staging = smem + kStages * kStageBytes;
    uint64_t* bars = (uint64_t*)(staging + kEpilogueWarps * 2 * kBuffer);
    uint32_t* tmem_slot = (uint32_t*)(bars + 2 * kStages + 4 + 2 * kEpilogueWarps);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const uint32_t sbase = smem_u32(smem), bar0 = smem_u32(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (kStages + s); };
    auto tfull_bar = [&](int b) { return bar0 + 8u * (2 * kStages + b); };
    auto tempty_bar = [&](int b) { return bar0 + 8u * (2 * kStages + 2 + b); };
    auto res_bar = [&](int w, int k) { return bar0 + 8u * (2 * kStages + 4 + 2 * w + k); };
    const Product& p = q.p;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full_bar(s), rank == 0 ? 2 : 1);  // CTA 0: its own producer and the peer's forward
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(tfull_bar(b), 1);
            mbar_init(tempty_bar(b), 2 * kEpilogueWarps);
        }
        for (int w = 0; w < kEpilogueWarps; ++w)
            for (int k = 0; k < 2; ++k) mbar_init(res_bar(w, k), 1);
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs' barriers are initialised before anyone signals across
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    grid_wait();
    grid_trigger();
    const int num_tiles = q.m_tiles * q.n_tiles;
    const int cluster_id = blockIdx.x >> 1, nclusters = gridDim.x >> 1;
    bool failed = false;

    if (warp == 0) {
        if (lane == 0) {
            constexpr int bk = F8 ? 128 : 64;
            int stage = 0;
            uint32_t phase = 0;
            long long issued = 0;
            for (int tile = cluster_id; tile < num_tiles && !failed && !q.stall; tile += nclusters) {
                int mt, nt;
                pair_coords(tile, q.m_tiles, q.n_tiles, mt, nt);
                const int row0 = mt * 256 + (int)rank * 128;
                const int col0 = GATED ? nt * 128 : nt * 256 + (int)rank * 128;
                for (int kb = 0; kb < q.kb_total; ++kb) {
                    if (!mbar_wait(empty_bar(stage), phase ^ 1, q.wait_limit)) {
                        failed = true;
                        break;
                    }
                    const int seg = kb >= q.kb_seg, k = kb - (seg ? q.kb_seg : 0);
                    mbar_arrive_expect_tx(full_bar(stage), kStageBytes);
                    const uint32_t a_dst = sbase + stage * kStageBytes;
                    load_rows(a_dst, &q.a[seg], full_bar(stage), p.a_mn, k, bk, row0, 128);
                    load_rows(a_dst + kHalf, &q.b[GATED ? rank : seg], full_bar(stage), p.b_mn, k, bk, col0, 128);
                    ++issued;
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
            // Never leave with loads in flight.
            const long long last = issued < kStages ? issued : kStages;
            for (long long i = 0; i < last; ++i) {
                const long long n = issued - 1 - i;
                if (!mbar_wait(full_bar((int)(n % kStages)), (uint32_t)((n / kStages) & 1), q.wait_limit)) failed = true;
            }
        }
    } else if (warp == 1 && rank == 1) {
        if (lane == 0) {
            // forward every completed stage of this CTA to CTA 0's full barrier
            int stage = 0;
            uint32_t phase = 0;
            for (int tile = cluster_id; tile < num_tiles && !failed; tile += nclusters) {
                for (int kb = 0; kb < q.kb_total; ++kb) {
                    if (!mbar_wait(full_bar(stage), phase, q.wait_limit)) {
                        failed = true;
                        break;
                    }
                    mbar_arrive_cluster_relaxed(cluster_addr(full_bar(stage), 0));
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const Walk wa = walk_of(p.a_mn), wb = walk_of(p.b_mn);
            int stage = 0;
            uint32_t phase = 0;
            int t = 0;
            for (int tile = cluster_id; tile < num_tiles && !failed; tile += nclusters, ++t) {
                const int b = t & 1;
                if (!mbar_wait(tempty_bar(b), ((t >> 1) & 1) ^ 1, q.wait_limit)) {
                    failed = true;
                    break;
                }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + (uint32_t)(b * 256);
                for (int kb = 0; kb < q.kb_total; ++kb) {
                    if (!mbar_wait(full_bar(stage), phase, q.wait_limit)) {
                        failed = true;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a_s = sbase + stage * kStageBytes, b_s = a_s + kHalf;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        mma<2, F8>(d_tmem, walk_desc(a_s, wa, i), walk_desc(b_s, wb, i), q.idesc, (kb | i) != 0);
                    tc2_commit(cluster_addr(empty_bar(stage), 0));
                    tc2_commit(cluster_addr(empty_bar(stage), 1));
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1;
                    }
                }
                if (failed) break;
                tc2_commit(cluster_addr(tfull_bar(b), 0));
                tc2_commit(cluster_addr(tfull_bar(b), 1));
            }
        }
    } else {
        failed = pair_epilogue<DT, GATED>(q, staging, tmem_base, bar0, rank);
    }

    if (failed) *(volatile int*)q.status = 1;
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the pair's MMAs and signals are done before TMEM is freed or a CTA exits
    tc_fence_after();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
}

// ---------------------------------------------------------------- tile kernel
// One CTA: 128 output columns (gated: 64 outputs, their gate columns in the
// first half and their up columns in the second) against `tok` rows of x, over
// its share of the k-blocks. The accumulator's lanes are output columns and its
// columns rows of x; it goes to shared memory as [row of x][128] over the ring,
// where the CTAs of the cluster add up each other's shares in rank order, some of
// the rows each.
__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

__device__ __forceinline__ float ld_cluster1(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// Four values at float index i of the tile, added over the cluster's CTAs in rank order.
__device__ __forceinline__ float4 tile_sum4(uint32_t sbase, int splits, int i) {
    float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const uint32_t at = sbase + 4u * (uint32_t)i;
    if (splits == 1) {
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(t.x), "=f"(t.y), "=f"(t.z), "=f"(t.w)
                     : "r"(at)
                     : "memory");
        return t;
    }
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
        const float4 v = ld_cluster(cluster_addr(at, s));
        t.x += v.x, t.y += v.y, t.z += v.z, t.w += v.w;
    }
    return t;
}

// Four consecutive elements of DT, 8 or 16 bytes.
template <int DT>
struct Four {
    using Raw = typename std::conditional<DT == TTC_F32, uint4, uint2>::type;
    static constexpr int kSize = DT == TTC_F32 ? 4 : 2;
    static __device__ __forceinline__ Raw* at(const void* base, long long i) {
        return reinterpret_cast<Raw*>(static_cast<char*>(const_cast<void*>(base)) + i * kSize);
    }
    static __device__ __forceinline__ float4 load(const void* base, long long i) {
        const Raw r = *at(base, i);
        if constexpr (DT == TTC_F32) {
            return make_float4(__uint_as_float(r.x), __uint_as_float(r.y), __uint_as_float(r.z), __uint_as_float(r.w));
        } else {
            using T = typename std::conditional<DT == TTC_BF16, __nv_bfloat16, __half>::type;
            const T *a = reinterpret_cast<const T*>(&r.x), *b = reinterpret_cast<const T*>(&r.y);
            return make_float4(to_f32(a[0]), to_f32(a[1]), to_f32(b[0]), to_f32(b[1]));
        }
    }
    static __device__ __forceinline__ void store(void* base, long long i, const float (&v)[4]) {
        if constexpr (DT == TTC_F32) {
            *at(base, i) = pack16<TTC_F32>(v);
        } else {
            using T = typename std::conditional<DT == TTC_BF16, __nv_bfloat16, __half>::type;
            *at(base, i) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
        }
    }
};

// Rows [r0, r1) of the tile's result, a lane four columns: a warp reads a row of
// the tile (gated: two half rows) with one 512-byte access from each CTA of the
// cluster and writes it with one, four rows on their way at a time. Eight columns
// a thread with every choice made per row took 9 of the 22 us of 256 x 4096 x 4096.
template <int DT, bool GATED>
__device__ __forceinline__ void tile_finish(const ProductParams& q, uint32_t sbase, int m0, int n0, int r0, int r1) {
    const ProductEpilogue& e = q.p.epi;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int j = GATED ? lane & 15 : lane, col = n0 + 4 * j;
    constexpr int kStep = (GATED ? 2 : 1) * kThreads / 32;  // rows of all warps
    constexpr int kAhead = 4;
    float4 s0 = make_float4(1, 1, 1, 1), s1 = s0, bias = make_float4(0, 0, 0, 0);
    if (e.row_scales) {
        s0 = *reinterpret_cast<const float4*>(e.col_scales[0] + col);
        if (GATED) s1 = *reinterpret_cast<const float4*>(e.col_scales[1] + col);
    }
    if (e.bias) bias = Four<DT>::load(e.bias, col);
    for (int r = r0 + (GATED ? 2 * warp + (lane >> 4) : warp); r < r1; r += kAhead * kStep) {
        float v[kAhead][4], u[kAhead][4];
        auto each = [&](auto f) {
#pragma unroll
            for (int a = 0; a < kAhead; ++a)
                if (r + a * kStep < r1) f(a, m0 + r + a * kStep);
        };
        auto get = [](float (&to)[4], const float4& x) { to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w; };
        if (!GATED && e.residual)
            each([&](int a, int row) { get(u[a], Four<DT>::load(e.residual, row * e.ldr + col)); });
        each([&](int a, int row) { get(v[a], tile_sum4(sbase, q.splits, (row - m0) * 128 + 4 * j)); });
        if (GATED) each([&](int a, int row) { get(u[a], tile_sum4(sbase, q.splits, (row - m0) * 128 + 64 + 4 * j)); });
        if (e.row_scales)
            each([&](int a, int row) {
                const float rs = e.row_scales[row];
                v[a][0] *= rs * s0.x, v[a][1] *= rs * s0.y, v[a][2] *= rs * s0.z, v[a][3] *= rs * s0.w;
                if (GATED) u[a][0] *= rs * s1.x, u[a][1] *= rs * s1.y, u[a][2] *= rs * s1.z, u[a][3] *= rs * s1.w;
            });
        if (GATED) {
            if (e.gate)
                each([&](int a, int row) {
                    Four<DT>::store(e.gate, row * e.ldp + col, v[a]);
                    Four<DT>::store(e.up, row * e.ldp + col, u[a]);
                });
        } else {
            if (e.bias)
                each([&](int a, int) { v[a][0] += bias.x, v[a][1] += bias.y, v[a][2] += bias.z, v[a][3] += bias.w; });
            if (e.pre) each([&](int a, int row) { Four<DT>::store(e.pre, row * e.ldp + col, v[a]); });
        }
        if (e.act != TTC_ACT_NONE) {
            float all[4 * kAhead];
#pragma unroll
            for (int i = 0; i < 4 * kAhead; ++i) all[i] = v[i / 4][i % 4];
            activate_all<4 * kAhead>(e.act, all);
#pragma unroll
            for (int i = 0; i < 4 * kAhead; ++i) v[i / 4][i % 4] = all[i];
        }
        if (GATED)
            each([&](int a, int) { v[a][0] *= u[a][0], v[a][1] *= u[a][1], v[a][2] *= u[a][2], v[a][3] *= u[a][3]; });
        else if (e.residual)
            each([&](int a, int) { v[a][0] += u[a][0], v[a][1] += u[a][1], v[a][2] += u[a][2], v[a][3] += u[a][3]; });
        each([&](int a, int row) {
            void* out = e.out;
            int k = col;
            if (!GATED && e.split_rows > 0 && row >= e.split_rows) {
                row -= e.split_rows + e.split_skip;
                if (row < 0) return;
                out = e.out2;
            } else if (!GATED && e.split_cols > 0 && col >= e.split_cols) {  // the seam is in no tile that comes here
                k -= e.split_cols + e.split_skip;
                out = e.out2;
            }
            Four<DT>::store(out, row * e.ldo + k, v[a]);
        });
    }
}

// The same for unaligned tensors and the last columns: a lane a column, eight
// rows at a time. Eight of the warps share the tile: four (gated: two) side by
// side, the others on the rows between.
template <int DT, bool GATED>
__device__ __noinline__ void tile_finish_columns(const ProductParams& q, uint32_t sbase, int m0, int n0, int r0, int r1) {
    constexpr int kAcross = GATED ? 2 : 4, kStep = 8 / kAcross;
    const ProductEpilogue& e = q.p.epi;
    const int warp = threadIdx.x >> 5, c = (warp % kAcross) * 32 + (threadIdx.x & 31), col = n0 + c;
    if (warp >= 8 || col >= q.p.N) return;
    const float s0 = e.row_scales ? e.col_scales[0][col] : 1.0f;
    const float s1 = GATED && e.row_scales ? e.col_scales[1][col] : 1.0f;
    const float bias = bias_at(e, col);
#pragma unroll 1
    for (int r = r0 + warp / kAcross; r < r1; r += 8 * kStep) {
        const int count = min(8, (r1 - r + kStep - 1) / kStep);
        float v[8] = {}, u[8] = {};
        for (int s = 0; s < q.splits; ++s) {  // the cluster's shares in rank order
            const uint32_t from = (q.splits == 1 ? sbase : cluster_addr(sbase, s)) + 4u * (uint32_t)(r * 128 + c);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < count) {
                    v[i] += ld_cluster1(from + 4u * (uint32_t)(i * kStep * 128));
                    if (GATED) u[i] += ld_cluster1(from + 4u * (uint32_t)(i * kStep * 128 + 64));
                }
        }
        finish_column<DT, GATED>(e, m0 + r, kStep, count, col, v, u, s0, s1, bias);
    }
}

// N = 2: both products of a backward pass, which do not wait for one another. One
// launch and dbias without a second one: 79 x 976 x 512 with silu and bias 20.5 ->
// 13.6 us a call, 104 x 440 x 1240 21.2 -> 13.7.
template <bool F8, int N>
__global__ void __launch_bounds__(kThreads) tile_kernel(const __grid_constant__ ProductSet<N> set) {
    const int which = N == 2 && blockIdx.x >= set.second;
    const ProductParams& q = set.q[which];
    const int block = (int)(blockIdx.x - (which ? set.second : 0));
    if (N == 2 && block >= q.m_tiles * q.n_tiles * q.splits) return;  // (splits is 1 here)
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int stage_bytes = kHalf + q.tok * kRow, stages = q.stages;
    uint64_t* bars = (uint64_t*)(smem + stages * stage_bytes);
    uint32_t* tmem_slot = (uint32_t*)(bars + 2 * stages + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t sbase = smem_u32(smem), bar0 = smem_u32(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (stages + s); };
    const uint32_t done_bar = bar0 + 8u * (2 * stages);
    const Product& p = q.p;
    const int splits = q.splits, split = splits > 1 ? (int)cluster_rank() : 0;
    const int tile = block / splits;
    const int m0 = tile % q.m_tiles * q.tok, n0 = tile / q.m_tiles * (p.gated ? 64 : 128);
    const int kb0 = (int)((long long)q.kb_total * split / splits);
    const int kb1 = (int)((long long)q.kb_total * (split + 1) / splits);
    const uint32_t tmem_cols = q.tok <= 32 ? 32 : q.tok <= 64 ? 64 : q.tok <= 128 ? 128 : 256;
    bool failed = false;

    // The first loads go out before the block has met: the barriers they need
    // are this thread's own.
    constexpr int bk = F8 ? 128 : 64;
    auto load = [&](int kb, int stage) {
        const int seg = kb >= q.kb_seg, k = kb - (seg ? q.kb_seg : 0);
        const uint32_t dst = sbase + stage * stage_bytes, bar = full_bar(stage);
        mbar_arrive_expect_tx(bar, stage_bytes);
        if (p.gated) {
            load_rows(dst, &q.b[0], bar, p.b_mn, k, bk, n0, 64);
            load_rows(dst + kHalf / 2, &q.b[1], bar, p.b_mn, k, bk, n0, 64);
        } else {
            load_rows(dst, &q.b[seg], bar, p.b_mn, k, bk, n0, 128);
        }
        load_rows(dst + kHalf, &q.a[seg], bar, p.a_mn, k, bk, m0, q.tok);
    };
    int issued = 0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(done_bar, 1);
        mbar_fence_init();
        grid_wait();
        if (!q.stall)
            for (; issued < stages && kb0 + issued < kb1; ++issued) load(kb0 + issued, issued);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    grid_trigger();

    if (warp == 0) {
        if (lane == 0 && !q.stall) {
            int stage = 0;  // the ring is full, or everything is on its way
            uint32_t phase = 0;
            for (int kb = kb0 + issued; kb < kb1; ++kb) {
                if (!mbar_wait(empty_bar(stage), phase, q.wait_limit)) {
                    failed = true;
                    break;
                }
                load(kb, stage);
                ++issued;
                if (++stage == stages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            const int last = issued < stages ? issued : stages;  // never leave with loads in flight
            for (int i = 0; i < last; ++i) {
                const int n = issued - 1 - i;
                if (!mbar_wait(full_bar(n % stages), (uint32_t)((n / stages) & 1), q.wait_limit)) failed = true;
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const Walk ww = walk_of(p.b_mn), wx = walk_of(p.a_mn);
            int stage = 0;
            uint32_t phase = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(full_bar(stage), phase, q.wait_limit)) {
                    failed = true;
                    break;
                }
                tc_fence_after();
                const uint32_t w_s = sbase + stage * stage_bytes, x_s = w_s + kHalf;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    mma<1, F8>(tmem_base, walk_desc(w_s, ww, i), walk_desc(x_s, wx, i), q.idesc, kb > kb0 || i > 0);
                tc_commit(empty_bar(stage));
                if (++stage == stages) {
                    stage = 0;
                    phase ^= 1;
                }
            }
            if (!failed) tc_commit(done_bar);
        }
    }
    const int rows = min(q.tok, p.M - m0);
    float* const part = reinterpret_cast<float*>(smem);  // [row of x][128] over the ring
    if (warp >= 2) {
        const int quarter = warp & 3;
        if (__all_sync(0xffffffffu, mbar_wait(done_bar, 0, q.wait_limit))) {
            // every load has landed and every instruction has read its stage: the ring is free
            tc_fence_after();
            for (int c = (warp - 2) / 4 * 16; c < rows; c += 32) {
                uint32_t r[16];
                tc_ld_32x32b_x16(tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)c, r);
                tc_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) part[(c + j) * 128 + quarter * 32 + lane] = __uint_as_float(r[j]);
            }
        } else {
            failed = true;
        }
    }
    grid_wait();
    if (failed) *(volatile int*)q.status = 1;
    tc_fence_before();
    __syncthreads();
    if (splits > 1) cluster_sync();
    tc_fence_after();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(tmem_cols)
                     : "memory");

    const int share = (rows + splits - 1) / splits;  // rows that this CTA finishes
    const int r0 = split * share, r1 = min(rows, r0 + share);
    const bool seam = p.epi.split_cols > 0 && n0 < p.epi.split_cols + p.epi.split_skip && n0 + 128 > p.epi.split_cols;
    const bool columns = !p.epi.vec || seam || n0 + (p.gated ? 64 : 128) > p.N;
    auto finish = [&](auto dt, auto gated) {
        if (columns)
            tile_finish_columns<dt(), gated()>(q, sbase, m0, n0, r0, r1);
        else
            tile_finish<dt(), gated()>(q, sbase, m0, n0, r0, r1);
    };
    auto typed = [&](auto dt) {
        if (p.gated)
            finish(dt, std::true_type());
        else
            finish(dt, std::false_type());
    };
    if (p.epi.out_dtype == TTC_BF16)
        typed(std::integral_constant<int, TTC_BF16>());
    else if (p.epi.out_dtype == TTC_F16)
        typed(std::integral_constant<int, TTC_F16>());
    else
        typed(std::integral_constant<int, TTC_F32>());
    if (splits > 1) {  // nobody leaves while its shared memory is still read
        __syncwarp();
        cluster_sync();
    }
}

// ------------------------------------------------------------ padded operands
// TMA wants 16-byte aligned addresses and row pitches. Other operands are
// copied once per call, rows padded to 16 bytes (the padding is never read).
bool aligned16(const Operand& o, int es) { return (uintptr_t)o.ptr % 16 == 0 && (o.ld * es) % 16 == 0; }

struct Copy {
    const uint8_t* src;
    uint8_t* dst;
    long long src_pitch, dst_pitch;  // bytes
    unsigned rows, segments;         // segments of kSegment bytes a row
    int bytes;                       // of a row
};
constexpr int kMaxOperands = 8;  // of two products
struct Copies {
    Copy c[kMaxOperands];
    int n;
    unsigned blocks;  // segments of all rows of all copies
};
constexpr int kSegment = 4096;  // 256 threads, four words each

// A block a segment of a row, in 32-bit words: a word that starts inside a source
// word is put together from two, so that a row is read and written in whole lines
// wherever it starts. The first and last words of a row go byte by byte: nothing
// outside the row is read.
__global__ void __launch_bounds__(256) pad_rows_kernel(const __grid_constant__ Copies all) {
    grid_wait();
    grid_trigger();
    for (unsigned b = blockIdx.x; b < all.blocks; b += gridDim.x) {
        unsigned k = b;
        int which = 0;
        while (k >= all.c[which].rows * all.c[which].segments) k -= all.c[which].rows * all.c[which].segments, ++which;
        const Copy& c = all.c[which];
        const unsigned row = k / c.segments;
        const uint8_t* src = c.src + row * c.src_pitch;
        uint8_t* dst = c.dst + row * c.dst_pitch;
        const int first = (int)(k - row * c.segments) * kSegment + threadIdx.x * 4;
        const int off = (int)((uintptr_t)src & 3);
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = first + i * 1024;
            w[i] = 0;
            if (at >= c.bytes) continue;
            if (at > 0 && at + 8 <= c.bytes) {
                const uint32_t* p = reinterpret_cast<const uint32_t*>(src + at - off);
                w[i] = off ? __funnelshift_r(p[0], p[1], 8 * off) : p[0];
            } else {
                for (int j = 0; j < 4 && at + j < c.bytes; ++j) w[i] |= (uint32_t)src[at + j] << (8 * j);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (first + i * 1024 < c.bytes) *reinterpret_cast<uint32_t*>(dst + first + i * 1024) = w[i];
    }
}

// The operands of a product with their stored shapes.
struct Stored {
    const Operand* o;
    long long rows, cols;  // as stored
};
int stored_operands(const Product& p, Stored (&s)[4]) {
    int n = 0;
    for (int i = 0; i < p.segs; ++i) s[n++] = {&p.a[i], p.a_mn ? p.K : p.M, p.a_mn ? p.M : p.K};
    for (int i = 0; i < (p.gated ? 2 : p.segs); ++i) s[n++] = {&p.b[i], p.b_mn ? p.K : p.N, p.b_mn ? p.N : p.K};
    return n;
}
long long padded_ld(long long cols, int es) { return (cols * es + 15) / 16 * 16 / es; }

int make_map(CUtensorMap* map, const Product& p, const Operand& o, int width, bool mn, int box_rows) {
    const bool f8 = p.dtype == TTC_E4M3;
    const int es = dtype_size(p.dtype);
    const unsigned long long dims[2] = {(unsigned long long)(mn ? width : p.K), (unsigned long long)(mn ? p.K : width)};
    const unsigned long long strides[1] = {(unsigned long long)o.ld};
    const unsigned box[2] = {(unsigned)(kRow / es), (unsigned)(mn ? 64 : box_rows)};
    const CUtensorMapDataType type = f8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    return encode_tensor_map(map, type, es, o.ptr, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// The pair kernel's output side: boxes of 32 rows x 128 bytes.
int make_output_maps(ProductParams& q) {
    const Product& p = q.p;
    const ProductEpilogue& e = p.epi;
    const int es = dtype_size(e.out_dtype);
    auto map = [&](CUtensorMap* m, const void* ptr, long long ld, int rows, int cols) -> int {
        const unsigned long long dims[2] = {(unsigned long long)cols, (unsigned long long)rows};
        const unsigned long long strides[1] = {(unsigned long long)ld};
        const unsigned box[2] = {(unsigned)(kRow / es), 32};
        return encode_tensor_map(m, es == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, es, ptr,
                                 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    };
    const int rows = e.split_rows ? e.split_rows : p.M, cols = e.split_cols ? e.split_cols : p.N;
    if (int rc = map(&q.out, e.out, e.ldo, rows, cols)) return rc;
    if (e.out2)
        if (int rc = map(&q.out2, e.out2, e.ldo, rows, cols)) return rc;
    if (e.gate) {
        if (int rc = map(&q.aside, e.gate, e.ldp, p.M, p.N)) return rc;
        if (int rc = map(&q.out2, e.up, e.ldp, p.M, p.N)) return rc;
    }
    if (e.pre)
        if (int rc = map(&q.aside, e.pre, e.ldp, p.M, p.N)) return rc;
    return e.residual ? map(&q.residual, e.residual, e.ldr, p.M, p.N) : TTC_OK;
}

unsigned instruction(const Product& p, bool a_mn, bool b_mn, int m, int n) {
    const unsigned fmt = p.dtype == TTC_BF16 ? 1u : 0u;  // kind::f16: f16 0, bf16 1; kind::f8f6f4: e4m3 0
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((unsigned)a_mn << 15) | ((unsigned)b_mn << 16) |
           ((unsigned)(n >> 3) << 17) | ((unsigned)(m >> 4) << 24);
}

template <bool F8, bool GATED, int DT>
int launch_pair_as(ProductParams& q) {
    auto kernel = pair_kernel<F8, GATED, DT>;
    static OncePerDevice once;
    static int most[kMaxDevices] = {};
    cudaLaunchConfig_t cfg;
    std::memset(&cfg, 0, sizeof cfg);
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    cfg.numAttrs = launch_attributes(attr, 2);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = kPairSmem;
    cfg.stream = rt().stream;
    int& clusters = most[rt().device];
    if (int rc = once(rt().device, [&]() -> int {
            TTC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem));
            cfg.gridDim = dim3(2 * (rt().sm_count / 2), 1, 1);
            if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess || clusters < 1) {
                cudaGetLastError();
                clusters = rt().sm_count / 2;
            }
            return TTC_OK;
        }))
        return rc;
    const long long tiles = (long long)q.m_tiles * q.n_tiles;
    cfg.gridDim = dim3(2u * (unsigned)std::min<long long>(tiles, clusters), 1, 1);
    TTC_CUDA(cudaLaunchKernelEx(&cfg, kernel, q));
    count_launch();
    return TTC_OK;
}

// An instantiation for each kind of epilogue: the kernel's speed at small K is that
// of fetching the epilogue's instructions.
template <bool F8>
int launch_pair(ProductParams& q) {
    auto typed = [&](auto gated) {
        switch (q.p.epi.out_dtype) {
            case TTC_BF16: return launch_pair_as<F8, gated(), TTC_BF16>(q);
            case TTC_F16: return launch_pair_as<F8, gated(), TTC_F16>(q);
            default: return launch_pair_as<F8, gated(), TTC_F32>(q);
        }
    };
    return q.p.gated ? typed(std::true_type()) : typed(std::false_type());
}

constexpr int kTileExtra = 1024 + 256;  // shared memory beside the ring: alignment, barriers

// A launch of tile_kernel but for its arguments.
struct TileLaunch {
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    TileLaunch(unsigned blocks, int cluster, int ring) {
        std::memset(&cfg, 0, sizeof cfg);
        cfg.attrs = attr;
        cfg.numAttrs = launch_attributes(attr, cluster);
        cfg.blockDim = dim3(kThreads, 1, 1);
        cfg.dynamicSmemBytes = (size_t)ring + kTileExtra;
        cfg.stream = rt().stream;
        cfg.gridDim = dim3(blocks, 1, 1);
    }
};

// Blocks that run at once, in clusters, with a ring of kFullRing bytes: fewer than
// the SMs where a cluster has to fit into what earlier ones leave of a group of SMs.
constexpr int kMaxSplits = 8;
constexpr int kFullRing = 200 * 1024, kHalfRing = 104 * 1024;
bool half_ring_holds(int tok) { return 3 * (kHalf + tok * kRow) <= kHalfRing; }  // three stages
template <bool F8, int N>
int tile_blocks_at_once(int cluster, int* blocks) {
    static OncePerDevice once;
    static int most[kMaxDevices][kMaxSplits + 1] = {};
    auto kernel = tile_kernel<F8, N>;
    if (int rc = once(rt().device, [&]() -> int {
            TTC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448));
            for (int c = 1; c <= kMaxSplits; ++c) {
                const TileLaunch l(rt().sm_count / c * c, c, kFullRing);
                int n = 0;
                if (cudaOccupancyMaxActiveClusters(&n, kernel, &l.cfg) != cudaSuccess || n < 1) {
                    cudaGetLastError();
                    n = rt().sm_count / c;
                }
                most[rt().device][c] = n * c;
            }
            return TTC_OK;
        }))
        return rc;
    *blocks = most[rt().device][cluster];
    return TTC_OK;
}

// The operands that must be copied and where each goes; one that several products
// read is copied once.
struct Padding {
    struct Entry {
        Operand o;
        long long rows, cols;
        size_t at;
    } e[kMaxOperands];
    int n = 0;
    size_t bytes = 0;
    int find(const Stored& s) const {
        int j = 0;
        while (j < n && !(e[j].o.ptr == s.o->ptr && e[j].o.ld == s.o->ld && e[j].rows == s.rows && e[j].cols == s.cols)) ++j;
        return j;
    }
};
Padding padding_of(const Product* products, int count) {
    Padding pad;
    for (int k = 0; k < count; ++k) {
        Stored s[4];
        const int n = stored_operands(products[k], s), es = dtype_size(products[k].dtype);
        for (int i = 0; i < n; ++i) {
            if (aligned16(*s[i].o, es) || pad.find(s[i]) < pad.n) continue;
            pad.e[pad.n++] = {*s[i].o, s[i].rows, s[i].cols, pad.bytes};
            pad.bytes += align256((size_t)s[i].rows * padded_ld(s[i].cols, es) * es);
        }
    }
    return pad;
}

// Copies what must be copied and has the products read the copies.
int pad_operands(Product* products, int count, void* scratch) {
    const Padding pad = padding_of(products, count);
    if (!pad.n) return TTC_OK;
    const int es = dtype_size(products[0].dtype);
    Copies copies = {};
    long long segments = 0;
    for (int j = 0; j < pad.n; ++j) {
        const Padding::Entry& e = pad.e[j];
        const int bytes = (int)e.cols * es;
        const Copy c = {(const uint8_t*)e.o.ptr, (uint8_t*)scratch + e.at, e.o.ld * es, padded_ld(e.cols, es) * es,
                        (unsigned)e.rows, (unsigned)((bytes + kSegment - 1) / kSegment), bytes};
        copies.c[copies.n++] = c;
        segments += (long long)c.rows * c.segments;
    }
    if (segments > INT32_MAX) return set_error(TTC_ERR_UNSUPPORTED, "tt_cuda: unaligned operands are too large");
    for (int k = 0; k < count; ++k) {
        Stored s[4];
        const int n = stored_operands(products[k], s);
        for (int i = 0; i < n; ++i) {
            if (aligned16(*s[i].o, es)) continue;
            const Padding::Entry& e = pad.e[pad.find(s[i])];
            *const_cast<Operand*>(s[i].o) = {(char*)scratch + e.at, padded_ld(e.cols, es)};
        }
    }
    copies.blocks = (unsigned)segments;
    count_launch();
    const dim3 grid((unsigned)std::min<long long>(segments, 64ll * rt().sm_count));
    return launch_overlapped(pad_rows_kernel, grid, 256, 1, copies);
}

// tile_kernel's shape for q.p, and whether pair_kernel is expected to be faster.
int plan_product(ProductParams& q, bool* pair) {
    const Product& p = q.p;
    const int sms = rt().sm_count, bk = kRow / dtype_size(p.dtype);
    q.kb_seg = (p.K + bk - 1) / bk;
    q.kb_total = q.kb_seg * p.segs;
    if (int rc = device_status_ptr(&q.status)) return rc;
    q.stall = stall_test("linear") ? 1 : 0;
    q.wait_limit = q.stall ? kStallTestLimitCycles : kWaitLimitCycles;

    // tile_kernel's shape. Rows a tile: all of x up to 256; fewer where even eight
    // CTAs a tile would leave SMs idle (256 x 1024 x 512: 18.3 us with 8 tiles of
    // 256 rows, 6.2 with 64 tiles of 32). CTAs a tile: until the SMs have one
    // each, and two each for few rows, whose CTAs spend their time waiting for the
    // weight (1 x 4096 x 16384: 24.2 us with 256 CTAs, 28.0 with 128, side by side; 64 x 4096 x
    // 4096: 13.1 us with 128, 15.8 with 256), while every share has at least
    // four k-blocks (two for a few rows, where joining the shares is quick). One CTA
    // an SM takes any number of shares whose clusters run at once (256 x 4608 x 4608:
    // three 20.9 us, two 25.0, four in two rounds 34.1); two an SM take powers of two
    // (clusters of five or seven leave SMs out: 32 x 5120 x 5120 four 14.8, seven 22.4).
    const int unit = p.a_mn ? 64 : 16, width = p.gated ? 64 : 128;
    const int least = p.M <= 16 ? 2 : 4;
    q.n_tiles = (p.N + width - 1) / width;
    const int most_splits = std::max(1, std::min(kMaxSplits, q.kb_total / least));
    q.tok = std::min(256, (p.M + unit - 1) / unit * unit);
    auto tiles = [&] { return ((long long)p.M + q.tok - 1) / q.tok * q.n_tiles; };
    while (q.tok > std::max(32, unit) && tiles() * most_splits < sms) q.tok = (q.tok / 2 + unit - 1) / unit * unit;
    for (q.splits = most_splits; q.splits > 1; --q.splits) {
        int at_once = 0;
        if (int rc = tile_blocks_at_once<false, 1>(q.splits, &at_once)) return rc;
        if (q.tok <= 32 && (q.splits & (q.splits - 1))) continue;
        if (tiles() * q.splits <= (q.tok <= 32 ? 2 * sms : half_ring_holds(q.tok) ? sms : at_once)) break;
    }

    // Which kernel: the shorter estimate, from k-blocks times their measured cost
    // (0.35 us for a pair's 256 x 256, up to 0.42 us for a tile's 128 x 256, both
    // 128 bytes deep) and what starting and ending takes (6 us, and 4 to 9 us with
    // the rows of the tile). Measured, pair / tile, in bf16: 256 x 4096 x 4096 28.4
    // / 18.9 us, 512 rows 28.4 / 24.8, 768 rows 30.2 / 33.8, 1024 rows 29.5 / 34.4;
    // 128 x 16384 x 4096 33.8 / 31.4, 256 rows 34.6 / 41.4; 512 x 2048 x 16384 89.7
    // / 37.0; 2048^3 18.8 / 22.6.
    const int pair_width = p.gated ? 128 : 256;
    const long long pair_m = ((long long)p.M + 255) / 256, pair_n = ((long long)p.N + pair_width - 1) / pair_width;
    if (pair_m * pair_n > INT32_MAX / 2 || tiles() * q.splits > INT32_MAX / 2)
        return set_error(TTC_ERR_UNSUPPORTED, "tt_cuda: too many output tiles");
    auto rounds = [](long long n, long long at_once) { return (double)((n + at_once - 1) / at_once); };
    const double pair_us = 6.0 + 0.35 * q.kb_total * rounds(pair_m * pair_n, sms / 2);
    const double tile_us = 3.5 + 5.5 * q.tok / 256 + 0.42 * (128 + q.tok) / 384 * rounds(q.kb_total, q.splits) *
                                                         rounds(tiles() * q.splits, sms);
    *pair = pair_us < tile_us;
    if (!*pair) q.m_tiles = (p.M + q.tok - 1) / q.tok;
    return TTC_OK;
}

int run_pair(ProductParams& q) {
    const Product& p = q.p;
    q.m_tiles = (p.M + 255) / 256;
    q.n_tiles = p.gated ? (p.N + 127) / 128 : (p.N + 255) / 256;
    q.idesc = instruction(p, p.a_mn, p.b_mn, 256, 256);
    for (int i = 0; i < p.segs; ++i)
        if (int rc = make_map(&q.a[i], p, p.a[i], p.M, p.a_mn, 128)) return rc;
    for (int i = 0; i < (p.gated ? 2 : p.segs); ++i)
        if (int rc = make_map(&q.b[i], p, p.b[i], p.N, p.b_mn, 128)) return rc;
    if (p.epi.vec)
        if (int rc = make_output_maps(q)) return rc;
    return p.dtype == TTC_E4M3 ? launch_pair<true>(q) : launch_pair<false>(q);
}

template <bool F8, int N>
int run_tiles(ProductSet<N>& set) {
    int cluster = 1;
    for (const ProductParams& q : set.q) cluster = std::max(cluster, q.splits);
    unsigned blocks = 0;
    bool small = true;
    for (ProductParams& q : set.q) {
        if (&q != set.q) set.second = blocks;
        const unsigned tiles = (unsigned)q.m_tiles * q.n_tiles * q.splits;
        blocks += (tiles + cluster - 1) / cluster * cluster;
        small = small && half_ring_holds(q.tok);
    }
    // The ring: half an SM's shared memory where not all CTAs run at once otherwise
    // and that holds three stages, so that two meet on an SM and one's loads run
    // under the other's start and end (4 x 16384 x 4096 gated, side by side: 45 us, 51 with the
    // whole of it; 32 x 2048 x 8192 in 16 clusters of 8, of which 15 fit: 11.4 and
    // 22.4); else most of it.
    int at_once = 0;
    if (int rc = tile_blocks_at_once<F8, N>(cluster, &at_once)) return rc;
    const int room = small && blocks > (unsigned)at_once ? kHalfRing : kFullRing;
    int ring = 0;
    for (ProductParams& q : set.q) {
        const Product& p = q.p;
        q.stages = std::min(12, room / (kHalf + q.tok * kRow));
        ring = std::max(ring, q.stages * (kHalf + q.tok * kRow));
        q.idesc = instruction(p, p.b_mn, p.a_mn, 128, q.tok);
        for (int i = 0; i < p.segs; ++i)
            if (int rc = make_map(&q.a[i], p, p.a[i], p.M, p.a_mn, q.tok)) return rc;
        for (int i = 0; i < (p.gated ? 2 : p.segs); ++i)
            if (int rc = make_map(&q.b[i], p, p.b[i], p.N, p.b_mn, p.gated ? 64 : 128)) return rc;
    }
    const TileLaunch l(blocks, cluster, ring);
    TTC_CUDA(cudaLaunchKernelEx(&l.cfg, tile_kernel<F8, N>, set));
    count_launch();
    return TTC_OK;
}

}  // namespace

size_t product_scratch(const Product* products, int count) { return padding_of(products, count).bytes; }

int run_products(const Product* given, int count, void* scratch) {
    if (rt().device < 0 || rt().device >= kMaxDevices)
        return set_error(TTC_ERR_UNSUPPORTED, "tt_cuda: device %d", rt().device);
    Product products[2];
    for (int k = 0; k < count; ++k) products[k] = given[k];
    if (int rc = pad_operands(products, count, scratch)) return rc;
    ProductSet<2> both;
    std::memset(&both, 0, sizeof both);
    bool pair[2] = {};
    for (int k = 0; k < count; ++k) {
        both.q[k].p = products[k];
        if (int rc = plan_product(both.q[k], &pair[k])) return rc;
    }
    // Together only where neither product's sums are split differently than alone.
    const int s0 = both.q[0].splits, s1 = both.q[1].splits;
    if (count == 2 && !pair[0] && !pair[1] && (s0 == s1 || s0 == 1 || s1 == 1)) return run_tiles<false, 2>(both);
    for (int k = 0; k < count; ++k) {
        if (pair[k]) {
            if (int rc = run_pair(both.q[k])) return rc;
            continue;
        }
        ProductSet<1> one;
        one.second = 0;
        one.q[0] = both.q[k];
        if (int rc = products[k].dtype == TTC_E4M3 ? run_tiles<true, 1>(one) : run_tiles<false, 1>(one)) return rc;
    }
    return TTC_OK;
}

}  // namespace ttc
