// The clear half's matrix product on the fifth-generation tensor cores.
//
// One persistent block per SM walks 128 x BN output tiles. Warp 0 streams the operands' 64-k blocks through a ring of
// shared-memory stages with the TMA engine (either operand may have k or its rows adjacent in memory: the instruction
// descriptor says which, nothing is transposed on the way); warp 1 issues the products (tcgen05.mma, 128 x BN x 16) into
// one of two TMEM accumulators; the other warps take the finished accumulator out of TMEM, apply the epilogue in 32 bits
// and store through shared memory, while the next tile's products run.
//
// Waits are bounded (mma::wait): a role that gives up tells the others, the loads and products in flight are waited for
// (bounded as well), TMEM is freed and the block ends; pcb_device_timeouts counts it.
#include "clear_gemm.h"

#include <cstring>

#include "mma.cuh"

namespace pcb {
namespace clear {

using namespace mma;

__device__ unsigned int g_gemm_timeouts;

namespace {

constexpr int SMS = 148;
constexpr int BM = 128, BK = 64;
constexpr float LOG2E = 1.4426950408889634f;

// A tile is 128 x BN by one block, or 256 x BN by a pair (128 rows of A and half of B's rows in each block's shared memory:
// per product each SM reads a third less of it than alone, and half of B crosses from L2 once instead of twice)
template <int BN, int CTAS>
struct Shape {
    static constexpr int B_ROWS = BN / CTAS;
    static constexpr int A_BYTES = BM * BK * 2, B_BYTES = B_ROWS * BK * 2, STAGE = A_BYTES + B_BYTES;
    static constexpr int EWARPS = BN == 64 ? 4 : 8;         // epilogue warps: 4 cover the 128 lanes, 8 halve the columns
    static constexpr int STAGES = BN == 64 ? 8 : STAGE == 32768 ? 5 : 6;
    static constexpr int COLS = BN / (EWARPS / 4);          // columns of one epilogue warp
    static constexpr int THREADS = 64 + 32 * EWARPS;
    static constexpr int TMEM = 2 * BN;
    static constexpr int STAGING = 4096;                    // per epilogue warp: 32 rows x 128 bytes, out and in
    static constexpr size_t SMEM = 1024 + STAGES * STAGE + EWARPS * (2 * STAGING + 128) + 512;
};

struct alignas(64) Params {
    CUtensorMap a, b, y, extra_map;
    int m, n, k;
    int a_mn, b_mn, a_panels, b_panels, bf16;
    int tiles_m, tiles_n, splits, kblocks, kper;  // k blocks in all and of one split
    Act act;
    const void* bias;
    const void* extra;
    void* y_ptr;
    int64_t extra_pitch, y_pitch;
    int bias_type, extra_type, y_type, y_tma, extra_tma, accumulate;
    const float* alpha;
    float* row_sums;
    const VocabRow* rows;
    int col0;
    const int64_t* targets;
    float2* parts;
    float* hit;
};

// ------------------------------------------------------------------------------------------------ epilogue pieces
// GELU z Phi(z) and its slope Phi(z) + z phi(z), two values at a time. Phi from Abramowitz and Stegun 7.1.26 (absolute error
// below 1.5e-7 in erf): for x = |z| / sqrt 2, h = erfc(x) / 2 = (a1 t + ... + a5 t^5) exp(-x^2) / 2, t = 1 / (1 + 0.3275911 x);
// z Phi(z) = max(z, 0) - |z| h, Phi(z) = 1/2 + sign(z) (1/2 - h). A reciprocal and an exponential per value.
__device__ __forceinline__ f32x2 half_erfc(f32x2 z, f32x2 size, f32x2& gauss) {
    float x0, x1, e0, e1;
    parts(fma2(size, both(0.3275911f * 0.70710678118654752f), both(1.0f)), x0, x1);
    const f32x2 t = two(rcp(x0), rcp(x1));
    parts(mul2(mul2(z, both(-0.5f * LOG2E)), z), e0, e1);
    gauss = two(ex2(e0), ex2(e1));
    f32x2 q = fma2(t, both(0.5f * 1.061405429f), both(0.5f * -1.453152027f));
    q = fma2(q, t, both(0.5f * 1.421413741f));
    q = fma2(q, t, both(0.5f * -0.284496736f));
    q = fma2(q, t, both(0.5f * 0.254829592f));
    return mul2(mul2(q, t), gauss);
}
__device__ __forceinline__ f32x2 gelu2(f32x2 z) {
    float z0, z1;
    parts(z, z0, z1);
    const f32x2 size = two(fabsf(z0), fabsf(z1));
    f32x2 g;
    const f32x2 h = half_erfc(z, size, g);
    return fma2(mul2(size, both(-1.0f)), h, two(fmaxf(z0, 0.0f), fmaxf(z1, 0.0f)));
}
__device__ __forceinline__ f32x2 gelu_slope2(f32x2 z) {
    float z0, z1, r0, r1;
    parts(z, z0, z1);
    f32x2 g;
    const f32x2 h = half_erfc(z, two(fabsf(z0), fabsf(z1)), g);
    parts(fma2(h, both(-1.0f), both(0.5f)), r0, r1);
    const f32x2 cdf = add2(two(copysignf(r0, z0), copysignf(r1, z1)), both(0.5f));
    return fma2(mul2(z, both(0.3989422804014327f)), g, cdf);
}
template <int ACT, bool SLOPE>
__device__ __forceinline__ f32x2 act2(const Act& a, f32x2 z) {
    if (ACT == PCB_ACT_GELU) return SLOPE ? gelu_slope2(z) : gelu2(z);
    if (ACT == PCB_ACT_POLY) {
        const f32x2 u = mul2(z, both(a.inv_bound));
        f32x2 r = SLOPE ? both(a.d[6]) : both(a.c[7]);
#pragma unroll
        for (int i = SLOPE ? 5 : 6; i >= 0; --i) r = fma2(r, u, both(SLOPE ? a.d[i] : a.c[i]));
        return r;
    }
    return z;
}

// Sum over the warp's lanes of each of 32 values: lane l returns the sum of v[l], in a fixed order
__device__ __forceinline__ float lane_sums(float* v) {
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int w = 16; w; w >>= 1) {
        const bool up = lane & w;
#pragma unroll
        for (int j = 0; j < w; ++j) {
            const float keep = up ? v[j + w] : v[j], give = up ? v[j] : v[j + w];
            v[j] = keep + __shfl_xor_sync(~0u, give, w);
        }
    }
    return v[0];
}

// 32 x 32 values of a row-major array at (row0, col0), rows and columns past the end as zero, in 32 bits into the warp's
// staging buffer as a box of the TMA engine would lie there; read along the rows (lane = column). For arrays that the engine
// cannot read.
__device__ __noinline__ void load_block(const void* p, int64_t pitch, int type, int row0, int col0, int m, int n, unsigned char* stage) {
    const int lane = threadIdx.x % 32;
    const bool in = col0 + lane < n;
#pragma unroll 16
    for (int r = 0; r < 32; ++r)
        *(float*)(stage + r * 128 + ((lane / 4) ^ (r & 7)) * 16 + lane % 4 * 4) =
            in && row0 + r < m ? load(p, (int64_t)(row0 + r) * pitch + col0 + lane, type) : 0.0f;
    __syncwarp();
}
// A box of the staging buffer (32 rows x 128 bytes, 16-byte pieces swizzled by the row) to rows that the engine cannot write
__device__ __noinline__ void store_block(const unsigned char* stage, bool narrow, void* y, int64_t pitch, int rows, int cols, bool add) {
    const int lane = threadIdx.x % 32;
    for (int r = 0; r < rows; ++r) {
        const unsigned char* row = stage + r * 128;
        for (int c = lane; c < min(cols, narrow ? 64 : 32); c += 32) {
            if (narrow) {
                ((uint16_t*)y)[r * pitch + c] = *(const uint16_t*)(row + ((c / 8) ^ (r & 7)) * 16 + c % 8 * 2);
            } else {
                const float v = *(const float*)(row + ((c / 4) ^ (r & 7)) * 16 + c % 4 * 4);
                float* at = (float*)y + r * pitch + c;
                *at = add ? *at + v : v;
            }
        }
    }
    __syncwarp();
}

// ------------------------------------------------------------------------------------------------ the kernel
template <int BN, int CTAS, int EPI, int ACT>
__global__ void __launch_bounds__(Shape<BN, CTAS>::THREADS, 1) product(const __grid_constant__ Params p) {
    using S = Shape<BN, CTAS>;
    extern __shared__ unsigned char raw[];
    unsigned char* base = (unsigned char*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    unsigned char* staging = base + S::STAGES * S::STAGE;
    float* bias_s = (float*)(staging + S::EWARPS * 2 * S::STAGING);
    uint64_t* full = (uint64_t*)(bias_s + S::EWARPS * 32);
    uint64_t* empty = full + S::STAGES;
    uint64_t* acc_full = empty + S::STAGES;
    uint64_t* acc_empty = acc_full + 2;
    uint64_t* extra_full = acc_empty + 2;
    uint64_t* drain = extra_full + S::EWARPS;
    uint32_t* tmem_at = (uint32_t*)(drain + 1);
    volatile int* dead = (volatile int*)(tmem_at + 1);
    const int warp = warp_index(), lane = threadIdx.x % 32;
    const uint32_t rank = CTAS == 2 ? cluster_rank() : 0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], S::EWARPS * CTAS);
        }
        for (int i = 0; i < S::EWARPS; ++i) mbar_init(&extra_full[i], 1);
        mbar_init(drain, 1);
        mbar_init_fence();
        *dead = 0;
        prefetch_map(&p.a);
        prefetch_map(&p.b);
    }
    if (warp == 1) tmem_alloc<CTAS>(tmem_at, S::TMEM);
    fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync();
    fence_after();
    const uint32_t tmem = *tmem_at;
    pdl_wait();
    pdl_release();

    const int tiles = p.tiles_m * p.tiles_n * p.splits;
    const int first_tile = blockIdx.x / CTAS, stride = gridDim.x / CTAS;
    if (warp == 0) {
        Ring<S::STAGES> r;
        int loaded = 0;
        bool ok = true, ready = true;
        for (int tile = first_tile; tile < tiles && ok; tile += stride) {
            const int sp = tile / (p.tiles_m * p.tiles_n), mn = tile % (p.tiles_m * p.tiles_n);
            const int m0 = (mn % p.tiles_m * CTAS + rank) * BM, n0 = mn / p.tiles_m * BN + rank * S::B_ROWS;
            const int kb0 = sp * p.kper, kb1 = min(p.kblocks, kb0 + p.kper);
            for (int kb = kb0; kb < kb1; ++kb, ++loaded, r.next()) {
                // a fresh barrier's preceding phase counts as done: the first round does not wait
                if (!__all_sync(~0u, ready)) ok = wait_warp(&empty[r.stage], r.phase ^ 1, dead, &g_gemm_timeouts);
                if (!ok) break;
                Ring<S::STAGES> ahead = r;
                ahead.next();
                ready = peek(&empty[ahead.stage], ahead.phase ^ 1);
                unsigned char* sa = base + r.stage * S::STAGE;
                unsigned char* sb = sa + S::A_BYTES;
                uint64_t* bar = &full[r.stage];
                // a pair's loads all complete on the first block's barrier, whose warp issues the products
                const uint32_t pair_bar = CTAS == 2 ? cluster_addr(bar, 0) : 0;
                if (elect()) {
                    if (rank == 0) mbar_expect(bar, CTAS * S::STAGE);
                    auto box = [&](void* dst, const CUtensorMap* map, int x, int y, int z) {
                        if (CTAS == 2) tma_load_pair(dst, map, x, y, z, pair_bar);
                        else tma_load(dst, map, x, y, z, bar);
                    };
                    // rows adjacent: 64 x 64 panels, together in one box where the rows are whole panels (operand_map)
                    if (!p.a_mn) box(sa, &p.a, kb * BK, m0, 0);
                    else if (p.a_panels) box(sa, &p.a, 0, kb * BK, m0 / 64);
                    else
                        for (int j = 0; j < BM / 64; ++j) box(sa + j * 8192, &p.a, m0 + 64 * j, kb * BK, 0);
                    if (!p.b_mn) box(sb, &p.b, kb * BK, n0, 0);
                    else if (p.b_panels) box(sb, &p.b, 0, kb * BK, n0 / 64);
                    else
                        for (int j = 0; j < S::B_ROWS / 64; ++j) box(sb + j * 8192, &p.b, n0 + 64 * j, kb * BK, 0);
                }
                __syncwarp();
            }
        }
        if (!ok && rank == 0)  // the loads in flight: a pair's complete here, before the cluster's end
            for (int i = max(0, loaded - S::STAGES); i < loaded; ++i) mbar_wait(&full[i % S::STAGES], (i / S::STAGES) & 1);
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t idesc = instr_desc(p.bf16, p.a_mn, p.b_mn, BM * CTAS, BN);
            const uint32_t a_lbo = p.a_mn ? 8192 : 16, a_step = (p.a_mn ? 2048 : 32) >> 4;
            const uint32_t b_lbo = p.b_mn ? 8192 : 16, b_step = (p.b_mn ? 2048 : 32) >> 4;
            const uint64_t a_desc = smem_desc(smem_addr(base), a_lbo, 1024), b_desc = smem_desc(smem_addr(base + S::A_BYTES), b_lbo, 1024);
            Ring<S::STAGES> r;
            Ring<2> out;
            bool ok = true, ready = false;
            for (int tile = first_tile; tile < tiles && ok; tile += stride, out.next()) {
                const int sp = tile / (p.tiles_m * p.tiles_n);
                const int kb0 = sp * p.kper, kb1 = min(p.kblocks, kb0 + p.kper);
                ok = wait_warp(&acc_empty[out.stage], out.phase ^ 1, dead, &g_gemm_timeouts);
                if (!ok) break;
                fence_after();
                const uint32_t acc = tmem + out.stage * BN;
                for (int kb = kb0; kb < kb1; ++kb, r.next()) {
                    if (!__all_sync(~0u, ready)) ok = wait_warp(&full[r.stage], r.phase, dead, &g_gemm_timeouts);
                    if (!ok) break;
                    fence_after();
                    Ring<S::STAGES> ahead = r;
                    ahead.next();
                    ready = peek(&full[ahead.stage], ahead.phase);
                    const uint64_t da = a_desc + (uint32_t)(r.stage * (S::STAGE >> 4)), db = b_desc + (uint32_t)(r.stage * (S::STAGE >> 4));
                    if (elect()) {
#pragma unroll
                        for (int q = 0; q < BK / 16; ++q) mma_ss<CTAS>(acc, da + q * a_step, db + q * b_step, idesc, kb > kb0 || q > 0);
                        mma_commit<CTAS>(&empty[r.stage]);
                        if (kb + 1 == kb1) mma_commit<CTAS>(&acc_full[out.stage]);
                    }
                    __syncwarp();
                }
            }
            if (!ok) {  // the products in flight
                if (elect()) mma_commit<CTAS>(drain);
                mbar_wait(drain, 0);
            }
        }
    } else {
        const int ew = warp - 2, quad = warp % 4, half = ew / 4;
        unsigned char* stage = staging + ew * 2 * S::STAGING;
        unsigned char* in = stage + S::STAGING;  // `extra`'s boxes: 32 rows x 128 bytes, the next one on its way
        float* bias = bias_s + ew * 32;
        const float alpha = p.alpha ? *p.alpha : 1.0f;
        const uint32_t leader_empty[2] = {CTAS == 2 ? cluster_addr(&acc_empty[0], 0) : 0, CTAS == 2 ? cluster_addr(&acc_empty[1], 0) : 0};
        auto release = [&](int buf) {  // this warp has the accumulator's values
            fence_before();
            if (lane) return;
            if (CTAS == 2) mbar_arrive_cluster(leader_empty[buf]);
            else mbar_arrive(&acc_empty[buf]);
        };
        // the boxes of `extra` in the order that they are used: box e of a tile covers columns [e ecols, ...) of the warp's
        constexpr bool USES_EXTRA = EPI == EPI_STORE || EPI == EPI_DZ;
        const bool extra_tma = USES_EXTRA && p.extra_tma;
        const int ecols = p.extra_type == PCB_F32 ? 32 : 64;
        int fetched = 0;
        auto fetch = [&](int tile, int e) {
            if (!extra_tma || lane) return;
            while (USES_EXTRA) {  // the next box with columns inside: of this tile, or the first of the next
                if (tile >= tiles) return;
                const int mn = tile % (p.tiles_m * p.tiles_n);
                const int x = mn / p.tiles_m * BN + half * S::COLS + e * ecols;
                if (e * ecols < S::COLS && x < p.n) {
                    const int y = (mn % p.tiles_m * CTAS + rank) * BM + quad * 32;
                    fence_async_smem();
                    mbar_expect(&extra_full[ew], S::STAGING);
                    tma_load(in, &p.extra_map, x, y, &extra_full[ew]);
                    return;
                }
                tile += stride;
                e = 0;
            }
        };
        fetch(first_tile, 0);
        int t = 0;
        for (int tile = first_tile; tile < tiles; tile += stride, ++t) {
            const int sp = tile / (p.tiles_m * p.tiles_n), mn = tile % (p.tiles_m * p.tiles_n);
            const int m0 = (mn % p.tiles_m * CTAS + rank) * BM, tn = mn / p.tiles_m, n0 = tn * BN;
            const int buf = t & 1, row0 = m0 + quad * 32, row = row0 + lane, first = n0 + half * S::COLS;
            auto bias_of = [&](int col) { return col + lane < p.n ? load(p.bias, col + lane, p.bias_type) : 0.0f; };
            float next_bias = 0.0f;
            if (USES_EXTRA && p.bias) next_bias = bias_of(first);
            if (!wait_warp<true>(&acc_full[buf], (t / 2) & 1, dead, &g_gemm_timeouts)) break;
            fence_after();
            const uint32_t acc = tmem + buf * BN + half * S::COLS + ((uint32_t)(quad * 32) << 16);
            const int chunks = min(S::COLS / 32, max(0, (p.n - first + 31) / 32));
            float top = -INFINITY, sum = 0.0f, lse2 = 0.0f, weight = 0.0f;
            int target = -1;  // the row's column among this warp's, if it is there
            if (EPI == EPI_DL && row < p.m) {
                const VocabRow vr = p.rows[row];
                lse2 = vr.lse2, weight = vr.weight, target = vr.target - p.col0 - first;
            }
            if (EPI == EPI_LSE && row < p.m) {
                const int64_t at = p.targets[row] - first;
                target = at >= 0 && at < S::COLS ? (int)at : -1;
            }
            uint32_t held[16];
            for (int c = 0; c < chunks; ++c) {
                const int col0 = first + 32 * c;
                float v[32];
                tmem_ld32(acc + 32 * c, v);
                ld_wait();
                if (c == chunks - 1) release(buf);
                const bool has_target = (EPI == EPI_LSE || EPI == EPI_DL) && __any_sync(~0u, (unsigned)(target - 32 * c) < 32u);
                if (EPI == EPI_LSE) {
                    if (has_target) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (target == 32 * c + j && col0 + j < p.n) p.hit[row] = v[j];
                    }
                    if (col0 + 32 > p.n) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = col0 + j < p.n ? v[j] : -INFINITY;
                    }
                    float m4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                    for (int j = 4; j < 32; ++j) m4[j % 4] = fmaxf(m4[j % 4], v[j]);
                    const float nt = fmaxf(top, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * LOG2E);
                    f32x2 s2[2] = {0, 0};
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        float a, b;
                        parts(fma2(two(v[j], v[j + 1]), both(LOG2E), both(-nt)), a, b);
                        s2[j / 2 % 2] = add2(s2[j / 2 % 2], two(ex2(a), ex2(b)));
                    }
                    float a, b;
                    parts(add2(s2[0], s2[1]), a, b);
                    sum = fmaf(sum, ex2(top - nt), a + b);
                    top = nt;
                    continue;
                }
                if (EPI == EPI_STORE || EPI == EPI_DZ) {
                    if (p.bias) {
                        __syncwarp();
                        bias[lane] = next_bias;
                        __syncwarp();
                        if (c + 1 < chunks) next_bias = bias_of(col0 + 32);
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const float4 q = *(const float4*)(bias + j);
                            parts(add2(two(v[j], v[j + 1]), two(q.x, q.y)), v[j], v[j + 1]);
                            parts(add2(two(v[j + 2], v[j + 3]), two(q.z, q.w)), v[j + 2], v[j + 3]);
                        }
                    }
                    if (ACT != PCB_ACT_NONE) {
#pragma unroll
                        for (int j = 0; j < 32; j += 2) parts(act2<ACT, EPI == EPI_DZ>(p.act, two(v[j], v[j + 1])), v[j], v[j + 1]);
                    }
                    if (p.extra) {
                        const bool wide = !extra_tma || p.extra_type == PCB_F32;
                        if (!extra_tma) {
                            if (lane == 0) bulk_wait_read();
                            __syncwarp();
                            load_block(p.extra, p.extra_pitch, p.extra_type, row0, col0, p.m, p.n, stage);
                        } else if (wide || c % 2 == 0) {
                            if (!wait_warp(&extra_full[ew], fetched++ & 1, dead, &g_gemm_timeouts)) break;
                        }
                        const uint4* irow = (const uint4*)((extra_tma ? in : stage) + lane * 128);
                        auto join = [&](int j, float e0, float e1) {
                            const f32x2 a = two(v[j], v[j + 1]), e = two(e0, e1);
                            parts(EPI == EPI_DZ ? mul2(a, e) : add2(a, e), v[j], v[j + 1]);
                        };
                        if (wide) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const uint4 q = irow[j ^ (lane & 7)];
                                join(4 * j, __uint_as_float(q.x), __uint_as_float(q.y));
                                join(4 * j + 2, __uint_as_float(q.z), __uint_as_float(q.w));
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const uint4 q = irow[(j + (c % 2) * 4) ^ (lane & 7)];
                                const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    float e[2];
                                    unpack2(w[i], p.bf16, e);
                                    join(8 * j + 2 * i, e[0], e[1]);
                                }
                            }
                        }
                        __syncwarp();
                        if (extra_tma && (wide || c % 2 || c + 1 == chunks)) fetch(tile, wide ? c + 1 : c / 2 + 1);
                    }
                    if (EPI == EPI_STORE && p.alpha) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] *= alpha;
                    }
                }
                if (EPI == EPI_DL) {
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        float a, b;
                        parts(fma2(two(v[j], v[j + 1]), both(LOG2E), both(-lse2)), a, b);
                        parts(mul2(two(ex2(a), ex2(b)), both(weight)), v[j], v[j + 1]);
                    }
                    if (has_target) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = target == 32 * c + j ? v[j] - weight : v[j];
                    }
                }
                // ---- to memory: the lane's row of 128 bytes in the staging buffer, 16-byte pieces swizzled by the row;
                // 64 columns of 16 bits fill it (the first 32 wait in registers: the buffer also serves `extra`)
                const bool narrow = p.y_type != PCB_F32;
                uint32_t now[16];
                if (narrow) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) now[j] = pack2(v[2 * j], v[2 * j + 1], p.y_type == PCB_BF16);
                }
                if (EPI == EPI_DZ && p.row_sums) {
                    const float s = lane_sums(v);
                    if (col0 + lane < p.n && row0 < p.m) p.row_sums[(int64_t)(row0 / 32) * p.n + col0 + lane] = s;
                }
                if (narrow && c % 2 == 0 && c + 1 < chunks) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) held[j] = now[j];
                    continue;
                }
                if (lane == 0) bulk_wait_read();
                __syncwarp();
                uint4* srow = (uint4*)(stage + lane * 128);
                if (narrow) {
                    if (c % 2) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            srow[j ^ (lane & 7)] = make_uint4(held[4 * j], held[4 * j + 1], held[4 * j + 2], held[4 * j + 3]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        srow[(j + (c % 2) * 4) ^ (lane & 7)] = make_uint4(now[4 * j], now[4 * j + 1], now[4 * j + 2], now[4 * j + 3]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        srow[j ^ (lane & 7)] = make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]),
                                                          __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]));
                }
                const int box0 = narrow ? col0 - (c % 2) * 32 : col0;
                if (p.y_tma) {
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0 && row0 < p.m) {
                        if (p.accumulate) tma_add(&p.y, box0, row0, sp, stage);
                        else tma_store(&p.y, box0, row0, sp, stage);
                        bulk_commit();
                    }
                } else {
                    __syncwarp();
                    const int64_t at = ((int64_t)sp * p.m + row0) * p.y_pitch + box0;
                    store_block(stage, narrow, (char*)p.y_ptr + at * (narrow ? 2 : 4), p.y_pitch, min(32, p.m - row0), p.n - box0, p.accumulate);
                }
            }
            if (chunks == 0) release(buf);
            if (EPI == EPI_LSE && row < p.m) p.parts[(int64_t)(tn * (S::EWARPS / 4) + half) * p.m + row] = make_float2(top, sum);
        }
        if (lane == 0) bulk_wait();
        if (*dead && extra_tma && lane == 0) mbar_wait(&extra_full[ew], fetched & 1);  // the box in flight
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync();
    fence_after();
    if (warp == 1) tmem_free<CTAS>(tmem, S::TMEM);
}

// y = alpha (act(sum of the splits + bias) + extra), the splits in order
__global__ void __launch_bounds__(256) join(const float* part, int splits, const __grid_constant__ Params p) {
    pdl_wait();
    pdl_release();
    const float alpha = p.alpha ? *p.alpha : 1.0f;
    const int64_t total = (int64_t)p.m * p.n;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        float v = 0.0f;
        for (int s = 0; s < splits; ++s) v += part[s * total + i];
        const int64_t r = i / p.n, c = i % p.n;
        if (p.bias) v += load(p.bias, c, p.bias_type);
        float skip;
        if (p.act.kind == PCB_ACT_GELU) parts(act2<PCB_ACT_GELU, false>(p.act, both(v)), v, skip);
        else if (p.act.kind == PCB_ACT_POLY) parts(act2<PCB_ACT_POLY, false>(p.act, both(v)), v, skip);
        if (p.extra) v += load(p.extra, r * p.extra_pitch + c, p.extra_type);
        store(p.y_ptr, r * p.y_pitch + c, p.y_type, v * alpha);
    }
}

__global__ void __launch_bounds__(256) copy_rows(const uint16_t* x, int64_t pitch, int64_t rows, int cols, uint16_t* y, int64_t to) {
    pdl_wait();
    pdl_release();
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < rows * to; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / to, c = i % to;
        y[i] = c < cols ? x[r * pitch + c] : (uint16_t)0;
    }
}

// ------------------------------------------------------------------------------------------------ host side
typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                           const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                           CUtensorMapFloatOOBfill);
Encode encoder() {
    static Encode f = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return (Encode)p;
    }();
    return f;
}

}  // namespace

int encode_map(CUtensorMap* map, int type, const void* p, int dims, const uint64_t* size, const uint64_t* stride_bytes,
               const uint32_t* box) {
    const Encode f = encoder();
    if (!f) return report(PCB_BAD_ARGS, "the driver has no cuTensorMapEncodeTiled");
    const CUtensorMapDataType t = type == PCB_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                  : type == PCB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                     : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
    const CUresult r = f(map, t, (cuuint32_t)dims, const_cast<void*>(p), size, stride_bytes, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : report(PCB_BAD_ARGS, "cuTensorMapEncodeTiled failed with %d", (int)r);
}

namespace {

// an operand's map, three dimensions always: boxes of 64 adjacent values by `tile` rows (k adjacent), of 64 adjacent rows by
// 64 k (rows adjacent), or of tile / 64 such panels where the rows are a multiple of 64 (each copy costs its issuing warp
// some 80 cycles)
bool panels(const Operand& o, int rows) { return !o.k_adjacent && rows % 64 == 0; }
int operand_map(CUtensorMap* map, const Operand& o, int type, int rows, int k, int tile) {
    const uint64_t pitch = (uint64_t)o.pitch * 2;
    if (panels(o, rows)) {
        const uint64_t size[3] = {64, (uint64_t)k, (uint64_t)rows / 64}, stride[2] = {pitch, 128};
        const uint32_t box[3] = {64, BK, (uint32_t)tile / 64};
        return encode_map(map, type, o.p, 3, size, stride, box);
    }
    const uint64_t size[3] = {(uint64_t)(o.k_adjacent ? k : rows), (uint64_t)(o.k_adjacent ? rows : k), 1};
    const uint64_t stride[2] = {pitch, pitch};
    const uint32_t box[3] = {64, (uint32_t)(o.k_adjacent ? tile : BK), 1};
    return encode_map(map, type, o.p, 3, size, stride, box);
}

// Tile and k splits, from estimated cycles: a 64-k block of a tile costs its products (512 cycles at a width of 256, the
// tensor core's rate) or its bytes into shared memory where they take longer, a tile about 1200 cycles of latency besides, a
// split its 32-bit traffic and the joining launch.
struct Plan {
    int bn, ctas, splits, kper;
};
Plan plan(int m, int n, int k, bool may_split) {
    struct Tile {
        int bn, ctas;
        double block;
    };
    static const Tile shapes[] = {{256, 2, 530}, {128, 2, 300}, {128, 1, 330}, {64, 1, 240}};
    const int kb = (k + BK - 1) / BK;
    Plan best{256, 2, 1, kb};
    double least = 1e300;
    for (const Tile& t : shapes) {
        const int64_t tm = ((int64_t)m + BM * t.ctas - 1) / (BM * t.ctas), tn = ((int64_t)n + t.bn - 1) / t.bn;
        for (int sp = 1; sp <= (may_split ? 16 : 1); sp *= 2) {
            const int per = (kb + sp - 1) / sp;
            if (sp > 1 && (per < 4 || (sp - 1) * per >= kb)) break;
            const int slots = SMS / t.ctas;
            const double waves = (double)((tm * tn * sp + slots - 1) / slots);
            double cost = waves * (per * t.block + t.bn * 2.0) + 1200 + (t.ctas == 2 ? 300 : 0);
            if (sp > 1) cost += 5000 + (double)m * n * 4 * sp * 2 / (SMS * 16.0);
            if (cost < least) least = cost, best = Plan{t.bn, t.ctas, sp, per};
        }
    }
    return best;
}

template <int BN, int CTAS, int EPI, int ACT>
int launch(const Params& p, cudaStream_t s) {
    using S = Shape<BN, CTAS>;
    static_assert(S::SMEM <= 232448, "shared memory");
    static const cudaError_t set = cudaFuncSetAttribute(product<BN, CTAS, EPI, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM);
    if (set != cudaSuccess) return (int)set;
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n * p.splits, slots = SMS / CTAS;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((tiles < slots ? tiles : slots) * CTAS));
    cfg.blockDim = dim3(S::THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = CTAS;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = CTAS == 2 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, product<BN, CTAS, EPI, ACT>, p);
    return PCB_LAUNCH_RESULT();
}
template <int EPI, int ACT>
int launch(const Plan& pl, const Params& p, cudaStream_t s) {
    if (pl.ctas == 2) return pl.bn == 256 ? launch<256, 2, EPI, ACT>(p, s) : launch<128, 2, EPI, ACT>(p, s);
    return pl.bn == 128 ? launch<128, 1, EPI, ACT>(p, s) : launch<64, 1, EPI, ACT>(p, s);
}

}  // namespace

size_t gemm_partial(int m, int n, int k) {
    const Plan pl = plan(m, n, k, true);
    return pl.splits > 1 ? (size_t)pl.splits * m * n : 0;
}
int vocab_parts(int m, int n) {
    const int bn = plan(m, n, 1 << 20, false).bn;
    return (n + bn - 1) / bn * (bn == 64 ? 1 : 2);
}

int gemm(const Gemm& g, cudaStream_t s) {
    // the column blocks of an EPI_LSE product follow vocab_parts, which does not know k
    const Plan pl = plan(g.m, g.n, g.epi == EPI_LSE ? 1 << 20 : g.k, g.epi == EPI_STORE && !g.accumulate && !g.whole);
    const int kb = (g.k + BK - 1) / BK;
    Params p;
    memset(&p, 0, sizeof p);
    if (int rc = operand_map(&p.a, g.a, g.type, g.m, g.k, BM)) return rc;
    if (int rc = operand_map(&p.b, g.b, g.type, g.n, g.k, pl.bn / pl.ctas)) return rc;
    p.m = g.m, p.n = g.n, p.k = g.k;
    p.a_mn = !g.a.k_adjacent, p.b_mn = !g.b.k_adjacent, p.a_panels = panels(g.a, g.m), p.b_panels = panels(g.b, g.n), p.bf16 = g.type == PCB_BF16;
    p.tiles_m = (int)(((int64_t)g.m + BM * pl.ctas - 1) / (BM * pl.ctas)), p.tiles_n = (g.n + pl.bn - 1) / pl.bn;
    p.splits = pl.splits, p.kblocks = kb, p.kper = pl.splits > 1 ? pl.kper : kb;
    p.act = g.act, p.bias = g.bias, p.bias_type = g.bias_type;
    p.extra = g.extra, p.extra_pitch = g.extra_pitch, p.extra_type = g.extra_type;
    p.y_ptr = g.y, p.y_pitch = g.y_pitch, p.y_type = g.y_type, p.accumulate = g.accumulate;
    p.alpha = g.alpha, p.row_sums = g.row_sums, p.rows = g.rows, p.col0 = g.col0, p.targets = g.targets, p.parts = g.parts, p.hit = g.hit;
    Params fin = p;
    if (pl.splits > 1) {  // 32-bit sums of each split, the epilogue in `join`
        p.act = Act{}, p.bias = nullptr, p.extra = nullptr, p.alpha = nullptr;
        p.y_ptr = g.partial, p.y_pitch = g.n, p.y_type = PCB_F32;
    }
    const size_t eb = type_bytes(p.y_type);
    // 16-byte aligned rows go through the TMA engine; others by rows of the staging buffer
    p.y_tma = g.epi != EPI_LSE && ((uintptr_t)p.y_ptr & 15) == 0 && p.y_pitch * eb % 16 == 0;
    if (p.y_tma) {
        const uint64_t size[3] = {(uint64_t)g.n, (uint64_t)g.m, (uint64_t)pl.splits};
        const uint64_t stride[2] = {(uint64_t)p.y_pitch * eb, (uint64_t)p.y_pitch * eb * g.m};
        const uint32_t box[3] = {(uint32_t)(128 / eb), 32, 1};
        if (int rc = encode_map(&p.y, p.y_type, p.y_ptr, 3, size, stride, box)) return rc;
    }
    if (p.extra && ((uintptr_t)p.extra & 15) == 0 && p.extra_pitch * type_bytes(p.extra_type) % 16 == 0) {
        const uint64_t size[2] = {(uint64_t)g.n, (uint64_t)g.m}, stride[1] = {(uint64_t)(p.extra_pitch * type_bytes(p.extra_type))};
        const uint32_t box[2] = {(uint32_t)(128 / type_bytes(p.extra_type)), 32};
        if (int rc = encode_map(&p.extra_map, p.extra_type, p.extra, 2, size, stride, box)) return rc;
        p.extra_tma = 1;
    }
    int rc;
    if (g.epi == EPI_LSE) rc = launch<EPI_LSE, 0>(pl, p, s);
    else if (g.epi == EPI_DL) rc = launch<EPI_DL, 0>(pl, p, s);
    else if (g.epi == EPI_DZ) rc = p.act.kind == PCB_ACT_GELU ? launch<EPI_DZ, PCB_ACT_GELU>(pl, p, s) : launch<EPI_DZ, PCB_ACT_POLY>(pl, p, s);
    else if (p.act.kind == PCB_ACT_GELU) rc = launch<EPI_STORE, PCB_ACT_GELU>(pl, p, s);
    else if (p.act.kind == PCB_ACT_POLY) rc = launch<EPI_STORE, PCB_ACT_POLY>(pl, p, s);
    else rc = launch<EPI_STORE, PCB_ACT_NONE>(pl, p, s);
    if (rc || pl.splits == 1) return rc;
    const int64_t blocks = ((int64_t)g.m * g.n + 255) / 256;
    launch_pdl(join, dim3((unsigned)(blocks < 8 * SMS ? blocks : 8 * SMS)), dim3(256), s, (const float*)g.partial, pl.splits, fin);
    return PCB_LAUNCH_RESULT();
}

size_t aligned_bytes(const void* p, int64_t pitch, int64_t rows, int64_t cols) {
    if (((uintptr_t)p & 15) == 0 && pitch % 8 == 0) return 0;
    return (size_t)rows * ((cols + 7) / 8 * 8) * 2;
}
int align_rows(const void** p, int64_t* pitch, int64_t rows, int64_t cols, void* to, cudaStream_t s) {
    if (!aligned_bytes(*p, *pitch, rows, cols)) return 0;
    const int64_t np = (cols + 7) / 8 * 8;
    const int64_t blocks = (rows * np + 255) / 256;
    launch_pdl(copy_rows, dim3((unsigned)(blocks < 16 * SMS ? blocks : 16 * SMS)), dim3(256), s, (const uint16_t*)*p, *pitch, rows,
               (int)cols, (uint16_t*)to, np);
    *p = to;
    *pitch = np;
    return PCB_LAUNCH_RESULT();
}

unsigned int gemm_timeouts() {
    unsigned int v = 0;
    return cudaMemcpyFromSymbol(&v, g_gemm_timeouts, sizeof v) == cudaSuccess ? v : ~0u;
}

}  // namespace clear
}  // namespace pcb
