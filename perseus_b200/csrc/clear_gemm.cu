// The clear half's matrix product D = A B^T on the fifth-generation tensor cores, with the operators' epilogues.
//
// Persistent blocks, one per SM, walk output tiles of 256 x 256 or 256 x 128 (by pairs of blocks) or 128 x 128 or 128 x 64 (by
// one). Two warps stream the operands' 64-k blocks, A's and B's, through a ring of shared-memory stages with the TMA engine
// (either operand may have k or its rows adjacent in memory: the instruction descriptor says which, nothing is transposed on
// the way; one warp for both took 520 cycles a block, as long as a large tile's products); warp 1 issues the products
// (tcgen05.mma) into one of two TMEM accumulators; eight warps (four for 64 columns) take the finished accumulator out of
// TMEM 32 columns at a time, apply the epilogue in 32 bits and store through shared memory, while the next tile's products
// run.
//
// What bounds it: a pair's 64-k block of a 256 x 256 tile takes 512 cycles of products, and the loop keeps to 505 to 520 of
// them; what falls is the clock (1.5 to 1.6 GHz with all tensor cores busy), so what costs energy costs time: 8192 x 8192 x
// 8192 730 us (1.51 PFLOP/s, 93 % of the measured library rate) with tiles in bands, 790 reading A again for each column.
// At k = 768 the epilogue shares the time: 8192 x 768 x 3072 31.4 us plain, 34.5 under the polynomial (36.4 with a bias), 41
// under GELU (two special functions per value), 44 with a 16-bit residual, 58 with a 32-bit one and result. Short products
// (1024 x 1024 x 1024 8 us) are set-up, one tile's loads and its epilogue.
// The accumulators are 32-bit and truncate: the error of a result grows with k, about 1.2e-9 k of it.
//
// Waits are bounded (mma::wait_warp): a role that gives up tells the others, the loads and products in flight are waited for
// (bounded as well), TMEM is freed and the block ends; pcb_device_timeouts counts it.
#include "clear_gemm.h"

#include <algorithm>
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
// the kernels' epilogues: EPI_STORE without and with `extra`, and the others
enum { KERNEL_STORE, KERNEL_ADD, KERNEL_DZ, KERNEL_LSE, KERNEL_DL };
enum { EXTRA_TMA = 1, EXTRA_COPY = 2, EXTRA_LOAD = 3 };  // how `extra` is read: boxes, 4-byte asynchronous copies, loads

// A tile is 128 x BN by one block, or 256 x BN by a pair (128 rows of A and half of B's rows in each block's shared memory:
// per product each SM reads a third less of it than alone, and half of B crosses from L2 once instead of twice)
template <int BN, int CTAS, int EPI>
struct Shape {
    static constexpr int B_ROWS = BN / CTAS;
    static constexpr int A_BYTES = BM * BK * 2, B_BYTES = B_ROWS * BK * 2, STAGE = A_BYTES + B_BYTES;
    static constexpr int EWARPS = BN == 64 ? 4 : 8;         // epilogue warps: 4 cover the 128 lanes, 8 halve the columns
    static constexpr int COLS = BN / (EWARPS / 4);          // columns of one epilogue warp
    // 64-k blocks that one turn of the products' loop takes. A turn's waiting, electing and committing cost some 150 cycles, a
    // product's issue 40: a block of a tile of 256 columns keeps the tensor core longer than that (512 cycles), one of 128
    // columns does not (2048 x 3072 x 768: 15.5 us by twos, 16.5 by ones; 8192 x 768 x 3072 by 256 columns 32.1 and 31.0)
    static constexpr int AT_ONCE = BN == 256 ? 1 : 2;
    static constexpr int THREADS = 96 + 32 * EWARPS;
    static constexpr int TMEM = 2 * BN;
    static constexpr int STAGING = 4096;                    // per epilogue warp and direction: 32 rows x 128 bytes
    static constexpr int BUFFERS = EPI == KERNEL_ADD || EPI == KERNEL_DZ ? 2 : 1;
    static constexpr int STAGES = BN == 64 ? 8 : STAGE == 32768 ? (BUFFERS == 2 ? 5 : 6) : (BUFFERS == 2 ? 6 : 8);
    static constexpr size_t SMEM = 1024 + STAGES * STAGE + EWARPS * (BUFFERS * STAGING + 128) + 512;
};

struct alignas(64) Params {
    CUtensorMap a, b, y, extra_map, part;
    int m, n, k;
    int a_mn, b_mn, a_panels, b_panels, bf16;
    int a_bytes;  // of one block's loads of A: fewer than the stage's where A has few rows
    int tiles_m, tiles_n, band, kblocks;
    // Units of work: tiles [0, whole) entire, then the other `tail` tiles in `splits` parts of `kper` k blocks: to 32-bit
    // sums that `join` finishes, or (slices) each part to its own y
    int whole, tail, splits, kper, slices;
    Act act;
    const void* bias;
    const void* extra;
    void* y_ptr;
    int64_t extra_pitch, y_pitch;
    int bias_type, extra_type, y_type, y_tma, extra_mode, accumulate;
    const float* alpha;
    float* row_sums;
    const float* sizes;
    int nsizes;
    float slope;
    float* unscale;
    const VocabRow* rows;
    int col0;
    const int64_t* targets;
    float2* parts;
    float* hit;
};

struct Unit {
    int tile, split, kb0, kb1, tm, tn;
    bool partial;
};
// Tile number `tile`'s row and column of tiles: down all rows of tiles, or (BANDS) down `band` of them at a time, column
// after column (`gemm` says when)
template <bool BANDS>
__device__ __forceinline__ void place(const Params& p, int tile, int& tm, int& tn) {
    int at = 0, h = p.tiles_m;
    if (BANDS) {
        const int per = p.band * p.tiles_n, b = tile / per;
        at = b * p.band, h = min(p.band, p.tiles_m - at), tile -= b * per;
    }
    tn = tile / h;
    tm = at + tile - tn * h;
}
template <bool BANDS>
__device__ __forceinline__ Unit unit_of(const Params& p, int u) {
    Unit w = {u, 0, 0, p.kblocks, 0, 0, false};
    if (u >= p.whole) {
        w.split = (u - p.whole) / p.tail;
        w.tile = u - w.split * p.tail;
        w.kb0 = w.split * p.kper;
        w.kb1 = min(p.kblocks, w.kb0 + p.kper);
        w.partial = !p.slices;
    }
    place<BANDS>(p, w.tile, w.tm, w.tn);
    return w;
}

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
    float z0, z1, f0, f1;
    parts(z, z0, z1);
    f32x2 g;
    const f32x2 h = half_erfc(z, two(fabsf(z0), fabsf(z1)), g);
    // |z| h at +inf is 0: a finite value for it there (-inf and NaN go through to NaN)
    asm("min.NaN.f32 %0, %1, 0f7F7FFFFF;" : "=f"(f0) : "f"(z0));
    asm("min.NaN.f32 %0, %1, 0f7F7FFFFF;" : "=f"(f1) : "f"(z1));
    return fma2(two(-fabsf(f0), -fabsf(f1)), h, two(fmaxf(z0, 0.0f), fmaxf(z1, 0.0f)));
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

// Sum over the warp's lanes of each of N values, in a fixed order: lane l returns the sum of v[l % N]
template <int N>
__device__ __forceinline__ float lane_sums(float* v) {
    const int lane = threadIdx.x % 32;
#pragma unroll
    for (int w = N / 2; w; w >>= 1) {
        const bool up = lane & w;
#pragma unroll
        for (int j = 0; j < w; ++j) {
            const float keep = up ? v[j + w] : v[j], give = up ? v[j] : v[j + w];
            v[j] = keep + __shfl_xor_sync(~0u, give, w);
        }
    }
#pragma unroll
    for (int w = N; w < 32; w <<= 1) v[0] += __shfl_xor_sync(~0u, v[0], w);
    return v[0];
}

// 32 x 32 values of a row-major array at (row0, col0), rows and columns past the end as zero, in 32 bits to where a box of
// the TMA engine would put them; along the rows (lane = column). For arrays that the engine cannot read: 32-bit values by
// asynchronous copies of 4 bytes (copy_wait, then __syncwarp), 16-bit ones by loads.
__device__ __forceinline__ uint32_t block_at(int r, int c) { return r * 128 + ((c / 4) ^ (r & 7)) * 16 + c % 4 * 4; }
__device__ __noinline__ void copy_block(const void* p, int64_t pitch, int row0, int col0, int m, int n, unsigned char* to) {
    const int lane = threadIdx.x % 32;
    const bool in = col0 + lane < n;
    const float* x = (const float*)p + (int64_t)row0 * pitch + col0 + lane;
#pragma unroll 8
    for (int r = 0; r < 32; ++r, x += pitch) {
        const bool here = in && row0 + r < m;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_addr(to + block_at(r, lane))), "l"(here ? (const void*)x : p),
                     "r"(here ? 4 : 0)
                     : "memory");
    }
}
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __noinline__ void load_block(const void* p, int64_t pitch, int type, int row0, int col0, int m, int n, unsigned char* to) {
    const int lane = threadIdx.x % 32;
    const bool in = col0 + lane < n;
    float v[32];
#pragma unroll
    for (int r = 0; r < 32; ++r) v[r] = in && row0 + r < m ? load(p, (int64_t)(row0 + r) * pitch + col0 + lane, type) : 0.0f;
#pragma unroll
    for (int r = 0; r < 32; ++r) *(float*)(to + block_at(r, lane)) = v[r];
    __syncwarp();
}
// A box of the staging buffer (32 rows x 128 bytes, 16-byte pieces swizzled by the row) to rows that the engine cannot write,
// eight rows at a time
__device__ __noinline__ void store_block(const unsigned char* stage, bool narrow, void* y, int64_t pitch, int rows, int cols, bool add) {
    const int lane = threadIdx.x % 32;
    for (int r0 = 0; r0 < rows; r0 += 8) {
        if (narrow) {
            uint16_t v[2][8];
#pragma unroll
            for (int r = 0; r < 8; ++r)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int c = lane + 32 * h;
                    v[h][r] = *(const uint16_t*)(stage + (r0 + r) * 128 + ((c / 8) ^ r) * 16 + c % 8 * 2);
                }
#pragma unroll
            for (int r = 0; r < 8; ++r)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (r0 + r < rows && lane + 32 * h < cols) ((uint16_t*)y)[(r0 + r) * pitch + lane + 32 * h] = v[h][r];
        } else {
            float v[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] = *(const float*)(stage + block_at(r0 + r, lane));
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                float* at = (float*)y + (r0 + r) * pitch + lane;
                if (r0 + r < rows && lane < cols) *at = add ? *at + v[r] : v[r];
            }
        }
    }
    __syncwarp();
}

// ------------------------------------------------------------------------------------------------ the kernel
template <int BN, int CTAS, int EPI, int ACT, bool BANDS>
__global__ void __launch_bounds__(Shape<BN, CTAS, EPI>::THREADS, 1) product(const __grid_constant__ Params p) {
    using S = Shape<BN, CTAS, EPI>;
    extern __shared__ unsigned char raw[];
    unsigned char* base = (unsigned char*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    unsigned char* staging = base + S::STAGES * S::STAGE;
    float* bias_s = (float*)(staging + S::EWARPS * S::BUFFERS * S::STAGING);
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
            mbar_init(&full[i], 2);  // A's warp and B's
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

    const int units = p.whole + p.tail * p.splits;
    const int first_unit = blockIdx.x / CTAS, stride = gridDim.x / CTAS;
    if (warp == 0 || warp == 2) {  // A's blocks and B's
        const bool b_side = warp == 2;
        const CUtensorMap* map = b_side ? &p.b : &p.a;
        // rows adjacent: 64 x 64 panels, together in one box where the rows are whole panels (operand_map)
        const int mn = b_side ? p.b_mn : p.a_mn, panels = b_side ? p.b_panels : p.a_panels;
        const int boxes = mn && !panels ? (b_side ? S::B_ROWS : BM) / 64 : 1;
        const uint32_t bytes = CTAS * (b_side ? S::B_BYTES : p.a_bytes);
        unsigned char* to = base + (b_side ? S::A_BYTES : 0);
        Ring<S::STAGES> r;
        int loaded = 0;
        bool ok = true, ready = true;
        for (int u = first_unit; u < units && ok; u += stride) {
            const Unit w = unit_of<BANDS>(p, u);
            const int row = b_side ? w.tn * BN + rank * S::B_ROWS : (w.tm * CTAS + rank) * BM;
            int x = !mn ? w.kb0 * BK : panels ? 0 : row, y = mn ? w.kb0 * BK : row;
            const int z = mn && panels ? row / 64 : 0, dx = mn ? 0 : BK, dy = mn ? BK : 0;
            for (int kb = w.kb0; kb < w.kb1; ++kb, ++loaded, x += dx, y += dy, r.next()) {
                // a fresh barrier's preceding phase counts as done: the first round does not wait
                if (!__all_sync(~0u, ready)) ok = wait_warp(&empty[r.stage], r.phase ^ 1, dead, &g_gemm_timeouts);
                if (!ok) break;
                Ring<S::STAGES> ahead = r;
                ahead.next();
                ready = peek(&empty[ahead.stage], ahead.phase ^ 1);
                unsigned char* at = to + r.stage * S::STAGE;
                uint64_t* bar = &full[r.stage];
                // a pair's loads all complete on the first block's barrier, whose warp issues the products
                const uint32_t pair_bar = CTAS == 2 ? cluster_addr(bar, 0) : 0;
                if (elect()) {
                    if (rank == 0) mbar_expect(bar, bytes);
                    auto box = [&](int j) {
                        if (CTAS == 2) tma_load_pair(at + j * 8192, map, x + 64 * j, y, z, pair_bar);
                        else tma_load(at + j * 8192, map, x + 64 * j, y, z, bar);
                    };
                    box(0);
                    for (int j = 1; j < boxes; ++j) box(j);
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
            for (int u = first_unit; u < units && ok; u += stride) {
                const Unit w = unit_of<BANDS>(p, u);
                if (w.kb0 >= w.kb1) continue;
                ok = wait_warp(&acc_empty[out.stage], out.phase ^ 1, dead, &g_gemm_timeouts);
                if (!ok) break;
                fence_after();
                const uint32_t acc = tmem + out.stage * BN;
                for (int kb = w.kb0; kb < w.kb1; kb += S::AT_ONCE) {
                    const bool two = S::AT_ONCE == 2 && kb + 1 < w.kb1;
                    Ring<S::STAGES> second = r;
                    second.next();
                    if (!__all_sync(~0u, ready)) {
                        ok = wait_warp(&full[r.stage], r.phase, dead, &g_gemm_timeouts);
                        if (two) ok = ok && wait_warp(&full[second.stage], second.phase, dead, &g_gemm_timeouts);
                    }
                    if (!ok) break;
                    fence_after();
                    const uint64_t da = a_desc + (uint32_t)(r.stage * (S::STAGE >> 4)), db = b_desc + (uint32_t)(r.stage * (S::STAGE >> 4));
                    const uint64_t da2 = a_desc + (uint32_t)(second.stage * (S::STAGE >> 4)), db2 = b_desc + (uint32_t)(second.stage * (S::STAGE >> 4));
                    uint64_t* done[2] = {&empty[r.stage], &empty[second.stage]};
                    r = second;
                    if (two) r.next();
                    ready = peek(&full[r.stage], r.phase);
                    if (S::AT_ONCE == 2) {
                        Ring<S::STAGES> ahead = r;
                        ahead.next();
                        ready = ready && peek(&full[ahead.stage], ahead.phase);
                    }
                    if (elect()) {
#pragma unroll
                        for (int q = 0; q < BK / 16; ++q) mma_ss<CTAS>(acc, da + q * a_step, db + q * b_step, idesc, kb > w.kb0 || q > 0);
                        mma_commit<CTAS>(done[0]);
                        if (two) {
#pragma unroll
                            for (int q = 0; q < BK / 16; ++q) mma_ss<CTAS>(acc, da2 + q * a_step, db2 + q * b_step, idesc, true);
                            mma_commit<CTAS>(done[1]);
                        }
                        if (kb + S::AT_ONCE >= w.kb1) mma_commit<CTAS>(&acc_full[out.stage]);
                    }
                    __syncwarp();
                }
                out.next();
            }
            if (!ok) {  // the products in flight
                if (elect()) mma_commit<CTAS>(drain);
                mbar_wait(drain, 0);
            }
        }
    } else {
        const int ew = warp - 3, quad = warp % 4, half = ew / 4;
        unsigned char* stage = staging + ew * S::BUFFERS * S::STAGING;
        unsigned char* in = stage + (S::BUFFERS - 1) * S::STAGING;  // `extra`'s boxes: 32 rows x 128 bytes, the next one on its way
        float* bias = bias_s + ew * 32;
        const float alpha = p.alpha ? *p.alpha : 1.0f;
        float factor = 1.0f;
        if (EPI == KERNEL_DZ && p.sizes) {
            float big = 0.0f;
            for (int i = lane; i < p.nsizes; i += 32) big = fmaxf(big, p.sizes[i]);
            for (int i = 16; i; i >>= 1) big = fmaxf(big, __shfl_xor_sync(~0u, big, i));
            big *= p.slope;
            const int e = big > 0.0f ? max(-100, min(100, 134 - (int)(__float_as_uint(big) >> 23))) : 0;  // big in [2^(7-e), 2^(8-e))
            factor = __uint_as_float((127 + e) << 23);
            if (blockIdx.x == 0 && ew == 0 && lane == 0) *p.unscale = __uint_as_float((127 - e) << 23);
        }
        const uint32_t leader_empty[2] = {CTAS == 2 ? cluster_addr(&acc_empty[0], 0) : 0, CTAS == 2 ? cluster_addr(&acc_empty[1], 0) : 0};
        auto release = [&](int buf) {  // this warp has the accumulator's values
            fence_before();
            if (lane) return;
            if (CTAS == 2) mbar_arrive_cluster(leader_empty[buf]);
            else mbar_arrive(&acc_empty[buf]);
        };
        // the boxes of `extra` in the order that they are used: box e of a tile covers columns [e ecols, ...) of the warp's
        constexpr int W = 32;  // columns at a time (16: 5 to 15 % slower)
        constexpr bool HAS_EXTRA = S::BUFFERS == 2, AFFINE = HAS_EXTRA || EPI == KERNEL_STORE;
        const bool extra_wide = p.extra_mode != EXTRA_TMA || p.extra_type == PCB_F32;
        const int ecols = extra_wide ? 32 : 64;
        int fetched = 0;
        auto fetch = [&](int u, int e) {
            if (p.extra_mode == EXTRA_LOAD) return;
            for (; HAS_EXTRA && u < units; u += stride, e = 0) {  // the next box with columns inside: of this unit, or the first of a later one
                const Unit w = unit_of<BANDS>(p, u);
                const int x = w.tn * BN + half * S::COLS + e * ecols;
                if (w.partial || e * ecols >= S::COLS || x >= p.n) continue;
                const int y = (w.tm * CTAS + rank) * BM + quad * 32;
                if (p.extra_mode == EXTRA_TMA) {
                    if (lane == 0) {
                        fence_async_smem();
                        mbar_expect(&extra_full[ew], S::STAGING);
                        tma_load(in, &p.extra_map, x, y, &extra_full[ew]);
                    }
                } else {
                    copy_block(p.extra, p.extra_pitch, y, x, p.m, p.n, in);
                }
                return;
            }
        };
        if constexpr (HAS_EXTRA) fetch(first_unit, 0);
        int t = 0;
        for (int u = first_unit; u < units; u += stride) {
            const Unit w = unit_of<BANDS>(p, u);
            if (w.kb0 >= w.kb1) continue;
            const int m0 = (w.tm * CTAS + rank) * BM, tn = w.tn, n0 = tn * BN;
            const int buf = t & 1, row0 = m0 + quad * 32, row = row0 + lane, first = n0 + half * S::COLS;
            auto bias_of = [&](int col) { return col + lane < p.n ? load(p.bias, col + lane, p.bias_type) : 0.0f; };
            float biases[S::COLS / 32];  // the lane's column of each 32, read while the products still run
            if (AFFINE && p.bias && !w.partial) {
#pragma unroll
                for (int i = 0; i < S::COLS / 32; ++i) biases[i] = bias_of(first + 32 * i);
            }
            if (!wait_warp<true>(&acc_full[buf], (t / 2) & 1, dead, &g_gemm_timeouts)) break;
            ++t;
            fence_after();
            const uint32_t acc = tmem + buf * BN + half * S::COLS + ((uint32_t)(quad * 32) << 16);
            const int chunks = min(S::COLS / W, max(0, (p.n - first + W - 1) / W));
            float top = -INFINITY, sum = 0.0f, lse = 0.0f, weight = 0.0f;
            int target = -1;  // the row's column among this warp's, if it is there
            bool off = false, any_off = false;
            if (EPI == KERNEL_DL && row < p.m) {
                const VocabRow vr = p.rows[row];
                lse = vr.lse, weight = vr.weight, target = vr.target - p.col0 - first, off = vr.off;
            }
            if (EPI == KERNEL_DL) any_off = __any_sync(~0u, off);
            if (EPI == KERNEL_LSE && row < p.m) {
                const int64_t at = p.targets[row] - first;
                target = at >= 0 && at < S::COLS ? (int)at : -1;
            }
            for (int c = 0; c < chunks; ++c) {
                const int col0 = first + W * c;
                float v[W];
                tmem_ld32(acc + W * c, v);
                ld_wait();
                if (c == chunks - 1) release(buf);
                const bool has_target = (EPI == KERNEL_LSE || EPI == KERNEL_DL) && __any_sync(~0u, (unsigned)(target - W * c) < (unsigned)W);
                if (EPI == KERNEL_LSE) {
                    if (has_target) {
#pragma unroll
                        for (int j = 0; j < W; ++j)
                            if (target == W * c + j && col0 + j < p.n) p.hit[row] = v[j];
                    }
                    if (col0 + W > p.n) {
#pragma unroll
                        for (int j = 0; j < W; ++j) v[j] = col0 + j < p.n ? v[j] : -INFINITY;
                    }
                    float m4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                    for (int j = 4; j < W; ++j) m4[j % 4] = fmaxf(m4[j % 4], v[j]);
                    // Differences first, to base 2 after: a finite logit times log2 e may not be finite. Where all are -inf so
                    // far, 0 in place of the maximum: they weigh nothing
                    const float nt = fmaxf(top, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]))), sub = nt == -INFINITY ? 0.0f : nt;
                    f32x2 s2[2] = {0, 0};
#pragma unroll
                    for (int j = 0; j < W; j += 2) {
                        float a, b;
                        parts(mul2(add2(two(v[j], v[j + 1]), both(-sub)), both(LOG2E)), a, b);
                        s2[j / 2 % 2] = add2(s2[j / 2 % 2], two(ex2(a), ex2(b)));
                    }
                    float a, b;
                    parts(add2(s2[0], s2[1]), a, b);
                    sum = fmaf(sum, ex2((top - sub) * LOG2E), a + b);
                    top = nt;
                    continue;
                }
                const bool partial = AFFINE && w.partial;  // 32-bit sums for `join`, in tiles of their own
                if (AFFINE && !partial) {
                    if (p.bias) {
                        if (W * c % 32 == 0) {
                            __syncwarp();
                            float b = biases[0];
#pragma unroll
                            for (int i = 1; i < S::COLS / 32; ++i) b = W * c / 32 == i ? biases[i] : b;
                            bias[lane] = b;
                            __syncwarp();
                        }
#pragma unroll
                        for (int j = 0; j < W; j += 4) {
                            const float4 q = *(const float4*)(bias + W * c % 32 + j);
                            parts(add2(two(v[j], v[j + 1]), two(q.x, q.y)), v[j], v[j + 1]);
                            parts(add2(two(v[j + 2], v[j + 3]), two(q.z, q.w)), v[j + 2], v[j + 3]);
                        }
                    }
                    if (ACT != PCB_ACT_NONE) {
#pragma unroll
                        for (int j = 0; j < W; j += 2) parts(act2<ACT, EPI == KERNEL_DZ>(p.act, two(v[j], v[j + 1])), v[j], v[j + 1]);
                    }
                    if constexpr (HAS_EXTRA) {
                        const int per = ecols / W, part = c % per;  // of a box
                        if (part == 0) {
                            if (p.extra_mode == EXTRA_LOAD) {
                                load_block(p.extra, p.extra_pitch, p.extra_type, row0, col0, p.m, p.n, in);
                            } else if (p.extra_mode == EXTRA_COPY) {
                                copy_wait();
                                __syncwarp();
                            } else if (!wait_warp(&extra_full[ew], fetched++ & 1, dead, &g_gemm_timeouts)) {
                                break;
                            }
                        }
                        const uint4* irow = (const uint4*)(in + lane * 128);
                        auto join = [&](int j, float e0, float e1) {
                            const f32x2 a = two(v[j], v[j + 1]), e = two(e0, e1);
                            parts(EPI == KERNEL_DZ ? mul2(a, e) : add2(a, e), v[j], v[j + 1]);
                        };
                        if (extra_wide) {
#pragma unroll
                            for (int j = 0; j < W / 4; ++j) {
                                const uint4 q = irow[(j + part * (W / 4)) ^ (lane & 7)];
                                join(4 * j, __uint_as_float(q.x), __uint_as_float(q.y));
                                join(4 * j + 2, __uint_as_float(q.z), __uint_as_float(q.w));
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < W / 8; ++j) {
                                const uint4 q = irow[(j + part * (W / 8)) ^ (lane & 7)];
                                const uint32_t x[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    float e[2];
                                    unpack2(x[i], p.bf16, e);
                                    join(8 * j + 2 * i, e[0], e[1]);
                                }
                            }
                        }
                        __syncwarp();
                        if (part + 1 == per || c + 1 == chunks) fetch(u, c / per + 1);
                    }
                    if (EPI != KERNEL_DZ && p.alpha) {
#pragma unroll
                        for (int j = 0; j < W; ++j) v[j] *= alpha;
                    }
                }
                if (EPI == KERNEL_DL) {
#pragma unroll
                    for (int j = 0; j < W; j += 2) {
                        float a, b;
                        parts(mul2(add2(two(v[j], v[j + 1]), both(-lse)), both(LOG2E)), a, b);
                        parts(mul2(two(ex2(a), ex2(b)), both(weight)), v[j], v[j + 1]);
                    }
                    if (has_target) {
#pragma unroll
                        for (int j = 0; j < W; ++j) v[j] = target == W * c + j ? v[j] - weight : v[j];
                    }
                    if (any_off) {
#pragma unroll
                        for (int j = 0; j < W; ++j) v[j] = off ? 0.0f : v[j];
                    }
                }
                if (EPI == KERNEL_DZ && p.row_sums) {
                    float t[W];
#pragma unroll
                    for (int j = 0; j < W; ++j) t[j] = row < p.m ? v[j] : 0.0f;  // rows past the end hold anything
                    const float s = lane_sums<W>(t);
                    if (lane < W && col0 + lane < p.n && row0 < p.m) p.row_sums[(int64_t)(row0 / 32) * p.n + col0 + lane] = s;
                }
                if (EPI == KERNEL_DZ) {
#pragma unroll
                    for (int j = 0; j < W; j += 2) parts(mul2(two(v[j], v[j + 1]), both(factor)), v[j], v[j + 1]);
                }
                // ---- to memory: the lane's row of 128 bytes in the staging buffer, 16-byte pieces swizzled by the row: 64
                // columns of 16 bits or 32 of 32 fill it
                const bool narrow = p.y_type != PCB_F32 && !partial;
                const int per = (narrow ? 64 : 32) / W, part = c % per;
                if (part == 0) {
                    if (lane == 0) bulk_wait_read();
                    __syncwarp();
                }
                uint4* srow = (uint4*)(stage + lane * 128);
                if (narrow) {
                    const bool bf16 = p.y_type == PCB_BF16;
#pragma unroll
                    for (int j = 0; j < W / 8; ++j)
                        srow[(j + part * (W / 8)) ^ (lane & 7)] =
                            make_uint4(pack2(v[8 * j], v[8 * j + 1], bf16), pack2(v[8 * j + 2], v[8 * j + 3], bf16),
                                       pack2(v[8 * j + 4], v[8 * j + 5], bf16), pack2(v[8 * j + 6], v[8 * j + 7], bf16));
                } else {
#pragma unroll
                    for (int j = 0; j < W / 4; ++j)
                        srow[(j + part * (W / 4)) ^ (lane & 7)] =
                            make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]),
                                       __float_as_uint(v[4 * j + 3]));
                }
                if (part + 1 < per && c + 1 < chunks) continue;
                fence_async_smem();
                __syncwarp();
                const int box0 = col0 - part * W;
                if (partial) {
                    if (lane == 0 && row0 < p.m) {
                        const int at = ((w.split * p.tail + w.tile - p.whole) * CTAS + (int)rank) * BM + quad * 32;
                        tma_store(&p.part, box0 - n0, at, 0, stage);
                        bulk_commit();
                    }
                } else if (p.y_tma) {
                    if (lane == 0 && row0 < p.m) {
                        if (p.accumulate) tma_add(&p.y, box0, row0, w.split, stage);
                        else tma_store(&p.y, box0, row0, w.split, stage);
                        bulk_commit();
                    }
                } else {
                    const int64_t at = ((int64_t)w.split * p.m + row0) * p.y_pitch + box0;
                    store_block(stage, narrow, (char*)p.y_ptr + at * (narrow ? 2 : 4), p.y_pitch, min(32, p.m - row0), p.n - box0, p.accumulate);
                }
            }
            if (chunks == 0) release(buf);
            if (EPI == KERNEL_LSE && row < p.m) p.parts[(int64_t)(tn * (S::EWARPS / 4) + half) * p.m + row] = make_float2(top, sum);
        }
        if (lane == 0) bulk_wait_read();  // the staging buffer stays until it is read; the grid's end completes the writes
        if (HAS_EXTRA) {  // the box in flight, where the warp gave up
            copy_wait();
            if (*dead && p.extra_mode == EXTRA_TMA && lane == 0) mbar_wait(&extra_full[ew], fetched & 1);
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if (CTAS == 2) cluster_sync();
    fence_after();
    if (warp == 1) tmem_free<CTAS>(tmem, S::TMEM);
}

// The split tiles: y = alpha (act(sum of the parts in order + bias) + extra). Four adjacent columns per thread, the parts
// read four at a time so that their latencies overlap (one after another, six parts cost 3 us of a 9 us call).
constexpr int JOIN_VALUES = 1024;  // of a tile per block
__global__ void __launch_bounds__(JOIN_VALUES / 4) join(const float* part, int bn, int tile_rows, const __grid_constant__ Params p) {
    const int groups = tile_rows * bn / JOIN_VALUES, i = blockIdx.x / groups, quads = bn / 4;
    const int e = blockIdx.x % groups * (JOIN_VALUES / 4) + threadIdx.x, tile = p.whole + i;
    int tm, tn;
    if (p.band) place<true>(p, tile, tm, tn);
    else place<false>(p, tile, tm, tn);
    const int64_t row = (int64_t)tm * tile_rows + e / quads, col = (int64_t)tn * bn + e % quads * 4;
    const int64_t step = (int64_t)p.tail * tile_rows * quads;
    pdl_wait();
    pdl_release();
    if (row >= p.m || col >= p.n) return;
    const float alpha = p.alpha ? *p.alpha : 1.0f;
    const float4* at = (const float4*)part + (int64_t)i * tile_rows * quads + e;
    float4 s = at[0];
    for (int k = 1; k < p.splits; k += 4) {
        float4 q[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (k + j < p.splits) q[j] = at[(k + j) * step];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (k + j < p.splits) s.x += q[j].x, s.y += q[j].y, s.z += q[j].z, s.w += q[j].w;
    }
    float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float skip;
        if (col + j >= p.n) break;
        if (p.bias) v[j] += load(p.bias, col + j, p.bias_type);
        if (p.act.kind == PCB_ACT_GELU) parts(act2<PCB_ACT_GELU, false>(p.act, both(v[j])), v[j], skip);
        else if (p.act.kind == PCB_ACT_POLY) parts(act2<PCB_ACT_POLY, false>(p.act, both(v[j])), v[j], skip);
        if (p.extra) v[j] += load(p.extra, row * p.extra_pitch + col + j, p.extra_type);
        v[j] *= alpha;
    }
    const int64_t to = row * p.y_pitch + col;
    if (p.y_tma && col + 3 < p.n) {  // rows on 16 bytes
        if (p.y_type == PCB_F32) ((float4*)p.y_ptr)[to / 4] = make_float4(v[0], v[1], v[2], v[3]);
        else ((uint2*)p.y_ptr)[to / 4] = make_uint2(pack2(v[0], v[1], p.bf16), pack2(v[2], v[3], p.bf16));
        return;
    }
    for (int j = 0; j < 4 && col + j < p.n; ++j) store(p.y_ptr, to + j, p.y_type, v[j]);
}

// Rows of 16-bit values to rows on 16 bytes, zeros up to the pitch; a warp per row, up to three matrices (blockIdx.y)
struct CopyJobs {
    const uint16_t* x[3];
    uint32_t* y[3];
    int64_t pitch[3], rows[3];
    int cols[3], to[3];
};
__global__ void __launch_bounds__(256) copy_rows(const __grid_constant__ CopyJobs j) {
    pdl_wait();
    pdl_release();
    const int b = blockIdx.y, lane = threadIdx.x % 32, words = j.to[b] / 2;
    for (int64_t r = blockIdx.x * 8ll + threadIdx.x / 32; r < j.rows[b]; r += gridDim.x * 8ll) {
        const uint16_t* x = j.x[b] + r * j.pitch[b];
        uint32_t* y = j.y[b] + r * words;
#pragma unroll 4
        for (int c = lane; c < words; c += 32) {
            const uint32_t lo = 2 * c < j.cols[b] ? x[2 * c] : 0, hi = 2 * c + 1 < j.cols[b] ? x[2 * c + 1] : 0;
            y[c] = lo | hi << 16;
        }
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

// Tile and splitting, from estimated nanoseconds, fitted to every tile and splitting of 20 shapes of 1 to 8192 rows, k 509 to
// 8192, 768 to 50000 columns (the choice is within 7 % of the fastest there). A 64-k block of a tile costs its
// products or their issue, up to a fifth more as more SMs are busy and the clock falls, or its bytes into shared memory at
// 16.5 TB/s for all SMs together. The tiles that do not fill a round over the SMs may split their k; that costs their 32-bit
// sums' way to L2 and back and a launch.
struct Plan {
    int bn, ctas, whole, splits, kper;
    double ns;
};
struct Tile {
    int bn, ctas;
    double block;      // ns of a 64-k block
    double next, last; // ns of what one tile, and the last one, add: first loads and the epilogue that does not overlap
};
constexpr Tile TILES[] = {{256, 2, 270, 600, 1800}, {128, 2, 175, 400, 1200}, {128, 1, 230, 400, 700}, {64, 1, 150, 300, 400}};
int a_rows(int m) { return m < BM ? (m + 7) / 8 * 8 : BM; }  // rows of A that a tile loads: what lies past them is not used
double block_ns(const Tile& t, int m, int64_t active) {
    const double sms = (double)(active * t.ctas), bytes = (a_rows(m) + t.bn / t.ctas) * BK * 2;
    return std::max(t.block * (1.0 + 0.2 * std::min(1.0, sms / 96)), bytes * sms / 16500);
}
double rounds(const Tile& t, int m, int64_t units, int kblocks) {
    const int64_t slots = SMS / t.ctas, full = units / slots, rest = units % slots;
    return full * (kblocks * block_ns(t, m, slots) + t.next) + (rest ? kblocks * block_ns(t, m, rest) + t.last : t.last - t.next);
}
// the way of `parts` tiles' 32-bit sums to L2 and back, and the launch that joins them
double join_cost(const Tile& t, int64_t parts) { return 1000.0 + 8.0 * t.bn + (double)parts * BM * t.ctas * t.bn * 8 / 13500; }
Plan plan(int m, int n, int k, bool may_split) {
    const int kb = (k + BK - 1) / BK;
    Plan best{256, 2, 0, 1, kb, 1e300};
    for (const Tile& t : TILES) {
        const int64_t tm = ((int64_t)m + BM * t.ctas - 1) / (BM * t.ctas), tn = ((int64_t)n + t.bn - 1) / t.bn;
        const int64_t tiles = tm * tn, slots = SMS / t.ctas, tail = tiles % slots, whole = tiles - tail;
        double ns = rounds(t, m, tiles, kb);
        if (ns < best.ns) best = Plan{t.bn, t.ctas, (int)tiles, 1, kb, ns};
        for (int sp = 2; may_split && tail && sp <= 16; ++sp) {
            const int per = (kb + sp - 1) / sp;
            if (per < 4 || (sp - 1) * per >= kb) continue;
            ns = whole / slots * (kb * block_ns(t, m, slots) + t.next) + rounds(t, m, tail * sp, per) + join_cost(t, tail * sp);
            if (ns < best.ns) best = Plan{t.bn, t.ctas, (int)whole, sp, per, ns};
        }
    }
    return best;
}
// k in `slices` parts to as many outputs: the tile for that many units
Plan plan_slices(int m, int n, int k, int slices) {
    const int kb = (k + BK - 1) / BK, per = (kb + slices - 1) / slices;
    Plan best{256, 2, 0, slices, per, 1e300};
    for (const Tile& t : TILES) {
        const int64_t tm = ((int64_t)m + BM * t.ctas - 1) / (BM * t.ctas), tn = ((int64_t)n + t.bn - 1) / t.bn;
        const double ns = rounds(t, m, tm * tn * slices, per) + (double)m * n * 8 * slices / 8000;
        if (ns < best.ns) best = Plan{t.bn, t.ctas, 0, slices, per, ns};
    }
    return best;
}

template <int BN, int CTAS, int EPI, int ACT, bool BANDS = false>
int launch(const Params& p, cudaStream_t s) {
    using S = Shape<BN, CTAS, EPI>;
    static_assert(S::SMEM <= 232448, "shared memory");
    static std::atomic<uint64_t> done{0};
    if (int rc = allow_smem((const void*)product<BN, CTAS, EPI, ACT, BANDS>, S::SMEM, done)) return rc;
    const int64_t units = (int64_t)p.whole + (int64_t)p.tail * p.splits, slots = SMS / CTAS;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((units < slots ? units : slots) * CTAS));
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
    cudaLaunchKernelEx(&cfg, product<BN, CTAS, EPI, ACT, BANDS>, p);
    return PCB_LAUNCH_RESULT();
}
template <int EPI, int ACT>
int launch(const Plan& pl, const Params& p, cudaStream_t s) {
    if (p.band) return launch<256, 2, EPI, ACT, true>(p, s);
    if (pl.ctas == 2) return pl.bn == 256 ? launch<256, 2, EPI, ACT>(p, s) : launch<128, 2, EPI, ACT>(p, s);
    return pl.bn == 128 ? launch<128, 1, EPI, ACT>(p, s) : launch<64, 1, EPI, ACT>(p, s);
}

}  // namespace

size_t gemm_partial(int m, int n, int k) {
    const Plan pl = plan(m, n, k, true);
    if (pl.splits == 1) return 0;
    const size_t rows = BM * pl.ctas;
    const size_t tiles = ((size_t)m + rows - 1) / rows * (((size_t)n + pl.bn - 1) / pl.bn);
    return (tiles - pl.whole) * pl.splits * rows * pl.bn;
}
double gemm_cost(int m, int n, int k, bool may_split) { return plan(m, n, k, may_split).ns; }
int gemm_slices(int m, int n, int k) {
    int best = 1;
    double least = 1e300;
    for (int s = 1; s <= 8; ++s) {
        const Plan p = plan_slices(m, n, k, s);
        if (s > 1 && (p.kper < 4 || (s - 1) * p.kper >= (k + BK - 1) / BK)) continue;  // every part has some of k
        if (p.ns < 0.97 * least) least = p.ns, best = s;
    }
    return best;
}
int vocab_parts(int m, int n) {
    const int bn = plan(m, n, 1 << 10, false).bn;
    return (n + bn - 1) / bn * (bn == 64 ? 1 : 2);
}

int gemm(const Gemm& g, cudaStream_t s) {
    // the column blocks of an EPI_LSE product follow vocab_parts, which does not know k
    const Plan pl = g.slices ? plan_slices(g.m, g.n, g.k, g.slices) : plan(g.m, g.n, g.epi == EPI_LSE ? 1 << 10 : g.k, g.epi == EPI_STORE && g.partial);
    const int rows = BM * pl.ctas;
    const int64_t tm = ((int64_t)g.m + rows - 1) / rows, tn = ((int64_t)g.n + pl.bn - 1) / pl.bn;
    if (tm * tn * pl.splits > INT32_MAX) return report(PCB_BAD_ARGS, "a product of %d x %d outputs", g.m, g.n);
    Params p;
    memset(&p, 0, sizeof p);
    const int arows = g.a.k_adjacent && pl.ctas == 1 ? a_rows(g.m) : BM;
    if (int rc = operand_map(&p.a, g.a, g.type, g.m, g.k, arows)) return rc;
    if (int rc = operand_map(&p.b, g.b, g.type, g.n, g.k, pl.bn / pl.ctas)) return rc;
    p.m = g.m, p.n = g.n, p.k = g.k;
    p.a_mn = !g.a.k_adjacent, p.b_mn = !g.b.k_adjacent, p.a_panels = panels(g.a, g.m), p.b_panels = panels(g.b, g.n);
    p.bf16 = g.type == PCB_BF16;
    p.a_bytes = arows * BK * 2;
    // Where A stays in L2, tiles go down all of its rows, column after column; a larger A is read again for each column, and
    // bands of 2048 rows, about square over a round, read less of both (8192 x 8192 x 8192: 730 us against 790,
    // 50000 x 4096 x 768: 225 against 263; 4096 x 768 x 50000, whose A takes 6 MB, 241 down all rows against 252)
    p.band = pl.bn == 256 && tm > 8 && 2.0 * g.m * g.k > 64e6 ? 8 : 0;
    p.tiles_m = (int)tm, p.tiles_n = (int)tn, p.kblocks = (g.k + BK - 1) / BK;
    p.whole = pl.whole, p.tail = (int)(tm * tn) - pl.whole, p.splits = pl.splits, p.kper = pl.kper, p.slices = g.slices;
    p.act = g.act, p.bias = g.bias, p.bias_type = g.bias_type;
    p.extra = g.extra, p.extra_pitch = g.extra_pitch, p.extra_type = g.extra_type;
    p.y_ptr = g.y, p.y_pitch = g.y_pitch, p.y_type = g.y_type, p.accumulate = g.accumulate;
    p.alpha = g.alpha, p.row_sums = g.row_sums, p.sizes = g.sizes, p.nsizes = g.nsizes, p.slope = g.slope, p.unscale = g.unscale, p.rows = g.rows, p.col0 = g.col0, p.targets = g.targets, p.parts = g.parts, p.hit = g.hit;
    const size_t eb = type_bytes(p.y_type);
    // 16-byte aligned rows go through the TMA engine, which writes whole 16 bytes: where a row's last ones are not all its own,
    // and in rows off 16 bytes, results go by rows of the staging buffer
    p.y_tma = g.epi != EPI_LSE && ((uintptr_t)p.y_ptr & 15) == 0 && p.y_pitch * eb % 16 == 0 && (g.padded || g.n * eb % 16 == 0);
    if (p.y_tma) {
        const uint64_t size[3] = {(uint64_t)g.n, (uint64_t)g.m, (uint64_t)(g.slices ? g.slices : 1)};
        const uint64_t stride[2] = {(uint64_t)p.y_pitch * eb, (uint64_t)p.y_pitch * eb * g.m};
        const uint32_t box[3] = {(uint32_t)(128 / eb), 32, 1};
        if (int rc = encode_map(&p.y, p.y_type, p.y_ptr, 3, size, stride, box)) return rc;
    }
    if (p.extra) {
        const size_t ee = type_bytes(p.extra_type);
        p.extra_mode = p.extra_type == PCB_F32 ? EXTRA_COPY : EXTRA_LOAD;
        if (((uintptr_t)p.extra & 15) == 0 && p.extra_pitch * ee % 16 == 0) {
            const uint64_t size[2] = {(uint64_t)g.n, (uint64_t)g.m}, stride[1] = {(uint64_t)(p.extra_pitch * ee)};
            const uint32_t box[2] = {(uint32_t)(128 / ee), 32};
            if (int rc = encode_map(&p.extra_map, p.extra_type, p.extra, 2, size, stride, box)) return rc;
            p.extra_mode = EXTRA_TMA;
        }
    }
    const bool split = !g.slices && pl.splits > 1;
    if (split) {
        const uint64_t size[3] = {(uint64_t)pl.bn, (uint64_t)p.tail * p.splits * rows, 1};
        const uint64_t stride[2] = {(uint64_t)pl.bn * 4, (uint64_t)pl.bn * 4 * size[1]};
        const uint32_t box[3] = {32, 32, 1};
        if (int rc = encode_map(&p.part, PCB_F32, g.partial, 3, size, stride, box)) return rc;
    }
    int rc;
    const int act = p.act.kind;
    if (g.epi == EPI_LSE) rc = launch<KERNEL_LSE, 0>(pl, p, s);
    else if (g.epi == EPI_DL) rc = launch<KERNEL_DL, 0>(pl, p, s);
    else if (g.epi == EPI_DZ) rc = act == PCB_ACT_GELU ? launch<KERNEL_DZ, PCB_ACT_GELU>(pl, p, s) : launch<KERNEL_DZ, PCB_ACT_POLY>(pl, p, s);
    else if (p.extra)
        rc = act == PCB_ACT_GELU   ? launch<KERNEL_ADD, PCB_ACT_GELU>(pl, p, s)
             : act == PCB_ACT_POLY ? launch<KERNEL_ADD, PCB_ACT_POLY>(pl, p, s)
                                   : launch<KERNEL_ADD, PCB_ACT_NONE>(pl, p, s);
    else
        rc = act == PCB_ACT_GELU   ? launch<KERNEL_STORE, PCB_ACT_GELU>(pl, p, s)
             : act == PCB_ACT_POLY ? launch<KERNEL_STORE, PCB_ACT_POLY>(pl, p, s)
                                   : launch<KERNEL_STORE, PCB_ACT_NONE>(pl, p, s);
    if (rc || !split) return rc;
    launch_pdl(join, dim3((unsigned)((int64_t)p.tail * rows * pl.bn / JOIN_VALUES)), dim3(JOIN_VALUES / 4), s, (const float*)g.partial, pl.bn, rows, p);
    return PCB_LAUNCH_RESULT();
}

size_t aligned_bytes(const void* p, int64_t pitch, int64_t rows, int64_t cols) {
    if (((uintptr_t)p & 15) == 0 && pitch % 8 == 0 && pitch < (1ll << 38)) return 0;  // a map's strides are below 2^40 bytes
    return (size_t)rows * ((cols + 7) / 8 * 8) * 2;
}
int align_rows(const Rows* r, int n, cudaStream_t s) {
    CopyJobs j;
    memset(&j, 0, sizeof j);
    int jobs = 0;
    int64_t most = 0;
    for (int i = 0; i < n; ++i) {
        if (!aligned_bytes(*r[i].p, *r[i].pitch, r[i].rows, r[i].cols)) continue;
        const int64_t to = (r[i].cols + 7) / 8 * 8;
        j.x[jobs] = (const uint16_t*)*r[i].p, j.y[jobs] = (uint32_t*)r[i].to, j.pitch[jobs] = *r[i].pitch;
        j.rows[jobs] = r[i].rows, j.cols[jobs] = (int)r[i].cols, j.to[jobs] = (int)to;
        most = std::max(most, r[i].rows);
        *r[i].p = r[i].to, *r[i].pitch = to;
        ++jobs;
    }
    if (!jobs) return 0;
    launch_pdl(copy_rows, dim3((unsigned)std::min<int64_t>((most + 7) / 8, 8 * SMS), jobs), dim3(256), s, j);
    return PCB_LAUNCH_RESULT();
}

unsigned int gemm_timeouts() {
    unsigned int v = 0;
    return cudaMemcpyFromSymbol(&v, g_gemm_timeouts, sizeof v) == cudaSuccess ? v : ~0u;
}

}  // namespace clear
}  // namespace pcb
