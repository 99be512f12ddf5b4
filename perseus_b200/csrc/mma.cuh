// The fifth-generation tensor core and the TMA engine's tiled copies, as the clear half's kernels use them (sm_100a,
// hand-written PTX): 128-row products of 16-bit operands into 32-bit accumulators in TMEM, operands in shared memory
// under the 128-byte swizzle (or the left one in TMEM), every completion on a shared-memory mbarrier. No multicast.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>

#include "arith.cuh"

namespace pcb {
namespace mma {

// ------------------------------------------------------------------------------------------------ TMA, tiled
// The box at (x, y) of a two-dimensional map; x times the element size is a multiple of 16 bytes. What lies outside the
// tensor reads as zero (loads) or is not written (stores; but along x they write whole 16 bytes: a tensor whose inner size
// is no multiple of them has to own what follows in the last).
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(smem_addr(bar))
        : "memory");
}
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
        : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, int x, int y, int z, const void* src) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x), "r"(y),
                 "r"(z), "r"(smem_addr(src))
                 : "memory");
}
// adds the box to what is there (32-bit floats); one writer per element and launch keeps the order fixed
__device__ __forceinline__ void tma_add(const CUtensorMap* map, int x, int y, int z, const void* src) {
    asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map),
                 "r"(x), "r"(y), "r"(z), "r"(smem_addr(src))
                 : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// the same by one block of a pair, completing on a barrier of either (`bar`: a cluster address)
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

// ------------------------------------------------------------------------------------------------ pairs of blocks
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// the cluster address of block `rank`'s copy of a shared-memory object
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// ------------------------------------------------------------------------------------------------ barriers
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// whether the phase is done, without waiting: asked for the next stage before this one's instructions are issued, the
// answer costs nothing when it is used
__device__ __forceinline__ bool peek(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// A bounded wait of a whole warp that also gives up when another role of the block has (`dead`, shared memory): false then,
// and counted. RELAXED waits (for a tile's worth of work, not for the next block) poll from one lane and sleep in between,
// so that the epilogue's warps leave the barriers' unit to the warps that feed the products; their limit leaves a tile some
// seconds (k may be millions).
constexpr uint32_t RELAXED_WAIT_LIMIT = 1u << 27;
template <bool RELAXED = false>
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* dead, unsigned int* timeouts) {
    bool ok = true;
    if (!RELAXED || threadIdx.x % 32 == 0) {
        for (uint32_t it = 1; !mbar_test(bar, parity); ++it) {
            if (RELAXED) __nanosleep(32);
            if ((it & 255) == 0 && *dead) {
                ok = false;
                break;
            }
            if (it >= (RELAXED ? RELAXED_WAIT_LIMIT : MBAR_WAIT_LIMIT)) {
                *dead = 1;
                atomicAdd(timeouts, 1u);
                ok = false;
                break;
            }
        }
    }
    return __all_sync(~0u, ok);
}

// One lane of a converged warp. The loops that feed the TMA engine and the tensor core run on whole warps, with only the
// instructions themselves under elect(): addresses, descriptors and phases then stay in uniform registers, which those
// instructions take. (Run on one lane, the loop's bookkeeping cost 280 cycles per 64-k block and each product was held up by
// moves into uniform registers: 8192 x 8192 x 8192 took 829 us.)
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ int warp_index() { return __shfl_sync(~0u, (int)threadIdx.x / 32, 0); }
// A ring of N stages: the stage, and the parity of its barriers' phase
template <int N>
struct Ring {
    int stage = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next() {
        if (++stage == N) stage = 0, phase ^= 1;
    }
};

// ------------------------------------------------------------------------------------------------ TMEM
// One warp (of each block of a pair) allocates `cols` (a power of two from 32 to 512) columns of 128 lanes x 32 bits, and
// frees them
template <int CTAS = 1>
__device__ __forceinline__ void tmem_alloc(uint32_t* at, uint32_t cols) {
    if (CTAS == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(at)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(at)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
}
template <int CTAS = 1>
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
    if (CTAS == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 32 columns of the warp's 32 lanes: thread = lane (row), register = column
__device__ __forceinline__ void tmem_ld32(uint32_t at, float* v) {
    uint32_t* r = (uint32_t*)v;
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
          "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, float* v) {
    uint32_t* r = (uint32_t*)v;
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at));
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::
            "r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}

// ------------------------------------------------------------------------------------------------ products
// Shared-memory operand under the 128-byte swizzle, in groups of 8 x 128 bytes (1024-byte aligned). K adjacent: rows of
// 64 k-values, 8-row groups `sbo` = 1024 bytes apart; 16 k-values further is 32 bytes further. M (N) adjacent: rows of 64
// m-values, one per k, 8-k groups `sbo` = 1024 bytes apart, the next 64 m-values `lbo` bytes on; 16 k-values further is
// 2048 bytes further.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}
// 32-bit accumulator, both operands bf16 or both f16; a_mn / b_mn: M / N adjacent in shared memory
__host__ __device__ constexpr uint32_t instr_desc(bool bf16, bool a_mn, bool b_mn, int m, int n) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
           ((uint32_t)(n / 8) << 17) | ((uint32_t)(m / 16) << 24);
}
// acc (TMEM) = or += A B^T over 16 k-values, issued by one thread. A pair's product has 256 rows, 128 of A and of the
// accumulator in each block, and half of B's rows in each: the first block's thread issues it, the operands lie at the same
// offsets in both
template <int CTAS = 1>
__device__ __forceinline__ void mma_ss(uint32_t acc, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    if (CTAS == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(acc),
            "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(acc),
            "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
            : "memory");
}
// the same with A in TMEM (two 16-bit k-values per 32-bit column)
__device__ __forceinline__ void mma_ts(uint32_t acc, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(acc),
        "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
// arrives on `bar` (of a pair: on both blocks') when this thread's products so far are done
template <int CTAS = 1>
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    if (CTAS == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                         smem_addr(bar)),
                     "h"((uint16_t)3)
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// ------------------------------------------------------------------------------------------------ 32-bit pieces
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two 32-bit values at a time (one instruction for both): x holds (lo, hi)
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 two(float lo, float hi) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ f32x2 both(float x) { return two(x, x); }
__device__ __forceinline__ void parts(f32x2 x, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// two values rounded to 16 bits, `lo` in the lower half
__device__ __forceinline__ uint32_t pack2(float lo, float hi, bool bf16) {
    uint32_t r;
    if (bf16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// and back: v[0] the lower half, v[1] the upper
__device__ __forceinline__ void unpack2(uint32_t x, bool bf16, float* v) {
    if (bf16) {
        v[0] = __uint_as_float(x << 16);
        v[1] = __uint_as_float(x & 0xFFFF0000u);
    } else {
        const float2 f = __half22float2(*(const __half2*)&x);
        v[0] = f.x, v[1] = f.y;
    }
}

}  // namespace mma
}  // namespace pcb
