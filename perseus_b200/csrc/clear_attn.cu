// Attention over packed prompts on the fifth-generation tensor cores (pcb_clear_attention).
//
// A block takes 128 rows of one K/V head of one sequence: consecutive tokens x the query heads that share the K/V head
// (a group is never split, so its keys and values are read once), and walks the keys up to the last one its tokens see, 128
// per copy and 64 per step. A step's scores S = Q K^T land in TMEM (128 rows x 64 keys, 32 bits, two buffers); four warps, one
// thread per row, turn them into weights, which go back over them in 16 bits as the left operand of O += P V. Softmax runs
// with a running maximum and sum: O is rescaled only when a row's maximum grew by more than 2^8 (weights stay below 2^8, in
// range for f16), which after the first steps is rare. Under polynomial weights there is no maximum, no sum and no rescaling.
// Two blocks share an SM: while one's warps compute weights, the other's products run.
//
// What bounds it: a warp's own chain (scores' arrival, maximum, exponentials, weights' way back), 1500 cycles a step, of which two
// overlap on an SM. 8192 tokens, 12 heads over 4 of 64: 159 us, 0.65 PFLOP/s, some 890 cycles a step of a block, against 256 of
// products and 384 on the special-function pipe (512 exponentials' worth of cycles, a quarter of them on the multiply-add pipe);
// under polynomial weights, without any exponentials, 153 us. 128 dims: 197 us, 1.04 PFLOP/s.
// More warps per row, three or four blocks of one buffer, and blocks that stay for many tiles measured slower (187, 195, 212,
// 171 us). Short sequences: a block costs some 4 us besides its steps (24 prompts of 1 to 1024 tokens: 45 us, 1350 blocks).
//
// Few rows against many keys (single tokens) split the keys over several blocks, joined in order by `join_splits`.
//
// A key block may reach into the next sequence, or hold keys that some rows do not see: their weights are zero, but zero
// times a value that is not finite is not zero. So rows whose result is not finite, and not for the keys that they see,
// are computed again key by key over those (`redo`): exact semantics at no cost where all values are finite.
#include <algorithm>
#include <cstring>

#include "clear_gemm.h"
#include "mma.cuh"

namespace pcb {
namespace clear {

using namespace mma;

int encode_map(CUtensorMap* map, int type, const void* p, int dims, const uint64_t* size, const uint64_t* stride_bytes,
               const uint32_t* box);

__device__ unsigned int g_attn_timeouts;

namespace {

constexpr int SMS = 148;
constexpr int ROWS = 128, KEYS = 128, STEP = 64;  // rows of a tile, keys of a copy, keys of a product
constexpr int SEQS = 128;  // sequences of one launch

struct Work {
    int32_t n;
    int32_t tile0[SEQS + 1];  // first tile (times kv_heads blocks) of each sequence, the longest sequences first
    int32_t q0[SEQS], nq[SEQS], k0[SEQS], nk[SEQS];
};
struct alignas(64) Params {
    CUtensorMap q, k, v;
    PcbClearAttention a;  // the operands as they lie, for redo
    int group, tokens;    // query heads of a K/V head, tokens of a 128-row tile
    int splits;
    float c;              // scores to base-2 exponents: |scale| log2 e
    int negate;           // scale < 0: the products are negated
    float coef[8];        // of the raw scores, the largest of the polynomial's own brought to 1
    float out_scale;
    float* part_o;        // splits > 1: [split][q row][head][dim] sums, and (maximum in base 2, sum of weights)
    float2* part_ml;
    int out_vec;          // out's rows take 16-byte stores
    Work w;
};

// TMEM columns of a block: two buffers of 64 keys' scores, each turned into weights in place (16 bits: its first 32
// columns), and the sums O
template <int DP>
struct Shape {
    static constexpr int HALF = 128 * 128;               // 128 rows of 64 values
    static constexpr int OPERAND = HALF * (DP / 64);     // 128 rows of DP
    static constexpr int RING = DP == 64 ? 4 : 2;        // K and V blocks in flight
    static constexpr uint32_t S = 0, O = 2 * STEP, TMEM = 256;
    static constexpr size_t SMEM = 1024 + OPERAND * (1 + RING) + 256;
};
constexpr int THREADS = 224;  // loads, scores, sums, and four warps with a row per thread

// A block's tile: the sequence (its rows q0.. and keys k0..), the K/V head, the tokens from t0 (the last ones first), the key blocks
struct Tile {
    int split, kh, nq, nk, q0, k0, t0, seen, b0, n;
};
__device__ __forceinline__ Tile tile_of(const Params& p) {
    Tile w;
    w.split = blockIdx.x % p.splits;
    const int item = blockIdx.x / p.splits, tile = item / p.a.kv_heads;
    w.kh = item % p.a.kv_heads;
    int lo = 0, hi = p.w.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (p.w.tile0[mid] <= tile) lo = mid;
        else hi = mid;
    }
    w.nq = p.w.nq[lo], w.nk = p.w.nk[lo], w.q0 = p.w.q0[lo], w.k0 = p.w.k0[lo];
    w.t0 = (p.w.tile0[lo + 1] - 1 - tile) * p.tokens;
    w.seen = p.a.causal ? min(w.nk, max(0, min(w.nq, w.t0 + p.tokens) + w.nk - w.nq)) : w.nk;  // keys of the last token
    const int blocks = (w.seen + KEYS - 1) / KEYS, per = (blocks + p.splits - 1) / p.splits;
    w.b0 = min(blocks, w.split * per), w.n = min(blocks, w.b0 + per) - w.b0;
    return w;
}
// Row r of a tile: its token, its query head, and how many keys it sees (0: not a row)
__device__ __forceinline__ void row_of(const Params& p, const Tile& w, int r, int& tok, int& head, int& limit) {
    tok = w.t0 + r / p.group, head = w.kh * p.group + r % p.group;
    limit = r >= p.group * p.tokens || tok >= w.nq ? 0 : p.a.causal ? min(w.nk, max(0, tok + w.nk - w.nq + 1)) : w.nk;
}

// What a split leaves to the join: the maximum and the sum of its weights. (-inf, 0) where the row sees none of its keys, (-inf,
// -1) where all scores that it sees are -inf, (-inf, NaN) where the sum is NaN: so is the row, wherever the others' maxima lie.
__device__ __forceinline__ float2 part_of(bool blind, float top, float sum) {
    return make_float2(blind || sum != sum ? -INFINITY : top, blind ? 0.0f : sum == 0.0f ? -1.0f : sum);
}

// ------------------------------------------------------------------------------------------------ rows again, key by key
// A warp looks at its rows of `again`, whose result is not finite though (under softmax) the sum of their weights is positive.
// Where keys that a row sees account for that, it stands: every dim that is not finite has a value that is not in V (under
// polynomial weights also a key or the query itself). The others, which hold 0 x Inf of keys that they do not see, or an overflow,
// are computed once more, each over those of the block's keys that it sees and nothing else, in 32 bits: two rows at a time,
// which share the loads, and 32 keys: lane l has key l's scores and weights, then dims l + 32 t of the sums. 8192 tokens, 12 heads
// over 4, Inf in the 1st value 1.1 ms, in the 4096th 9.8 ms (all rows after it computed again key by key: 468 and 403 ms).
template <int DP, bool POLY>
__device__ __forceinline__ void redo(const Params& p, uint32_t again) {
    constexpr int R = 2, T = DP / 32;  // four rows: 30 % less here, but the whole kernel 1 to 3 % slower
    const PcbClearAttention& a = p.a;
    const Tile w = tile_of(p);
    const int lane = threadIdx.x % 32, kh = w.kh, j0 = w.b0 * KEYS, j1 = (w.b0 + w.n) * KEYS;
    const int64_t q0 = w.q0, k0 = w.k0;
    const bool bf16 = a.type == PCB_BF16;
    int tok, head, limit;
    row_of(p, w, threadIdx.x / 32 % 4 * 32 + lane, tok, head, limit);
    {
        int first_v[T], first_k = INT32_MAX, last = j0;  // the first keys with a value that is not finite: of each dim, of any
        for (uint32_t i = again; i; i &= i - 1) last = max(last, min(j1, __shfl_sync(~0u, limit, __ffs(i) - 1)));
        const uint16_t exponent = bf16 ? 0x7F80 : 0x7C00;
        auto first = [&](const void* x, int64_t pitch, int64_t at, int t) {  // eight keys' loads at a time
            const uint16_t* col = (const uint16_t*)x + k0 * pitch + at + min(lane + 32 * t, a.dim - 1);
            int found = INT32_MAX;
            for (int j = j0; j < last; j += 8) {
                uint16_t v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = col[min(j + e, last - 1) * pitch];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if ((v[e] & exponent) == exponent) found = min(found, j + e);
            }
            return found;
        };
#pragma unroll
        for (int t = 0; t < T; ++t) {
            first_v[t] = first(a.v, a.v_pitch, kh * a.v_head, t);
            if (POLY) first_k = min(first_k, first(a.k, a.k_pitch, kh * a.k_head, t));
        }
        first_k = __reduce_min_sync(~0u, first_k);
        for (uint32_t i = again; i; i &= i - 1) {
            const int src = __ffs(i) - 1, lim = __shfl_sync(~0u, limit, src), hd = __shfl_sync(~0u, head, src);
            const int64_t qr = q0 + __shfl_sync(~0u, tok, src), row = ((int64_t)w.split * a.q_rows + qr) * a.heads + hd;
            bool scores = POLY && first_k < lim, unexplained = false;  // a score that is not finite: with two coefficients, all dims
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const int d = lane + 32 * t;
                if (d >= a.dim) continue;
                if (POLY) scores |= !isfinite(load(a.q, qr * a.q_pitch + hd * a.q_head + d, a.type));
                const float y = p.splits > 1 ? p.part_o[row * a.dim + d] : load(a.out, qr * a.out_pitch + hd * a.out_head + d, a.type);
                unexplained |= !isfinite(y) && first_v[t] >= lim;
            }
            if (!__any_sync(~0u, unexplained) || (__any_sync(~0u, scores) && a.ncoef > 1)) again &= ~(1u << src);
        }
    }
    const bool wide = (((uintptr_t)a.q | (uintptr_t)a.k) & 15) == 0 && ((a.q_pitch | a.q_head | a.k_pitch | a.k_head | a.dim) & 7) == 0;
    const uint16_t* v_col[T];
#pragma unroll
    for (int t = 0; t < T; ++t) v_col[t] = (const uint16_t*)a.v + k0 * a.v_pitch + kh * a.v_head + min(lane + 32 * t, a.dim - 1);
    while (again) {
        int64_t qr[R];
        int hd[R], lim[R], end = j0;
        bool live[R];
        float o[R][T] = {}, top[R], sum[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int src = again ? __ffs(again) - 1 : 0;
            live[r] = again != 0;
            again &= again - 1;
            qr[r] = q0 + __shfl_sync(~0u, tok, src);
            hd[r] = __shfl_sync(~0u, head, src);
            lim[r] = min(j1, __shfl_sync(~0u, limit, src));
            if (!live[r]) qr[r] = qr[0], hd[r] = hd[0], lim[r] = j0;
            end = max(end, lim[r]);
            top[r] = -INFINITY, sum[r] = 0.0f;
        }
        for (int j = j0; j < end; j += 32) {
            const int n = min(32, end - j);
            float s[R] = {};
            if (lane < n) {
                const int64_t k_at = (k0 + j + lane) * a.k_pitch + kh * a.k_head;
                if (wide) {
#pragma unroll 4
                    for (int d = 0; d < a.dim; d += 8) {
                        const uint4 y = *(const uint4*)((const uint16_t*)a.k + k_at + d);
                        const uint32_t ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                        for (int r = 0; r < R; ++r) {
                            const uint4 x = *(const uint4*)((const uint16_t*)a.q + qr[r] * a.q_pitch + hd[r] * a.q_head + d);
                            const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float u[2], v[2];
                                unpack2(xs[i], bf16, u);
                                unpack2(ys[i], bf16, v);
                                s[r] = fmaf(u[1], v[1], fmaf(u[0], v[0], s[r]));
                            }
                        }
                    }
                } else {
                    for (int d = 0; d < a.dim; ++d) {
                        const float y = load(a.k, k_at + d, a.type);
#pragma unroll
                        for (int r = 0; r < R; ++r) s[r] = fmaf(load(a.q, qr[r] * a.q_pitch + hd[r] * a.q_head + d, a.type), y, s[r]);
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) {  // scores to weights
                if (POLY) {
                    const float x = s[r] * a.scale;
                    s[r] = a.coef[a.ncoef - 1];
                    for (int i = a.ncoef - 2; i >= 0; --i) s[r] = fmaf(s[r], x, a.coef[i]);
                } else {
                    s[r] = j + lane < lim[r] ? (a.scale < 0.0f ? -s[r] : s[r]) * p.c : -INFINITY;
                    float nt = s[r];
                    for (int m = 16; m; m >>= 1) nt = fmaxf(nt, __shfl_xor_sync(~0u, nt, m));
                    nt = fmaxf(top[r], nt);
                    const float f = top[r] == -INFINITY ? 0.0f : exp2f(top[r] - nt);
                    s[r] = nt == -INFINITY ? (s[r] == s[r] ? 0.0f : s[r]) : exp2f(s[r] - nt);
                    float more = s[r];
                    for (int m = 16; m; m >>= 1) more += __shfl_xor_sync(~0u, more, m);
                    sum[r] = sum[r] * f + more;
                    for (int t = 0; t < T; ++t) o[r][t] *= f;
                    top[r] = nt;
                }
            }
            for (int i = 0; i < n; i += 8) {  // eight keys' loads at a time
                uint16_t v[8][T];
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int t = 0; t < T; ++t) v[e][t] = v_col[t][min(j + i + e, end - 1) * a.v_pitch];
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float weight = __shfl_sync(~0u, s[r], i + e);
                        if (j + i + e < lim[r]) {
#pragma unroll
                            for (int t = 0; t < T; ++t) {
                                const float x = bf16 ? __uint_as_float(v[e][t] << 16) : __half2float(__ushort_as_half(v[e][t]));
                                o[r][t] = fmaf(weight, x, o[r][t]);
                            }
                        }
                    }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (!live[r]) continue;
            const int64_t row = ((int64_t)w.split * a.q_rows + qr[r]) * a.heads + hd[r];
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const int d = lane + 32 * t;
                if (d >= a.dim) continue;
                if (p.splits > 1) p.part_o[row * a.dim + d] = o[r][t];
                else store(a.out, qr[r] * a.out_pitch + hd[r] * a.out_head + d, a.type, POLY ? o[r][t] : o[r][t] / sum[r]);
            }
            if (p.splits > 1 && lane == 0) p.part_ml[row] = part_of(false, top[r], sum[r]);
        }
    }
}

// 2^x for two values on the multiply-add pipe: the special-function pipe gives 16 exponentials per cycle and SM, half of what
// the products need at 64 dims, so a quarter of them is computed here (8192 tokens, 12 heads over 4: 164 us without, 156 with
// a quarter, 166 with half; at 128 dims the products take as long as the exponentials, and it costs 1 %). x = n + f with n the nearest integer (in the low bits of
// x + 1.5 2^23), |f| <= 1/2; 2^f by the polynomial of least relative error of degree 4 (2.6e-6, a thousandth of the weights'
// rounding), times 2^n. x stays at -126 from below, and the result there is subtracted from all: a key that is masked (x = -inf)
// or far below weighs exactly 0, or V values near bfloat16's largest would show through 2^-126. NaN stays NaN.
__device__ __forceinline__ f32x2 exp2_fma(f32x2 x) {
    float x0, x1, t0, t1;
    parts(x, x0, x1);
    asm("max.NaN.f32 %0, %1, 0fC2FC0000;" : "=f"(x0) : "f"(x0));  // -126
    asm("max.NaN.f32 %0, %1, 0fC2FC0000;" : "=f"(x1) : "f"(x1));
    x = two(x0, x1);
    const f32x2 t = add2(x, both(12582912.0f));
    const f32x2 f = fma2(add2(t, both(-12582912.0f)), both(-1.0f), x);
    f32x2 p = fma2(f, both(0.009570102207362652f), both(0.05591785907745361f));
    p = fma2(p, f, both(0.240247443318367f));
    p = fma2(p, f, both(0.6931217908859253f));
    p = fma2(p, f, both(0.9999992847442627f));
    parts(t, t0, t1);
    const f32x2 n = two(__uint_as_float(0x3F800000u + (__float_as_uint(t0) << 23)), __uint_as_float(0x3F800000u + (__float_as_uint(t1) << 23)));
    return fma2(p, n, both(__uint_as_float(0x807FFFFAu)));  // -0.9999992847442627 2^-126: f = 0, n = -126
}

// ------------------------------------------------------------------------------------------------ the kernel
template <int DP, bool POLY>
__global__ void __launch_bounds__(THREADS, 2) attend(const __grid_constant__ Params p) {
    using S = Shape<DP>;
    extern __shared__ unsigned char raw[];
    unsigned char* base = (unsigned char*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    unsigned char* ring = base + S::OPERAND;
    uint64_t* q_full = (uint64_t*)(ring + S::RING * S::OPERAND);
    uint64_t* full = q_full + 1;
    uint64_t* empty = full + S::RING;
    uint64_t* s_full = empty + S::RING;
    uint64_t* p_ready = s_full + 2;
    uint64_t* pv_done = p_ready + 2;
    uint64_t* drain = pv_done + 2;
    uint32_t* tmem_at = (uint32_t*)(drain + 2);
    volatile int* dead = (volatile int*)(tmem_at + 1);
    const int warp = warp_index(), lane = threadIdx.x % 32;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        for (int i = 0; i < S::RING; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_ready[i], 4);
            mbar_init(&pv_done[i], 1);
        }
        mbar_init(&drain[0], 1);
        mbar_init(&drain[1], 1);
        mbar_init_fence();
        *dead = 0;
        prefetch_map(&p.q);
        prefetch_map(&p.k);
        prefetch_map(&p.v);
    }
    if (warp == 1) tmem_alloc(tmem_at, S::TMEM);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_at;
    pdl_wait();
    pdl_release();

    const Tile w = tile_of(p);
    const int kh = w.kh, k0 = w.k0, b0 = w.b0, n = w.n;
    const int least = p.a.causal ? min(w.nk, max(0, w.t0 + w.nk - w.nq + 1)) : w.nk;               // keys of the first token
    const int steps = n > 0 ? (min(w.seen, (b0 + n) * KEYS) - b0 * KEYS + STEP - 1) / STEP : 0;  // products of 64 keys

    uint32_t again = 0;  // rows of a softmax warp that `redo` computes
    if (warp == 0) {
        if (n > 0) {
            if (elect()) {
                mbar_expect(q_full, (DP / 64) * 128 * p.group * p.tokens);
                for (int h = 0; h < DP / 64; ++h) tma_load(base + h * S::HALF, &p.q, 64 * h, kh * p.group, w.q0 + w.t0, q_full);
            }
            __syncwarp();
            Ring<S::RING> rg;
            int i = 0;
            bool ok = true;
            for (; i < 2 * n; ++i, rg.next()) {  // K and V in turn
                ok = wait_warp(&empty[rg.stage], rg.phase ^ 1, dead, &g_attn_timeouts);
                if (!ok) break;
                if (elect()) {
                    mbar_expect(&full[rg.stage], S::OPERAND);
                    for (int h = 0; h < DP / 64; ++h)
                        tma_load(ring + rg.stage * S::OPERAND + h * S::HALF, i % 2 ? &p.v : &p.k, 64 * h, kh, k0 + (b0 + i / 2) * KEYS,
                                 &full[rg.stage]);
                }
                __syncwarp();
            }
            if (!ok) {  // the loads in flight
                mbar_wait(q_full, 0);
                for (int f = max(0, i - S::RING); f < i; ++f) mbar_wait(&full[f % S::RING], (f / S::RING) & 1);
            }
        }
    } else if (warp <= 2) {
        // Two warps issue the products, one the scores and one the sums: each of these loops costs its warp some 500 cycles
        // a step in waits and issue, and both in one warp (1530 cycles) kept everything else waiting.
        if (n > 0) {
            const bool bf16 = p.a.type == PCB_BF16;
            const int ksteps = (p.a.dim + 15) / 16, nd = (p.a.dim + 15) / 16 * 16;
            constexpr uint32_t NEXT = S::OPERAND >> 4;
            Ring<S::RING> rg;  // the K (or V) block in use: every other one of the ring
            bool ok = true, ready = false;
            if (warp == 1) {  // S[i % 2] = Q K^T over the 64 keys of step i, in place of weights already used
                const uint32_t is = instr_desc(bf16, false, false, ROWS, STEP) | (p.negate ? 1u << 13 : 0u);
                const uint64_t dq = smem_desc(smem_addr(base), 16, 1024), dk0 = smem_desc(smem_addr(ring), 16, 1024);
                ok = wait_warp(q_full, 0, dead, &g_attn_timeouts);
                for (int i = 0; i < steps && ok; ++i) {
                    if (i % 2 == 0 && !__all_sync(~0u, ready)) ok = wait_warp(&full[rg.stage], rg.phase, dead, &g_attn_timeouts);
                    if (i >= 2) ok = ok && wait_warp(&pv_done[i % 2], (i - 2) / 2 & 1, dead, &g_attn_timeouts);
                    if (!ok) break;
                    fence_after();
                    const uint64_t dk = dk0 + rg.stage * NEXT + (uint32_t)(i % 2 * (STEP * 128) >> 4);
                    if (elect()) {
#pragma unroll
                        for (int s = 0; s < DP / 16; ++s) {
                            const uint32_t off = ((s / 4) * S::HALF + (s % 4) * 32) >> 4;
                            if (s < ksteps) mma_ss(tmem + S::S + i % 2 * STEP, dq + off, dk + off, is, s > 0);
                        }
                        mma_commit(&s_full[i % 2]);
                        if (i % 2 || i + 1 == steps) mma_commit(&empty[rg.stage]);
                    }
                    __syncwarp();
                    if (i % 2) {
                        rg.next(), rg.next();
                        ready = peek(&full[rg.stage], rg.phase);
                    }
                }
            } else {  // O += P[i % 2] V
                const uint32_t ipv = instr_desc(bf16, false, true, ROWS, nd);
                const uint64_t dv0 = smem_desc(smem_addr(ring), S::HALF, 1024);
                rg.next();
                for (int i = 0; i < steps && ok; ++i) {
                    if (i % 2 == 0 && !__all_sync(~0u, ready)) ok = wait_warp(&full[rg.stage], rg.phase, dead, &g_attn_timeouts);
                    ok = ok && wait_warp(&p_ready[i % 2], i / 2 & 1, dead, &g_attn_timeouts);
                    if (!ok) break;
                    fence_after();
                    const uint64_t dv = dv0 + rg.stage * NEXT + (uint32_t)(i % 2 * (STEP * 128) >> 4);
                    if (elect()) {
#pragma unroll
                        for (int s = 0; s < STEP / 16; ++s)
                            mma_ts(tmem + S::O, tmem + S::S + i % 2 * STEP + 8 * s, dv + (uint32_t)(s * 2048 >> 4), ipv, i > 0 || s > 0);
                        mma_commit(&pv_done[i % 2]);
                        if (i % 2 || i + 1 == steps) mma_commit(&empty[rg.stage]);
                    }
                    __syncwarp();
                    if (i % 2) {
                        rg.next(), rg.next();
                        ready = peek(&full[rg.stage], rg.phase);
                    }
                }
            }
            if (!ok) {  // the products in flight
                if (elect()) mma_commit(&drain[warp - 1]);
                mbar_wait(&drain[warp - 1], 0);
            }
        }
    } else {
        const int quad = warp % 4, r = quad * 32 + lane;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        int tok, head, limit;
        row_of(p, w, r, tok, head, limit);
        const bool mine = r < p.group * p.tokens && tok < w.nq;
        const bool bf16 = p.a.type == PCB_BF16;
        float top = -INFINITY, sum = 0.0f;
        bool ok = true;
        bool ready = false;
        for (int i = 0; i < steps; ++i) {
            if (!__all_sync(~0u, ready)) ok = wait_warp(&s_full[i % 2], i / 2 & 1, dead, &g_attn_timeouts);
            if (!ok) break;
            fence_after();
            const uint32_t at_s = tmem + S::S + i % 2 * STEP + lanes;
            float s[STEP];
            tmem_ld32(at_s, s);
            tmem_ld32(at_s + 32, s + 32);
            ld_wait();
            const int at = b0 * KEYS + i * STEP, left = limit - at;
            const bool masked = at + STEP > least;
            // 32 weights in 16 bits (their one rounding: the products with V take 16-bit operands), two per column
            auto put = [&](int h) {
                uint32_t w[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) w[j] = pack2(s[32 * h + 2 * j], s[32 * h + 2 * j + 1], bf16);
                tmem_st16(at_s + 16 * h, w);
            };
            if (POLY) {
#pragma unroll
                for (int j = 0; j < STEP; j += 2) {
                    const f32x2 x = two(s[j], s[j + 1]);
                    f32x2 r = both(p.coef[7]);
#pragma unroll
                    for (int e = 6; e >= 0; --e) r = fma2(r, x, both(p.coef[e]));
                    parts(r, s[j], s[j + 1]);
                }
                if (masked) {
#pragma unroll
                    for (int j = 0; j < STEP; ++j) s[j] = j < left ? s[j] : 0.0f;
                }
            } else {
                if (masked) {
#pragma unroll
                    for (int j = 0; j < STEP; ++j) s[j] = j < left ? s[j] : -INFINITY;
                }
                float m4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int j = 4; j + 7 < STEP; j += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) m4[e] = fmaxf(fmaxf(m4[e], s[j + e]), s[j + 4 + e]);
#pragma unroll
                for (int j = STEP - 4; j < STEP; ++j) m4[j % 4] = fmaxf(m4[j % 4], s[j]);
                const float big = fmaxf(top, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * p.c);
                const bool grew = big > top + 8.0f;
                if (__any_sync(~0u, grew)) {
                    const float f = grew ? ex2(top - big) : 1.0f;
                    if (i > 0) {
                        ok = wait_warp(&pv_done[(i - 1) % 2], (i - 1) / 2 & 1, dead, &g_attn_timeouts);
                        if (!ok) break;
                        fence_after();
#pragma unroll 1
                        for (int h = 0; h < DP / 16; ++h) {
                            float o[16];
                            tmem_ld16(tmem + S::O + lanes + 16 * h, o);
                            ld_wait();
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] *= f;
                            tmem_st16(tmem + S::O + lanes + 16 * h, (uint32_t*)o);
                        }
                    }
                    sum *= f;
                    if (grew) top = big;
                }
                const f32x2 c = both(p.c), sub = both(top == -INFINITY ? 0.0f : -top);
                f32x2 s2[2] = {0, 0};
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int j = 32 * h; j < 32 * h + 32; j += 2) {
                        const f32x2 x = fma2(two(s[j], s[j + 1]), c, sub);
                        f32x2 e;
                        if (DP == 64 && j / 2 % 4 == 3) {
                            e = exp2_fma(x);
                        } else {
                            float x0, x1;
                            parts(x, x0, x1);
                            e = two(ex2(x0), ex2(x1));
                        }
                        parts(e, s[j], s[j + 1]);
                        s2[j / 2 % 2] = add2(s2[j / 2 % 2], e);
                    }
                    put(h);
                }
                float x0, x1;
                parts(add2(s2[0], s2[1]), x0, x1);
                sum += x0 + x1;
            }
            if (POLY) put(0), put(1);
            ready = i + 1 < steps && peek(&s_full[(i + 1) % 2], (i + 1) / 2 & 1);
            st_wait();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_ready[i % 2]);
        }
        if (ok && steps > 0) ok = wait_warp(&pv_done[(steps - 1) % 2], (steps - 1) / 2 & 1, dead, &g_attn_timeouts);
        fence_after();
        if (ok) {
            const int64_t qrow = w.q0 + tok;
            // sees none of these keys: zeros, whatever the keys that other rows see have left in O (0 x Inf)
            const bool blind = limit <= b0 * KEYS;
            const float scale = POLY ? p.out_scale : p.splits > 1 ? 1.0f : 1.0f / sum;
            const int64_t prow = ((int64_t)w.split * p.a.q_rows + qrow) * p.a.heads + head;
            const int64_t orow = qrow * p.a.out_pitch + head * p.a.out_head;
            bool odd = false;
#pragma unroll 1
            for (int h = 0; h < DP / 32; ++h) {
                float o[32];
                if (n > 0) {
                    tmem_ld32(tmem + S::O + lanes + 32 * h, o);
                    ld_wait();
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    o[i] = blind ? 0.0f : o[i] * scale;
                    odd |= !(fabsf(o[i]) <= 3.4e38f) && 32 * h + i < p.a.dim;
                }
                if (!mine) continue;
                if (p.splits > 1) {
                    for (int i = 0; i < 32; ++i)
                        if (32 * h + i < p.a.dim) p.part_o[prow * p.a.dim + 32 * h + i] = o[i];
                } else if (p.out_vec) {
                    uint4* to = (uint4*)((uint16_t*)p.a.out + orow + 32 * h);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (32 * h + 8 * i < p.a.dim)
                            to[i] = make_uint4(pack2(o[8 * i], o[8 * i + 1], bf16), pack2(o[8 * i + 2], o[8 * i + 3], bf16),
                                               pack2(o[8 * i + 4], o[8 * i + 5], bf16), pack2(o[8 * i + 6], o[8 * i + 7], bf16));
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (32 * h + i < p.a.dim) store(p.a.out, orow + 32 * h + i, p.a.type, o[i]);
                }
            }
            if (mine && p.splits > 1) p.part_ml[prow] = part_of(blind, top, sum);
            // a sum of weights that is NaN, or 0, is the row's result (NaN): only keys that it sees take part in it
            again = __ballot_sync(~0u, mine && odd && (POLY || sum > 0.0f));
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 1) tmem_free(tmem, S::TMEM);
    if (again) redo<DP, POLY>(p, again);  // last, where nothing else lives in registers
}

// The splits of a row joined in order: a warp per (query, head)
__global__ void __launch_bounds__(256) join_splits(PcbClearAttention a, int splits, const float* part_o, const float2* part_ml) {
    pdl_wait();
    pdl_release();
    const int64_t rows = a.q_rows * a.heads, row = blockIdx.x * 8ll + threadIdx.x / 32;
    if (row >= rows) return;
    const int lane = threadIdx.x % 32;
    float top = -INFINITY, sum = 0.0f, o[4] = {};
    bool seen = false;
    if (!a.ncoef)
        for (int s = 0; s < splits; ++s) top = fmaxf(top, part_ml[s * rows + row].x);
    for (int s = 0; s < splits; ++s) {
        const float2 ml = part_ml[s * rows + row];
        const float f = a.ncoef ? 1.0f : ml.x == -INFINITY ? (ml.y == ml.y ? 0.0f : ml.y) : exp2f(ml.x - top);
        seen |= ml.y != 0.0f;
        if (f == 0.0f) continue;
        sum += ml.y * f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
            if (lane + 32 * t < a.dim) o[t] = fmaf(f, part_o[(s * rows + row) * a.dim + lane + 32 * t], o[t]);
    }
    const float f = a.ncoef ? 1.0f : sum == 0.0f ? (seen ? NAN : 0.0f) : 1.0f / sum;  // scores of -inf alone have no softmax
    const int64_t at = row / a.heads * a.out_pitch + row % a.heads * a.out_head;
    for (int t = 0; t < 4; ++t)
        if (lane + 32 * t < a.dim) store(a.out, at + lane + 32 * t, a.type, o[t] * f);
}

// [row][head][dim] at any strides to rows of `heads` x `to` adjacent values, zeros past dim
__global__ void __launch_bounds__(256) copy_heads(const uint16_t* x, int64_t pitch, int64_t head, int64_t rows, int heads, int dim,
                                                  uint16_t* y, int to) {
    pdl_wait();
    pdl_release();
    const int64_t total = rows * heads * to;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int d = (int)(i % to), h = (int)(i / to % heads);
        y[i] = d < dim ? x[i / to / heads * pitch + h * head + d] : (uint16_t)0;
    }
}

// ------------------------------------------------------------------------------------------------ host side
// One of q, k, v as the TMA engine can read it (16-byte aligned first element and strides, none of zero between several),
// or a copy
struct Heads {
    const void* p;
    int64_t pitch, head, rows;
    int heads;
    bool copy;
};
Heads heads_of(const void* p, int64_t pitch, int64_t head, int64_t rows, int heads, int dim) {
    Heads h{p, pitch, head, rows, heads, false};
    if (heads == 1) h.head = (dim + 7) / 8 * 8;
    if (rows == 1) h.pitch = heads * ((dim + 7) / 8 * 8);
    h.copy = ((uintptr_t)p & 15) || h.pitch % 8 || h.head % 8 || h.pitch == 0 || h.head == 0 || h.pitch >= (1ll << 38) ||
             h.head >= (1ll << 38);
    return h;
}
size_t copy_bytes(const Heads& h, int dim) { return h.copy ? (size_t)h.rows * h.heads * ((dim + 7) / 8 * 8) * 2 : 0; }
int make_copy(Heads& h, int dim, void* to, cudaStream_t s) {
    if (!h.copy) return 0;
    const int dp = (dim + 7) / 8 * 8;
    const int64_t blocks = (h.rows * h.heads * dp + 255) / 256;
    launch_pdl(copy_heads, dim3((unsigned)std::min<int64_t>(blocks, 16 * SMS)), dim3(256), s, (const uint16_t*)h.p, h.pitch, h.head,
               h.rows, h.heads, dim, (uint16_t*)to, dp);
    h.p = to, h.pitch = (int64_t)h.heads * dp, h.head = dp;
    return PCB_LAUNCH_RESULT();
}
int heads_map(CUtensorMap* map, const Heads& h, int type, int dim, int box_heads, int box_rows) {
    const uint64_t size[3] = {(uint64_t)dim, (uint64_t)h.heads, (uint64_t)h.rows};
    const uint64_t stride[2] = {(uint64_t)h.head * 2, (uint64_t)h.pitch * 2};
    const uint32_t box[3] = {64, (uint32_t)box_heads, (uint32_t)box_rows};
    return encode_map(map, type, h.p, 3, size, stride, box);
}

// Splits of the keys: as many as fill two blocks per SM, each with at least two key blocks, when the tiles alone do not. One
// launch's worth of sequences only: more of them are walked whole, launch after launch, though with few K/V heads (129 to 295
// single tokens of one) their tiles do not fill the SMs either.
int splits_of(const PcbClearAttention* a) {
    const int tokens = ROWS / (a->heads / a->kv_heads);
    int64_t tiles = 0;
    int longest = 0;
    for (int b = 0; b < a->nseq; ++b) {
        tiles += ((int64_t)a->q_lens[b] + tokens - 1) / tokens;
        if (a->q_lens[b]) longest = std::max(longest, a->k_lens[b]);
    }
    tiles *= a->kv_heads;
    const int blocks = (longest + KEYS - 1) / KEYS;
    if (tiles == 0 || tiles >= 2 * SMS || a->nseq > SEQS) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>({(2 * SMS + tiles - 1) / tiles, blocks / 2, 64}));
}

struct Ws {
    size_t bytes;
    Heads q, k, v;
    void *qc, *kc, *vc;
    int splits;
    float* part_o;
    float2* part_ml;
};
Ws attn_ws(const PcbClearAttention* a, void* ws) {
    Carve c(ws);
    Ws r;
    r.q = heads_of(a->q, a->q_pitch, a->q_head, a->q_rows, a->heads, a->dim);
    r.k = heads_of(a->k, a->k_pitch, a->k_head, a->k_rows, a->kv_heads, a->dim);
    r.v = heads_of(a->v, a->v_pitch, a->v_head, a->k_rows, a->kv_heads, a->dim);
    r.qc = c.take<char>(copy_bytes(r.q, a->dim));
    r.kc = c.take<char>(copy_bytes(r.k, a->dim));
    r.vc = c.take<char>(copy_bytes(r.v, a->dim));
    r.splits = splits_of(a);
    const size_t rows = r.splits > 1 ? (size_t)r.splits * a->q_rows * a->heads : 0;
    r.part_o = c.take<float>(rows * a->dim);
    r.part_ml = c.take<float2>(rows);
    r.bytes = c.used;
    return r;
}

template <int DP, bool POLY>
int launch(const Params& p, int64_t blocks, cudaStream_t s) {
    using S = Shape<DP>;
    static_assert(2 * (S::SMEM + 1024) <= 233472, "two blocks per SM");
    static std::atomic<uint64_t> done{0};
    if (int rc = allow_smem((const void*)attend<DP, POLY>, S::SMEM, done)) return rc;
    launch_pdl_smem(attend<DP, POLY>, dim3((unsigned)blocks), dim3(THREADS), S::SMEM, s, p);
    return PCB_LAUNCH_RESULT();
}

__global__ void __launch_bounds__(256) zero_out(PcbClearAttention a) {
    pdl_wait();
    pdl_release();
    const int64_t total = a.q_rows * a.heads * a.dim;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256)
        store(a.out, i / a.dim / a.heads * a.out_pitch + i / a.dim % a.heads * a.out_head + i % a.dim, a.type, 0.0f);
}

}  // namespace

unsigned int attn_timeouts() {
    unsigned int v = 0;
    return cudaMemcpyFromSymbol(&v, g_attn_timeouts, sizeof v) == cudaSuccess ? v : ~0u;
}

}  // namespace clear
}  // namespace pcb

using namespace pcb;
using namespace pcb::clear;

extern "C" {

int64_t pcb_clear_attention_ws(const PcbClearAttention* a) {
    if (int rc = bad_attention(a)) return rc;
    return a->q_rows && a->k_rows ? (int64_t)attn_ws(a, nullptr).bytes : 0;
}
int pcb_clear_attention(const PcbClearAttention* a, void* ws, size_t ws_bytes, cudaStream_t s) {
    if (int rc = bad_attention(a)) return rc;
    if (!a->q_rows) return 0;
    if (!a->k_rows) {
        launch_pdl(zero_out, dim3(4 * SMS), dim3(256), s, *a);
        return PCB_LAUNCH_RESULT();
    }
    Ws w = attn_ws(a, ws);
    if (int rc = bad_ws("clear_attention", ws, ws_bytes, w.bytes)) return rc;
    if (int rc = make_copy(w.q, a->dim, w.qc, s)) return rc;
    if (int rc = make_copy(w.k, a->dim, w.kc, s)) return rc;
    if (int rc = make_copy(w.v, a->dim, w.vc, s)) return rc;
    Params p;
    memset(&p, 0, offsetof(Params, w));
    p.a = *a;
    p.group = a->heads / a->kv_heads;
    p.tokens = ROWS / p.group;
    p.splits = w.splits;
    // a scale of zero keeps masked scores at -inf in the exponent
    p.c = std::max(std::fabs(a->scale) * 1.4426950408889634f, 1e-37f);
    p.negate = a->ncoef == 0 && a->scale < 0.0f;
    double big = 0.0, pw = 1.0;
    for (int i = 0; i < a->ncoef; ++i) big = std::max(big, (double)std::fabs(a->coef[i]));
    if (big == 0.0) big = 1.0;
    for (int i = 0; i < a->ncoef; ++i, pw *= a->scale) p.coef[i] = (float)(a->coef[i] * pw / big);
    p.out_scale = (float)big;
    p.part_o = w.part_o, p.part_ml = w.part_ml;
    p.out_vec = ((uintptr_t)a->out & 15) == 0 && a->out_pitch % 8 == 0 && a->out_head % 8 == 0 && a->dim % 8 == 0;
    if (int rc = heads_map(&p.q, w.q, a->type, a->dim, p.group, p.tokens)) return rc;
    if (int rc = heads_map(&p.k, w.k, a->type, a->dim, 1, KEYS)) return rc;
    if (int rc = heads_map(&p.v, w.v, a->type, a->dim, 1, KEYS)) return rc;
    int32_t q0 = 0, k0 = 0;
    for (int first = 0; first < a->nseq; first += SEQS) {
        const int n = std::min(a->nseq - first, SEQS);
        int32_t order[SEQS], q[SEQS], k[SEQS];
        for (int i = 0; i < n; ++i) {
            order[i] = i, q[i] = q0, k[i] = k0;
            q0 += a->q_lens[first + i], k0 += a->k_lens[first + i];
        }
        std::stable_sort(order, order + n, [&](int x, int y) { return a->k_lens[first + x] > a->k_lens[first + y]; });
        Work& wk = p.w;
        wk.n = 0;
        int64_t tiles = 0;
        for (int i = 0; i < n; ++i) {
            const int b = order[i], nq = a->q_lens[first + b];
            if (!nq) continue;
            wk.tile0[wk.n] = (int32_t)tiles;
            wk.q0[wk.n] = q[b], wk.nq[wk.n] = nq, wk.k0[wk.n] = k[b], wk.nk[wk.n] = a->k_lens[first + b];
            tiles += (nq + p.tokens - 1) / p.tokens;
            ++wk.n;
        }
        wk.tile0[wk.n] = (int32_t)tiles;
        const int64_t blocks = tiles * a->kv_heads * p.splits;
        if (!blocks) continue;
        if (blocks > INT32_MAX) return report(PCB_BAD_ARGS, "clear_attention: %lld blocks in one launch", (long long)blocks);
        const int rc = a->dim <= 64 ? (a->ncoef ? launch<64, true>(p, blocks, s) : launch<64, false>(p, blocks, s))
                                    : (a->ncoef ? launch<128, true>(p, blocks, s) : launch<128, false>(p, blocks, s));
        if (rc) return rc;
    }
    if (p.splits == 1) return 0;
    const int64_t rows = a->q_rows * a->heads;
    launch_pdl(join_splits, dim3((unsigned)((rows + 7) / 8)), dim3(256), s, *a, p.splits, (const float*)p.part_o, (const float2*)p.part_ml);
    return PCB_LAUNCH_RESULT();
}

}  // extern "C"
