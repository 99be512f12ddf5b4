// Shared by the clear half's translation units (clear_*.cu): 16-bit element access, argument checks, the workspace.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cmath>
#include <cstdint>

#include "arith.cuh"
#include "kernels.h"

namespace pcb {
// records the message of pcb_last_error and returns `code` (evaluator.cu)
int report(int code, const char* fmt, ...);

namespace clear {

// ------------------------------------------------------------------------------------------------ elements
// Element i of a PCB_BF16 / PCB_F16 / PCB_F32 array in 32 bits, and back with one rounding
__device__ __forceinline__ float load(const void* p, size_t i, int type) {
    if (type == PCB_F32) return ((const float*)p)[i];
    return type == PCB_BF16 ? __bfloat162float(((const __nv_bfloat16*)p)[i]) : __half2float(((const __half*)p)[i]);
}
__device__ __forceinline__ void store(void* p, size_t i, int type, float v) {
    if (type == PCB_F32) ((float*)p)[i] = v;
    else if (type == PCB_BF16) ((__nv_bfloat16*)p)[i] = __float2bfloat16(v);
    else ((__half*)p)[i] = __float2half(v);
}
inline size_t type_bytes(int type) { return type == PCB_F32 ? 4 : 2; }

// ------------------------------------------------------------------------------------------------ activations
// PCB_ACT_POLY: value sum c[i] u^i and slope sum d[i] u^i at u = z inv_bound
struct Act {
    int kind;
    float inv_bound;
    float c[8], d[7];
};
inline Act make_act(int kind, float bound, const float* coef) {
    Act a = {kind, 1.0f, {}, {}};
    if (kind != PCB_ACT_POLY) return a;
    a.inv_bound = 1.0f / bound;
    for (int i = 0; i < 8; ++i) a.c[i] = coef[i];
    for (int i = 1; i < 8; ++i) a.d[i - 1] = (float)((double)i * coef[i] / bound);
    return a;
}

// ------------------------------------------------------------------------------------------------ checks
// The largest size: rows and columns of tiles that reach past the last one are counted in 32 bits
constexpr int32_t MOST = INT32_MAX - 1024;
inline bool is16(int type) { return type == PCB_BF16 || type == PCB_F16; }
inline bool known(int type, int call) { return type == call || type == PCB_F32; }
// a pointer that is not a multiple of its elements' size
inline bool off(const void* p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) != 0; }
inline bool poly_ok(int kind, float bound, const float* coef) {
    if (kind != PCB_ACT_POLY) return true;
    if (!(bound > 0.0f) || !std::isfinite(bound)) return false;
    for (int i = 0; i < 8; ++i)
        if (!std::isfinite(coef[i])) return false;
    return true;
}
inline int bad_linear(const PcbClearLinear* a) {
    if (!a) return report(PCB_BAD_ARGS, "clear_linear: null arguments");
    if (a->m < 0 || a->k < 1 || a->n < 0 || a->m > MOST || a->k > MOST || a->n > MOST)
        return report(PCB_BAD_ARGS, "clear_linear: m %d, k %d, n %d", a->m, a->k, a->n);
    if (!is16(a->type)) return report(PCB_BAD_ARGS, "clear_linear: type %d is not PCB_BF16 or PCB_F16", a->type);
    if (a->act < 0 || a->act > PCB_ACT_POLY || !poly_ok(a->act, a->bound, a->coef))
        return report(PCB_BAD_ARGS, "clear_linear: act %d, bound %g", a->act, (double)a->bound);
    if ((a->bias && !known(a->bias_type, a->type)) || (a->residual && !known(a->residual_type, a->type)) ||
        !known(a->y_type, a->type))
        return report(PCB_BAD_ARGS, "clear_linear: bias, residual and y are of the call's type or PCB_F32");
    if (a->m == 0 || a->n == 0) return 0;
    if (!a->x || !a->w || !a->y) return report(PCB_BAD_ARGS, "clear_linear: null x, w or y");
    if (off(a->x, 2) || off(a->w, 2) || off(a->y, type_bytes(a->y_type)) || off(a->bias, a->bias ? type_bytes(a->bias_type) : 1) ||
        off(a->residual, a->residual ? type_bytes(a->residual_type) : 1))
        return report(PCB_BAD_ARGS, "clear_linear: a pointer is off its elements' size");
    if (a->x_pitch < a->k || a->w_pitch < (a->w_cols ? a->k : a->n) || a->y_pitch < a->n ||
        (a->residual && a->residual_pitch < a->n))
        return report(PCB_BAD_ARGS, "clear_linear: a pitch is below its row's elements");
    return 0;
}
inline int bad_grad(const PcbClearLinearGrad* a) {
    if (!a) return report(PCB_BAD_ARGS, "clear_linear_grad: null arguments");
    if (a->m < 0 || a->k < 1 || a->n < 1 || a->m > MOST || a->k > MOST || a->n > MOST)
        return report(PCB_BAD_ARGS, "clear_linear_grad: m %d, k %d, n %d", a->m, a->k, a->n);
    if (!is16(a->type)) return report(PCB_BAD_ARGS, "clear_linear_grad: type %d is not PCB_BF16 or PCB_F16", a->type);
    if (a->act < 0 || a->act > PCB_ACT_POLY || !poly_ok(a->act, a->bound, a->coef))
        return report(PCB_BAD_ARGS, "clear_linear_grad: act %d, bound %g", a->act, (double)a->bound);
    if ((a->bias && !known(a->bias_type, a->type)) || (a->db && !known(a->db_type, a->type)))
        return report(PCB_BAD_ARGS, "clear_linear_grad: bias and db are of the call's type or PCB_F32");
    if (a->m > 0 && (!a->dy || !a->x || !a->w)) return report(PCB_BAD_ARGS, "clear_linear_grad: null dy, x or w");
    if (off(a->dy, 2) || off(a->x, 2) || off(a->w, 2) || off(a->dx, 2) || off(a->dw, 2) ||
        off(a->bias, a->bias ? type_bytes(a->bias_type) : 1) || off(a->db, a->db ? type_bytes(a->db_type) : 1))
        return report(PCB_BAD_ARGS, "clear_linear_grad: a pointer is off its elements' size");
    const int64_t wrow = a->w_cols ? a->k : a->n;
    if ((a->m > 0 && (a->dy_pitch < a->n || a->x_pitch < a->k || a->w_pitch < wrow)) || (a->dx && a->dx_pitch < a->k) ||
        (a->dw && a->dw_pitch < wrow))
        return report(PCB_BAD_ARGS, "clear_linear_grad: a pitch is below its row's elements");
    return 0;
}
inline int bad_attention(const PcbClearAttention* a) {
    if (!a) return report(PCB_BAD_ARGS, "clear_attention: null arguments");
    if (a->nseq < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads || a->heads / a->kv_heads > 128 ||
        a->dim < 1 || a->dim > 128)
        return report(PCB_BAD_ARGS, "clear_attention: %d sequences, %d heads over %d (a multiple, at most 128 each), dim %d (1..128)",
                      a->nseq, a->heads, a->kv_heads, a->dim);
    if (!is16(a->type)) return report(PCB_BAD_ARGS, "clear_attention: type %d is not PCB_BF16 or PCB_F16", a->type);
    if (a->ncoef < 0 || a->ncoef > 8 || !std::isfinite(a->scale))
        return report(PCB_BAD_ARGS, "clear_attention: %d coefficients (0..8), scale %g", a->ncoef, (double)a->scale);
    for (int i = 0; i < a->ncoef; ++i)
        if (!std::isfinite(a->coef[i])) return report(PCB_BAD_ARGS, "clear_attention: coefficient %d is not finite", i);
    if (a->nseq > 0 && (!a->q_lens || !a->k_lens)) return report(PCB_BAD_ARGS, "clear_attention: null lengths");
    if (a->q_rows > MOST || a->k_rows > MOST) return report(PCB_BAD_ARGS, "clear_attention: over %d tokens", MOST);
    int64_t qs = 0, ks = 0;
    for (int b = 0; b < a->nseq; ++b) {
        if (a->q_lens[b] < 0 || a->k_lens[b] < 0)
            return report(PCB_BAD_ARGS, "clear_attention: sequence %d has %d queries, %d keys", b, a->q_lens[b], a->k_lens[b]);
        qs += a->q_lens[b];
        ks += a->k_lens[b];
    }
    if (qs != a->q_rows || ks != a->k_rows)
        return report(PCB_BAD_ARGS, "clear_attention: lengths sum to %lld and %lld, q has %lld rows and k %lld", (long long)qs,
                      (long long)ks, (long long)a->q_rows, (long long)a->k_rows);
    if ((qs && (!a->q || !a->out)) || (qs && ks && (!a->k || !a->v)))
        return report(PCB_BAD_ARGS, "clear_attention: null q, k, v or out");
    if (off(a->q, 2) || off(a->k, 2) || off(a->v, 2) || off(a->out, 2))
        return report(PCB_BAD_ARGS, "clear_attention: a pointer is off its elements' size");
    const int64_t strides[] = {a->q_pitch, a->q_head, a->k_pitch, a->k_head, a->v_pitch, a->v_head, a->out_pitch, a->out_head};
    for (int64_t st : strides)
        if (st < 0) return report(PCB_BAD_ARGS, "clear_attention: negative stride");
    return 0;
}
inline int bad_vocab(const PcbClearVocab* a, bool grad) {
    const char* who = grad ? "clear_vocab_grad" : "clear_vocab_loss";
    if (!a) return report(PCB_BAD_ARGS, "%s: null arguments", who);
    if (a->rows < 0 || a->vocab < 1 || a->dim < 1 || a->rows > MOST || a->vocab > MOST || a->dim > MOST)
        return report(PCB_BAD_ARGS, "%s: %d rows, vocabulary of %d, dim %d", who, a->rows, a->vocab, a->dim);
    if (!is16(a->type)) return report(PCB_BAD_ARGS, "%s: type %d is not PCB_BF16 or PCB_F16", who, a->type);
    if (a->rows > 0 && (!a->h || !a->w || !a->targets || !a->lse || (!grad && !a->loss)))
        return report(PCB_BAD_ARGS, "%s: null h, w, targets, lse or loss", who);
    if (off(a->h, 2) || off(a->w, 2) || off(a->targets, 8) || off(a->loss, 4) || off(a->lse, 4))
        return report(PCB_BAD_ARGS, "%s: a pointer is off its elements' size", who);
    if (a->rows > 0 && (a->h_pitch < a->dim || a->w_pitch < a->dim))
        return report(PCB_BAD_ARGS, "%s: a pitch is below its row's elements", who);
    return 0;
}
inline int bad_vocab_grad(const PcbClearVocabGrad* a) {
    if (!a) return report(PCB_BAD_ARGS, "clear_vocab_grad: null arguments");
    if (int rc = bad_vocab(&a->v, true)) return rc;
    if (a->v.rows > 0 && !a->weight) return report(PCB_BAD_ARGS, "clear_vocab_grad: null weight");
    if (off(a->weight, 4) || off(a->dh, 2) || off(a->dw, 2))
        return report(PCB_BAD_ARGS, "clear_vocab_grad: a pointer is off its elements' size");
    if ((a->dh && a->dh_pitch < a->v.dim) || (a->dw && a->dw_pitch < a->v.dim))
        return report(PCB_BAD_ARGS, "clear_vocab_grad: a pitch is below its row's elements");
    return 0;
}

// ------------------------------------------------------------------------------------------------ launching
// Lets a kernel use `bytes` of dynamic shared memory on the current device, once per device (`done`: the kernel's own)
inline int allow_smem(const void* kernel, size_t bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return 0;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return (int)e;
}

// ------------------------------------------------------------------------------------------------ workspace
// Carves 256-byte aligned pieces off the caller's workspace; with a null base it only counts.
struct Carve {
    char* base;
    size_t used = 0;
    explicit Carve(void* p) : base((char*)p) {}
    template <class T>
    T* take(size_t n) {
        T* r = base ? (T*)(base + used) : nullptr;
        used += (n * sizeof(T) + 255) / 256 * 256;
        return r;
    }
};
inline int bad_ws(const char* who, const void* ws, size_t have, size_t need) {
    if (need && (!ws || have < need || ((uintptr_t)ws & 255)))
        return report(PCB_BAD_ARGS, "%s: workspace of %zu bytes at %p, %zu at a 256-byte boundary needed", who, have, ws, need);
    return 0;
}

}  // namespace clear
}  // namespace pcb
