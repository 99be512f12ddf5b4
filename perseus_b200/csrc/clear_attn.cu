// Attention over packed prompts (pcb_clear_attention). First form: one warp per query.
#include "clear.h"

namespace pcb {
namespace clear {

// ------------------------------------------------------------------------------------------------ attention
// One warp per (query, head); lane l holds dims l, l + 32, ...; softmax with a running maximum and sum. starts: the
// sequences' first rows come from walking the lengths, passed as blocks of up to SEQS sequences per launch.
constexpr int SEQS = 256;
struct Seqs {
    int32_t n;
    int32_t q0[SEQS + 1], k0[SEQS + 1];
};
__global__ void __launch_bounds__(128) attend_rows(PcbClearAttention a, Seqs sq) {
    const int64_t first = sq.q0[0];
    const int64_t item = blockIdx.x * 4ll + threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    const int64_t row = first + item / a.heads;
    const int head = (int)(item % a.heads);
    if (row >= sq.q0[sq.n]) return;
    int b = 0;
    while (row >= sq.q0[b + 1]) ++b;
    const int nq = sq.q0[b + 1] - sq.q0[b], nk = sq.k0[b + 1] - sq.k0[b];
    const int64_t i = row - sq.q0[b];
    const int64_t seen = a.causal ? min((int64_t)nk, i + nk - nq + 1) : nk;
    const int kh = head / (a.heads / a.kv_heads);
    float q[4], o[4] = {}, top = -INFINITY, sum = 0.0f;
    for (int t = 0; t < 4; ++t) {
        const int d = lane + 32 * t;
        q[t] = d < a.dim ? load(a.q, row * a.q_pitch + head * a.q_head + d, a.type) : 0.0f;
    }
    for (int64_t j = 0; j < seen; ++j) {
        const int64_t kr = sq.k0[b] + j;
        float s = 0.0f;
        for (int t = 0; t < 4; ++t) {
            const int d = lane + 32 * t;
            if (d < a.dim) s = fmaf(q[t], load(a.k, kr * a.k_pitch + kh * a.k_head + d, a.type), s);
        }
        for (int m = 16; m; m >>= 1) s += __shfl_xor_sync(~0u, s, m);
        s *= a.scale;
        float p;
        if (a.ncoef) {
            p = a.coef[a.ncoef - 1];
            for (int c = a.ncoef - 2; c >= 0; --c) p = fmaf(p, s, a.coef[c]);
        } else {
            const float nt = fmaxf(top, s), f = top == -INFINITY ? 0.0f : expf(top - nt);
            p = nt == -INFINITY ? 0.0f : expf(s - nt);
            sum = sum * f + p;
            for (int t = 0; t < 4; ++t) o[t] *= f;
            top = nt;
        }
        for (int t = 0; t < 4; ++t) {
            const int d = lane + 32 * t;
            if (d < a.dim) o[t] = fmaf(p, load(a.v, kr * a.v_pitch + kh * a.v_head + d, a.type), o[t]);
        }
    }
    const float f = a.ncoef ? 1.0f : seen > 0 ? 1.0f / sum : 0.0f;
    for (int t = 0; t < 4; ++t) {
        const int d = lane + 32 * t;
        if (d < a.dim) store(a.out, row * a.out_pitch + head * a.out_head + d, a.type, o[t] * f);
    }
}

}  // namespace clear
}  // namespace pcb

using namespace pcb;
using namespace pcb::clear;

extern "C" {

int64_t pcb_clear_attention_ws(const PcbClearAttention* a) { return bad_attention(a); }
int pcb_clear_attention(const PcbClearAttention* a, void*, size_t, cudaStream_t s) {
    if (int rc = bad_attention(a)) return rc;
    int32_t q0 = 0, k0 = 0;
    for (int b0 = 0; b0 < a->nseq; b0 += SEQS) {
        Seqs sq;
        sq.n = a->nseq - b0 < SEQS ? a->nseq - b0 : SEQS;
        for (int i = 0; i < sq.n; ++i) {
            sq.q0[i] = q0, sq.k0[i] = k0;
            q0 += a->q_lens[b0 + i], k0 += a->k_lens[b0 + i];
        }
        sq.q0[sq.n] = q0, sq.k0[sq.n] = k0;
        const int64_t items = (int64_t)(q0 - sq.q0[0]) * a->heads;
        if (!items) continue;
        attend_rows<<<(unsigned)((items + 3) / 4), 128, 0, s>>>(*a, sq);
        if (int rc = PCB_LAUNCH_RESULT()) return rc;
    }
    return 0;
}

}  // extern "C"
