// The clear half of the model (include/pcb200.h section 4): matrix product with bias, activation and residual, its
// gradients, attention over packed prompts, and the vocabulary loss with its gradients. First form: one tiled product
// kernel in 32-bit arithmetic that every operator's contraction goes through, and one warp per query for the attention.
#include "clear.h"

namespace pcb {
namespace clear {

// ------------------------------------------------------------------------------------------------ product
// Operand of a product: element (row, k) at p[row * rs + k * ks]
struct Mat {
    const void* p;
    int64_t rs, ks;
    int type;
};
enum Epi { EPI_LINEAR, EPI_DZ, EPI_STORE, EPI_ADD };
struct Out {
    void* y;
    int64_t pitch;
    int type;
    const void* bias;
    int bias_type;
    const void* extra;  // LINEAR: the residual (or null); DZ: dy
    int64_t extra_pitch;
    int extra_type;
    Act a;
};

// y[m][n] = epilogue(sum_k A(m, k) B(n, k)): 64 x 64 outputs per block of 256 threads (4 x 4 each), k in steps of 16
// through shared memory in 32 bits
template <int EPI>
__global__ void __launch_bounds__(256) product(Mat A, Mat B, int M, int N, int K, Out o) {
    __shared__ float sa[16][65], sb[16][65];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int64_t m0 = (int64_t)blockIdx.x * 64, n0 = (int64_t)blockIdx.y * 64;
    float acc[4][4] = {};
    for (int k0 = 0; k0 < K; k0 += 16) {
        for (int i = threadIdx.x; i < 1024; i += 256) {
            // the index that is adjacent in memory runs fastest over the threads
            const int ka = A.ks == 1 ? i % 16 : i / 64, ra = A.ks == 1 ? i / 16 : i % 64;
            const int kb = B.ks == 1 ? i % 16 : i / 64, rb = B.ks == 1 ? i / 16 : i % 64;
            sa[ka][ra] = m0 + ra < M && k0 + ka < K ? load(A.p, (m0 + ra) * A.rs + (int64_t)(k0 + ka) * A.ks, A.type) : 0.0f;
            sb[kb][rb] = n0 + rb < N && k0 + kb < K ? load(B.p, (n0 + rb) * B.rs + (int64_t)(k0 + kb) * B.ks, B.type) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty + 16 * i], sb[k][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
            if (m >= M || n >= N) continue;
            float v = acc[i][j];
            if (EPI == EPI_LINEAR || EPI == EPI_DZ) {
                if (o.bias) v += load(o.bias, n, o.bias_type);
                const float e = o.extra ? load(o.extra, m * o.extra_pitch + n, o.extra_type) : 0.0f;
                v = EPI == EPI_DZ ? e * act_slope(o.a, v) : act(o.a, v) + e;
            }
            if (EPI == EPI_ADD) v += load(o.y, m * o.pitch + n, o.type);
            store(o.y, m * o.pitch + n, o.type, v);
        }
}
template <int EPI>
int run_product(const Mat& A, const Mat& B, int M, int N, int K, const Out& o, cudaStream_t s) {
    const dim3 g((unsigned)((M + 63) / 64), (unsigned)((N + 63) / 64));
    product<EPI><<<g, 256, 0, s>>>(A, B, M, N, K, o);
    return PCB_LAUNCH_RESULT();
}

// out[n] = sum_m x[m][n] in a fixed order: 32 columns per block, 8 row lanes joined in shared memory
__global__ void __launch_bounds__(256) column_sum(const void* x, int64_t pitch, int type, int M, int N, void* out, int out_type) {
    __shared__ float part[8][32];
    const int c = threadIdx.x % 32, r = threadIdx.x / 32;
    const int64_t n = (int64_t)blockIdx.x * 32 + c;
    float s = 0.0f;
    if (n < N)
        for (int64_t m = r; m < M; m += 8) s += load(x, m * pitch + n, type);
    part[r][c] = s;
    __syncthreads();
    if (r == 0 && n < N) {
        for (int i = 1; i < 8; ++i) s += part[i][c];
        store(out, n, out_type, s);
    }
}
__global__ void convert(const float* x, int64_t rows, int64_t cols, void* y, int64_t pitch, int type) {
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * blockDim.x)
        store(y, i / cols * pitch + i % cols, type, x[i]);
}
__global__ void fill_rows(void* y, int64_t rows, int64_t cols, int64_t pitch, int type) {
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * blockDim.x)
        store(y, i / cols * pitch + i % cols, type, 0.0f);
}

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

// ------------------------------------------------------------------------------------------------ vocabulary loss
// One block per row over a piece of logits (32 bits): the running maximum and sum of the row, the target's logit; with
// the last piece the row's lse and loss.
__global__ void __launch_bounds__(256) vocab_rows(const float* l, int P, int v0, PcbClearVocab a, float2* state, float* hit, int last) {
    const int64_t r = blockIdx.x;
    __shared__ float red[256];
    const float* x = l + r * P;
    const int cols = min(P, a.vocab - v0);
    const bool begin = v0 == 0;
    float m = -INFINITY;
    for (int i = threadIdx.x; i < cols; i += 256) m = fmaxf(m, x[i]);
    red[threadIdx.x] = m;
    __syncthreads();
    for (int w = 128; w; w >>= 1) {
        if (threadIdx.x < w) red[threadIdx.x] = fmaxf(red[threadIdx.x], red[threadIdx.x + w]);
        __syncthreads();
    }
    m = begin ? red[0] : fmaxf(red[0], state[r].x);
    __syncthreads();
    float s = 0.0f;
    for (int i = threadIdx.x; i < cols; i += 256) s += expf(x[i] - m);
    red[threadIdx.x] = s;
    __syncthreads();
    for (int w = 128; w; w >>= 1) {
        if (threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x) return;
    s = red[0] + (begin ? 0.0f : state[r].y * expf(state[r].x - m));
    state[r] = make_float2(m, s);
    const int64_t t = a.targets[r];
    if (begin) hit[r] = NAN;
    if (t >= v0 && t < v0 + cols) hit[r] = x[t - v0];
    if (last) {
        const float lse = m + logf(s);
        a.lse[r] = lse;
        a.loss[r] = t == a.ignore ? 0.0f : lse - hit[r];
    }
}
// logits in place to their gradients
__global__ void __launch_bounds__(256) vocab_slopes(float* l, int P, int v0, PcbClearVocab a, const float* weight) {
    const int64_t r = blockIdx.x;
    const int64_t t = a.targets[r];
    const float lse = a.lse[r], g = weight[r];
    for (int i = threadIdx.x; i < P; i += 256) {
        float* x = l + r * P + i;
        *x = v0 + i >= a.vocab || t == a.ignore ? 0.0f : g * (expf(*x - lse) - (t == v0 + i ? 1.0f : 0.0f));
    }
}
// Columns of one piece: the piece's 32-bit logits take at most 256 MiB, at least 64 columns
int piece(int rows, int vocab) {
    const int64_t fit = (256ll << 20) / 4 / (rows > 0 ? rows : 1);
    const int64_t p = fit < 64 ? 64 : fit / 64 * 64;
    return (int)(p < vocab ? p : vocab);
}

}  // namespace clear
}  // namespace pcb

using namespace pcb;
using namespace pcb::clear;

extern "C" {

int64_t pcb_clear_linear_ws(const PcbClearLinear* a) { return bad_linear(a); }
int pcb_clear_linear(const PcbClearLinear* a, void*, size_t, cudaStream_t s) {
    if (int rc = bad_linear(a)) return rc;
    if (!a->m || !a->n) return 0;
    const Mat A{a->x, a->x_pitch, 1, a->type};
    const Mat B = a->w_cols ? Mat{a->w, a->w_pitch, 1, a->type} : Mat{a->w, 1, a->w_pitch, a->type};
    const Out o{a->y, a->y_pitch, a->y_type, a->bias, a->bias_type, a->residual, a->residual_pitch, a->residual_type,
                make_act(a->act, a->bound, a->coef)};
    return run_product<EPI_LINEAR>(A, B, a->m, a->n, a->k, o, s);
}

static size_t grad_ws(const PcbClearLinearGrad* a, Carve& c, float** dz) {
    *dz = a->act ? c.take<float>((size_t)a->m * a->n) : nullptr;
    return c.used;
}
int64_t pcb_clear_linear_grad_ws(const PcbClearLinearGrad* a) {
    if (int rc = bad_grad(a)) return rc;
    Carve c(nullptr);
    float* dz;
    return (int64_t)grad_ws(a, c, &dz);
}
int pcb_clear_linear_grad(const PcbClearLinearGrad* a, void* ws, size_t ws_bytes, cudaStream_t s) {
    if (int rc = bad_grad(a)) return rc;
    Carve c(ws);
    float* dzp;
    if (int rc = bad_ws("clear_linear_grad", ws, ws_bytes, grad_ws(a, c, &dzp))) return rc;
    const Mat x{a->x, a->x_pitch, 1, a->type}, xt{a->x, 1, a->x_pitch, a->type};
    const Mat wn = a->w_cols ? Mat{a->w, a->w_pitch, 1, a->type} : Mat{a->w, 1, a->w_pitch, a->type};  // rows n, along k
    const Mat wk = a->w_cols ? Mat{a->w, 1, a->w_pitch, a->type} : Mat{a->w, a->w_pitch, 1, a->type};  // rows k, along n
    Mat dz{a->dy, a->dy_pitch, 1, a->type};
    if (a->act && a->m) {
        const Out o{dzp, a->n, PCB_F32, a->bias, a->bias_type, a->dy, a->dy_pitch, a->type, make_act(a->act, a->bound, a->coef)};
        if (int rc = run_product<EPI_DZ>(x, wn, a->m, a->n, a->k, o, s)) return rc;
        dz = Mat{dzp, a->n, 1, PCB_F32};
    }
    const Mat dzt{dz.p, 1, dz.rs, dz.type};
    Out o{};
    o.type = a->type;
    if (a->dx && a->m) {
        o.y = a->dx, o.pitch = a->dx_pitch;
        if (int rc = run_product<EPI_STORE>(dz, wk, a->m, a->k, a->n, o, s)) return rc;
    }
    if (a->dw) {
        o.y = a->dw, o.pitch = a->dw_pitch;
        if (int rc = a->w_cols ? run_product<EPI_STORE>(dzt, xt, a->n, a->k, a->m, o, s)
                               : run_product<EPI_STORE>(xt, dzt, a->k, a->n, a->m, o, s))
            return rc;
    }
    if (a->db) {
        column_sum<<<(a->n + 31) / 32, 256, 0, s>>>(dz.p, dz.rs, dz.type, a->m, a->n, a->db, a->db_type);
        return PCB_LAUNCH_RESULT();
    }
    return 0;
}

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

int64_t pcb_clear_vocab_loss_ws(const PcbClearVocab* a) {
    if (int rc = bad_vocab(a, false)) return rc;
    Carve c(nullptr);
    c.take<float>((size_t)a->rows * piece(a->rows, a->vocab));
    c.take<float2>(a->rows);
    c.take<float>(a->rows);
    return (int64_t)c.used;
}
int pcb_clear_vocab_loss(const PcbClearVocab* a, void* ws, size_t ws_bytes, cudaStream_t s) {
    if (int rc = bad_vocab(a, false)) return rc;
    if (int rc = bad_ws("clear_vocab_loss", ws, ws_bytes, (size_t)pcb_clear_vocab_loss_ws(a))) return rc;
    if (!a->rows) return 0;
    const int P = piece(a->rows, a->vocab);
    Carve c(ws);
    float* l = c.take<float>((size_t)a->rows * P);
    float2* state = c.take<float2>(a->rows);
    float* hit = c.take<float>(a->rows);
    Out o{};
    o.y = l, o.pitch = P, o.type = PCB_F32;
    for (int v0 = 0; v0 < a->vocab; v0 += P) {
        const int cols = a->vocab - v0 < P ? a->vocab - v0 : P;
        const Mat w{(const char*)a->w + 2 * v0 * a->w_pitch, a->w_pitch, 1, a->type};
        if (int rc = run_product<EPI_STORE>(Mat{a->h, a->h_pitch, 1, a->type}, w, a->rows, cols, a->dim, o, s)) return rc;
        vocab_rows<<<a->rows, 256, 0, s>>>(l, P, v0, *a, state, hit, v0 + P >= a->vocab);
        if (int rc = PCB_LAUNCH_RESULT()) return rc;
    }
    return 0;
}

int64_t pcb_clear_vocab_grad_ws(const PcbClearVocabGrad* a) {
    if (int rc = bad_vocab_grad(a)) return rc;
    Carve c(nullptr);
    c.take<float>((size_t)a->v.rows * piece(a->v.rows, a->v.vocab));
    c.take<float>((size_t)a->v.rows * a->v.dim);
    return (int64_t)c.used;
}
int pcb_clear_vocab_grad(const PcbClearVocabGrad* a, void* ws, size_t ws_bytes, cudaStream_t s) {
    if (int rc = bad_vocab_grad(a)) return rc;
    if (int rc = bad_ws("clear_vocab_grad", ws, ws_bytes, (size_t)pcb_clear_vocab_grad_ws(a))) return rc;
    const PcbClearVocab& v = a->v;
    if (!v.rows) {
        if (!a->dw) return 0;
        fill_rows<<<1024, 256, 0, s>>>(a->dw, v.vocab, v.dim, a->dw_pitch, v.type);
        return PCB_LAUNCH_RESULT();
    }
    const int P = piece(v.rows, v.vocab);
    Carve c(ws);
    float* l = c.take<float>((size_t)v.rows * P);
    float* dh = c.take<float>((size_t)v.rows * v.dim);
    const Mat h{v.h, v.h_pitch, 1, v.type}, ht{v.h, 1, v.h_pitch, v.type};
    for (int v0 = 0; v0 < v.vocab; v0 += P) {
        const int cols = v.vocab - v0 < P ? v.vocab - v0 : P;
        const void* wp = (const char*)v.w + 2 * v0 * v.w_pitch;
        Out o{};
        o.y = l, o.pitch = P, o.type = PCB_F32;
        if (int rc = run_product<EPI_STORE>(h, Mat{wp, v.w_pitch, 1, v.type}, v.rows, cols, v.dim, o, s)) return rc;
        vocab_slopes<<<v.rows, 256, 0, s>>>(l, P, v0, v, a->weight);
        if (int rc = PCB_LAUNCH_RESULT()) return rc;
        if (a->dh) {
            o.y = dh, o.pitch = v.dim;
            const Mat L{l, P, 1, PCB_F32}, W{wp, 1, v.w_pitch, v.type};
            if (int rc = v0 ? run_product<EPI_ADD>(L, W, v.rows, v.dim, cols, o, s) : run_product<EPI_STORE>(L, W, v.rows, v.dim, cols, o, s))
                return rc;
        }
        if (a->dw) {
            o.y = (char*)a->dw + 2 * v0 * a->dw_pitch, o.pitch = a->dw_pitch, o.type = v.type;
            if (int rc = run_product<EPI_STORE>(Mat{l, 1, P, PCB_F32}, ht, cols, v.dim, v.rows, o, s)) return rc;
        }
    }
    if (!a->dh) return 0;
    convert<<<1024, 256, 0, s>>>(dh, v.rows, v.dim, a->dh, a->dh_pitch, v.type);
    return PCB_LAUNCH_RESULT();
}

}  // extern "C"
