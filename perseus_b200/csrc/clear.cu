// The clear half's operators on the product of clear_gemm.cu (include/pcb200.h section 4): linear, its gradients, and the
// vocabulary loss with its gradients.
#include <algorithm>
#include <cstring>
#include <utility>

#include "clear_gemm.h"

namespace pcb {
namespace clear {

// ------------------------------------------------------------------------------------------------ column sums
// Sums over the rows of a matrix, in two launches of fixed order: 256 rows of 64 columns per block, more where a grid would
// have over 65535 blocks along the rows (a warp along the columns, two per lane, eight row lanes joined in shared memory),
// then the blocks' sums the same way. The first may run beside the
// product launched before it, from which it reads nothing (`beside`): it then waits for that one only before it ends.
constexpr int SUM_ONCE = 1024;  // up to SUM_ONCE rows one launch does: beside a product it costs no time
constexpr int sum_rows_of(int m) { return std::max(256, m / 65535 + 1); }
constexpr int sum_parts(int m) { return m / sum_rows_of(m) + (m % sum_rows_of(m) != 0); }
__global__ void __launch_bounds__(256) sum_rows(const void* x, int64_t pitch, int type, int m, int n, int rows, float* part, void* out,
                                                int out_type, bool beside) {
    __shared__ float2 red[8][32];
    if (!beside) pdl_wait();
    pdl_release();
    const int c = threadIdx.x % 32, r = threadIdx.x / 32;
    const int64_t col = blockIdx.x * 64ll + 2 * c, r0 = (int64_t)blockIdx.y * rows, r1 = min((int64_t)m, r0 + rows);
    float2 s = make_float2(0.0f, 0.0f);
    const bool wide = type == PCB_F32, pairs = pitch % 2 == 0 && ((uintptr_t)x & (wide ? 7 : 3)) == 0 && col + 1 < n;
    if (pairs && wide) {
#pragma unroll 8
        for (int64_t i = r0 + r; i < r1; i += 8) {
            const float2 v = *(const float2*)((const float*)x + i * pitch + col);
            s.x += v.x, s.y += v.y;
        }
    } else if (pairs) {
#pragma unroll 8
        for (int64_t i = r0 + r; i < r1; i += 8) {
            const uint32_t w = *(const uint32_t*)((const uint16_t*)x + i * pitch + col);
            float2 v;
            if (type == PCB_BF16) v = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
            else v = __half22float2(*(const __half2*)&w);
            s.x += v.x, s.y += v.y;
        }
    } else {
#pragma unroll 4
        for (int64_t i = r0 + r; i < r1; i += 8) {
            if (col < n) s.x += load(x, i * pitch + col, type);
            if (col + 1 < n) s.y += load(x, i * pitch + col + 1, type);
        }
    }
    red[r][c] = s;
    __syncthreads();
    if (r == 0) {
        for (int i = 1; i < 8; ++i) s.x += red[i][c].x, s.y += red[i][c].y;
        for (int e = 0; e < 2; ++e)
            if (col + e < n) {
                if (part) part[(int64_t)blockIdx.y * n + col + e] = e ? s.y : s.x;
                else store(out, col + e, out_type, e ? s.y : s.x);
            }
    }
    if (beside) pdl_wait();  // later launches may rely on everything before this one
}
int run_sum(const void* x, int64_t pitch, int type, int m, int n, float* part, void* out, int out_type, bool beside, cudaStream_t s) {
    const dim3 g((n + 63) / 64, part ? sum_parts(m) : 1);
    launch_pdl(sum_rows, g, dim3(256), s, x, pitch, type, m, n, part ? sum_rows_of(m) : m, part, out, out_type, beside);
    return PCB_LAUNCH_RESULT();
}

// The largest finite size of a float16 matrix's values, one per block: a warp along a row, eight adjacent values per lane
// where the rows lie on 16 bytes. The operand dz of a gradient is scaled by it (linear_grad below).
constexpr int SIZE_BLOCKS = 296;
__global__ void __launch_bounds__(1024) largest(const uint16_t* x, int64_t pitch, int m, int n, float* sizes) {
    __shared__ uint32_t red[32];
    pdl_wait();
    pdl_release();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const bool wide = ((uintptr_t)x & 15) == 0 && pitch % 8 == 0;
    uint32_t big = 0;
    auto take = [&](uint32_t bits) {
        bits &= 0x7FFF;
        if (bits < 0x7C00) big = max(big, bits);
    };
    for (int64_t r = blockIdx.x * 32ll + warp; r < m; r += gridDim.x * 32ll) {
        const uint16_t* row = x + r * pitch;
        const int whole = wide ? n / 8 * 8 : 0;
#pragma unroll 4
        for (int c = 8 * lane; c < whole; c += 256) {
            const uint4 q = *(const uint4*)(row + c);
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) take(w[i]), take(w[i] >> 16);
        }
        for (int c = whole + lane; c < n; c += 32) take(row[c]);
    }
    big = __reduce_max_sync(~0u, big);
    if (lane == 0) red[warp] = big;
    __syncthreads();
    if (warp) return;
    big = __reduce_max_sync(~0u, red[lane]);
    if (lane == 0) sizes[blockIdx.x] = __half2float(__ushort_as_half((unsigned short)big));
}

// zeros: the gradients of no rows
__global__ void __launch_bounds__(256) zero_rows(void* y, int64_t rows, int64_t cols, int64_t pitch, int type) {
    pdl_wait();
    pdl_release();
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * 256)
        store(y, i / cols * pitch + i % cols, type, 0.0f);
}
int run_zero(void* y, int64_t rows, int64_t cols, int64_t pitch, int type, cudaStream_t s) {
    launch_pdl(zero_rows, dim3(1184), dim3(256), s, y, rows, cols, pitch, type);
    return PCB_LAUNCH_RESULT();
}

// ------------------------------------------------------------------------------------------------ vocabulary
// A maximum and a sum of exponentials below it, joined with another. A side without terms, or whose terms are all
// -inf, adds nothing; NaN goes through the sum.
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float2 join_lse(float2 a, float2 b) {
    const float top = fmaxf(a.x, b.x);
    const float fa = a.x == -INFINITY ? (a.y == a.y ? 0.0f : a.y) : a.y * exp2f((a.x - top) * LOG2E);
    const float fb = b.x == -INFINITY ? (b.y == b.y ? 0.0f : b.y) : b.y * exp2f((b.x - top) * LOG2E);
    return make_float2(top, fa + fb);
}
// lse and loss from the column blocks' maxima and sums: 8 rows per block, 128 lanes over the column blocks (few rows against a
// large vocabulary are all latency: 16 rows against 50000 took 5 us of 28 with 32 lanes)
__global__ void __launch_bounds__(1024) join_parts(const float2* part, int nparts, const float* hit, PcbClearVocab a) {
    __shared__ float2 red[32][8];
    pdl_wait();
    pdl_release();
    const int x = threadIdx.x % 8, y = threadIdx.x / 8, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int64_t row = blockIdx.x * 8ll + x;
    float2 v = make_float2(-INFINITY, 0.0f);
    if (row < a.rows) {
#pragma unroll 4
        for (int i = y; i < nparts; i += 128) v = join_lse(v, part[(int64_t)i * a.rows + row]);
    }
    for (int w = 8; w < 32; w *= 2) v = join_lse(v, make_float2(__shfl_xor_sync(~0u, v.x, w), __shfl_xor_sync(~0u, v.y, w)));
    if (lane < 8) red[warp][lane] = v;
    __syncthreads();
    if (warp) return;
    v = red[lane / 8][x];
    for (int i = 4 + lane / 8; i < 32; i += 4) v = join_lse(v, red[i][x]);
    for (int w = 8; w < 32; w *= 2) v = join_lse(v, make_float2(__shfl_xor_sync(~0u, v.x, w), __shfl_xor_sync(~0u, v.y, w)));
    if (lane >= 8 || row >= a.rows) return;
    const float lse = v.x + logf(v.y);
    const int64_t t = a.targets[row];
    a.lse[row] = lse;
    a.loss[row] = t == a.ignore ? 0.0f : t >= 0 && t < a.vocab ? lse - hit[row] : NAN;
}

// What the gradient's pieces need of each row, and the factor that brings the largest weight to 8192 (the products, in 32
// bits, are scaled back): f16 slopes then keep their relative precision down to 2^-27 of the largest, and the largest ones,
// the targets' (p - 1) weight, which are much alike, lie just below a power of two, where rounding to 16 bits errs least (with
// a power of two as the factor they lay anywhere in the binade: up to twice the error)
__global__ void __launch_bounds__(1024) prepare_rows(PcbClearVocab a, const float* weight, VocabRow* rows, float* unscale) {
    __shared__ float red[32];
    pdl_wait();
    pdl_release();
    float big = 0.0f;
    for (int64_t i = threadIdx.x; i < a.rows; i += 1024)
        if (a.targets[i] != a.ignore) big = fmaxf(big, fabsf(weight[i]));
    for (int w = 16; w; w >>= 1) big = fmaxf(big, __shfl_xor_sync(~0u, big, w));
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = big;
    __syncthreads();
    big = red[threadIdx.x % 32];
    for (int w = 16; w; w >>= 1) big = fmaxf(big, __shfl_xor_sync(~0u, big, w));
    const float scale = big > 0.0f && big <= 3.4e38f ? fminf(8192.0f / big, 1e38f) : 1.0f;
    const int64_t i = blockIdx.x * 1024ll + threadIdx.x;
    if (blockIdx.x == 0 && threadIdx.x == 0) *unscale = 1.0f / scale;
    if (i >= a.rows) return;
    const int64_t t = a.targets[i];
    rows[i] = VocabRow{a.lse[i], t == a.ignore ? 0.0f : weight[i] * scale,
                       t >= 0 && t < a.vocab ? (int32_t)t : -1, t == a.ignore && !isfinite(a.lse[i])};
}
// y = factor * (the sum of `slices` matrices x of pitch `from`, in order), rounded
__global__ void __launch_bounds__(256) finish(const float* x, int slices, int64_t rows, int cols, int64_t from, const float* factor, void* y,
                                              int64_t pitch, int type) {
    pdl_wait();
    pdl_release();
    const float f = *factor;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
        for (int c = threadIdx.x; c < cols; c += 256) {
            float s = x[r * from + c];
            for (int i = 1; i < slices; ++i) s += x[(i * rows + r) * from + c];
            store(y, r * pitch + c, type, s * f);
        }
}

// The pieces of the vocabulary: at most 256 MiB of slopes (16 bits) each, and of the widths that fit, alike but for the last and
// multiples of 256, the one whose three products fill the SMs best (rows x columns, columns x dim, and rows x dim with k in
// `slices` parts). Pieces that stay in L2 are no faster, and each costs some 20 us of products starting and ending: the
// gradients of 4096 x 50000 x 768 take 1040 us at 24 MiB, 818 at 48, 790 at 96, 722 at 256 and 703 in one piece of 410.
struct Pieces {
    int cols, slices;
};
Pieces pieces_of(int rows, int vocab, int dim, bool dh, bool dw) {
    const int64_t fit = (256ll << 20) / 2 / rows;
    const int64_t most = fit < 256 ? 256 : fit / 256 * 256, least = (vocab + most - 1) / most;
    Pieces best{(int)most, 1};
    double ns = 1e300;
    for (int64_t n = least; n <= least + 6; ++n) {
        const int cols = (int)(((vocab + n - 1) / n + 255) / 256 * 256);
        const int full = vocab / cols, rest = vocab % cols, slices = gemm_slices(rows, dim, cols);
        double t = 0.0;
        for (const auto& [count, width] : {std::pair<int, int>{full, cols}, {1, rest}})
            if (count && width)
                t += count * (gemm_cost(rows, width, dim, false) + (dw ? gemm_cost(width, dim, rows, true) : 0.0) +
                              (dh ? gemm_cost(rows, dim, (width + slices - 1) / slices, false) : 0.0) + 18000.0);
        if (t < ns) ns = t, best = Pieces{cols, slices};
    }
    return best;
}

}  // namespace clear
}  // namespace pcb

using namespace pcb;
using namespace pcb::clear;

// ================================================================================================ linear
namespace {
struct LinearWs {
    size_t bytes;
    void *x, *w;
    float* partial;
};
LinearWs linear_ws(const PcbClearLinear* a, void* ws) {
    Carve c(ws);
    LinearWs r;
    r.x = c.take<char>(aligned_bytes(a->x, a->x_pitch, a->m, a->k));
    r.w = c.take<char>(aligned_bytes(a->w, a->w_pitch, a->w_cols ? a->n : a->k, a->w_cols ? a->k : a->n));
    r.partial = c.take<float>(gemm_partial(a->m, a->n, a->k));
    r.bytes = c.used;
    return r;
}

struct GradWs {
    size_t bytes;
    void *dy, *x, *w, *dz;
    int64_t dz_pitch;
    float *sums, *partial, *sizes, *unscale;  // sizes, unscale: null unless dz is scaled
};
GradWs grad_ws(const PcbClearLinearGrad* a, void* ws) {
    Carve c(ws);
    GradWs r;
    const bool products = a->dx || a->dw;
    r.dy = c.take<char>(products && !a->act ? aligned_bytes(a->dy, a->dy_pitch, a->m, a->n) : 0);
    r.x = c.take<char>(a->dw || a->act ? aligned_bytes(a->x, a->x_pitch, a->m, a->k) : 0);
    r.w = c.take<char>(a->dx || a->act ? aligned_bytes(a->w, a->w_pitch, a->w_cols ? a->n : a->k, a->w_cols ? a->k : a->n) : 0);
    r.dz_pitch = ((int64_t)a->n + 7) / 8 * 8;
    r.dz = c.take<uint16_t>(a->act ? (size_t)a->m * r.dz_pitch : 0);
    r.sums = c.take<float>(a->db ? ((size_t)(a->act ? ((int64_t)a->m + 31) / 32 : sum_parts(a->m)) * a->n) : 0);
    const size_t px = a->dx ? gemm_partial(a->m, a->k, a->n) : 0;
    const size_t pw = !a->dw ? 0 : a->w_cols ? gemm_partial(a->n, a->k, a->m) : gemm_partial(a->k, a->n, a->m);
    r.partial = c.take<float>(px > pw ? px : pw);  // the products run one after the other
    const bool scaled = a->act && products && a->type == PCB_F16;
    r.sizes = scaled ? c.take<float>(SIZE_BLOCKS) : nullptr;
    r.unscale = scaled ? c.take<float>(1) : nullptr;
    r.bytes = c.used;
    return r;
}

struct VocabWs {
    size_t bytes;
    void *h, *w, *slopes;
    float2* parts;
    float *hit, *unscale, *dh, *partial;
    VocabRow* rows;
    int piece, slices;
    int64_t slope_pitch, dh_pitch;
};
VocabWs loss_ws(const PcbClearVocab* a, void* ws) {
    Carve c(ws);
    VocabWs r{};
    r.h = c.take<char>(aligned_bytes(a->h, a->h_pitch, a->rows, a->dim));
    r.w = c.take<char>(aligned_bytes(a->w, a->w_pitch, a->vocab, a->dim));
    r.parts = c.take<float2>((size_t)vocab_parts(a->rows, a->vocab) * a->rows);
    r.hit = c.take<float>(a->rows);
    r.bytes = c.used;
    return r;
}
VocabWs vgrad_ws(const PcbClearVocabGrad* a, void* ws) {
    const PcbClearVocab& v = a->v;
    Carve c(ws);
    VocabWs r{};
    r.h = c.take<char>(aligned_bytes(v.h, v.h_pitch, v.rows, v.dim));
    r.w = c.take<char>(aligned_bytes(v.w, v.w_pitch, v.vocab, v.dim));
    const Pieces pc = pieces_of(v.rows, v.vocab, v.dim, a->dh, a->dw);
    r.piece = pc.cols;
    r.slices = pc.slices;
    r.slope_pitch = r.piece;
    r.dh_pitch = (v.dim + 3) / 4 * 4;
    r.slopes = c.take<uint16_t>((size_t)v.rows * r.slope_pitch);
    r.rows = c.take<VocabRow>(v.rows);
    r.unscale = c.take<float>(1);
    r.dh = c.take<float>(a->dh && r.piece < v.vocab ? (size_t)r.slices * v.rows * r.dh_pitch : 0);
    size_t part = 0;
    for (int v0 = 0; v0 < v.vocab; v0 += r.piece) {
        const int cols = v.vocab - v0 < r.piece ? v.vocab - v0 : r.piece;
        const size_t pw = a->dw ? gemm_partial(cols, v.dim, v.rows) : 0;
        const size_t ph = a->dh && r.piece >= v.vocab ? gemm_partial(v.rows, v.dim, cols) : 0;
        part = pw > part ? pw : part;
        part = ph > part ? ph : part;
        if (v0 == 0 && r.piece < v.vocab) v0 = (v.vocab - 1) / r.piece * r.piece - r.piece;  // the first and the last piece differ
    }
    r.partial = c.take<float>(part);
    r.bytes = c.used;
    return r;
}
Gemm product_of(const Operand& a, const Operand& b, int m, int n, int k, int type) {
    Gemm g;
    memset(&g, 0, sizeof g);
    g.a = a, g.b = b, g.m = m, g.n = n, g.k = k, g.type = type, g.y_type = type;
    return g;
}
}  // namespace

extern "C" {

int64_t pcb_clear_linear_ws(const PcbClearLinear* a) {
    if (int rc = bad_linear(a)) return rc;
    return a->m && a->n ? (int64_t)linear_ws(a, nullptr).bytes : 0;
}
int pcb_clear_linear(const PcbClearLinear* a, void* ws, size_t ws_bytes, cudaStream_t s) {
    if (int rc = bad_linear(a)) return rc;
    if (!a->m || !a->n) return 0;
    const LinearWs w = linear_ws(a, ws);
    if (int rc = bad_ws("clear_linear", ws, ws_bytes, w.bytes)) return rc;
    Operand x{a->x, a->x_pitch, true}, wt{a->w, a->w_pitch, a->w_cols != 0};
    const Rows rows[] = {{&x.p, &x.pitch, a->m, a->k, w.x}, {&wt.p, &wt.pitch, a->w_cols ? a->n : a->k, a->w_cols ? a->k : a->n, w.w}};
    if (int rc = align_rows(rows, 2, s)) return rc;
    Gemm g = product_of(x, wt, a->m, a->n, a->k, a->type);
    g.y = a->y, g.y_pitch = a->y_pitch, g.y_type = a->y_type;
    g.act = make_act(a->act, a->bound, a->coef);
    g.bias = a->bias, g.bias_type = a->bias_type;
    g.extra = a->residual, g.extra_pitch = a->residual_pitch, g.extra_type = a->residual_type;
    g.partial = w.partial;
    return gemm(g, s);
}

int64_t pcb_clear_linear_grad_ws(const PcbClearLinearGrad* a) {
    if (int rc = bad_grad(a)) return rc;
    return a->m ? (int64_t)grad_ws(a, nullptr).bytes : 0;
}
int pcb_clear_linear_grad(const PcbClearLinearGrad* a, void* ws, size_t ws_bytes, cudaStream_t s) {
    if (int rc = bad_grad(a)) return rc;
    if (!a->m) {
        if (a->dw)
            if (int rc = run_zero(a->dw, a->w_cols ? a->n : a->k, a->w_cols ? a->k : a->n, a->dw_pitch, a->type, s)) return rc;
        return a->db ? run_zero(a->db, 1, a->n, a->n, a->db_type, s) : 0;
    }
    const GradWs w = grad_ws(a, ws);
    if (int rc = bad_ws("clear_linear_grad", ws, ws_bytes, w.bytes)) return rc;
    Operand x{a->x, a->x_pitch, true}, wt{a->w, a->w_pitch, a->w_cols != 0}, dz{a->dy, a->dy_pitch, true};
    Rows rows[3];
    int nrows = 0;
    if (a->dw || a->act) rows[nrows++] = Rows{&x.p, &x.pitch, a->m, a->k, w.x};
    if (a->dx || a->act) rows[nrows++] = Rows{&wt.p, &wt.pitch, a->w_cols ? a->n : a->k, a->w_cols ? a->k : a->n, w.w};
    if (!a->act && (a->dx || a->dw)) rows[nrows++] = Rows{&dz.p, &dz.pitch, a->m, a->n, w.dy};
    if (int rc = align_rows(rows, nrows, s)) return rc;
    if (a->act) {
        // dz in 16 bits (its one rounding: the products with x and W take 16-bit operands), and the sums of its rows from the
        // same 32-bit values. dy of a mean over thousands of rows lies where float16 has few bits left or none, so dz is
        // scaled by a power of two that brings the largest dy, times the largest slope, to 2^8: 2^-22 of it still has all
        // bits, and slopes past the polynomial's bound have a factor of 256 left. The products are scaled back in 32 bits.
        Gemm g = product_of(x, wt, a->m, a->n, a->k, a->type);
        g.epi = EPI_DZ;
        g.y = w.dz, g.y_pitch = w.dz_pitch, g.padded = true;
        g.act = make_act(a->act, a->bound, a->coef);
        g.bias = a->bias, g.bias_type = a->bias_type;
        g.extra = a->dy, g.extra_pitch = a->dy_pitch, g.extra_type = a->type;
        g.row_sums = a->db ? w.sums : nullptr;
        if (w.sizes) {
            const int blocks = std::min(a->m / 32 + 1, SIZE_BLOCKS);
            launch_pdl(largest, dim3(blocks), dim3(1024), s, (const uint16_t*)a->dy, a->dy_pitch, a->m, a->n, w.sizes);
            if (int rc = PCB_LAUNCH_RESULT()) return rc;
            g.sizes = w.sizes, g.nsizes = blocks, g.unscale = w.unscale;
            g.slope = a->act == PCB_ACT_GELU ? 1.13f : 0.0f;
            for (int i = 0; i < 7; ++i) g.slope += std::fabs(g.act.d[i]);
        }
        if (int rc = gemm(g, s)) return rc;
        dz = Operand{w.dz, w.dz_pitch, true};
        if (a->db)
            if (int rc = run_sum(w.sums, a->n, PCB_F32, (a->m + 31) / 32, a->n, nullptr, a->db, a->db_type, false, s)) return rc;
    }
    if (a->dx) {
        Gemm g = product_of(dz, Operand{wt.p, wt.pitch, a->w_cols == 0}, a->m, a->k, a->n, a->type);
        g.y = a->dx, g.y_pitch = a->dx_pitch, g.partial = w.partial, g.alpha = w.unscale;
        if (int rc = gemm(g, s)) return rc;
    }
    if (a->db && !a->act) {  // beside the product before it, if there is one
        const bool once = a->m <= SUM_ONCE;
        if (int rc = run_sum(a->dy, a->dy_pitch, a->type, a->m, a->n, once ? nullptr : w.sums, a->db, a->db_type, a->dx != nullptr, s)) return rc;
        if (!once)
            if (int rc = run_sum(w.sums, a->n, PCB_F32, sum_parts(a->m), a->n, nullptr, a->db, a->db_type, false, s)) return rc;
    }
    if (!a->dw) return 0;
    const Operand xr{x.p, x.pitch, false}, dr{dz.p, dz.pitch, false};
    Gemm g = a->w_cols ? product_of(dr, xr, a->n, a->k, a->m, a->type) : product_of(xr, dr, a->k, a->n, a->m, a->type);
    g.y = a->dw, g.y_pitch = a->dw_pitch, g.partial = w.partial, g.alpha = w.unscale;
    return gemm(g, s);
}

// ================================================================================================ vocabulary loss
int64_t pcb_clear_vocab_loss_ws(const PcbClearVocab* a) {
    if (int rc = bad_vocab(a, false)) return rc;
    return a->rows ? (int64_t)loss_ws(a, nullptr).bytes : 0;
}
int pcb_clear_vocab_loss(const PcbClearVocab* a, void* ws, size_t ws_bytes, cudaStream_t s) {
    if (int rc = bad_vocab(a, false)) return rc;
    if (!a->rows) return 0;
    const VocabWs w = loss_ws(a, ws);
    if (int rc = bad_ws("clear_vocab_loss", ws, ws_bytes, w.bytes)) return rc;
    Operand h{a->h, a->h_pitch, true}, wt{a->w, a->w_pitch, true};
    const Rows rows[] = {{&h.p, &h.pitch, a->rows, a->dim, w.h}, {&wt.p, &wt.pitch, a->vocab, a->dim, w.w}};
    if (int rc = align_rows(rows, 2, s)) return rc;
    Gemm g = product_of(h, wt, a->rows, a->vocab, a->dim, a->type);
    g.epi = EPI_LSE;
    g.targets = a->targets, g.parts = w.parts, g.hit = w.hit;
    if (int rc = gemm(g, s)) return rc;
    launch_pdl(join_parts, dim3((a->rows + 7) / 8), dim3(1024), s, (const float2*)w.parts, vocab_parts(a->rows, a->vocab),
               (const float*)w.hit, *a);
    return PCB_LAUNCH_RESULT();
}

int64_t pcb_clear_vocab_grad_ws(const PcbClearVocabGrad* a) {
    if (int rc = bad_vocab_grad(a)) return rc;
    return a->v.rows ? (int64_t)vgrad_ws(a, nullptr).bytes : 0;
}
int pcb_clear_vocab_grad(const PcbClearVocabGrad* a, void* ws, size_t ws_bytes, cudaStream_t s) {
    if (int rc = bad_vocab_grad(a)) return rc;
    const PcbClearVocab& v = a->v;
    if (!v.rows) return a->dw ? run_zero(a->dw, v.vocab, v.dim, a->dw_pitch, v.type, s) : 0;
    const VocabWs w = vgrad_ws(a, ws);
    if (int rc = bad_ws("clear_vocab_grad", ws, ws_bytes, w.bytes)) return rc;
    Operand h{v.h, v.h_pitch, true}, wt{v.w, v.w_pitch, true};
    const Rows rows[] = {{&h.p, &h.pitch, v.rows, v.dim, w.h}, {&wt.p, &wt.pitch, v.vocab, v.dim, w.w}};
    if (int rc = align_rows(rows, 2, s)) return rc;
    launch_pdl(prepare_rows, dim3((v.rows + 1023) / 1024), dim3(1024), s, v, a->weight, w.rows, w.unscale);
    if (int rc = PCB_LAUNCH_RESULT()) return rc;
    const bool whole = w.piece >= v.vocab;
    for (int v0 = 0; v0 < v.vocab; v0 += w.piece) {
        const int cols = v.vocab - v0 < w.piece ? v.vocab - v0 : w.piece;
        const void* wp = (const char*)wt.p + 2 * (int64_t)v0 * wt.pitch;
        Gemm g = product_of(h, Operand{wp, wt.pitch, true}, v.rows, cols, v.dim, v.type);
        g.epi = EPI_DL;
        g.y = w.slopes, g.y_pitch = w.slope_pitch, g.padded = true, g.rows = w.rows, g.col0 = v0;
        if (int rc = gemm(g, s)) return rc;
        if (a->dh) {
            g = product_of(Operand{w.slopes, w.slope_pitch, true}, Operand{wp, wt.pitch, false}, v.rows, v.dim, cols, v.type);
            if (whole) g.y = a->dh, g.y_pitch = a->dh_pitch, g.alpha = w.unscale, g.partial = w.partial;
            else g.y = w.dh, g.y_pitch = w.dh_pitch, g.y_type = PCB_F32, g.padded = true, g.slices = w.slices, g.accumulate = v0 > 0;
            if (int rc = gemm(g, s)) return rc;
        }
        if (a->dw) {
            g = product_of(Operand{w.slopes, w.slope_pitch, false}, Operand{h.p, h.pitch, false}, cols, v.dim, v.rows, v.type);
            g.y = (char*)a->dw + 2 * (int64_t)v0 * a->dw_pitch, g.y_pitch = a->dw_pitch, g.alpha = w.unscale, g.partial = w.partial;
            if (int rc = gemm(g, s)) return rc;
        }
    }
    if (!a->dh || whole) return 0;
    launch_pdl(finish, dim3((unsigned)std::min(v.rows, 4096)), dim3(256), s, (const float*)w.dh, w.slices, (int64_t)v.rows, v.dim, w.dh_pitch,
               (const float*)w.unscale, a->dh, a->dh_pitch, v.type);
    return PCB_LAUNCH_RESULT();
}

}  // extern "C"
