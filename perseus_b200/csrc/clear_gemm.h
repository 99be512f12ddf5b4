// The product behind the clear half's operators: D[m][n] = sum_k A(m, k) B(n, k) with an epilogue (clear_gemm.cu).
#pragma once
#include "clear.h"

namespace pcb {
namespace clear {

// A 16-bit operand: `rows` rows along m (or n) and `k` values. k_adjacent: row r's k-values are adjacent at p + r pitch;
// otherwise the rows are, at p + k pitch.
struct Operand {
    const void* p;
    int64_t pitch;
    bool k_adjacent;
};

enum Epilogue {
    EPI_STORE,  // y = alpha * (act(D + bias) + extra)
    EPI_DZ,     // y = extra * act'(D + bias), times a power of two if `sizes` is given, and the sums of each 32 rows of its
                // columns in 32 bits (without that factor)
    EPI_LSE,    // the maximum and the sum of exponentials of each row of a column block, the target's logit
    EPI_DL,     // y = weight (exp(D - lse) - [n = target])
};

// What EPI_DL needs of a row
struct VocabRow {
    float lse, weight;
    int32_t target;  // -1: none
    int32_t off;     // an ignored row whose lse is not finite: its slopes are 0, not 0 x NaN
};

struct Gemm {
    Operand a, b;
    int m, n, k;
    int type;  // of the operands
    Epilogue epi;
    void* y;
    int64_t y_pitch;
    int y_type;
    bool padded;      // y is scratch: its rows may be written past n up to the pitch
    int slices;       // EPI_STORE into 32 bits: > 0: k in this many parts, part i's sums at y + i m y_pitch
    bool accumulate;  // with slices: y += (one writer per element; a part without k is left as it is)
    Act act;
    const void* bias;
    int bias_type;
    const void* extra;
    int64_t extra_pitch;
    int extra_type;
    const float* alpha;     // one value on the device, or null
    float* row_sums;        // EPI_DZ: [ceil(m / 32)][n], or null
    const float* sizes;     // EPI_DZ: `nsizes` values of which the largest, times `slope`, the factor brings to [2^7, 2^8), or null
    int nsizes;
    float slope;
    float* unscale;         // EPI_DZ with `sizes`: one over the factor
    const VocabRow* rows;   // EPI_DL
    int col0;               // EPI_DL: the vocabulary entry of this product's first column
    const int64_t* targets; // EPI_LSE
    float2* parts;          // EPI_LSE: [vocab_parts(n)][m] (maximum, sum of exponentials below it)
    float* hit;             // EPI_LSE: [m], written where the target lies in this product's columns
    float* partial;         // EPI_STORE: workspace of gemm_partial() values; null: no splitting
};

// 32-bit values of workspace that an EPI_STORE product wants (the tiles of its last, partly filled round over the SMs split
// their k), and the estimated time of a product in nanoseconds
size_t gemm_partial(int m, int n, int k);
double gemm_cost(int m, int n, int k, bool may_split);
// parts of k that fill the SMs for an m x n product (for `slices`)
int gemm_slices(int m, int n, int k);
int gemm(const Gemm& g, cudaStream_t s);
// column blocks of an EPI_LSE product over n columns
int vocab_parts(int m, int n);

// An operand as the TMA engine can read it: first element and pitch on 16 bytes, as it lies or copied to `to` (null when
// only counting). aligned_bytes: the copy's size, 0 where none is needed.
struct Rows {
    const void** p;
    int64_t* pitch;
    int64_t rows, cols;
    void* to;
};
size_t aligned_bytes(const void* p, int64_t pitch, int64_t rows, int64_t cols);
int align_rows(const Rows* r, int n, cudaStream_t s);  // n <= 3, one launch

unsigned int gemm_timeouts();

}  // namespace clear
}  // namespace pcb
