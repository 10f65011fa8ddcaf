// Internal launch interface of the classification-head operators (head_api.cpp and the head_*.hip kernels).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <cmath>

namespace pngpd {

constexpr int64_t HEAD_MAX_LD = (int64_t)1 << 23;            // bytes between rows: 256 rows stay below 2^31
constexpr int64_t HEAD_MAX_EXTENT = HEAD_MAX_LD / 4;         // elements of a dense row

// One operand of a product out[m][n] = sum_k A(m,k) B(n,k).
// k_contiguous: element (r, k) sits at p[r * ld + k]; otherwise at p[k * ld + r] (the operand lies transposed).
// Both take rows as head_direct() describes them; head_set_up() makes such rows of others.
struct HeadOperand {
    const void* p;
    int64_t ld;
    bool k_contiguous;
};
// 16-byte aligned rows whose dense extent is whole 16-byte chunks (or has zeros behind it up to one), and distances that
// keep a tile's offsets below 2^31
inline bool head_direct(const void* p, int64_t ld, int64_t extent, size_t size) {
    const int64_t c = 16 / (int64_t)size;
    return ((uintptr_t)p & 15) == 0 && ld % c == 0 && extent % c == 0 && ld <= HEAD_MAX_LD / (int64_t)size;
}

// Partial sums lie in rows of whole 16-byte chunks.
__host__ __device__ inline int64_t head_partial_ld(int64_t N) { return (N + 3) & ~(int64_t)3; }

// A LINEAR product of so few rows takes them, and the weight's, as they lie.
constexpr int64_t HEAD_FEW_ROWS = 4;

// What becomes of a product's 32-bit sums.
enum { HEAD_EPI_LINEAR = 0, HEAD_EPI_DZ = 1, HEAD_EPI_SCALED = 2, HEAD_EPI_STATS = 3 };
struct HeadEpilogue {
    int kind = HEAD_EPI_SCALED;
    // LINEAR: out = act(acc + bias[n]) + residual[m][n]; z (may be NULL, dense [M][N]) receives acc + bias
    const void* bias = nullptr;
    const void* residual = nullptr;
    int64_t ld_residual = 0;
    int act = 0;
    void* z = nullptr;
    // DZ: out = (exp(acc + bias[n] - lse[m]) - smooth - (target[m] == n + first_n ? 1 - eps : 0)) * row_weight[m]; rows of
    // ld_out, zeros behind column N
    const float* lse = nullptr;
    const float* row_weight = nullptr;
    const int64_t* target = nullptr;
    int64_t first_n = 0;
    float smooth = 0.f, one_minus_eps = 1.f;
    float* col_part = nullptr;  // may be NULL; [head_dz_parts][N]: sums of blocks of rows, of the values before they are rounded
    // SCALED: out = scale[0] * (acc + add[m][n]); scale NULL: 1; add NULL: 0 (32-bit, dense [M][N])
    const float* scale = nullptr;
    const float* add = nullptr;
    // STATS: stats[i][m] = maximum, sum of exp(z - maximum) and sum of row m's logits z = acc + bias in the i-th block of
    // columns; target_logit[m] = z[m][target[m]] where that is a column
    float4* stats = nullptr;
    float* target_logit = nullptr;
    bool want_logit_sum = false;
    // the output (all but STATS): of the operands' type, or 32-bit floats when out_f32
    void* out = nullptr;
    int64_t ld_out = 0;
    bool out_f32 = false;
};

// How a product is cut: tile shape, cuts of the contraction (joined by a second kernel from 32-bit partial sums).
struct HeadPlan {
    int shape, splits, tiles_m, tiles_n;
    int64_t k_split;
    size_t partial_bytes;
    int stats_blocks;           // blocks of columns a STATS epilogue writes
    double us;                  // what it should take
};
HeadPlan head_plan(int type, int64_t M, int64_t N, int64_t K, int kind);

// partial: head_plan(...).partial_bytes.  keep: the sums are left in partial (head_kept_bytes)
hipError_t head_product(int type, int64_t M, int64_t N, int64_t K, const HeadOperand& a, const HeadOperand& b,
                        const HeadEpilogue& e, float* partial, bool keep, hipStream_t s);
// Both gradients of a product, dx = dz W and dW = dz^T x (SCALED epilogues), in one launch where they are small.
struct HeadGradient {
    int64_t M, N, K;
    HeadOperand a, b;
    HeadEpilogue e;
    float* partial;             // of its own
};
hipError_t head_gradients(int type, const HeadGradient& x, const HeadGradient& w, hipStream_t s);
// Kept sums of a STATS product, and the DZ epilogue from them.
size_t head_kept_bytes(int type, int64_t M, int64_t N, int64_t K);
hipError_t head_kept(int type, int64_t M, int64_t N, int64_t K, const HeadEpilogue& e, const float* kept, hipStream_t s);
// Blocks of rows whose column sums a DZ product of this plan (kept: head_kept) leaves in col_part, and their sum times scale[0].
int64_t head_dz_parts(int type, int64_t M, int64_t N, const HeadPlan& plan, bool kept);
hipError_t head_col_sums(int type, int64_t parts, int64_t N, const float* part, const float* scale, void* out, hipStream_t s);

// dst[r][0 .. ld) = src[r][0 .. cols) and zeros behind them.  dst is 16-byte aligned, ld whole chunks.  With a target, rows
// whose target is ignored or no class become zeros whatever they hold.
struct HeadLayOut {
    const void* src;
    int64_t rows, cols, ld_src;
    void* dst;
    int64_t ld;
    bool live_rows_only;
};
// row_weight[t] = weight of row t in the loss's gradient divided by out_scale[0]: the one weight of all rows, the largest of
// them (16-bit types), or 1
struct HeadRowWeights {
    const int64_t* target;
    int64_t T, V, ignore_index;
    int reduction;
    const float* dloss;
    float *row_weight, *out_scale;
    float label_factor;         // 16-bit types: of all weights (head_label_factor)
    float* parts;               // head_row_parts(T) times three floats
};
// Many rows: their count, and the largest of their weights, come from this many workgroups in a launch in front (0: from one,
// beside those that lay operands out).
int64_t head_row_parts(int64_t T);
// c in (1/2, 1] with c (1 - eps) a power of two (1 where eps is)
inline float head_label_factor(float eps) {
    int e;
    const float m = std::frexp(1.f - eps, &e);
    return m > 0.5f ? 0.5f / m : 1.f;
}
// Up to two matrices laid out and the rows' weights, in one launch; each may be NULL, all NULL launches nothing.
hipError_t head_set_up(int type, const HeadLayOut* a, const HeadLayOut* b, const HeadRowWeights* w, hipStream_t s);
// dz[m][n] = dy[m][n] * act'(z[m][n]) (z dense; act NONE: dy itself) into dz (may be NULL; rows of ld_dz, whole chunks, zeros
// behind column N), and into sums (may be NULL) the columns' sums, by way of part: 32-bit [head_col_parts][N]
size_t head_col_parts(int type, int64_t M, int64_t N);
hipError_t head_grad_rows(int type, int64_t M, int64_t N, const void* dy, int64_t ld_dy, const void* z, int act, void* dz,
                          int64_t ld_dz, float* part, void* sums, hipStream_t s);

// a fill kernel, not a memset: the call may be captured
hipError_t head_zero(void* p, size_t bytes, hipStream_t s);

hipError_t head_dropout(int type, int64_t rows, int64_t cols, const void* x, int64_t ldx, const void* residual,
                        int64_t ldr, void* y, double p, uint64_t seed, uint64_t offset, const int64_t* rng_dev,
                        hipStream_t s);

// lse[t] and the loss of every row from its statistics; the batch's loss from its rows'
// (batch: not NULL, and one launch does both where that is as quick; head_loss_at_once() says whether it did)
bool head_loss_at_once(int64_t T, int blocks);
hipError_t head_row_loss(int64_t T, int64_t V, int blocks, const float4* stats, const float* target_logit, const int64_t* target,
                         int64_t ignore_index, float eps, float* row_loss, float* lse, int reduction, float* batch, hipStream_t s);
// used (may be NULL) receives the number of rows that are not ignored; parts: head_batch_parts(T) pairs of doubles
int64_t head_batch_parts(int64_t T);
hipError_t head_batch_loss(int64_t T, const float* row_loss, const int64_t* target, int64_t ignore_index, int reduction, float* loss,
                           float* used, double2* parts, hipStream_t s);

// The loss over at most HEAD_FEW classes, operands with any strides.  logits: what is kept for the backward pass, head_few_room
// floats a row (NULL: forward only).
constexpr int64_t HEAD_FEW = 8;
inline int64_t head_few_room(int64_t V) { return V <= 4 ? 4 : 8; }
struct HeadFew {
    int64_t T, V, D;
    const void* x;
    int64_t ldx;
    const void* w;
    int64_t ldw;
    const void* bias;           // may be NULL
    const int64_t* target;
    int64_t ignore_index;
    float eps;
    float* logits;
};
hipError_t head_few_loss(int type, const HeadFew& g, float* row_loss, float* lse, hipStream_t s);
// part: head_few_part_bytes; used: what head_batch_loss left (for the mean)
size_t head_few_part_bytes(int type, int64_t T, int64_t V, int64_t D);
hipError_t head_few_grad(int type, const HeadFew& g, const float* lse, const float* used, const float* dloss, int reduction, void* dx,
                         void* dw, void* db, float* part, hipStream_t s);
}  // namespace pngpd
