// Internal launch interface of the classification-head operators (head_api.cpp and the head_*.hip kernels).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace pngpd {

// One operand of a product out[m][n] = sum_k A(m,k) B(n,k).  Rows (m or n) are `rows`, the contraction index is k.
// k_contiguous: element (r, k) sits at p[r * ld + k]; otherwise at p[k * ld + r] (the operand lies transposed).
struct HeadOperand {
    const void* p;
    int64_t ld;
    bool k_contiguous;
};

// What becomes of a product's 32-bit sums.
enum { HEAD_EPI_LINEAR = 0, HEAD_EPI_DZ = 1, HEAD_EPI_SCALED = 2 };
struct HeadEpilogue {
    int kind = HEAD_EPI_SCALED;
    // LINEAR: out = act(acc + bias[n]) + residual[m][n]; z (may be NULL) receives acc + bias, rows ld_out_z = N
    const void* bias = nullptr;
    const void* residual = nullptr;
    int64_t ld_residual = 0;
    int act = 0;
    void* z = nullptr;
    // DZ: out = (exp(acc + bias[n] - lse[m]) - smooth - (target[m] == n + first_n ? 1 - eps : 0)) * row_weight[m]
    const float* lse = nullptr;
    const float* row_weight = nullptr;
    const int64_t* target = nullptr;
    int64_t first_n = 0;
    float smooth = 0.f, one_minus_eps = 1.f;
    // SCALED: out = scale[0] * (acc + add[m][n]); scale NULL: 1; add NULL: 0 (32-bit, rows of N)
    const float* scale = nullptr;
    const float* add = nullptr;
    // the output: `type` as the operands, or 32-bit floats when out_f32
    void* out = nullptr;
    int64_t ld_out = 0;
    bool out_f32 = false;
};

hipError_t head_product(int type, int64_t M, int64_t N, int64_t K, const HeadOperand& a, const HeadOperand& b,
                        const HeadEpilogue& e, hipStream_t s);

// dz[m][n] = dy[m][n] * act'(z[m][n]) (rows of N)
hipError_t head_act_backward(int type, int64_t M, int64_t N, const void* dy, int64_t ld_dy, const void* z, int act,
                             void* dz, hipStream_t s);
// out[n] = scale * sum_m a[m][n]; part: 32-bit [head_col_sum_parts(M)][N]
int64_t head_col_sum_parts(int64_t M);
hipError_t head_col_sum(int type, int64_t M, int64_t N, const void* a, int64_t ld, float* part, const float* scale,
                        void* out, hipStream_t s);

// a fill kernel, not a memset: the call may be captured
hipError_t head_zero(void* p, size_t bytes, hipStream_t s);

hipError_t head_dropout(int type, int64_t rows, int64_t cols, const void* x, int64_t ldx, const void* residual,
                        int64_t ldr, void* y, double p, uint64_t seed, uint64_t offset, const int64_t* rng_dev,
                        hipStream_t s);

// Running statistics of a row of logits over the pieces of the vocabulary.
struct HeadRowStats {
    float *max, *sum, *target_logit, *logit_sum;      // [T] each
};
hipError_t head_stats_piece(int64_t T, int64_t n, const float* logits, int64_t ld, int64_t first_n,
                            const int64_t* target, const HeadRowStats& st, bool first, hipStream_t s);
hipError_t head_loss_finish(int64_t T, int64_t V, const int64_t* target, int64_t ignore_index, float eps, int reduction,
                            const HeadRowStats& st, float* loss, float* lse, hipStream_t s);
// row_weight[t] = weight of row t in the gradient divided by 2^e, out_scale[0] = 2^e (type f16 only, else 2^e = 1)
hipError_t head_row_weights(int type, int64_t T, int64_t V, const int64_t* target, int64_t ignore_index, int reduction,
                            const float* dloss, float* row_weight, float* out_scale, hipStream_t s);

// out[t] = x[t] where row_weight[t] != 0, zeros elsewhere (rows of D): what a padding row holds stays out of sums
hipError_t head_live_rows(int type, int64_t T, int64_t D, const void* x, int64_t ldx, const float* row_weight, void* out,
                          hipStream_t s);

}  // namespace pngpd
