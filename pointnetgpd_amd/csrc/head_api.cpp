// C-ABI of the classification-head operators: checks of arguments, workspace layout, sequencing of the kernels.
#include <hip/hip_runtime.h>

#include "api_common.h"
#include "head.h"
#include "pngpd.h"

namespace {

using pngpd::fail;
using pngpd::HeadEpilogue;
using pngpd::HeadOperand;

constexpr int64_t MAX_SIZE = 2147483647;
constexpr int64_t MAX_CLASSES = (int64_t)1 << 24;
constexpr size_t PIECE_BYTES = (size_t)256 << 20;      // of the logits' gradients at a time, or as much as x and weight take
constexpr size_t STATS_BYTES = (size_t)256 << 20;      // of rows' statistics at a time

inline size_t esize(int type) { return type == PNGPD_TYPE_F32 ? 4 : 2; }
inline bool type_ok(int type) { return type >= PNGPD_TYPE_F32 && type <= PNGPD_TYPE_F16; }

struct Bump {
    char* base;
    size_t off = 0;
    explicit Bump(void* b) : base((char*)b) {}
    void* take(size_t bytes) {
        char* p = base ? base + off : nullptr;
        off += (bytes + 255) & ~(size_t)255;
        return p;
    }
};

int check_sizes(const char* who, int type, int64_t rows, int64_t a, int64_t b) {
    if (!type_ok(type)) return fail(PNGPD_ERR_INVALID, "%s: unknown type %d", who, type);
    if (rows < 0 || rows > MAX_SIZE || a < 1 || a > MAX_SIZE || b < 1 || b > MAX_SIZE)
        return fail(PNGPD_ERR_SHAPE, "%s: sizes %lld, %lld, %lld", who, (long long)rows, (long long)a, (long long)b);
    return PNGPD_OK;
}

int check_linear(const char* who, int type, int64_t M, int64_t N, int64_t K, int act) {
    int rc = check_sizes(who, type, M, N, K);
    if (rc) return rc;
    if (N > pngpd::HEAD_MAX_EXTENT || K > pngpd::HEAD_MAX_EXTENT)
        return fail(PNGPD_ERR_SHAPE, "%s: N = %lld, K = %lld, at most %lld", who, (long long)N, (long long)K, (long long)pngpd::HEAD_MAX_EXTENT);
    if (act < PNGPD_ACT_NONE || act > PNGPD_ACT_SILU) return fail(PNGPD_ERR_INVALID, "%s: unknown activation %d", who, act);
    return PNGPD_OK;
}

// A launch holds fewer than 2^23 tiles of a product's output, 256 x 256 (16 bits) or 128 x 128 (float32) at most.
int check_tiles(const char* who, int type, int64_t M, int64_t N) {
    const int64_t side = type == PNGPD_TYPE_F32 ? 128 : 256;
    if ((double)((M + side - 1) / side) * (double)((N + side - 1) / side) < 8388608.0) return PNGPD_OK;
    return fail(PNGPD_ERR_SHAPE, "%s: a product of %lld x %lld has more than 2^23 tiles", who, (long long)M, (long long)N);
}

int check_ld(const char* who, const char* name, int64_t ld, int64_t least) {
    if (ld < least || ld > ((int64_t)1 << 40)) return fail(PNGPD_ERR_SHAPE, "%s: %s = %lld for rows of %lld", who, name, (long long)ld, (long long)least);
    return PNGPD_OK;
}

int check_ws(const char* who, const void* ws, size_t have, size_t need) {
    if (need == 0) return PNGPD_OK;
    if (!ws) return fail(PNGPD_ERR_INVALID, "%s: NULL workspace", who);
    if (((uintptr_t)ws & 15) != 0) return fail(PNGPD_ERR_INVALID, "%s: the workspace must be aligned to 16 bytes", who);
    if (have < need) return fail(PNGPD_ERR_WORKSPACE, "%s: workspace of %zu bytes, needs %zu", who, have, need);
    return PNGPD_OK;
}

// rows of `extent` elements as the products take them: whole 16-byte chunks
inline int64_t padded(int64_t extent, int type) {
    const int64_t c = 16 / (int64_t)esize(type);
    return (extent + c - 1) / c * c;
}

// An operand as the products take it: itself, or a copy in `room` (rows of padded(extent)).
struct Rows {
    const void* p;
    int64_t ld;
};
inline bool direct(const void* p, int64_t ld, int64_t extent, int type) { return pngpd::head_direct(p, ld, extent, esize(type)); }
// Itself, or where head_set_up() has to lay it out first (`job` then is what it takes).
Rows direct_rows(int type, int64_t rows, int64_t extent, const void* p, int64_t ld, void* room, pngpd::HeadLayOut* job, bool* needed) {
    *needed = !direct(p, ld, extent, type);
    if (!*needed) return Rows{p, ld};
    *job = pngpd::HeadLayOut{p, rows, extent, ld, room, padded(extent, type), false};
    return Rows{room, job->ld};
}

inline size_t max2(size_t a, size_t b) { return a > b ? a : b; }

struct LinearWs {
    void *x, *w, *dz;           // laid out, if they have to be
    float *part, *partial;
    float* partial_w;           // the weight's gradient's own
    size_t bytes;
    // copy_*: x, weight or dz (dy where there is no activation) is not as the products take it
    LinearWs(void* base, int type, int64_t M, int64_t N, int64_t K, bool backward, bool copy_x, bool copy_w, bool copy_dz) {
        Bump b(base);
        dz = nullptr;
        part = partial = partial_w = nullptr;
        x = w = nullptr;
        if (M > 0) {
            if (copy_x) x = b.take((size_t)M * padded(K, type) * esize(type));
            if (copy_w) w = b.take((size_t)N * padded(K, type) * esize(type));
            size_t cut = pngpd::head_plan(type, M, N, K, pngpd::HEAD_EPI_LINEAR).partial_bytes;
            if (backward) {
                if (copy_dz) dz = b.take((size_t)M * padded(N, type) * esize(type));
                part = (float*)b.take((size_t)pngpd::head_col_parts(type, M, N) * N * 4);
                cut = pngpd::head_plan(type, M, K, N, pngpd::HEAD_EPI_SCALED).partial_bytes;
                partial_w = (float*)b.take(pngpd::head_plan(type, N, K, M, pngpd::HEAD_EPI_SCALED).partial_bytes);
            }
            partial = (float*)b.take(cut);
        }
        bytes = b.off;
    }
};

inline size_t loss_budget(int type, int64_t T, int64_t V, int64_t D) { return max2(PIECE_BYTES, ((size_t)T + (size_t)V) * (size_t)D * esize(type)); }

struct LossWs {
    int64_t rows_at_once;      // rows whose statistics are formed at a time (forward)
    int64_t piece;             // columns of the vocabulary whose gradients are formed at a time
    void *x, *w, *tile;        // laid out; gradients of a piece's logits, [T][padded(piece)]
    float4* stats;
    float *target_logit, *row_loss, *row_weight, *scale, *part, *dx_sum, *partial;
    double2* loss_parts;
    float* row_parts;
    float* partial_w;          // the weight's gradient's own
    pngpd::HeadPlan dz, dz_last;      // of a piece's logits, and of the last piece's where that is smaller
    size_t bytes;
    LossWs(void* base, int type, int64_t T, int64_t V, int64_t D, bool backward, bool copy_x, bool copy_w) {
        Bump b(base);
        const int64_t rows = T > 0 ? T : 1, dp = padded(D, type);
        const size_t e = esize(type);
        x = copy_x || backward ? b.take((size_t)rows * dp * e) : nullptr;      // the gradients take a copy without padding rows
        w = copy_w ? b.take((size_t)V * dp * e) : nullptr;
        tile = nullptr;
        stats = nullptr;
        target_logit = row_loss = row_weight = scale = part = dx_sum = partial = partial_w = row_parts = nullptr;
        loss_parts = nullptr;
        piece = V;
        rows_at_once = rows;
        if (!backward) {
            // 64 columns a block at least; a product of 2^34 elements stays inside a grid
            int64_t at_once = (int64_t)(STATS_BYTES / sizeof(float4)) / ((V + 63) / 64) / 256 * 256;
            const int64_t most = ((int64_t)1 << 34) / V / 256 * 256;
            if (at_once > most) at_once = most;
            if (at_once < 256) at_once = 256;
            rows_at_once = rows < at_once ? rows : at_once;
            const int64_t last = rows % rows_at_once ? rows % rows_at_once : rows_at_once;
            size_t cut = 0, blocks = 0;
            for (int64_t n : {rows_at_once, last}) {
                const pngpd::HeadPlan p = pngpd::head_plan(type, n, V, D, pngpd::HEAD_EPI_STATS);
                blocks = max2(blocks, (size_t)p.stats_blocks * n);
                cut = max2(cut, p.partial_bytes);
            }
            stats = (float4*)b.take(blocks * sizeof(float4));
            target_logit = (float*)b.take((size_t)rows * 4);
            row_loss = (float*)b.take((size_t)rows * 4);
            loss_parts = (double2*)b.take((size_t)pngpd::head_batch_parts(rows) * sizeof(double2));
            partial = (float*)b.take(cut);
        } else {
            piece = (int64_t)(loss_budget(type, rows, V, D) / ((size_t)rows * e)) / 256 * 256;
            if (piece < 256) piece = 256;
            if (piece > pngpd::HEAD_MAX_EXTENT) piece = pngpd::HEAD_MAX_EXTENT;
            if (piece > V) piece = V;
            const int64_t last = V % piece ? V % piece : piece;
            tile = b.take((size_t)rows * padded(piece, type) * e);
            row_weight = (float*)b.take((size_t)rows * 4);
            scale = (float*)b.take(4);
            row_parts = (float*)b.take((size_t)pngpd::head_row_parts(rows) * 12);
            if (piece < V) dx_sum = (float*)b.take((size_t)rows * D * 4);
            size_t cut = 0, cut_w = 0, sums = 0;
            for (int64_t n : {piece, last}) {
                pngpd::HeadPlan& p = n == piece ? dz : dz_last;
                p = pngpd::head_plan(type, rows, n, D, pngpd::HEAD_EPI_DZ);
                for (bool kept : {false, true}) sums = max2(sums, (size_t)pngpd::head_dz_parts(type, rows, n, p, kept) * n * 4);
                cut = max2(cut, p.partial_bytes);
                cut_w = max2(cut_w, pngpd::head_plan(type, n, D, rows, pngpd::HEAD_EPI_SCALED).partial_bytes);
                cut = max2(cut, pngpd::head_plan(type, rows, D, n, pngpd::HEAD_EPI_SCALED).partial_bytes);
            }
            part = (float*)b.take(sums);
            partial = (float*)b.take(cut);
            partial_w = (float*)b.take(cut_w);
        }
        bytes = b.off;
    }
};

int check_loss(const char* who, int type, int64_t T, int64_t V, int64_t D, const void* x, int64_t ldx, const void* w, int64_t ldw,
               const int64_t* target, float eps, int reduction) {
    int rc = check_sizes(who, type, T, V, D);
    if (rc) return rc;
    if (D > pngpd::HEAD_MAX_EXTENT) return fail(PNGPD_ERR_SHAPE, "%s: D = %lld, at most %lld", who, (long long)D, (long long)pngpd::HEAD_MAX_EXTENT);
    if (V > MAX_CLASSES) return fail(PNGPD_ERR_SHAPE, "%s: V = %lld, at most %lld", who, (long long)V, (long long)MAX_CLASSES);
    if (!w || (T > 0 && (!x || !target))) return fail(PNGPD_ERR_INVALID, "%s: NULL argument", who);
    if ((rc = check_ld(who, "ldx", ldx, D)) || (rc = check_ld(who, "ldw", ldw, D))) return rc;
    if (!(eps >= 0.f && eps <= 1.f)) return fail(PNGPD_ERR_INVALID, "%s: label_smoothing %g", who, (double)eps);
    if (reduction < PNGPD_REDUCE_NONE || reduction > PNGPD_REDUCE_SUM) return fail(PNGPD_ERR_INVALID, "%s: unknown reduction %d", who, reduction);
    return PNGPD_OK;
}

// Few classes have kernels of their own, which take x and the weight as they lie: the rows' losses, and the parts of the gradients
// where the logits were kept (the general products serve those that were not).
struct FewForwardWs {
    float* row_loss;
    double2* loss_parts;
    size_t bytes;
    FewForwardWs(void* base, int64_t T) {
        Bump b(base);
        row_loss = (float*)b.take((size_t)T * 4);
        loss_parts = (double2*)b.take((size_t)pngpd::head_batch_parts(T) * sizeof(double2));
        bytes = b.off;
    }
};
size_t few_backward_bytes(int type, int64_t T, int64_t V, int64_t D) {
    Bump b(nullptr);
    b.take(pngpd::head_few_part_bytes(type, T, V, D));
    return b.off;
}

constexpr size_t FEW_HEAD = 256;       // bytes in front of few classes' kept logits: the number of rows that count

// What the forward pass keeps for the backward pass, or 0.  Few classes: their logits, at most 32 bytes a row.  More: the
// 32-bit logits (without the bias) where they are one piece of the gradients' and forming them again should take longer than
// writing and reading them at 4.5 TB/s, with a launch that costs a little more.  Training, kept and formed again, in us:
// 4096 x 2048 -> 32768 in bfloat16 1620 and 1822, 4096 x 4096 -> 32768 2718 and 3332, 4096 x 1024 -> 32768 1103 and 1146,
// 1023 x 1000 -> 10007 in float32 581 and 684, 8192 x 4096 -> 16 in bfloat16 (where x is what costs) 121 and 138; the worst
// found is 2048 x 1024 -> 32768 in bfloat16, 573 and 559.
size_t kept_bytes(int type, int64_t T, int64_t V, int64_t D) {
    if (V <= pngpd::HEAD_FEW) {
        const size_t bytes = FEW_HEAD + (size_t)T * pngpd::head_few_room(V) * 4;
        return T > 0 && bytes <= loss_budget(type, T, V, D) ? bytes : 0;
    }
    if (T < 1 || pngpd::head_plan(type, T, V, D, pngpd::HEAD_EPI_DZ).us < 8.0 + 8.0 * (double)T * (double)V / 4.5e6) return 0;
    if (LossWs(nullptr, type, T, V, D, false, false, false).rows_at_once < T || LossWs(nullptr, type, T, V, D, true, false, false).piece < V) return 0;
    const size_t bytes = pngpd::head_kept_bytes(type, T, V, D);
    return bytes <= loss_budget(type, T, V, D) / esize(type) * 4 ? bytes : 0;
}

// those that are asked for
hipError_t gradients(int type, const pngpd::HeadGradient& x, const pngpd::HeadGradient& w, hipStream_t s) {
    if (x.e.out && w.e.out) return pngpd::head_gradients(type, x, w, s);
    if (!x.e.out && !w.e.out) return hipSuccess;
    const pngpd::HeadGradient& g = x.e.out ? x : w;
    return pngpd::head_product(type, g.M, g.N, g.K, g.a, g.b, g.e, g.partial, false, s);
}

inline const void* at(const void* p, int64_t elements, int type) { return p ? (const char*)p + (size_t)elements * esize(type) : nullptr; }
inline void* at(void* p, int64_t elements, int type) { return p ? (char*)p + (size_t)elements * esize(type) : nullptr; }

}  // namespace

extern "C" {

size_t pngpd_linear_workspace_bytes(int type, int64_t M, int64_t N, int64_t K, int backward, int aligned) {
    if (check_linear("pngpd_linear_workspace_bytes", type, M, N, K, PNGPD_ACT_NONE)) return 0;
    const bool k = (!aligned || padded(K, type) != K) && (backward || M > pngpd::HEAD_FEW_ROWS);
    return LinearWs(nullptr, type, M, N, K, backward != 0, k, k, true).bytes;
}

int pngpd_linear_forward(int type, int64_t M, int64_t N, int64_t K, const void* x_dev, int64_t ldx, const void* weight_dev,
                         int64_t ldw, const void* bias_dev, int act, const void* residual_dev, int64_t ldr, void* y_dev,
                         void* z_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
    const char* who = "pngpd_linear_forward";
    int rc = check_linear(who, type, M, N, K, act);
    if (rc) return rc;
    if (M == 0) return PNGPD_OK;
    if (!x_dev || !weight_dev || !y_dev) return fail(PNGPD_ERR_INVALID, "%s: NULL argument", who);
    if ((rc = check_ld(who, "ldx", ldx, K)) || (rc = check_ld(who, "ldw", ldw, K))) return rc;
    if (residual_dev && (rc = check_ld(who, "ldr", ldr, N))) return rc;
    const bool few = M <= pngpd::HEAD_FEW_ROWS;
    if (!few && (rc = check_tiles(who, type, M, N))) return rc;
    LinearWs ws(workspace_dev, type, M, N, K, false, !few && !direct(x_dev, ldx, K, type), !few && !direct(weight_dev, ldw, K, type), false);
    if ((rc = check_ws(who, workspace_dev, workspace_bytes, ws.bytes))) return rc;
    HeadEpilogue e;
    e.kind = pngpd::HEAD_EPI_LINEAR;
    e.bias = bias_dev;
    e.residual = residual_dev;
    e.ld_residual = ldr;
    e.act = act;
    e.z = z_dev;
    e.out = y_dev;
    e.ld_out = N;
    hipStream_t s = (hipStream_t)stream;
    pngpd::HeadLayOut job_x, job_w;
    bool lay_x = false, lay_w = false;
    const Rows x = few ? Rows{x_dev, ldx} : direct_rows(type, M, K, x_dev, ldx, ws.x, &job_x, &lay_x);
    const Rows w = few ? Rows{weight_dev, ldw} : direct_rows(type, N, K, weight_dev, ldw, ws.w, &job_w, &lay_w);
    HIP_TRY(pngpd::head_set_up(type, lay_x ? &job_x : nullptr, lay_w ? &job_w : nullptr, nullptr, s));
    HIP_TRY(pngpd::head_product(type, M, N, K, HeadOperand{x.p, x.ld, true}, HeadOperand{w.p, w.ld, true}, e, ws.partial, false, s));
    return PNGPD_OK;
}

int pngpd_linear_backward(int type, int64_t M, int64_t N, int64_t K, const void* dy_dev, int64_t ld_dy, const void* z_dev,
                          const void* x_dev, int64_t ldx, const void* weight_dev, int64_t ldw, int act, void* dx_dev,
                          void* dweight_dev, void* dbias_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
    const char* who = "pngpd_linear_backward";
    int rc = check_linear(who, type, M, N, K, act);
    if (rc) return rc;
    hipStream_t s = (hipStream_t)stream;
    if (M == 0) {
        if (dweight_dev) HIP_TRY(pngpd::head_zero(dweight_dev, (size_t)N * K * esize(type), s));
        if (dbias_dev) HIP_TRY(pngpd::head_zero(dbias_dev, (size_t)N * esize(type), s));
        return PNGPD_OK;
    }
    if (!dy_dev || (act != PNGPD_ACT_NONE && !z_dev) || (dx_dev && !weight_dev) || (dweight_dev && !x_dev))
        return fail(PNGPD_ERR_INVALID, "%s: NULL argument", who);
    if ((rc = check_ld(who, "ld_dy", ld_dy, N))) return rc;
    if (dweight_dev && (rc = check_ld(who, "ldx", ldx, K))) return rc;
    if (dx_dev && (rc = check_ld(who, "ldw", ldw, K))) return rc;
    if ((dx_dev && (rc = check_tiles(who, type, M, K))) || (dweight_dev && (rc = check_tiles(who, type, N, K)))) return rc;
    LinearWs ws(workspace_dev, type, M, N, K, true, dweight_dev && !direct(x_dev, ldx, K, type),
                dx_dev && !direct(weight_dev, ldw, K, type), act != PNGPD_ACT_NONE || !direct(dy_dev, ld_dy, N, type));
    if ((rc = check_ws(who, workspace_dev, workspace_bytes, ws.bytes))) return rc;
    // one pass over dy (and z): dz where it is not dy as it lies, and the bias gradient's partial sums
    const bool same = act == PNGPD_ACT_NONE && direct(dy_dev, ld_dy, N, type);
    const Rows dz = same ? Rows{dy_dev, ld_dy} : Rows{ws.dz, padded(N, type)};
    if (!same || dbias_dev)
        HIP_TRY(pngpd::head_grad_rows(type, M, N, dy_dev, ld_dy, z_dev, act, same ? nullptr : ws.dz, dz.ld,
                                      ws.part, dbias_dev, s));
    pngpd::HeadLayOut job_x, job_w;
    bool lay_x = false, lay_w = false;
    Rows x{}, w{};
    if (dx_dev) w = direct_rows(type, N, K, weight_dev, ldw, ws.w, &job_w, &lay_w);
    if (dweight_dev) x = direct_rows(type, M, K, x_dev, ldx, ws.x, &job_x, &lay_x);
    HIP_TRY(pngpd::head_set_up(type, lay_x ? &job_x : nullptr, lay_w ? &job_w : nullptr, nullptr, s));
    pngpd::HeadGradient gx{M, K, N, HeadOperand{dz.p, dz.ld, true}, HeadOperand{w.p, w.ld, false}, HeadEpilogue{}, ws.partial};
    pngpd::HeadGradient gw{N, K, M, HeadOperand{dz.p, dz.ld, false}, HeadOperand{x.p, x.ld, false}, HeadEpilogue{}, ws.partial_w};
    gx.e.ld_out = gw.e.ld_out = K;
    gx.e.out = dx_dev;
    gw.e.out = dweight_dev;
    HIP_TRY(gradients(type, gx, gw, s));
    return PNGPD_OK;
}

int pngpd_dropout(int type, int64_t rows, int64_t cols, const void* x_dev, int64_t ldx, const void* residual_dev, int64_t ldr,
                  void* y_dev, double p, uint64_t seed, uint64_t offset, const int64_t* rng_dev, void* stream) {
    const char* who = "pngpd_dropout";
    int rc = PNGPD_OK;
    if (!type_ok(type)) return fail(PNGPD_ERR_INVALID, "%s: unknown type %d", who, type);
    if (rows < 0 || cols < 1 || (double)rows * (double)cols > 4398046511104.0 || cols > ((int64_t)1 << 40))
        return fail(PNGPD_ERR_SHAPE, "%s: %lld x %lld, at most 2^42 elements, 2^40 a row", who, (long long)rows, (long long)cols);
    if (!(p >= 0.0 && p <= 1.0)) return fail(PNGPD_ERR_INVALID, "%s: p = %g", who, p);
    if (rows == 0) return PNGPD_OK;
    if (!x_dev || !y_dev) return fail(PNGPD_ERR_INVALID, "%s: NULL argument", who);
    if ((rc = check_ld(who, "ldx", ldx, cols))) return rc;
    if (residual_dev && (rc = check_ld(who, "ldr", ldr, cols))) return rc;
    HIP_TRY(pngpd::head_dropout(type, rows, cols, x_dev, ldx, residual_dev, ldr, y_dev, p, seed, offset, rng_dev, (hipStream_t)stream));
    return PNGPD_OK;
}

size_t pngpd_linear_cross_entropy_workspace_bytes(int type, int64_t T, int64_t V, int64_t D, int backward, int aligned) {
    const void* some = &type;      // the sizes alone are checked
    if (check_loss("pngpd_linear_cross_entropy_workspace_bytes", type, T, V, D, some, D, some, D, (const int64_t*)some, 0.f, 0)) return 0;
    if (V <= pngpd::HEAD_FEW && !backward) return FewForwardWs(nullptr, T).bytes;
    if (V <= pngpd::HEAD_FEW && backward == 2 && kept_bytes(type, T, V, D)) return few_backward_bytes(type, T, V, D);
    const bool d = !aligned || padded(D, type) != D;
    return LossWs(nullptr, type, T, V, D, backward != 0, d, d).bytes;
}

size_t pngpd_linear_cross_entropy_kept_bytes(int type, int64_t T, int64_t V, int64_t D) {
    const void* some = &type;
    if (check_loss("pngpd_linear_cross_entropy_kept_bytes", type, T, V, D, some, D, some, D, (const int64_t*)some, 0.f, 0)) return 0;
    return kept_bytes(type, T, V, D);
}

int pngpd_linear_cross_entropy_forward(int type, int64_t T, int64_t V, int64_t D, const void* x_dev, int64_t ldx,
                                       const void* weight_dev, int64_t ldw, const void* bias_dev, const int64_t* target_dev,
                                       int64_t ignore_index, float label_smoothing, int reduction, float* loss_dev,
                                       float* lse_dev, void* kept_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
    const char* who = "pngpd_linear_cross_entropy_forward";
    int rc = check_loss(who, type, T, V, D, x_dev, ldx, weight_dev, ldw, target_dev, label_smoothing, reduction);
    if (rc) return rc;
    if ((T > 0 || reduction != PNGPD_REDUCE_NONE) && !loss_dev) return fail(PNGPD_ERR_INVALID, "%s: NULL loss", who);
    if (((uintptr_t)kept_dev & 15) != 0) return fail(PNGPD_ERR_INVALID, "%s: kept must be aligned to 16 bytes", who);
    if (T > 0 && !lse_dev) return fail(PNGPD_ERR_INVALID, "%s: NULL lse", who);
    hipStream_t s = (hipStream_t)stream;
    if (T > 0 && V <= pngpd::HEAD_FEW) {
        const bool rows = reduction == PNGPD_REDUCE_NONE;
        const FewForwardWs ws(workspace_dev, T);
        if ((rc = check_ws(who, workspace_dev, workspace_bytes, rows ? 0 : ws.bytes))) return rc;
        char* few = kept_bytes(type, T, V, D) ? (char*)kept_dev : nullptr;
        float* row_loss = rows ? loss_dev : ws.row_loss;
        const pngpd::HeadFew g{T, V, D, x_dev, ldx, weight_dev, ldw, bias_dev, target_dev, ignore_index, label_smoothing,
                               few ? (float*)(few + FEW_HEAD) : nullptr};
        HIP_TRY(pngpd::head_few_loss(type, g, row_loss, lse_dev, s));
        if (!rows) HIP_TRY(pngpd::head_batch_loss(T, row_loss, target_dev, ignore_index, reduction, loss_dev, (float*)few, ws.loss_parts, s));
        return PNGPD_OK;
    }
    LossWs ws(workspace_dev, type, T, V, D, false, !direct(x_dev, ldx, D, type), !direct(weight_dev, ldw, D, type));
    if (T > 0) {
        if ((rc = check_ws(who, workspace_dev, workspace_bytes, ws.bytes))) return rc;
        pngpd::HeadLayOut job_x, job_w;
        bool lay_x, lay_w;
        const Rows x = direct_rows(type, T, D, x_dev, ldx, ws.x, &job_x, &lay_x);
        const Rows w = direct_rows(type, V, D, weight_dev, ldw, ws.w, &job_w, &lay_w);
        HIP_TRY(pngpd::head_set_up(type, lay_x ? &job_x : nullptr, lay_w ? &job_w : nullptr, nullptr, s));
        float* row_loss = reduction == PNGPD_REDUCE_NONE ? loss_dev : ws.row_loss;
        float* kept = kept_bytes(type, T, V, D) ? (float*)kept_dev : nullptr;
        for (int64_t t = 0; t < T; t += ws.rows_at_once) {
            const int64_t n = T - t < ws.rows_at_once ? T - t : ws.rows_at_once;
            const bool whole = n == T;
            HeadEpilogue e;
            e.kind = pngpd::HEAD_EPI_STATS;
            e.bias = bias_dev;
            e.target = target_dev + t;
            e.stats = ws.stats;
            e.target_logit = ws.target_logit;
            e.want_logit_sum = label_smoothing > 0.f;
            HIP_TRY(pngpd::head_product(type, n, V, D, HeadOperand{at(x.p, t * x.ld, type), x.ld, true}, HeadOperand{w.p, w.ld, true}, e,
                                        kept ? kept : ws.partial, kept != nullptr, s));
            const int blocks = pngpd::head_plan(type, n, V, D, pngpd::HEAD_EPI_STATS).stats_blocks;
            HIP_TRY(pngpd::head_row_loss(n, V, blocks, ws.stats, ws.target_logit, target_dev + t, ignore_index, label_smoothing,
                                         row_loss + t, lse_dev + t, reduction,
                                         whole && reduction != PNGPD_REDUCE_NONE ? loss_dev : nullptr, s));
            if (whole && reduction != PNGPD_REDUCE_NONE && pngpd::head_loss_at_once(n, blocks)) return PNGPD_OK;
        }
    }
    if (reduction != PNGPD_REDUCE_NONE) HIP_TRY(pngpd::head_batch_loss(T, ws.row_loss, target_dev, ignore_index, reduction, loss_dev, nullptr, ws.loss_parts, s));
    return PNGPD_OK;
}

int pngpd_linear_cross_entropy_backward(int type, int64_t T, int64_t V, int64_t D, const void* x_dev, int64_t ldx,
                                        const void* weight_dev, int64_t ldw, const void* bias_dev, const int64_t* target_dev,
                                        int64_t ignore_index, float label_smoothing, int reduction, const float* lse_dev,
                                        const void* kept_dev, const float* dloss_dev, void* dx_dev, void* dweight_dev, void* dbias_dev,
                                        void* workspace_dev, size_t workspace_bytes, void* stream) {
    const char* who = "pngpd_linear_cross_entropy_backward";
    int rc = check_loss(who, type, T, V, D, x_dev, ldx, weight_dev, ldw, target_dev, label_smoothing, reduction);
    if (rc) return rc;
    hipStream_t s = (hipStream_t)stream;
    if (T == 0) {
        if (dweight_dev) HIP_TRY(pngpd::head_zero(dweight_dev, (size_t)V * D * esize(type), s));
        if (dbias_dev) HIP_TRY(pngpd::head_zero(dbias_dev, (size_t)V * esize(type), s));
        return PNGPD_OK;
    }
    if (!lse_dev || !dloss_dev) return fail(PNGPD_ERR_INVALID, "%s: NULL argument", who);
    if (((uintptr_t)kept_dev & 15) != 0) return fail(PNGPD_ERR_INVALID, "%s: kept must be aligned to 16 bytes", who);
    const float* kept = kept_bytes(type, T, V, D) ? (const float*)kept_dev : nullptr;
    if (kept && V <= pngpd::HEAD_FEW) {
        if ((rc = check_ws(who, workspace_dev, workspace_bytes, few_backward_bytes(type, T, V, D)))) return rc;
        const pngpd::HeadFew g{T, V, D, x_dev, ldx, weight_dev, ldw, bias_dev, target_dev, ignore_index, label_smoothing,
                               const_cast<float*>(kept) + FEW_HEAD / 4};
        HIP_TRY(pngpd::head_few_grad(type, g, lse_dev, kept, dloss_dev, reduction, dx_dev, dweight_dev, dbias_dev, (float*)workspace_dev, s));
        return PNGPD_OK;
    }
    LossWs ws(workspace_dev, type, T, V, D, true, !direct(x_dev, ldx, D, type), !direct(weight_dev, ldw, D, type));
    if ((rc = check_tiles(who, type, T, ws.piece)) || (rc = check_tiles(who, type, T, D)) || (rc = check_tiles(who, type, ws.piece, D))) return rc;
    if ((rc = check_ws(who, workspace_dev, workspace_bytes, ws.bytes))) return rc;
    const HeadOperand x{ws.x, padded(D, type), true}, xt{ws.x, padded(D, type), false};
    const pngpd::HeadRowWeights weights{target_dev, T, V, ignore_index, reduction, dloss_dev, ws.row_weight, ws.scale,
                                        pngpd::head_label_factor(label_smoothing), ws.row_parts};
    const pngpd::HeadLayOut job_x{x_dev, T, D, ldx, ws.x, x.ld, true};      // what padding rows hold stays out of the sums
    pngpd::HeadLayOut job_w;
    bool lay_w;
    const Rows whole = direct_rows(type, V, D, weight_dev, ldw, ws.w, &job_w, &lay_w);
    HIP_TRY(pngpd::head_set_up(type, &job_x, lay_w ? &job_w : nullptr, &weights, s));
    for (int64_t v = 0; v < V; v += ws.piece) {
        const int64_t n = V - v < ws.piece ? V - v : ws.piece, np = padded(n, type);
        const void* w = at(whole.p, v * whole.ld, type);
        HeadEpilogue e;
        e.kind = pngpd::HEAD_EPI_DZ;
        e.bias = at(bias_dev, v, type);
        e.lse = lse_dev;
        e.row_weight = ws.row_weight;
        e.target = target_dev;
        e.first_n = v;
        e.smooth = label_smoothing / (float)V;
        e.one_minus_eps = 1.f - label_smoothing;
        e.out = ws.tile;
        e.ld_out = np;
        e.col_part = dbias_dev ? ws.part : nullptr;
        if (kept) HIP_TRY(pngpd::head_kept(type, T, V, D, e, kept, s));
        else HIP_TRY(pngpd::head_product(type, T, n, D, x, HeadOperand{w, whole.ld, true}, e, ws.partial, false, s));
        if (dbias_dev)
            HIP_TRY(pngpd::head_col_sums(type, pngpd::head_dz_parts(type, T, n, n == ws.piece ? ws.dz : ws.dz_last, kept != nullptr), n, ws.part, ws.scale,
                                         at(dbias_dev, v, type), s));
        const bool last = v + n == V;
        pngpd::HeadGradient gx{T, D, n, HeadOperand{ws.tile, np, true}, HeadOperand{w, whole.ld, false}, HeadEpilogue{}, ws.partial};
        pngpd::HeadGradient gw{n, D, T, HeadOperand{ws.tile, np, false}, xt, HeadEpilogue{}, ws.partial_w};
        gx.e.ld_out = gw.e.ld_out = D;
        gx.e.add = v > 0 ? ws.dx_sum : nullptr;
        gx.e.out_f32 = !last;
        gx.e.scale = last ? ws.scale : nullptr;
        gx.e.out = !dx_dev || last ? dx_dev : (void*)ws.dx_sum;
        gw.e.scale = ws.scale;
        gw.e.out = at(dweight_dev, v * D, type);
        HIP_TRY(gradients(type, gx, gw, s));
    }
    return PNGPD_OK;
}

}  // extern "C"
