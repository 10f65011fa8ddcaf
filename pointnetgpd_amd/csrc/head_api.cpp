// C-ABI of the classification-head operators: checks of arguments, workspace layout, sequencing of the kernels.
#include <hip/hip_runtime.h>

#include "api_common.h"
#include "head.h"
#include "pngpd.h"

namespace {

using pngpd::fail;
using pngpd::HeadEpilogue;
using pngpd::HeadOperand;
using pngpd::HeadRowStats;

constexpr int64_t MAX_SIZE = 2147483647;
constexpr size_t PIECE_BYTES = (size_t)256 << 20;      // of logits (forward) or their gradients (backward) at a time

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

struct LinearWs {
    void* dz;
    float* part;
    size_t bytes;
    LinearWs(void* base, int type, int64_t M, int64_t N, int64_t K, bool backward) {
        Bump b(base);
        dz = nullptr;
        part = nullptr;
        if (backward && M > 0) {
            dz = b.take((size_t)M * N * esize(type));
            part = (float*)b.take((size_t)pngpd::head_col_sum_parts(M) * N * 4);
        }
        (void)K;
        bytes = b.off;
    }
};

struct LossWs {
    int64_t piece;             // columns of the vocabulary at a time
    void* tile;                // logits (32-bit, forward) or their gradients (of the type, backward): [T, piece]
    HeadRowStats st;
    float *row_weight, *scale, *part, *dx_sum;
    void* x;
    size_t bytes;
    LossWs(void* base, int type, int64_t T, int64_t V, int64_t D, bool backward) {
        Bump b(base);
        const int64_t rows = T > 0 ? T : 1;
        const size_t e = backward ? esize(type) : 4;
        piece = (int64_t)(PIECE_BYTES / ((size_t)rows * e)) / 256 * 256;
        if (piece < 256) piece = 256;
        if (piece > V) piece = V;
        tile = b.take((size_t)rows * piece * e);
        st = HeadRowStats{};
        row_weight = scale = part = dx_sum = nullptr;
        x = nullptr;
        if (!backward) {
            float* p = (float*)b.take((size_t)rows * 4 * 4);
            st = HeadRowStats{p, p + rows, p + 2 * rows, p + 3 * rows};
        } else {
            row_weight = (float*)b.take((size_t)rows * 4);
            scale = (float*)b.take(4);
            x = b.take((size_t)rows * D * esize(type));
            part = (float*)b.take((size_t)pngpd::head_col_sum_parts(T) * piece * 4);
            if (piece < V) dx_sum = (float*)b.take((size_t)rows * D * 4);
        }
        bytes = b.off;
    }
};

int check_loss(const char* who, int type, int64_t T, int64_t V, int64_t D, const void* x, int64_t ldx, const void* w, int64_t ldw,
               const int64_t* target, float eps, int reduction) {
    int rc = check_sizes(who, type, T, V, D);
    if (rc) return rc;
    if (!w || (T > 0 && (!x || !target))) return fail(PNGPD_ERR_INVALID, "%s: NULL argument", who);
    if ((rc = check_ld(who, "ldx", ldx, D)) || (rc = check_ld(who, "ldw", ldw, D))) return rc;
    if (!(eps >= 0.f && eps <= 1.f)) return fail(PNGPD_ERR_INVALID, "%s: label_smoothing %g", who, (double)eps);
    if (reduction < PNGPD_REDUCE_NONE || reduction > PNGPD_REDUCE_SUM) return fail(PNGPD_ERR_INVALID, "%s: unknown reduction %d", who, reduction);
    return PNGPD_OK;
}

inline const void* at(const void* p, int64_t elements, int type) { return p ? (const char*)p + (size_t)elements * esize(type) : nullptr; }
inline void* at(void* p, int64_t elements, int type) { return p ? (char*)p + (size_t)elements * esize(type) : nullptr; }

}  // namespace

extern "C" {

size_t pngpd_linear_workspace_bytes(int type, int64_t M, int64_t N, int64_t K, int backward) {
    if (check_sizes("pngpd_linear_workspace_bytes", type, M, N, K)) return 0;
    return LinearWs(nullptr, type, M, N, K, backward != 0).bytes;
}

int pngpd_linear_forward(int type, int64_t M, int64_t N, int64_t K, const void* x_dev, int64_t ldx, const void* weight_dev,
                         int64_t ldw, const void* bias_dev, int act, const void* residual_dev, int64_t ldr, void* y_dev,
                         void* z_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
    const char* who = "pngpd_linear_forward";
    int rc = check_sizes(who, type, M, N, K);
    if (rc) return rc;
    if (act < PNGPD_ACT_NONE || act > PNGPD_ACT_SILU) return fail(PNGPD_ERR_INVALID, "%s: unknown activation %d", who, act);
    if (M == 0) return PNGPD_OK;
    if (!x_dev || !weight_dev || !y_dev) return fail(PNGPD_ERR_INVALID, "%s: NULL argument", who);
    if ((rc = check_ld(who, "ldx", ldx, K)) || (rc = check_ld(who, "ldw", ldw, K))) return rc;
    if (residual_dev && (rc = check_ld(who, "ldr", ldr, N))) return rc;
    LinearWs ws(workspace_dev, type, M, N, K, false);
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
    HIP_TRY(pngpd::head_product(type, M, N, K, HeadOperand{x_dev, ldx, true}, HeadOperand{weight_dev, ldw, true}, e, (hipStream_t)stream));
    return PNGPD_OK;
}

int pngpd_linear_backward(int type, int64_t M, int64_t N, int64_t K, const void* dy_dev, int64_t ld_dy, const void* z_dev,
                          const void* x_dev, int64_t ldx, const void* weight_dev, int64_t ldw, int act, void* dx_dev,
                          void* dweight_dev, void* dbias_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
    const char* who = "pngpd_linear_backward";
    int rc = check_sizes(who, type, M, N, K);
    if (rc) return rc;
    if (act < PNGPD_ACT_NONE || act > PNGPD_ACT_SILU) return fail(PNGPD_ERR_INVALID, "%s: unknown activation %d", who, act);
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
    LinearWs ws(workspace_dev, type, M, N, K, true);
    if ((rc = check_ws(who, workspace_dev, workspace_bytes, ws.bytes))) return rc;
    const void* dz = dy_dev;
    int64_t ld_dz = ld_dy;
    if (act != PNGPD_ACT_NONE) {
        HIP_TRY(pngpd::head_act_backward(type, M, N, dy_dev, ld_dy, z_dev, act, ws.dz, s));
        dz = ws.dz;
        ld_dz = N;
    }
    if (dbias_dev) HIP_TRY(pngpd::head_col_sum(type, M, N, dz, ld_dz, ws.part, nullptr, dbias_dev, s));
    HeadEpilogue e;
    e.kind = pngpd::HEAD_EPI_SCALED;
    e.ld_out = K;
    if (dx_dev) {
        e.out = dx_dev;
        HIP_TRY(pngpd::head_product(type, M, K, N, HeadOperand{dz, ld_dz, true}, HeadOperand{weight_dev, ldw, false}, e, s));
    }
    if (dweight_dev) {
        e.out = dweight_dev;
        HIP_TRY(pngpd::head_product(type, N, K, M, HeadOperand{dz, ld_dz, false}, HeadOperand{x_dev, ldx, false}, e, s));
    }
    return PNGPD_OK;
}

int pngpd_dropout(int type, int64_t rows, int64_t cols, const void* x_dev, int64_t ldx, const void* residual_dev, int64_t ldr,
                  void* y_dev, double p, uint64_t seed, uint64_t offset, const int64_t* rng_dev, void* stream) {
    const char* who = "pngpd_dropout";
    int rc = check_sizes(who, type, rows, cols, 1);
    if (rc) return rc;
    if (!(p >= 0.0 && p <= 1.0)) return fail(PNGPD_ERR_INVALID, "%s: p = %g", who, p);
    if (rows == 0) return PNGPD_OK;
    if (!x_dev || !y_dev) return fail(PNGPD_ERR_INVALID, "%s: NULL argument", who);
    if ((rc = check_ld(who, "ldx", ldx, cols))) return rc;
    if (residual_dev && (rc = check_ld(who, "ldr", ldr, cols))) return rc;
    HIP_TRY(pngpd::head_dropout(type, rows, cols, x_dev, ldx, residual_dev, ldr, y_dev, p, seed, offset, rng_dev, (hipStream_t)stream));
    return PNGPD_OK;
}

size_t pngpd_linear_cross_entropy_workspace_bytes(int type, int64_t T, int64_t V, int64_t D, int backward) {
    if (check_sizes("pngpd_linear_cross_entropy_workspace_bytes", type, T, V, D)) return 0;
    return LossWs(nullptr, type, T, V, D, backward != 0).bytes;
}

int pngpd_linear_cross_entropy_forward(int type, int64_t T, int64_t V, int64_t D, const void* x_dev, int64_t ldx,
                                       const void* weight_dev, int64_t ldw, const void* bias_dev, const int64_t* target_dev,
                                       int64_t ignore_index, float label_smoothing, int reduction, float* loss_dev,
                                       float* lse_dev, void* workspace_dev, size_t workspace_bytes, void* stream) {
    const char* who = "pngpd_linear_cross_entropy_forward";
    int rc = check_loss(who, type, T, V, D, x_dev, ldx, weight_dev, ldw, target_dev, label_smoothing, reduction);
    if (rc) return rc;
    if ((T > 0 || reduction != PNGPD_REDUCE_NONE) && !loss_dev) return fail(PNGPD_ERR_INVALID, "%s: NULL loss", who);
    if (T > 0 && !lse_dev) return fail(PNGPD_ERR_INVALID, "%s: NULL lse", who);
    hipStream_t s = (hipStream_t)stream;
    LossWs ws(workspace_dev, type, T, V, D, false);
    if (T > 0) {
        if ((rc = check_ws(who, workspace_dev, workspace_bytes, ws.bytes))) return rc;
        for (int64_t v = 0; v < V; v += ws.piece) {
            const int64_t n = V - v < ws.piece ? V - v : ws.piece;
            HeadEpilogue e;
            e.kind = pngpd::HEAD_EPI_LINEAR;
            e.bias = at(bias_dev, v, type);
            e.out = ws.tile;
            e.ld_out = n;
            e.out_f32 = true;
            HIP_TRY(pngpd::head_product(type, T, n, D, HeadOperand{x_dev, ldx, true}, HeadOperand{at(weight_dev, v * ldw, type), ldw, true}, e, s));
            HIP_TRY(pngpd::head_stats_piece(T, n, (const float*)ws.tile, n, v, target_dev, ws.st, v == 0, s));
        }
    } else if (reduction == PNGPD_REDUCE_NONE) {
        return PNGPD_OK;
    }
    HIP_TRY(pngpd::head_loss_finish(T, V, target_dev, ignore_index, label_smoothing, reduction, ws.st, loss_dev, lse_dev, s));
    return PNGPD_OK;
}

int pngpd_linear_cross_entropy_backward(int type, int64_t T, int64_t V, int64_t D, const void* x_dev, int64_t ldx,
                                        const void* weight_dev, int64_t ldw, const void* bias_dev, const int64_t* target_dev,
                                        int64_t ignore_index, float label_smoothing, int reduction, const float* lse_dev,
                                        const float* dloss_dev, void* dx_dev, void* dweight_dev, void* dbias_dev,
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
    LossWs ws(workspace_dev, type, T, V, D, true);
    if ((rc = check_ws(who, workspace_dev, workspace_bytes, ws.bytes))) return rc;
    HIP_TRY(pngpd::head_row_weights(type, T, V, target_dev, ignore_index, reduction, dloss_dev, ws.row_weight, ws.scale, s));
    HIP_TRY(pngpd::head_live_rows(type, T, D, x_dev, ldx, ws.row_weight, ws.x, s));
    const HeadOperand x{ws.x, D, true};
    for (int64_t v = 0; v < V; v += ws.piece) {
        const int64_t n = V - v < ws.piece ? V - v : ws.piece;
        const void* w = at(weight_dev, v * ldw, type);
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
        e.ld_out = n;
        HIP_TRY(pngpd::head_product(type, T, n, D, x, HeadOperand{w, ldw, true}, e, s));
        if (dbias_dev) HIP_TRY(pngpd::head_col_sum(type, T, n, ws.tile, n, ws.part, ws.scale, at(dbias_dev, v, type), s));
        HeadEpilogue g;
        g.kind = pngpd::HEAD_EPI_SCALED;
        g.ld_out = D;
        if (dweight_dev) {
            g.out = at(dweight_dev, v * D, type);
            g.scale = ws.scale;
            HIP_TRY(pngpd::head_product(type, n, D, T, HeadOperand{ws.tile, n, false}, HeadOperand{ws.x, D, false}, g, s));
        }
        if (dx_dev) {
            const bool last = v + n == V;
            g.add = v > 0 ? ws.dx_sum : nullptr;
            g.out_f32 = !last;
            g.scale = last ? ws.scale : nullptr;
            g.out = last ? dx_dev : (void*)ws.dx_sum;
            HIP_TRY(pngpd::head_product(type, T, D, n, HeadOperand{ws.tile, n, true}, HeadOperand{w, ldw, false}, g, s));
        }
    }
    return PNGPD_OK;
}

}  // extern "C"
