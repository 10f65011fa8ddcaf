// Linear cross entropy over a few classes (at most 8): the weight is as small as a tile's row, so the products are bound by
// reading x, and by launches.
//
// Forward: 16 rows a workgroup, its waves side by side over the contraction, classes and rows as the two sides of a 16 x 16
// matrix instruction; the waves' sums are joined in order and every row's loss follows in registers.  The logits stay with the
// caller (4 or 8 floats a row).  Backward: one pass over x that forms dz from the kept logits, writes dx and sums dz^T x over
// the workgroup's rows; nothing is rounded between.  256 x 256 -> 3 in float32 takes 2 + 2 launches of 3 to 5 us, where the
// general products take 2 + 5 of 3 to 10.
#include "head.h"
#include "head_math.h"
#include "head_tile.h"

namespace pngpd {
namespace {

constexpr int TILE = 16;        // rows of a forward workgroup
constexpr int AHEAD = 8;
constexpr int BLOCK = 256;      // rows whose dz a backward workgroup has at a time

// 16 bytes from p, `valid` elements of them there, zeros behind
template <typename E>
__device__ __forceinline__ i32x4 chunk_of(const E* p, int64_t valid) {
    constexpr int C = 16 / sizeof(E);
    typedef __attribute__((ext_vector_type(16 / sizeof(E)))) E V;
    V v;
    if (valid >= C) {
        __builtin_memcpy(&v, p, 16);
        return __builtin_bit_cast(i32x4, v);
    }
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = i < valid ? p[i] : (E)0.f;
    return __builtin_bit_cast(i32x4, v);
}

// VP: classes a row has room for, 4 or 8
template <typename E, int VP>
__global__ __launch_bounds__(256) void few_loss_kernel(HeadFew g, float* row_loss, float* lse) {
    constexpr int C = 16 / sizeof(E);
    __shared__ f32x4 share[4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), t = lane & 15, q = lane >> 4;
    const int V = (int)g.V;
    const E* bias = (const E*)g.bias;
    const int64_t steps = (g.D + 4 * C - 1) / (4 * C), whole = g.D / (4 * C);
    // rows and classes beyond the last repeat it: what comes of them is not used
    const E* w = (const E*)g.w + (t < V ? t : V - 1) * g.ldw;
    for (int64_t m0 = (int64_t)blockIdx.x * TILE; m0 < g.T; m0 += (int64_t)gridDim.x * TILE) {
        const int64_t m = m0 + t;
        const E* x = (const E*)g.x + (m < g.T ? m : g.T - 1) * g.ldx;
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        // eight steps' loads at once; those beyond the last whole step repeat it and count as zeros
        for (int64_t s = wave; s < whole; s += 4 * AHEAD) {
            i32x4 fw[AHEAD], fx[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int64_t at = s + 4 * j < whole ? s + 4 * j : whole - 1, d = (at * 4 + q) * C;
                fw[j] = chunk_of<E>(w + d, C);
                fx[j] = chunk_of<E>(x + d, C);
            }
            fence();      // or the compiler takes them one by one
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const bool real = s + 4 * j < whole;
                acc = mma16<E>(real ? fw[j] : i32x4{}, real ? fx[j] : i32x4{}, acc);
            }
        }
        for (int64_t s = whole + (wave - whole & 3); s < steps; s += 4) {
            const int64_t d = (s * 4 + q) * C;
            acc = mma16<E>(chunk_of<E>(w + d, g.D - d), chunk_of<E>(x + d, g.D - d), acc);
        }
        share[wave][lane] = acc;
        __syncthreads();
        if (wave == 0) {
            const f32x4 sum = share[0][lane] + share[1][lane] + share[2][lane] + share[3][lane];
            const int64_t y = m < g.T ? g.target[m] : -1;
            f32x4 z;
            float mx = -__builtin_inff(), es = 0.f, zs = 0.f, zy = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = 4 * q + i;
                z[i] = n < V ? sum[i] + (bias ? to_f32(bias[n]) : 0.f) : -__builtin_inff();
                if (n < V) zs += z[i];
                if (n < V && n == y) zy = z[i];
                mx = __builtin_fmaxf(mx, z[i]);
            }
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16));
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32));
#pragma unroll
            for (int i = 0; i < 4; ++i) es += z[i] == -__builtin_inff() ? 0.f : __expf(z[i] - mx);
#pragma unroll
            for (int o = 16; o <= 32; o <<= 1) {
                es += __shfl_xor(es, o);
                zs += __shfl_xor(zs, o);
                zy += __shfl_xor(zy, o);
            }
            if (m < g.T) {
                if (g.logits && 4 * q < VP) *(f32x4*)(g.logits + m * VP + 4 * q) = z;
                if (q == 0) {
                    const float l = mx + logf(es);
                    lse[m] = l;
                    float loss = 0.f;
                    if (y != g.ignore_index) {
                        loss = y >= 0 && y < V ? l - (1.f - g.eps) * zy : __builtin_nanf("");
                        if (g.eps > 0.f) loss -= g.eps / (float)V * zs;
                    }
                    row_loss[m] = loss;
                }
            }
        }
        __syncthreads();
    }
}

struct FewGrad {
    const float *lse, *dloss, *used;
    int reduction;
    void *dx, *dw, *db;         // each may be NULL
    float* part;                // [parts][V][D] and [parts][V], unless there is one part
    int lanes;                  // 2^lanes threads side by side over chunks of columns
    int64_t rows;               // of a part
};

template <typename E, int VP>
__global__ __launch_bounds__(256) void few_grad_kernel(HeadFew g, FewGrad o) {
    constexpr int C = 16 / sizeof(E);
    typedef __attribute__((ext_vector_type(16 / sizeof(E)))) E Vec;
    typedef __attribute__((ext_vector_type(VP))) float Row;
    __shared__ Row dz[BLOCK];
    __shared__ bool live[BLOCK];
    __shared__ float share[256][C + 1];
    const int wide = 1 << o.lanes, side = 256 >> o.lanes, row = threadIdx.x >> o.lanes;
    const int64_t col = ((int64_t)blockIdx.x * wide + (threadIdx.x & (wide - 1))) * C;
    const int64_t m0 = (int64_t)blockIdx.y * o.rows, m1 = m0 + o.rows < g.T ? m0 + o.rows : g.T;
    const int V = (int)g.V;
    const float smooth = g.eps / (float)V;
    Vec w[VP];
    if (o.dx) {
#pragma unroll
        for (int n = 0; n < VP; ++n) w[n] = __builtin_bit_cast(Vec, chunk_of<E>((const E*)g.w + n * g.ldw + col, n < V ? g.D - col : 0));
    }
    float acc[VP][C] = {}, db[VP] = {};
    for (int64_t base = m0; base < m1; base += BLOCK) {
        __syncthreads();
        const int64_t m = base + threadIdx.x;
        if (m < m1) {
            const int64_t y = g.target[m];
            const bool on = y != g.ignore_index && y >= 0 && y < V;
            float weight = o.dloss[o.reduction == PNGPD_REDUCE_NONE ? m : 0];
            if (o.reduction == PNGPD_REDUCE_MEAN) weight /= o.used[0];
            const float l = o.lse[m];
            const Row z = *(const Row*)(g.logits + m * VP);
            Row d;
#pragma unroll
            for (int n = 0; n < VP; ++n) {
                d[n] = on && n < V ? (exp2_f(LOG2E * (z[n] - l)) - smooth - (n == y ? 1.f - g.eps : 0.f)) * weight : 0.f;
                db[n] += d[n];
            }
            dz[threadIdx.x] = d;
            live[threadIdx.x] = on;
        }
        __syncthreads();
        if (col < g.D) {
            const int rows = (int)(m1 - base < BLOCK ? m1 - base : BLOCK);
            const auto one = [&](int r, Vec x) {
                const Row d = dz[r];
                const bool on = live[r];
                if (!on) x = Vec{};      // what rows without a gradient hold stays out of the sums
#pragma unroll
                for (int n = 0; n < VP; ++n)
#pragma unroll
                    for (int i = 0; i < C; ++i) acc[n][i] = __builtin_fmaf(d[n], (float)x[i], acc[n][i]);
                if (o.dx) {
                    Eight v = {};
#pragma unroll
                    for (int n = 0; n < VP; ++n)
#pragma unroll
                        for (int i = 0; i < C; ++i) v.v[i] = __builtin_fmaf(d[n], (float)w[n][i], v.v[i]);
                    E* dx = (E*)o.dx + (base + r) * g.D + col;
                    Vec out;
#pragma unroll
                    for (int i = 0; i < C; ++i) out[i] = (E)(on ? v.v[i] : 0.f);
                    if (col + C <= g.D) __builtin_memcpy(dx, &out, 16);
                    else
#pragma unroll
                        for (int i = 0; i < C; ++i)
                            if (col + i < g.D) dx[i] = out[i];
                }
            };
            const E* x = (const E*)g.x + base * g.ldx + col;
            if (col + C <= g.D) {
#pragma unroll 4
                for (int r = row; r < rows; r += side) one(r, __builtin_bit_cast(Vec, chunk_of<E>(x + r * g.ldx, C)));
            } else {
                for (int r = row; r < rows; r += side) one(r, __builtin_bit_cast(Vec, chunk_of<E>(x + r * g.ldx, g.D - col)));
            }
        }
    }
    const bool whole = gridDim.y == 1;
    if (o.dw) {
#pragma unroll
        for (int n = 0; n < VP; ++n) {
            if (n >= V) break;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < C; ++i) share[threadIdx.x][i] = acc[n][i];
            __syncthreads();
            for (int c = threadIdx.x; c < wide * C; c += 256) {
                const int64_t d = (int64_t)blockIdx.x * wide * C + c;
                if (d >= g.D) continue;
                float s = 0.f;
                for (int r = 0; r < side; ++r) s += share[(r << o.lanes) + c / C][c % C];
                if (whole) ((E*)o.dw)[n * g.D + d] = from_f32<E>(s);
                else o.part[((int64_t)blockIdx.y * V + n) * g.D + d] = s;
            }
        }
    }
    if (o.db && blockIdx.x == 0) {
        __syncthreads();
#pragma unroll
        for (int n = 0; n < VP; ++n) {
            const float s = wave_sum(db[n]);
            if ((threadIdx.x & 63) == 0) share[threadIdx.x >> 6][n % C] = s;      // 4 floats a row at least: two turns of 4 classes
            __syncthreads();
            if (threadIdx.x == 0 && n < V) {
                const float v = share[0][n % C] + share[1][n % C] + share[2][n % C] + share[3][n % C];
                if (whole) ((E*)o.db)[n] = from_f32<E>(v);
                else o.part[(int64_t)gridDim.y * V * g.D + (int64_t)blockIdx.y * V + n] = v;
            }
            __syncthreads();
        }
    }
}

// dw and db from their parts: 32 elements by 8 shares of the parts a workgroup
template <typename E>
__global__ __launch_bounds__(256) void few_join_kernel(int parts, int64_t N, int64_t V, const float* part, E* dw, E* db) {
    __shared__ float share[8][32];
    const int c = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t n = (int64_t)blockIdx.x * 32 + c;
    const float* p = n < N ? part + n : part + parts * N + (n - N);
    const int64_t step = n < N ? N : V;
    float s = 0.f;
    if (n < N + V && (n < N ? dw != nullptr : db != nullptr)) {
#pragma unroll 8
        for (int i = w; i < parts; i += 8) s += p[i * step];
    }
    share[w][c] = s;
    __syncthreads();
    if (w || n >= N + V) return;
    for (int i = 1; i < 8; ++i) s += share[i][c];
    if (n < N && dw) dw[n] = from_f32<E>(s);
    if (n >= N && db) db[n - N] = from_f32<E>(s);
}

// How the backward pass is cut: threads side by side over a row's chunks, 1024 workgroups, but four turns of each thread at
// least (a part's sums are written and read again).
struct FewCut {
    int lanes;
    unsigned blocks;
    int64_t parts, rows;
};
FewCut few_cut(int64_t T, int64_t D, int chunk) {
    FewCut c;
    const int64_t chunks = (D + chunk - 1) / chunk;
    c.lanes = 0;
    while (c.lanes < 6 && (1 << c.lanes) < chunks) ++c.lanes;
    c.blocks = (unsigned)((chunks + (1 << c.lanes) - 1) >> c.lanes);
    const int64_t side = 256 >> c.lanes, most = (T + 4 * side - 1) / (4 * side);
    int64_t parts = 1024 / c.blocks;
    if (parts > most) parts = most;
    if (parts > 256) parts = 256;
    if (parts < 1) parts = 1;
    c.rows = ((T + parts - 1) / parts + side - 1) / side * side;
    c.parts = (T + c.rows - 1) / c.rows;
    return c;
}

template <typename E>
hipError_t few_loss(const HeadFew& g, float* row_loss, float* lse, hipStream_t s) {
    const int64_t tiles = (g.T + TILE - 1) / TILE;
    const unsigned grid = (unsigned)(tiles < 65536 ? tiles : 65536);
    if (g.V <= 4) few_loss_kernel<E, 4><<<grid, 256, 0, s>>>(g, row_loss, lse);
    else few_loss_kernel<E, 8><<<grid, 256, 0, s>>>(g, row_loss, lse);
    return hipGetLastError();
}

template <typename E>
hipError_t few_grad(const HeadFew& g, const float* lse, const float* used, const float* dloss, int reduction, void* dx, void* dw,
                    void* db, float* part, hipStream_t s) {
    const FewCut c = few_cut(g.T, g.D, 16 / sizeof(E));
    const FewGrad o{lse, dloss, used, reduction, dx, dw, db, part, c.lanes, c.rows};
    const dim3 grid(c.blocks, (unsigned)c.parts);
    if (g.V <= 4) few_grad_kernel<E, 4><<<grid, 256, 0, s>>>(g, o);
    else few_grad_kernel<E, 8><<<grid, 256, 0, s>>>(g, o);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || c.parts == 1 || (!dw && !db)) return e;
    const int64_t N = g.V * g.D;
    few_join_kernel<E><<<(unsigned)((N + g.V + 31) / 32), 256, 0, s>>>((int)c.parts, N, g.V, part, (E*)dw, (E*)db);
    return hipGetLastError();
}

}  // namespace

size_t head_few_part_bytes(int type, int64_t T, int64_t V, int64_t D) {
    const FewCut c = few_cut(T, D, type == PNGPD_TYPE_F32 ? 4 : 8);
    return c.parts > 1 ? (size_t)c.parts * V * (D + 1) * 4 : 0;
}

hipError_t head_few_loss(int type, const HeadFew& g, float* row_loss, float* lse, hipStream_t s) {
    switch (type) {
        case PNGPD_TYPE_F32: return few_loss<float>(g, row_loss, lse, s);
        case PNGPD_TYPE_BF16: return few_loss<bf16_t>(g, row_loss, lse, s);
        case PNGPD_TYPE_F16: return few_loss<f16_t>(g, row_loss, lse, s);
        default: return hipErrorInvalidValue;
    }
}

hipError_t head_few_grad(int type, const HeadFew& g, const float* lse, const float* used, const float* dloss, int reduction, void* dx,
                         void* dw, void* db, float* part, hipStream_t s) {
    switch (type) {
        case PNGPD_TYPE_F32: return few_grad<float>(g, lse, used, dloss, reduction, dx, dw, db, part, s);
        case PNGPD_TYPE_BF16: return few_grad<bf16_t>(g, lse, used, dloss, reduction, dx, dw, db, part, s);
        case PNGPD_TYPE_F16: return few_grad<f16_t>(g, lse, used, dloss, reduction, dx, dw, db, part, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace pngpd
