// Products of the classification head: the choice of a tile shape, the joining of split contractions, and the passes that
// lay operands out.
#include "head.h"
#include "head_math.h"
#include "head_tile.h"

namespace pngpd {
namespace {

// ---- joining partial sums --------------------------------------------------------------------------------------------------------

// 8 neighbouring columns of a row a thread: the cuts of the contraction added in order, then the epilogue.  Bound by memory: the
// logits' gradients of 4096 x 32768 from kept sums (537 MB read, 268 written) take 148 us, 5.4 TB/s.
template <typename E, int KIND, int THREADS>
__global__ __launch_bounds__(THREADS) void join_kernel(int64_t M, int64_t N, int64_t groups, int splits, const float* partial, HeadEpilogue e) {
    const int64_t total = M * groups;
    for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < total; i += (int64_t)gridDim.x * THREADS) {
        const int64_t m = i / groups, n = (i - m * groups) * 8;
        const int64_t have = N - n;
        const int valid = (int)(have < 0 ? 0 : have < 8 ? have : 8);
        Eight v = {};
#pragma unroll 4
        for (int s = 0; s < splits; ++s) add8(v, load8(partial + ((int64_t)s * M + m) * head_partial_ld(N) + n, valid));
        const int64_t room = (KIND == TILE_DZ ? e.ld_out : N) - n;
        const int real = (int)(room < 8 ? room : 8);
        finish8<E, KIND>(e, N, m, n, real, load_columns<E, KIND>(e, N, n), load_ahead<E, KIND>(e, N, m, n, real), v);
    }
}

// a row a workgroup, or a wave where rows are short (LANES): statistics of its logits, formed from the cuts of the contraction.
// Eight logits at a time share one rescaling of the sum; 1023 rows of 10007 sums (41 MB) take 12 us, 29 with one at a time.
template <typename E, int LANES>
__global__ __launch_bounds__(256) void join_stats_kernel(int64_t M, int64_t N, int splits, const float* partial, HeadEpilogue e) {
    __shared__ float4 share[4];
    const int64_t m = LANES == 64 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (m >= M) return;
    const int64_t y = e.target[m];
    const E* bias = (const E*)e.bias;
    float mx = -__builtin_inff(), sum = 0.f, zs = 0.f;
    for (int64_t n = (threadIdx.x & (LANES - 1)) * 8; n < N; n += LANES * 8) {
        const int valid = N - n < 8 ? (int)(N - n) : 8;
        Eight z = {};
#pragma unroll 4
        for (int s = 0; s < splits; ++s) add8(z, load8(partial + ((int64_t)s * M + m) * head_partial_ld(N) + n, valid));
        if (bias) add8(z, load8(bias + n, valid));
        float top = mx, part = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i >= valid) z.v[i] = -__builtin_inff();
            else zs += z.v[i];
            if (n + i == y) e.target_logit[m] = z.v[i];
            top = __builtin_fmaxf(top, z.v[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) part += z.v[i] == -__builtin_inff() ? 0.f : __expf(z.v[i] - top);
        sum = sum * (mx == top ? 1.f : __expf(mx - top)) + part;
        mx = top;
    }
    const float top = wave_max(mx);
    sum = wave_sum(sum * (mx == top ? 1.f : __expf(mx - top)));
    zs = wave_sum(zs);
    if (LANES == 64) {
        if ((threadIdx.x & 63) == 0) e.stats[m] = make_float4(top, sum, zs, 0.f);
        return;
    }
    if ((threadIdx.x & 63) == 0) share[threadIdx.x >> 6] = make_float4(top, sum, zs, 0.f);
    __syncthreads();
    if (threadIdx.x == 0) {
        float4 v = share[0];
        for (int w = 1; w < 4; ++w) {
            const float4 u = share[w];
            const float t = __builtin_fmaxf(v.x, u.x);
            v.y = v.y * (v.x == t ? 1.f : __expf(v.x - t)) + u.y * (u.x == t ? 1.f : __expf(u.x - t));
            v.x = t;
            v.z += u.z;
        }
        e.stats[m] = v;
    }
}

// How a pass over [M, N] is cut when it also sums columns: 2^lanes threads of a workgroup side by side over chunks of
// columns, the others over rows, `parts` blocks of `rows` rows, `turns` turns of the threads at least.
struct ColumnCut {
    int lanes;
    unsigned blocks;
    int64_t parts, rows;
};
ColumnCut column_cut(int64_t M, int64_t N, int chunk, int turns, int most_lanes) {
    if (M < 1) M = 1;
    ColumnCut c;
    const int64_t chunks = (N + chunk - 1) / chunk;
    c.lanes = 0;
    while (c.lanes < most_lanes && (1 << c.lanes) < chunks) ++c.lanes;
    c.blocks = (unsigned)((chunks + (1 << c.lanes) - 1) >> c.lanes);
    const int64_t side = 256 >> c.lanes;                        // rows at a time
    int64_t parts = 2048 / c.blocks;                            // enough workgroups to fill the chip
    const int64_t most = (M + turns * side - 1) / (turns * side);
    if (parts > most) parts = most;
    if (parts > 256) parts = 256;
    if (parts < 1) parts = 1;
    c.rows = ((M + parts - 1) / parts + side - 1) / side * side;
    c.parts = (M + c.rows - 1) / c.rows;
    return c;
}

// The logits' gradients from partial sums together with their columns' sums before they are rounded, a part of col_part a block
// of rows.  Bound by memory: 4096 x 32768 from kept sums in bfloat16 (805 MB) takes 202 us, 4.0 TB/s (210 with at most 64 groups
// of columns side by side); join_kernel and a pass over its rounded output took 149 + 56.  One turn a thread is enough where rows
// are few: each reads every cut of the contraction (300 x 4096 -> 40: 6 us; with four the training step took 7 us more).
ColumnCut dz_cut(int64_t M, int64_t ld_out) { return column_cut(M, ld_out, 8, 1, 8); }

template <typename E>
__global__ __launch_bounds__(256) void join_dz_kernel(int64_t M, int64_t N, int splits, const float* partial, HeadEpilogue e, int lanes,
                                                      int64_t rows) {
    __shared__ float share[256][9];
    const int wide = 1 << lanes, side = 256 >> lanes;
    const int64_t n = ((int64_t)blockIdx.x * wide + (threadIdx.x & (wide - 1))) * 8;
    const int64_t m0 = (int64_t)blockIdx.y * rows, m1 = m0 + rows < M ? m0 + rows : M;
    const int64_t have = N - n, room = e.ld_out - n;
    const int valid = (int)(have < 0 ? 0 : have < 8 ? have : 8), real = (int)(room < 8 ? room : 8);
    Eight sums = {};
    if (real > 0) {
        const Columns col = load_columns<E, TILE_DZ>(e, N, n);
        for (int64_t m = m0 + (threadIdx.x >> lanes); m < m1; m += side) {
            Eight v = {};
#pragma unroll 4
            for (int s = 0; s < splits; ++s) add8(v, load8(partial + ((int64_t)s * M + m) * head_partial_ld(N) + n, valid));
            finish8<E, TILE_DZ>(e, N, m, n, real, col, load_ahead<E, TILE_DZ>(e, N, m, n, real), v);
            add8(sums, v);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) share[threadIdx.x][i] = sums.v[i];
    __syncthreads();
    for (int c = threadIdx.x; c < wide * 8; c += 256) {
        const int64_t k = (int64_t)blockIdx.x * wide * 8 + c;
        if (k >= N) continue;
        float v = 0.f;
        for (int r = 0; r < side; ++r) v += share[(r << lanes) + c / 8][c % 8];
        e.col_part[(int64_t)blockIdx.y * N + k] = v;
    }
}

template <typename E>
hipError_t join(int64_t M, int64_t N, int splits, const float* partial, const HeadEpilogue& e, hipStream_t s) {
    if (e.kind == HEAD_EPI_DZ && e.col_part) {
        const ColumnCut c = dz_cut(M, e.ld_out);
        join_dz_kernel<E><<<dim3(c.blocks, (unsigned)c.parts), 256, 0, s>>>(M, N, splits, partial, e, c.lanes, c.rows);
        return hipGetLastError();
    }
    const int64_t groups = ((e.kind == HEAD_EPI_DZ ? e.ld_out : N) + 7) / 8;
    // little to join: small workgroups, so that its loads leave from many compute units
    const bool few = M * groups < 65536;
    const int64_t threads = few ? 64 : 256, blocks = (M * groups + threads - 1) / threads;
    const unsigned grid = (unsigned)(blocks < 65536 ? blocks : 65536);
#define PNGPD_JOIN(KIND)                                                                                          \
    if (few) join_kernel<E, KIND, 64><<<grid, 64, 0, s>>>(M, N, groups, splits, partial, e);              \
    else join_kernel<E, KIND, 256><<<grid, 256, 0, s>>>(M, N, groups, splits, partial, e)
    switch (e.kind) {
        case HEAD_EPI_LINEAR: PNGPD_JOIN(TILE_LINEAR); break;
        case HEAD_EPI_DZ: PNGPD_JOIN(TILE_DZ); break;
        case HEAD_EPI_SCALED: PNGPD_JOIN(TILE_SCALED); break;
        default:
            if (N <= 512) join_stats_kernel<E, 64><<<(unsigned)((M + 3) / 4), 256, 0, s>>>(M, N, splits, partial, e);
            else join_stats_kernel<E, 256><<<(unsigned)M, 256, 0, s>>>(M, N, splits, partial, e);
    }
#undef PNGPD_JOIN
    return hipGetLastError();
}

// ---- one to four rows -----------------------------------------------------------------------------------------------------------

// y[m][n] for up to MR rows m: a wave takes NR rows of the weight, its lanes 16-byte chunks of them side by side, and adds its
// lanes' 32-bit fma chains at the end.  Rows may start at any element.  Bound by reading the weight once: 4096 x 4096 bf16
// (33.5 MB) for one row, 5.1 us a launch where the caches hold the weight, 7.6 us from the last-level cache (four weights in turn),
// 8.6 us (3.9 TB/s) from memory; 8.5 instead of 5.1 before its loads were kept together.
constexpr int64_t FEW_M = HEAD_FEW_ROWS;

template <typename E, int MR, int NR>
__global__ __launch_bounds__(256) void rows_kernel(int M, int64_t N, int64_t K, const E* x, int64_t ldx, const E* w, int64_t ldw,
                                                   HeadEpilogue e) {
    constexpr int C = 16 / sizeof(E), U = MR * NR > 8 ? 2 : 4;
    typedef E chunk __attribute__((ext_vector_type(16 / sizeof(E)), aligned(sizeof(E))));
    const int lane = threadIdx.x & 63;
    const int64_t n0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * NR;
    if (n0 >= N) return;
    const E *px[MR], *pw[NR];
#pragma unroll
    for (int m = 0; m < MR; ++m) px[m] = x + (m < M ? m : 0) * ldx;
#pragma unroll
    for (int r = 0; r < NR; ++r) pw[r] = w + (n0 + r < N ? n0 + r : n0) * ldw;
    float acc[MR][NR] = {};
    const int64_t chunks = K / C;
    int64_t c = lane;
    for (; c + (U - 1) * 64 < chunks; c += U * 64) {
        chunk a[U][MR], b[U][NR];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int r = 0; r < NR; ++r) b[u][r] = ((const chunk*)pw[r])[c + u * 64];
#pragma unroll
            for (int m = 0; m < MR; ++m) a[u][m] = ((const chunk*)px[m])[c + u * 64];
        }
        fence();      // or the compiler puts every load next to its use, and they wait for one another
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < C; ++i)
#pragma unroll
                for (int m = 0; m < MR; ++m)
#pragma unroll
                    for (int r = 0; r < NR; ++r) acc[m][r] = __builtin_fmaf((float)a[u][m][i], (float)b[u][r][i], acc[m][r]);
    }
    for (; c < chunks; c += 64) {
        chunk a[MR], b[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) b[r] = ((const chunk*)pw[r])[c];
#pragma unroll
        for (int m = 0; m < MR; ++m) a[m] = ((const chunk*)px[m])[c];
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int m = 0; m < MR; ++m)
#pragma unroll
                for (int r = 0; r < NR; ++r) acc[m][r] = __builtin_fmaf((float)a[m][i], (float)b[r][i], acc[m][r]);
    }
    if (lane < (int)(K - chunks * C)) {
        const int64_t k = chunks * C + lane;
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
            for (int r = 0; r < NR; ++r) acc[m][r] = __builtin_fmaf((float)px[m][k], (float)pw[r][k], acc[m][r]);
    }
    float mine = 0.f;
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const float v = wave_sum(acc[m][r]);
            if (lane == m * NR + r) mine = v;
        }
    const int m = lane / NR;
    const int64_t n = n0 + lane % NR;
    if (lane >= MR * NR || m >= M || n >= N) return;
    const Columns col = load_columns<E, TILE_LINEAR>(e, n + 1, n);
    Eight v = {{mine}};
    finish8<E, TILE_LINEAR>(e, N, m, n, 1, col, load_ahead<E, TILE_LINEAR>(e, N, m, n, 1), v);
}

template <typename E, int MR>
hipError_t rows(int M, int64_t N, int64_t K, const HeadOperand& a, const HeadOperand& b, const HeadEpilogue& e, hipStream_t s) {
    // four rows of the weight a wave once that leaves a wave for every SIMD
#define PNGPD_ROWS(NR) \
    rows_kernel<E, MR, NR><<<(unsigned)((N + 4 * NR - 1) / (4 * NR)), 256, 0, s>>>(M, N, K, (const E*)a.p, a.ld, (const E*)b.p, b.ld, e)
    if (N >= 4096) PNGPD_ROWS(4);
    else if (N >= 2048) PNGPD_ROWS(2);
    else PNGPD_ROWS(1);
#undef PNGPD_ROWS
    return hipGetLastError();
}

template <typename E>
TileArgs tile_args(const HeadPlan& p, int64_t M, int64_t N, int64_t K, const HeadOperand& a, const HeadOperand& b, const HeadEpilogue& e,
                   float* partial) {
    TileArgs g{};
    g.M = M;
    g.N = N;
    g.K = K;
    g.a = (const char*)a.p;
    g.b = (const char*)b.p;
    g.lda = a.ld * (int64_t)sizeof(E);
    g.ldb = b.ld * (int64_t)sizeof(E);
    g.tiles_m = p.tiles_m;
    g.tiles_n = p.tiles_n;
    g.splits = p.splits;
    g.k_split = p.k_split;
    g.partial = partial;
    g.e = e;
    return g;
}

template <typename E>
hipError_t product(int type, int64_t M, int64_t N, int64_t K, const HeadOperand& a, const HeadOperand& b, const HeadEpilogue& e,
                   float* partial, bool keep, hipStream_t s) {
    if (M <= FEW_M && e.kind == HEAD_EPI_LINEAR) {
        if (M == 1) return rows<E, 1>((int)M, N, K, a, b, e, s);
        if (M == 2) return rows<E, 2>((int)M, N, K, a, b, e, s);
        return rows<E, 4>((int)M, N, K, a, b, e, s);
    }
    const HeadPlan p = head_plan(type, M, N, K, e.kind);
    if (p.tiles_m == 0) return hipErrorInvalidValue;
    const TileArgs g = tile_args<E>(p, M, N, K, a, b, e, p.splits > 1 || keep ? partial : nullptr);
    const bool parts = p.splits > 1;
    const int kind = parts ? TILE_PARTIAL
                     : e.kind == HEAD_EPI_LINEAR ? TILE_LINEAR
                     : e.kind == HEAD_EPI_DZ     ? TILE_DZ
                     : e.kind == HEAD_EPI_STATS  ? TILE_STATS
                                                 : TILE_SCALED;
    hipError_t err;
    if constexpr (__is_same(E, float)) err = launch_tile_f32(p.shape, kind, a.k_contiguous, b.k_contiguous, g, s);
    else if constexpr (__is_same(E, bf16_t)) err = launch_tile_bf16(p.shape, kind, a.k_contiguous, b.k_contiguous, g, s);
    else err = launch_tile_f16(p.shape, kind, a.k_contiguous, b.k_contiguous, g, s);
    if (err != hipSuccess || !parts) return err;
    return join<E>(M, N, p.splits, partial, e, s);
}

// A(m,k) of x's gradient is dense in its contraction, the other three operands are not.
template <typename E>
hipError_t gradients(int type, const HeadGradient& x, const HeadGradient& w, hipStream_t s) {
    const HeadPlan px = head_plan(type, x.M, x.N, x.K, HEAD_EPI_SCALED), pw = head_plan(type, w.M, w.N, w.K, HEAD_EPI_SCALED);
    const int64_t grid = (int64_t)px.tiles_m * px.tiles_n * px.splits + (int64_t)pw.tiles_m * pw.tiles_n * pw.splits;
    if (px.shape != SHAPE_64 || pw.shape != SHAPE_64 || grid >= (int64_t)1 << 23) {
        const hipError_t err = product<E>(type, w.M, w.N, w.K, w.a, w.b, w.e, w.partial, false, s);
        return err != hipSuccess ? err : product<E>(type, x.M, x.N, x.K, x.a, x.b, x.e, x.partial, false, s);
    }
    const TileArgs gx = tile_args<E>(px, x.M, x.N, x.K, x.a, x.b, x.e, x.partial), gw = tile_args<E>(pw, w.M, w.N, w.K, w.a, w.b, w.e, w.partial);
    hipError_t err;
    if constexpr (__is_same(E, float)) err = launch_pair_f32(gx, gw, s);
    else if constexpr (__is_same(E, bf16_t)) err = launch_pair_bf16(gx, gw, s);
    else err = launch_pair_f16(gx, gw, s);
    if (err == hipSuccess && pw.splits > 1) err = join<E>(w.M, w.N, pw.splits, w.partial, w.e, s);
    if (err == hipSuccess && px.splits > 1) err = join<E>(x.M, x.N, px.splits, x.partial, x.e, s);
    return err;
}

// ---- passes over whole matrices -----------------------------------------------------------------------------------------------------

template <typename T>
struct Chunk {
    static constexpr int C = 16 / sizeof(T);
    typedef __attribute__((ext_vector_type(16 / sizeof(T)))) T V;
    // up to C values from p, `valid` of them there, zeros behind
    __device__ static __forceinline__ V load(const T* p, int64_t valid) {
        V v;
        if (valid >= C) {
            __builtin_memcpy(&v, p, 16);
            return v;
        }
#pragma unroll
        for (int i = 0; i < C; ++i) v[i] = i < valid ? p[i] : (T)0.f;
        return v;
    }
};

// How many of the loss's rows count, and the largest gradient up and down among those that have one.
struct RowSums {
    float used, up, down;
};
__device__ __forceinline__ RowSums row_sums(const HeadRowWeights& w, int64_t first, int64_t last) {
    RowSums r = {};
#pragma unroll 8
    for (int64_t t = first + threadIdx.x; t < last; t += 256) {
        const int64_t y = w.target[t];
        r.used += y != w.ignore_index ? 1.f : 0.f;
        if (w.reduction == PNGPD_REDUCE_NONE && y != w.ignore_index && y >= 0 && y < w.V) {
            r.up = __builtin_fmaxf(r.up, w.dloss[t]);
            r.down = __builtin_fmaxf(r.down, -w.dloss[t]);
        }
    }
    return r;
}
// over a workgroup of 256
__device__ __forceinline__ RowSums join_rows(RowSums r) {
    __shared__ RowSums share[4];
    r.used = wave_sum(r.used);
    r.up = wave_max(r.up);
    r.down = wave_max(r.down);
    if ((threadIdx.x & 63) == 0) share[threadIdx.x >> 6] = r;
    __syncthreads();
    r = share[0];
    for (int i = 1; i < 4; ++i) {
        r.used += share[i].used;
        r.up = __builtin_fmaxf(r.up, share[i].up);
        r.down = __builtin_fmaxf(r.down, share[i].down);
    }
    return r;
}

// Up to 4096 rows one workgroup counts them and writes their weights, beside those that lay operands out; more are counted by up
// to 256 workgroups in a launch of their own, and written by as many.  Training in bfloat16, one workgroup and many, in us: 8192 x
// 2048 -> 64 with rows' own weights 88 and 71, 8192 x 1024 -> 16 66 and 60, 8192 x 16 -> 16 41 and 41, 2^20 x 16 -> 64 2810 and 400.
constexpr int64_t ROWS_ALONE = 4096, ROW_PARTS = 256;
inline int64_t rows_of_part(int64_t T) { return T <= 1024 * ROW_PARTS ? 1024 : (T + ROW_PARTS - 1) / ROW_PARTS; }

__global__ __launch_bounds__(256) void row_parts_kernel(HeadRowWeights w, int64_t rows) {
    const int64_t first = blockIdx.x * rows;
    const RowSums r = join_rows(row_sums(w, first, first + rows < w.T ? first + rows : w.T));
    if (threadIdx.x == 0) ((RowSums*)w.parts)[blockIdx.x] = r;
}

// Gradient weights of the loss's rows: workgroup `block` of those that write them, `rows` each
__device__ __forceinline__ void row_weights(const HeadRowWeights& w, int block, int64_t rows, int parts, bool bits16, bool half) {
    RowSums r = {};
    if (!parts) r = row_sums(w, 0, w.T);
    else if (threadIdx.x < parts) r = ((const RowSums*)w.parts)[threadIdx.x];
    r = join_rows(r);
    const float g = r.up >= r.down ? r.up : -r.down;      // the largest in size, with its sign
    // Operands of 16 bits: one weight for all rows stays out of dz and goes into the products' 32-bit sums, or p - 1 of the labels
    // would be rounded the same way in every row (off by up to 2^-9 in one direction in bfloat16).  Rows' own weights are divided
    // by the largest for the same reason, so that equal ones, the usual case, become 1; a row's quotient with another is rounded
    // with its dz.  Smoothed labels hold p - (1 - eps): dz is formed times the factor in (1/2, 1] that makes 1 - eps a power of two
    // (eps = 0.1 in bfloat16: 0.9 is off by 0.0017 of itself, in every row).  Half precision: the largest weight becomes at most
    // 2^14, |dz| <= 2 times that is inside its range, and a probability of 2^-37 still is a number.
    const bool one = w.reduction != PNGPD_REDUCE_NONE, shared = bits16 && g != 0.f && __builtin_fabsf(g) < __builtin_inff();
    const float top_weight = (half ? 16384.f : 1.f) * (bits16 ? w.label_factor : 1.f);
    float all = one ? w.dloss[0] : 0.f;
    if (w.reduction == PNGPD_REDUCE_MEAN) all *= 1.f / __builtin_fmaxf(r.used, 1.f);
    // an infinite gradient goes into dz, so that rows that have none keep their zeros
    const bool apart = one && __builtin_fabsf(all) < __builtin_inff();
    const int64_t first = block * rows, last = first + rows < w.T ? first + rows : w.T;
#pragma unroll 8
    for (int64_t t = first + threadIdx.x; t < last; t += 256) {
        const int64_t y = w.target[t];
        const bool live = y != w.ignore_index && y >= 0 && y < w.V;
        w.row_weight[t] = !live ? 0.f : apart ? top_weight : one ? all : shared ? w.dloss[t] / g * top_weight : w.dloss[t];
    }
    if (block == 0 && threadIdx.x == 0) w.out_scale[0] = apart ? all / top_weight : shared ? g / top_weight : 1.f;
}

struct LayOutRun {
    HeadLayOut m;
    int64_t blocks;        // of 256 chunks
    unsigned grid;
};

// Workgroups 0 .. a.grid lay out a, the next b.grid b, the last ones the rows' weights: a thread a 16-byte chunk of the
// destination; at most HEAD_MAX_LD / 16 chunks a row.  Bound by memory: 8192 x 4096 in bfloat16 (134 MB both ways) 33 us, 4.1 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void set_up_kernel(LayOutRun a, LayOutRun b, HeadRowWeights w, int64_t rows, int parts) {
    constexpr int C = Chunk<T>::C;
    if (blockIdx.x >= a.grid + b.grid) {
        row_weights(w, blockIdx.x - a.grid - b.grid, rows, parts, sizeof(T) == 2, __is_same(T, f16_t));
        return;
    }
    const bool second = blockIdx.x >= a.grid;
    const LayOutRun& u = second ? b : a;
    const unsigned per_row = (unsigned)(u.m.ld / C);
    for (int64_t block = second ? blockIdx.x - a.grid : blockIdx.x; block < u.blocks; block += u.grid) {
        const int64_t first = block * 256, r0 = first / per_row;      // uniform
        const unsigned off = (unsigned)(first - r0 * per_row) + threadIdx.x, d = off / per_row;
        const int64_t r = r0 + d, c = (int64_t)(off - d * per_row) * C;
        if (r >= u.m.rows) continue;
        bool live = true;
        if (u.m.live_rows_only) {
            const int64_t y = w.target[r];
            live = y != w.ignore_index && y >= 0 && y < w.V;
        }
        typename Chunk<T>::V v = {};
        if (live) v = Chunk<T>::load((const T*)u.m.src + r * u.m.ld_src + c, u.m.cols - c);
        *(typename Chunk<T>::V*)((T*)u.m.dst + r * u.m.ld + c) = v;
    }
}

template <typename T>
hipError_t set_up(const HeadLayOut* a, const HeadLayOut* b, const HeadRowWeights* w, hipStream_t s) {
    constexpr int C = Chunk<T>::C;
    auto run = [](const HeadLayOut* m) {
        LayOutRun r{};
        if (!m) return r;
        r.m = *m;
        r.blocks = (m->rows * (m->ld / C) + 255) / 256;
        r.grid = (unsigned)(r.blocks < (1 << 22) ? r.blocks : 1 << 22);
        return r;
    };
    const LayOutRun ra = run(a), rb = run(b);
    const int parts = w ? (int)head_row_parts(w->T) : 0;
    const int64_t rows = !w ? 0 : parts ? rows_of_part(w->T) : w->T;
    if (parts) {
        row_parts_kernel<<<(unsigned)parts, 256, 0, s>>>(*w, rows);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    const unsigned grid = ra.grid + rb.grid + (w ? parts ? parts : 1 : 0);
    if (grid == 0) return hipSuccess;
    set_up_kernel<T><<<grid, 256, 0, s>>>(ra, rb, w ? *w : HeadRowWeights{}, rows, parts);
    return hipGetLastError();
}

// One pass over dy and z, bound by memory, so the sums of the columns ride along: 8192 x 8192 in bfloat16 with gelu's slope
// (402 MB) takes 95 us, 4.2 TB/s (its exponential and reciprocal take about two thirds of that by themselves).
template <typename T, int ACT, bool WRITE>
__global__ __launch_bounds__(256) void grad_rows_kernel(int64_t M, int64_t N, const T* dy, int64_t ld, const T* z, T* dz,
                                                        int64_t ld_dz, float* part, int lanes, int64_t rows, T* sums) {
    constexpr int C = Chunk<T>::C;
    __shared__ float share[256][C + 1];
    const int wide = 1 << lanes, side = 256 >> lanes;
    const int64_t col = ((int64_t)blockIdx.x * wide + (threadIdx.x & (wide - 1))) * C;
    const int row = threadIdx.x >> lanes;
    const int64_t m0 = (int64_t)blockIdx.y * rows, m1 = m0 + rows < M ? m0 + rows : M;
    float sum[C] = {};
    if (col < N) {
#pragma unroll 2
        for (int64_t m = m0 + row; m < m1; m += side) {
            const typename Chunk<T>::V g = Chunk<T>::load(dy + m * ld + col, N - col);
            typename Chunk<T>::V o = g;
            if constexpr (ACT != PNGPD_ACT_NONE) {
                const typename Chunk<T>::V v = Chunk<T>::load(z + m * N + col, N - col);
#pragma unroll
                for (int i = 0; i < C; ++i) {
                    const float d = (float)g[i] * act_slope<ACT>((float)v[i]);
                    sum[i] += d;                          // before it is rounded
                    o[i] = col + i < N ? (T)d : (T)0.f;
                }
            } else {
#pragma unroll
                for (int i = 0; i < C; ++i) sum[i] += (float)g[i];
            }
            if constexpr (WRITE) *(typename Chunk<T>::V*)(dz + m * ld_dz + col) = o;
        }
    }
    if (!sums) return;
#pragma unroll
    for (int i = 0; i < C; ++i) share[threadIdx.x][i] = sum[i];
    __syncthreads();
    for (int c = threadIdx.x; c < wide * C; c += 256) {
        const int64_t n = (int64_t)blockIdx.x * wide * C + c;
        if (n >= N) continue;
        float s = 0.f;
        for (int r = 0; r < side; ++r) s += share[(r << lanes) + c / C][c % C];
        if (gridDim.y == 1) sums[n] = from_f32<T>(s);
        else part[(int64_t)blockIdx.y * N + n] = s;
    }
}

// COLS columns by 256 / COLS shares of the parts a workgroup
template <typename T, int COLS>
__global__ __launch_bounds__(256) void col_join_kernel(int64_t parts, int64_t N, const float* part, const float* scale, T* out) {
    constexpr int SHARES = 256 / COLS;
    __shared__ float share[SHARES][COLS];
    const int c = threadIdx.x % COLS, w = threadIdx.x / COLS;
    const int64_t n = (int64_t)blockIdx.x * COLS + c;
    float s = 0.f;
    if (n < N) {
#pragma unroll 8
        for (int64_t i = w; i < parts; i += SHARES) s += part[i * N + n];
    }
    share[w][c] = s;
    __syncthreads();
    if (w || n >= N) return;
    for (int i = 1; i < SHARES; ++i) s += share[i][c];
    out[n] = from_f32<T>(scale ? s * scale[0] : s);
}

// A tile's rows are a part: 2^20 rows are 16384 of them, which 32 shares join in 25 us and 8 in 91.
template <typename T>
hipError_t col_sums(int64_t parts, int64_t N, const float* part, const float* scale, void* out, hipStream_t s) {
    if (parts <= 256) col_join_kernel<T, 32><<<(unsigned)((N + 31) / 32), 256, 0, s>>>(parts, N, part, scale, (T*)out);
    else col_join_kernel<T, 8><<<(unsigned)((N + 7) / 8), 256, 0, s>>>(parts, N, part, scale, (T*)out);
    return hipGetLastError();
}

template <typename T>
hipError_t grad_rows(int64_t M, int64_t N, const void* dy, int64_t ld, const void* z, int act, void* dz, int64_t ld_dz, float* part,
                     void* sums, hipStream_t s) {
    constexpr int C = Chunk<T>::C;
    const ColumnCut c = column_cut(M, N, C, 4, 6);
    const dim3 grid(c.blocks, (unsigned)c.parts);
#define PNGPD_GRAD_ROWS(A, W) \
    grad_rows_kernel<T, A, W><<<grid, 256, 0, s>>>(M, N, (const T*)dy, ld, (const T*)z, (T*)dz, ld_dz, part, c.lanes, c.rows, (T*)sums)
    switch (act) {
        case PNGPD_ACT_NONE:
            if (dz) PNGPD_GRAD_ROWS(PNGPD_ACT_NONE, true);
            else PNGPD_GRAD_ROWS(PNGPD_ACT_NONE, false);
            break;
        case PNGPD_ACT_RELU: PNGPD_GRAD_ROWS(PNGPD_ACT_RELU, true); break;
        case PNGPD_ACT_GELU: PNGPD_GRAD_ROWS(PNGPD_ACT_GELU, true); break;
        case PNGPD_ACT_GELU_TANH: PNGPD_GRAD_ROWS(PNGPD_ACT_GELU_TANH, true); break;
        case PNGPD_ACT_SILU: PNGPD_GRAD_ROWS(PNGPD_ACT_SILU, true); break;
        default: return hipErrorInvalidValue;
    }
#undef PNGPD_GRAD_ROWS
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !sums || c.parts == 1) return e;
    return col_sums<T>(c.parts, N, part, nullptr, sums, s);
}

}  // namespace

size_t head_col_parts(int type, int64_t M, int64_t N) { return (size_t)column_cut(M, N, type == PNGPD_TYPE_F32 ? 4 : 8, 4, 6).parts; }

namespace {

// What a step of 128 bytes a row takes, in microseconds, with k tiles of a shape on every compute unit (measured on 256
// units, operands of normal numbers: 1.2 PFLOP/s for 256 x 256 tiles of 16-bit elements, 0.95 for 128 x 128 over matrices
// that the L2 does not hold - 1.28 where it does -, 0.6 to 0.7 for the small ones, 0.14 for floats).
double step_us(bool f32, int shape, int64_t k) {
    const double n = (double)k;
    if (f32) {
        if (shape == SHAPE_128) return 1.83 * n;
        return k <= 1 ? 0.58 : 0.48 * n;
    }
    switch (shape) {
        case SHAPE_256: return 1.7 * n;
        case SHAPE_128: return k <= 1 ? 0.55 : 1.1 * (double)((k + 1) / 2);
        case SHAPE_64: return k <= 1 ? 0.27 : 0.194 * n;
        default: return k <= 1 ? 0.31 : 0.235 * n;
    }
}
// What a tile takes besides: its first loads and its epilogue.
double tile_us(int shape) { return shape == SHAPE_256 ? 11.0 : shape == SHAPE_128 ? 9.0 : 4.0; }

}  // namespace

// The shape, and the number of cuts of the contraction, that should take the least time.  A cut contraction costs the
// joining kernel's 4 us and its traffic (32-bit sums written and read, at some 4 TB/s).
HeadPlan head_plan(int type, int64_t M, int64_t N, int64_t K, int kind) {
    const bool f32 = type == PNGPD_TYPE_F32;
    const int64_t step = f32 ? 32 : 64, steps = (K + step - 1) / step;
    HeadPlan p{};
    if (M <= FEW_M && kind == HEAD_EPI_LINEAR) return p;      // rows_kernel, nothing to join
    double best = 1e300;
    for (int shape = SHAPE_256; shape <= SHAPE_FEW_COLS; ++shape) {
        if (f32 && shape == SHAPE_256) continue;
        int bm, bn;
        shape_size(shape, &bm, &bn);
        const int64_t tm = (M + bm - 1) / bm, tn = (N + bn - 1) / bn, tiles = tm * tn;
        for (int64_t cuts = 1; cuts <= 32; ++cuts) {
            const int64_t per = (steps + cuts - 1) / cuts;
            if (cuts > 1 && (per < 4 || tiles >= 512)) break;
            if ((steps + per - 1) / per != cuts) continue;
            if (tiles * cuts >= (int64_t)1 << 23) continue;      // a grid holds 2^32 threads
            const int64_t k = (tiles * cuts + 255) / 256;
            double us = (double)per * step_us(f32, shape, k) + tile_us(shape) * (shape == SHAPE_256 ? (double)k : 1.0);
            if (cuts > 1) us += 4.0 + (double)cuts * (double)M * (double)N * 8e-6 / 4.0;
            if (us < best * 0.999) {
                best = p.us = us;
                p.shape = shape;
                p.splits = (int)cuts;
                p.tiles_m = (int)tm;
                p.tiles_n = (int)tn;
                p.k_split = per * step;
            }
        }
    }
    p.stats_blocks = p.splits > 1 ? 1 : p.tiles_n;
    p.partial_bytes = p.splits > 1 ? (size_t)p.splits * M * head_partial_ld(N) * 4 : 0;
    return p;
}

#define PNGPD_BY_TYPE(call)                                      \
    switch (type) {                                              \
        case PNGPD_TYPE_F32: { typedef float T; return call; }   \
        case PNGPD_TYPE_BF16: { typedef bf16_t T; return call; } \
        case PNGPD_TYPE_F16: { typedef f16_t T; return call; }   \
        default: return hipErrorInvalidValue;                    \
    }

hipError_t head_product(int type, int64_t M, int64_t N, int64_t K, const HeadOperand& a, const HeadOperand& b,
                        const HeadEpilogue& e, float* partial, bool keep, hipStream_t s) {
    PNGPD_BY_TYPE((product<T>(type, M, N, K, a, b, e, partial, keep, s)))
}
hipError_t head_gradients(int type, const HeadGradient& x, const HeadGradient& w, hipStream_t s) {
    PNGPD_BY_TYPE((gradients<T>(type, x, w, s)))
}
size_t head_kept_bytes(int type, int64_t M, int64_t N, int64_t K) {
    return (size_t)head_plan(type, M, N, K, HEAD_EPI_STATS).splits * M * head_partial_ld(N) * 4;
}
hipError_t head_kept(int type, int64_t M, int64_t N, int64_t K, const HeadEpilogue& e, const float* kept, hipStream_t s) {
    const int splits = head_plan(type, M, N, K, HEAD_EPI_STATS).splits;
    PNGPD_BY_TYPE((join<T>(M, N, splits, kept, e, s)))
}
int64_t head_row_parts(int64_t T) { return T <= ROWS_ALONE ? 0 : (T + rows_of_part(T) - 1) / rows_of_part(T); }
int64_t head_dz_parts(int type, int64_t M, int64_t N, const HeadPlan& p, bool kept) {
    const int64_t chunk = type == PNGPD_TYPE_F32 ? 4 : 8;
    return kept || p.splits > 1 ? dz_cut(M, (N + chunk - 1) / chunk * chunk).parts : p.tiles_m;
}
hipError_t head_col_sums(int type, int64_t parts, int64_t N, const float* part, const float* scale, void* out, hipStream_t s) {
    PNGPD_BY_TYPE((col_sums<T>(parts, N, part, scale, out, s)))
}
hipError_t head_set_up(int type, const HeadLayOut* a, const HeadLayOut* b, const HeadRowWeights* w, hipStream_t s) {
    PNGPD_BY_TYPE((set_up<T>(a, b, w, s)))
}
hipError_t head_grad_rows(int type, int64_t M, int64_t N, const void* dy, int64_t ld, const void* z, int act, void* dz,
                          int64_t ld_dz, float* part, void* sums, hipStream_t s) {
    PNGPD_BY_TYPE((grad_rows<T>(M, N, dy, ld, z, act, dz, ld_dz, part, sums, s)))
}

}  // namespace pngpd
