// One output tile of a product on the matrix units: out[m][n] = sum_k A(m,k) B(n,k), any operand order.
//
// The contraction runs in steps of 128 bytes a row (64 16-bit or 32 float elements).  A step's tiles go from global
// memory straight into LDS (16 bytes a lane, no registers), into the half of LDS the matrix instructions are not
// reading; one barrier a step.  Loads are buffer loads whose descriptor ends where the operand ends: rows behind the
// last one, and what a step has beyond the contraction, arrive as zeros and nothing outside an operand is ever read.
//
// LDS layouts, both written in linear order by the loads and permuted on the global side:
//   contraction dense  [row][8 chunks of 16 bytes], chunk c of row r at slot c ^ (r & 7): the 16 rows a fragment read
//                      touches spread over all banks.
//   rows dense         [k][row chunks], permuted by a function of k (tr_mix) so that the k rows one transposing read
//                      touches spread over the banks.  16-bit fragments come out of ds_read_b64_tr_b16, which hands
//                      lane t of 16 the column t of a 4 x 16 block.
// The n side is the matrix instruction's first operand, so a lane ends up with 4 neighbouring n of one m.
#pragma once
#include "head.h"
#include "head_math.h"
#include "kernels.h"

namespace pngpd {

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((address_space(3))) char lds_char;

struct TileArgs {
    int64_t M, N, K;
    const char *a, *b;
    int64_t lda, ldb;           // bytes between rows (k_contiguous) or between contraction steps
    int tiles_m, tiles_n, splits;
    int64_t k_split;            // contraction elements a split takes (a multiple of a step)
    float* partial;             // [split][M][N] when splits > 1
    HeadEpilogue e;
};

enum { TILE_LINEAR = 0, TILE_DZ = 1, TILE_SCALED = 2, TILE_PARTIAL = 3, TILE_STATS = 4 };

// ---- pieces of the kernel -------------------------------------------------------------------------------------------------

template <typename E>
__device__ __forceinline__ f32x4 mma16(const i32x4& a, const i32x4& b, f32x4 c) {
    if constexpr (__is_same(E, bf16_t)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else if constexpr (__is_same(E, f16_t)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    } else {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
        return c;
    }
}

// 16 bytes a lane from global memory to LDS at m0 + lane * 16.  Written out because the compiler holds back transposing
// LDS reads until every such load it knows of has landed, those into the other half of LDS included; stage_wait() is the
// wait that the data needs.  No register receives anything; m0 holds nothing else in these kernels (the compiler sets it in
// front of each use of its own).
__device__ __forceinline__ void stage_load(unsigned lds, unsigned voff, const i32x4& rsrc) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(lds), "v"(voff), "s"(rsrc) : "memory");
}
__device__ __forceinline__ void stage_wait() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory"); }

__device__ __forceinline__ i32x4 make_rsrc(const char* p, int64_t bytes) {
    const unsigned long long v = (unsigned long long)p;
    i32x4 r;
    r[0] = __builtin_amdgcn_readfirstlane((int)(unsigned)v);
    r[1] = __builtin_amdgcn_readfirstlane((int)((unsigned)(v >> 32) & 0xffffu));
    r[2] = __builtin_amdgcn_readfirstlane((int)(bytes < 0 ? 0 : bytes));
    r[3] = 0x00020000;
    return r;
}

// One operand of a tile: R rows, its loads and its fragment reads.  WAVES waves share the loads.
template <typename E, int R, bool KC, int WAVES>
struct TileOperand {
    static constexpr int SZ = sizeof(E), STEP = 128 / SZ, BYTES = R * 128, PIECES = BYTES / 1024;
    static constexpr int PER_WAVE = (PIECES + WAVES - 1) / WAVES;
    static constexpr int ROW_BYTES = R * SZ;             // of one contraction step, rows dense
    unsigned voff[PER_WAVE];
    unsigned beyond;                                     // bit i: piece i's chunk lies beyond the contraction in the last step

    // permutation of the chunk index of contraction step k (rows dense): in units of the columns one read takes, 2 chunks
    // (16 columns of 16 bits) or 4 (16 floats)
    __device__ static __forceinline__ int tr_mix(int k) {
        if constexpr (SZ == 2) return ROW_BYTES >= 256 ? (k & 3) | ((k >> 3) & 1) << 2 : ROW_BYTES >= 128 ? ((k >> 1) & 1) | ((k >> 3) & 1) << 1 : (k >> 3) & 1;
        return ROW_BYTES >= 256 ? (k >> 2) & 3 : (k >> 2) & 1;
    }

    __device__ __forceinline__ void init(int wave, int lane, int64_t ld) {
        beyond = 0;
#pragma unroll
        for (int i = 0; i < PER_WAVE; ++i) {
            const int p = wave + i * WAVES;
            const int o = p * 1024 + lane * 16;
            if constexpr (KC) {
                const int row = o / 128, c = ((o / 16) & 7) ^ (row & 7);
                voff[i] = (unsigned)(row * ld) + c * 16;
            } else {
                constexpr int U = SZ == 2 ? 2 : 4;
                const int k = o / ROW_BYTES, slot = (o % ROW_BYTES) / 16;
                const int c = ((slot / U) ^ tr_mix(k)) * U + slot % U;
                voff[i] = (unsigned)(k * ld) + c * 16;
            }
        }
    }
    // marks the chunks of the last step that lie beyond the contraction (`left` elements are left in it)
    __device__ __forceinline__ void init_tail(int wave, int lane, int left) {
        if constexpr (KC) {
#pragma unroll
            for (int i = 0; i < PER_WAVE; ++i) {
                const int o = (wave + i * WAVES) * 1024 + lane * 16;
                const int c = ((o / 16) & 7) ^ ((o / 128) & 7);
                if (c * (16 / SZ) >= left) beyond |= 1u << i;
            }
        }
    }
    // base: the tile's first element of this step; left: contraction elements from here on; rows: valid rows of the tile
    __device__ __forceinline__ void load(const char* base, int64_t ld, int64_t left, int rows, unsigned lds, int wave) {
        i32x4 rsrc;
        // an operand's dense extent is whole chunks, in itself or with zeros behind it (head_direct)
        constexpr int C = 16 / SZ;
        if constexpr (KC) rsrc = make_rsrc(base, (rows - 1) * ld + (left + C - 1) / C * 16);
        else rsrc = make_rsrc(base, ((left < STEP ? left : STEP) - 1) * ld + (rows + C - 1) / C * 16);
        const bool tail = KC && left < STEP;
#pragma unroll
        for (int i = 0; i < PER_WAVE; ++i) {
            if (PIECES % WAVES != 0 && wave + i * WAVES >= PIECES) break;
            unsigned v = voff[i];
            if (tail) v |= (beyond >> i & 1u) << 31;
            stage_load(lds + (wave + i * WAVES) * 1024, v, rsrc);
        }
    }
    // fragment of 16 rows from row0 (a multiple of 16), part ks (0 or 1) of the step
    __device__ static __forceinline__ i32x4 frag(const char* lds, int row0, int ks, int lane) {
        const int t = lane & 15, q = lane >> 4;
        if constexpr (KC) {
            return *(const i32x4*)(lds + (row0 + t) * 128 + (((ks * 4 + q) ^ (t & 7)) * 16));
        } else if constexpr (SZ == 2) {
            const int k = ks * 32 + 8 * q + (t >> 2);
            const char* p = lds + k * ROW_BYTES + ((((row0 >> 4) ^ tr_mix(8 * q + (t >> 2))) * 2 + ((t & 3) >> 1)) * 16) + (t & 1) * 8;
            // the step to k + 4 changes nothing in the permutation
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * ROW_BYTES));
            return __builtin_bit_cast(i32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            i32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = ks * 16 + 4 * q + j;
                v[j] = *(const int*)(lds + k * ROW_BYTES + ((((row0 >> 4) ^ tr_mix(4 * q)) * 4 + (t >> 2)) * 16) + (t & 3) * 4);
            }
            return v;
        }
    }
};

__device__ __forceinline__ float act_any(float z, int act) {
    switch (act) {
        case PNGPD_ACT_RELU: return act_f<PNGPD_ACT_RELU>(z);
        case PNGPD_ACT_GELU: return act_f<PNGPD_ACT_GELU>(z);
        case PNGPD_ACT_GELU_TANH: return act_f<PNGPD_ACT_GELU_TANH>(z);
        case PNGPD_ACT_SILU: return act_f<PNGPD_ACT_SILU>(z);
        default: return z;
    }
}

// Four neighbouring values of a row, as one access where `vec` says that every row starts suitably aligned.
template <typename T>
__device__ __forceinline__ f32x4 load4(const T* p, int valid, bool vec) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (vec && valid >= 4) {
        typedef __attribute__((ext_vector_type(4))) T t4;
        const t4 r = *(const t4*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (float)r[i];
    } else {
        for (int i = 0; i < 4; ++i)
            if (i < valid) v[i] = (float)p[i];
    }
    return v;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const f32x4& v, int valid, bool vec) {
    if (vec && valid >= 4) {
        typedef __attribute__((ext_vector_type(4))) T t4;
        t4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = (T)v[i];
        *(t4*)p = r;
    } else {
        for (int i = 0; i < 4; ++i)
            if (i < valid) p[i] = (T)v[i];
    }
}

// What becomes of 4 neighbouring sums of row m, from column n on (valid of them exist).
template <typename E, int KIND>
__device__ __forceinline__ void finish4(const HeadEpilogue& e, int64_t N, int64_t m, int64_t n, int valid, bool vec, f32x4 acc) {
    if constexpr (KIND == TILE_LINEAR) {
        if (e.bias) acc += load4((const E*)e.bias + n, valid, vec);
        if (e.z) {
            if (e.act == PNGPD_ACT_RELU) {
                E* z = (E*)e.z + m * N + n;
                for (int i = 0; i < 4; ++i)
                    if (i < valid) z[i] = keep_z<E, PNGPD_ACT_RELU>(acc[i]);
            } else {
                store4((E*)e.z + m * N + n, acc, valid, vec);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = act_any(acc[i], e.act);
        if (e.residual) acc += load4((const E*)e.residual + m * e.ld_residual + n, valid, vec);
        store4((E*)e.out + m * e.ld_out + n, acc, valid, vec);
    } else if constexpr (KIND == TILE_DZ) {
        const float w = e.row_weight[m], lse = e.lse[m];
        // the columns between N and the row's end are the zeros behind a dense extent; the bias ends at N
        const int real = (int)(N - n < 4 ? N - n : 4);
        if (e.bias) acc += load4((const E*)e.bias + n, real, vec);
        const int64_t y = e.target[m] - e.first_n - n;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p = __expf(acc[i] - lse) - e.smooth - (y == i ? e.one_minus_eps : 0.f);
            acc[i] = w == 0.f || i >= real ? 0.f : p * w;
        }
        store4((E*)e.out + m * e.ld_out + n, acc, valid, vec);
    } else {
        if (e.add) acc += load4(e.add + m * N + n, valid, vec);
        if (e.scale) acc *= e.scale[0];
        if (e.out_f32) store4((float*)e.out + m * e.ld_out + n, acc, valid, vec);
        else store4((E*)e.out + m * e.ld_out + n, acc, valid, vec);
    }
}

// rows of every matrix the epilogue touches start at a multiple of 4 elements
inline bool epilogue_vec(const HeadEpilogue& e, int64_t N, size_t sz) {
    auto ok = [](const void* p, int64_t ld, size_t size) { return !p || (((uintptr_t)p & (4 * size - 1)) == 0 && ld % 4 == 0); };
    return ok(e.out, e.ld_out, e.out_f32 ? 4 : sz) && ok(e.bias, 0, sz) && ok(e.residual, e.ld_residual, sz) && ok(e.z, N, sz) && ok(e.add, N, 4);
}

// ---- the kernel -------------------------------------------------------------------------------------------------------------

// BM x BN outputs by WM x WN waves; AK / BK: the contraction is dense in the m / n operand
template <typename E, int BM, int BN, int WM, int WN, bool AK, bool BK, int KIND>
__global__ __launch_bounds__(WM * WN * 64, 2) void product_tile_kernel(TileArgs g, bool vec) {
    constexpr int WAVES = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16, STEP = 128 / (int)sizeof(E);
    constexpr int STAGE = (BM + BN) * 128;
    typedef TileOperand<E, BM, AK, WAVES> OpA;
    typedef TileOperand<E, BN, BK, WAVES> OpB;
    extern __shared__ __attribute__((aligned(1024))) char smem[];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;

    // Workgroups go round the 8 XCDs: each XCD takes a run of neighbouring tiles, in groups of 8 rows of tiles, so that
    // the operands' tiles in its L2 serve as many products as they can.
    const int tiles = g.tiles_m * g.tiles_n;
    const int split = blockIdx.x / tiles;
    int id = blockIdx.x - split * tiles;
    {
        const int per = tiles / 8, rest = tiles % 8, x = id % 8, i = id / 8;
        id = x * per + (x < rest ? x : rest) + i;
    }
    const int group = 8 * g.tiles_n, gi = id / group, first = gi * 8;
    const int gm = g.tiles_m - first < 8 ? g.tiles_m - first : 8;
    const int tm = first + (id - gi * group) % gm, tn = (id - gi * group) / gm;
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int rows_m = (int)(g.M - m0 < BM ? g.M - m0 : BM), rows_n = (int)(g.N - n0 < BN ? g.N - n0 : BN);
    const int64_t k_begin = split * g.k_split;
    const int64_t k_end = k_begin + g.k_split < g.K ? k_begin + g.k_split : g.K;

    OpA oa;
    OpB ob;
    oa.init(wave, lane, g.lda);
    ob.init(wave, lane, g.ldb);
    const int tail = (int)((k_end - k_begin) % STEP);
    if (tail) {
        oa.init_tail(wave, lane, tail);
        ob.init_tail(wave, lane, tail);
    }
    const char* pa = g.a + (AK ? m0 * g.lda + k_begin * (int)sizeof(E) : k_begin * g.lda + m0 * (int)sizeof(E));
    const char* pb = g.b + (BK ? n0 * g.ldb + k_begin * (int)sizeof(E) : k_begin * g.ldb + n0 * (int)sizeof(E));
    const int64_t step_a = AK ? 128 : STEP * g.lda, step_b = BK ? 128 : STEP * g.ldb;
    const unsigned lds0 = (unsigned)(uintptr_t)(lds_char*)smem;

    f32x4 acc[FN][FM];
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    int64_t left = k_end - k_begin;
    int cur = 0;
    if (left > 0) {
        oa.load(pa, g.lda, left, rows_m, lds0, wave);
        ob.load(pb, g.ldb, left, rows_n, lds0 + BM * 128, wave);
    }
    while (left > 0) {
        stage_wait();      // this step's tiles are in LDS, and every wave is done reading the other half
        const int64_t next = left - STEP;
        if (next > 0) {
            pa += step_a;
            pb += step_b;
            const unsigned dst = lds0 + (cur ^ 1) * STAGE;
            oa.load(pa, g.lda, next, rows_m, dst, wave);
            ob.load(pb, g.ldb, next, rows_n, dst + BM * 128, wave);
        }
        const char* sa = smem + cur * STAGE;
        const char* sb = sa + BM * 128;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            i32x4 fa[FM], fb[FN];
#pragma unroll
            for (int j = 0; j < FM; ++j) fa[j] = OpA::frag(sa, (wm * FM + j) * 16, ks, lane);
#pragma unroll
            for (int i = 0; i < FN; ++i) fb[i] = OpB::frag(sb, (wn * FN + i) * 16, ks, lane);
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int j = 0; j < FM; ++j) acc[i][j] = mma16<E>(fb[i], fa[j], acc[i][j]);
        }
        cur ^= 1;
        left = next;
    }

    const int t = lane & 15, q = lane >> 4;
    if constexpr (KIND == TILE_STATS) {
        // a row's maximum, sum and target over this tile's columns: lane, then the 4 lanes of the row, then the waves
        __syncthreads();
        float4* share = (float4*)smem;      // [WN][BM]
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int r = (wm * FM + j) * 16 + t;
            const int64_t m = m0 + r;
            const int64_t y = m < g.M ? g.e.target[m] : -1;
            float mx = -__builtin_inff(), zs = 0.f;
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                const int64_t n = n0 + (wn * FN + i) * 16 + 4 * q;
                const int64_t have = g.N - n;
                const int valid = (int)(have < 0 ? 0 : have < 4 ? have : 4);
                if (g.e.bias) acc[i][j] += load4((const E*)g.e.bias + n, valid, vec);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (c >= valid) {
                        acc[i][j][c] = -__builtin_inff();
                        continue;
                    }
                    const float z = acc[i][j][c];
                    mx = __builtin_fmaxf(mx, z);
                    zs += z;
                    if (n + c == y) g.e.target_logit[m] = z;
                }
            }
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16));
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32));
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) s += acc[i][j][c] == -__builtin_inff() ? 0.f : __expf(acc[i][j][c] - mx);
            s += __shfl_xor(s, 16);
            s += __shfl_xor(s, 32);
            zs += __shfl_xor(zs, 16);
            zs += __shfl_xor(zs, 32);
            if (q == 0) share[wn * BM + r] = make_float4(mx, s, zs, 0.f);
        }
        __syncthreads();
        for (int r = threadIdx.x; r < rows_m; r += WAVES * 64) {
            float4 v = share[r];
            for (int w = 1; w < WN; ++w) {
                const float4 u = share[w * BM + r];
                const float mx = __builtin_fmaxf(v.x, u.x);
                v.y = v.y * (v.x == mx ? 1.f : __expf(v.x - mx)) + u.y * (u.x == mx ? 1.f : __expf(u.x - mx));
                v.x = mx;
                v.z += u.z;
            }
            g.e.stats[(int64_t)tn * g.M + m0 + r] = v;
        }
    } else {
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int64_t m = m0 + (wm * FM + j) * 16 + t;
            if (m >= g.M) continue;
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                const int64_t n = n0 + (wn * FN + i) * 16 + 4 * q;
                const int64_t have = (KIND == TILE_DZ ? g.e.ld_out : g.N) - n;
                if (have <= 0) continue;
                const int valid = (int)(have < 4 ? have : 4);
                if constexpr (KIND == TILE_PARTIAL) store4(g.partial + ((int64_t)split * g.M + m) * g.N + n, acc[i][j], valid, vec);
                else finish4<E, KIND>(g.e, g.N, m, n, valid, vec, acc[i][j]);
            }
        }
    }
}

// ---- launch -----------------------------------------------------------------------------------------------------------------

// tile shapes: 256 x 256 by 8 waves, 128 x 128, 32 x 128 (few rows) and 128 x 32 (few columns) by 4
enum { SHAPE_256 = 0, SHAPE_128 = 1, SHAPE_FEW_ROWS = 2, SHAPE_FEW_COLS = 3 };
inline void shape_size(int shape, int* bm, int* bn) {
    *bm = shape == SHAPE_256 ? 256 : shape == SHAPE_FEW_ROWS ? 32 : 128;
    *bn = shape == SHAPE_256 ? 256 : shape == SHAPE_FEW_COLS ? 32 : 128;
}

template <typename E, int BM, int BN, int WM, int WN, bool AK, bool BK, int KIND>
hipError_t launch_one(const TileArgs& g, bool vec, hipStream_t s) {
    constexpr int lds = 2 * (BM + BN) * 128;
    const auto kern = product_tile_kernel<E, BM, BN, WM, WN, AK, BK, KIND>;
    if (lds > 65536) {
        const hipError_t e = set_max_lds_once((const void*)kern, lds);
        if (e != hipSuccess) return e;
    }
    kern<<<(unsigned)(g.tiles_m * g.tiles_n * g.splits), WM * WN * 64, lds, s>>>(g, vec);
    return hipGetLastError();
}

template <typename E, bool AK, bool BK, int KIND>
hipError_t launch_shape(int shape, const TileArgs& g, bool vec, hipStream_t s) {
    switch (shape) {
        case SHAPE_256: return launch_one<E, 256, 256, 2, 4, AK, BK, KIND>(g, vec, s);
        case SHAPE_128: return launch_one<E, 128, 128, 2, 2, AK, BK, KIND>(g, vec, s);
        case SHAPE_FEW_ROWS: return launch_one<E, 32, 128, 1, 4, AK, BK, KIND>(g, vec, s);
        default: return launch_one<E, 128, 32, 4, 1, AK, BK, KIND>(g, vec, s);
    }
}

// forward products and logits: both operands dense in the contraction; dx: the second one transposed; dW: both
template <typename E>
hipError_t launch_tile(int shape, int kind, bool ak, bool bk, const TileArgs& g, bool vec, hipStream_t s) {
    if (ak && bk) {
        switch (kind) {
            case TILE_LINEAR: return launch_shape<E, true, true, TILE_LINEAR>(shape, g, vec, s);
            case TILE_DZ: return launch_shape<E, true, true, TILE_DZ>(shape, g, vec, s);
            case TILE_STATS: return launch_shape<E, true, true, TILE_STATS>(shape, g, vec, s);
            case TILE_PARTIAL: return launch_shape<E, true, true, TILE_PARTIAL>(shape, g, vec, s);
        }
    } else if (ak && !bk) {
        switch (kind) {
            case TILE_SCALED: return launch_shape<E, true, false, TILE_SCALED>(shape, g, vec, s);
            case TILE_PARTIAL: return launch_shape<E, true, false, TILE_PARTIAL>(shape, g, vec, s);
        }
    } else if (!ak && !bk) {
        switch (kind) {
            case TILE_SCALED: return launch_shape<E, false, false, TILE_SCALED>(shape, g, vec, s);
            case TILE_PARTIAL: return launch_shape<E, false, false, TILE_PARTIAL>(shape, g, vec, s);
        }
    }
    return hipErrorInvalidValue;
}

hipError_t launch_tile_f32(int shape, int kind, bool ak, bool bk, const TileArgs& g, bool vec, hipStream_t s);
hipError_t launch_tile_bf16(int shape, int kind, bool ak, bool bk, const TileArgs& g, bool vec, hipStream_t s);
hipError_t launch_tile_f16(int shape, int kind, bool ak, bool bk, const TileArgs& g, bool vec, hipStream_t s);

}  // namespace pngpd
