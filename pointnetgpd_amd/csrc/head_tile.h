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
//
// 16-bit: 256 x 256 tiles reach 1.24 PFLOP/s (8192 x 4096 x 8192 in 445 us, 488 with gelu_tanh and a residual), the library's bare
// product 1.40 to 1.43 on the same card.  Two things bound them.  The clock: the same product on zeros takes 330 us (library: 256 to
// 275).  And the tile's ends: one workgroup holds a compute unit (128 KB of LDS), so nothing covers its first loads and its
// epilogue, 11 us a tile beside 64 steps of 1.7.  Floats: 64 x 64 tiles, three to a compute unit, reach 0.14
// PFLOP/s of the matrix unit's 0.157 inside the loop, 0.13 over 4096 x 2048 x 2048.
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
    float* partial;             // [split][M][head_partial_ld(N)] when splits > 1; of a STATS product whose sums are kept; else NULL
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

// N pieces of 16 bytes a lane from global memory to LDS, the i-th at lds + i * STRIDE + lane * 16.  Written out because the
// compiler holds back transposing LDS reads until every such load it knows of has landed, those into other stages included;
// stage_wait() is the wait that the data needs.  No register receives anything; m0 holds nothing else in these kernels (the
// compiler sets it in front of each use of its own).
template <int N, int STRIDE>
__device__ __forceinline__ void stage_load(unsigned lds, const unsigned* voff, const i32x4& rsrc) {
#define PNGPD_FIRST "s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
#define PNGPD_NEXT(v) "\n\ts_add_u32 m0, m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 " v ", %2, 0 offen lds"
    if constexpr (N == 1) {
        asm volatile(PNGPD_FIRST : : "s"(lds), "v"(voff[0]), "s"(rsrc) : "memory");
    } else if constexpr (N == 2) {
        asm volatile(PNGPD_FIRST PNGPD_NEXT("%4") : : "s"(lds), "v"(voff[0]), "s"(rsrc), "n"(STRIDE), "v"(voff[1]) : "memory", "scc");
    } else {
        static_assert(N == 4, "pieces of a wave");
        asm volatile(PNGPD_FIRST PNGPD_NEXT("%4") PNGPD_NEXT("%5") PNGPD_NEXT("%6")
                     :
                     : "s"(lds), "v"(voff[0]), "s"(rsrc), "n"(STRIDE), "v"(voff[1]), "v"(voff[2]), "v"(voff[3])
                     : "memory", "scc");
    }
#undef PNGPD_FIRST
#undef PNGPD_NEXT
}
// All but the wave's last AHEAD loads have landed, and its LDS reads; then the barrier.  By the builtins, so that the compiler
// knows that nothing read from LDS is outstanding.
template <int AHEAD>
__device__ __forceinline__ void stage_wait() {
    asm volatile("" : : : "memory");
    __builtin_amdgcn_s_waitcnt((AHEAD & 15) | 7 << 4 | (AHEAD >> 4) << 14);      // vmcnt(AHEAD) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
}

__device__ __forceinline__ i32x4 make_rsrc(const char* p, int bytes) {
    const unsigned long long v = (unsigned long long)p;
    i32x4 r;
    r[0] = __builtin_amdgcn_readfirstlane((int)(unsigned)v);
    r[1] = __builtin_amdgcn_readfirstlane((int)((unsigned)(v >> 32) & 0xffffu));
    r[2] = __builtin_amdgcn_readfirstlane(bytes);
    r[3] = 0x00020000;
    return r;
}

// Keeps the order of what stands before and behind: the compiler would otherwise put the reads next to their uses, to save
// registers, and the loads together.
__device__ __forceinline__ void fence() { __builtin_amdgcn_sched_barrier(0); }

// One operand of a tile: R rows, its loads and its fragment reads.  WAVES waves share the loads.
template <typename E, int R, bool KC, int WAVES>
struct TileOperand {
    static constexpr int SZ = sizeof(E), STEP = 128 / SZ, BYTES = R * 128, PIECES = BYTES / 1024;
    static constexpr int PER_WAVE = PIECES / WAVES;
    static_assert(PIECES % WAVES == 0, "every wave issues as many loads");
    static constexpr int ROW_BYTES = R * SZ;             // of one contraction step, rows dense
    unsigned voff[PER_WAVE];                             // of the wave's pieces, WAVES apart
    unsigned beyond;                                     // bit 31: the lane's chunk lies beyond the contraction in its last step

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
            const int o = (wave + i * WAVES) * 1024 + lane * 16;
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
    __device__ __forceinline__ void init_tail(int lane, int left) {
        if constexpr (KC) {
            const int c = (lane & 7) ^ (lane >> 3);
            beyond = c * (16 / SZ) >= left ? 0x80000000u : 0u;
        }
    }
    // base: the tile's first element of this step; left: contraction elements from here on (none: zeros arrive); rows: valid
    // rows of the tile.  An operand's dense extent is whole chunks, in itself or with zeros behind it (head_direct).
    __device__ __forceinline__ void load(const char* base, unsigned ld, int left, int rows, unsigned lds, int wave) {
        constexpr int C = 16 / SZ;
        const int here = left < STEP ? left : STEP;
        const int bytes = KC ? (int)((rows - 1) * ld) + (here + C - 1) / C * 16 : (int)((here - 1) * ld) + (rows + C - 1) / C * 16;
        const i32x4 rsrc = make_rsrc(base, left > 0 ? bytes : 0);
        stage_load<PER_WAVE, WAVES * 1024>(lds + wave * 1024, voff, rsrc);
    }
    // From the last step on, if it is not a whole one: its chunks beyond the contraction become offsets beyond the descriptor.
    __device__ __forceinline__ void mask_tail() {
#pragma unroll
        for (int i = 0; i < PER_WAVE; ++i) voff[i] |= beyond;
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

// Eight neighbouring values of a row, as 16-byte accesses wherever they start: the hardware takes
// them at any element (4001 x 2001 -> 1999 bfloat16 training 171 us, 220 with an access an element in such rows).
struct Eight {
    float v[8];
};
template <typename T>
__device__ __forceinline__ Eight load8(const T* p, int valid) {
    constexpr int C = 16 / sizeof(T);
    typedef __attribute__((ext_vector_type(16 / sizeof(T)))) T chunk;
    Eight r;
    if (valid >= 8) {
#pragma unroll
        for (int k = 0; k < 8 / C; ++k) {
            chunk c;
            __builtin_memcpy(&c, p + k * C, 16);
#pragma unroll
            for (int i = 0; i < C; ++i) r.v[k * C + i] = (float)c[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = i < valid ? (float)p[i] : 0.f;
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const Eight& r, int valid) {
    constexpr int C = 16 / sizeof(T);
    typedef __attribute__((ext_vector_type(16 / sizeof(T)))) T chunk;
    if (valid >= 8) {
#pragma unroll
        for (int k = 0; k < 8 / C; ++k) {
            chunk c;
#pragma unroll
            for (int i = 0; i < C; ++i) c[i] = (T)r.v[k * C + i];
            __builtin_memcpy(p + k * C, &c, 16);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < valid) p[i] = (T)r.v[i];
    }
}
__device__ __forceinline__ void add8(Eight& a, const Eight& b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) a.v[i] += b.v[i];
}
template <int ACT>
__device__ __forceinline__ void act8(Eight& a) {
#pragma unroll
    for (int i = 0; i < 8; ++i) a.v[i] = act_f<ACT>(a.v[i]);
}

// exp(z - base), the difference first: it is exact for z near base, however large both are (a class masked by a bias of -1e30
// has a maximum of that size in its tile).
__device__ __forceinline__ float exp_of(float z, float base) { return exp2_f(LOG2E * (z - base)); }

// The epilogue of 8 neighbouring sums of a row, in the order a latency-bound loop wants it: what depends on the columns is
// loaded once (Columns), what depends on the row for several rows ahead (Ahead), then the sums are finished.
struct Columns {
    Eight bias;
    float scale;
};
template <typename E, int KIND>
__device__ __forceinline__ Columns load_columns(const HeadEpilogue& e, int64_t N, int64_t n) {
    Columns c = {};
    c.scale = 1.f;
    if constexpr (KIND == TILE_LINEAR || KIND == TILE_DZ) {
        if (e.bias) c.bias = load8((const E*)e.bias + n, (int)(N - n < 0 ? 0 : N - n < 8 ? N - n : 8));
    }
    if constexpr (KIND == TILE_SCALED) {
        if (e.scale) c.scale = e.scale[0];
    }
    return c;
}
struct Ahead {
    Eight more;             // LINEAR: residual; SCALED: what is added
    float weight, lse;      // DZ
    int label;
};
template <typename E, int KIND>
__device__ __forceinline__ Ahead load_ahead(const HeadEpilogue& e, int64_t N, int64_t m, int64_t n, int valid) {
    Ahead h = {};
    if constexpr (KIND == TILE_LINEAR) {
        if (e.residual) h.more = load8((const E*)e.residual + m * e.ld_residual + n, valid);
    } else if constexpr (KIND == TILE_DZ) {
        h.weight = e.row_weight[m];
        h.lse = e.lse[m];
        const int64_t y = e.target[m] - e.first_n - n;
        h.label = y >= 0 && y < 8 ? (int)y : -1;
    } else if constexpr (KIND == TILE_SCALED) {
        if (e.add) h.more = load8(e.add + m * N + n, valid);
    }
    return h;
}
template <typename E, int KIND>
__device__ __forceinline__ void finish8(const HeadEpilogue& e, int64_t N, int64_t m, int64_t n, int valid, const Columns& col,
                                        const Ahead& h, Eight& a) {
    if constexpr (KIND == TILE_LINEAR) {
        add8(a, col.bias);
        if (e.z) {
            E* z = (E*)e.z + m * N + n;
            if (sizeof(E) == 2 && e.act == PNGPD_ACT_RELU) {
                Eight k;
#pragma unroll
                for (int i = 0; i < 8; ++i) k.v[i] = (float)keep_z<E, PNGPD_ACT_RELU>(a.v[i]);
                store8(z, k, valid);
            } else {
                store8(z, a, valid);
            }
        }
        switch (e.act) {
            case PNGPD_ACT_RELU: act8<PNGPD_ACT_RELU>(a); break;
            case PNGPD_ACT_GELU: act8<PNGPD_ACT_GELU>(a); break;
            case PNGPD_ACT_GELU_TANH: act8<PNGPD_ACT_GELU_TANH>(a); break;
            case PNGPD_ACT_SILU: act8<PNGPD_ACT_SILU>(a); break;
        }
        if (e.residual) add8(a, h.more);
        store8((E*)e.out + m * e.ld_out + n, a, valid);
    } else if constexpr (KIND == TILE_DZ) {
        // What only some rows or columns have stands in branches of its own: an instruction on every element costs half a
        // microsecond a tile.
        if (e.bias) add8(a, col.bias);
        const float gone = e.smooth * h.weight;
#pragma unroll
        for (int i = 0; i < 8; ++i) a.v[i] = __builtin_fmaf(exp_of(a.v[i], h.lse), h.weight, -gone);
        if (h.label >= 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) a.v[i] = h.label == i ? __builtin_fmaf(-e.one_minus_eps, h.weight, a.v[i]) : a.v[i];
        }
        if (h.weight == 0.f || N - n < 8) {      // ignored rows; the columns between N and the row's end are the zeros behind it
#pragma unroll
            for (int i = 0; i < 8; ++i) a.v[i] = h.weight == 0.f || n + i >= N ? 0.f : a.v[i];
        }
        store8((E*)e.out + m * e.ld_out + n, a, valid);
    } else {
        if (e.add) add8(a, h.more);
#pragma unroll
        for (int i = 0; i < 8; ++i) a.v[i] *= col.scale;
        if (e.out_f32) store8((float*)e.out + m * e.ld_out + n, a, valid);
        else store8((E*)e.out + m * e.ld_out + n, a, valid);
    }
}

// ---- the kernel -------------------------------------------------------------------------------------------------------------

// BM x BN outputs by WM x WN waves; AK / BK: the contraction is dense in the m / n operand
template <typename E, int BM, int BN, int WM, int WN, bool AK, bool BK, int KIND, int RING>
__device__ __forceinline__ void product_tile(const TileArgs& g, int block) {
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
    const int split = block / tiles;
    int id = block - split * tiles;
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
        oa.init_tail(lane, tail);
        ob.init_tail(lane, tail);
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

    // Four parts a step: the two halves of the step's contraction, and of the wave's m fragments in each.  While the matrix
    // unit works on one part, the fragments of the next one come out of LDS.  The last part is carried over the barrier: its
    // fragments are in registers by then, so the matrix unit has work while the next step's first ones arrive.  The step's
    // loads stand between the matrix instructions of the first two parts: in a row at its start they keep all waves waiting
    // for the memory unit to take them (8192 x 4096 x 2048 with 256 x 256 tiles: 125 us), behind the middle they arrive too
    // late (136 us); so 120 us, and 170 instead of 180 us for 8192 x 8192 x 2048 on zeros, where the clock is not held back.
    constexpr int H = FM / 2;
    static_assert(FM % 2 == 0, "two halves of the m fragments");
    int left = (int)(k_end - k_begin);
    i32x4 fa[2][H], fb[2][FN];
    const auto read_a = [&](const char* base, int ks, int half, i32x4* f) {
#pragma unroll
        for (int j = 0; j < H; ++j) f[j] = OpA::frag(base, (wm * FM + half * H + j) * 16, ks, lane);
    };
    const auto read_b = [&](const char* base, int ks, i32x4* f) {
#pragma unroll
        for (int i = 0; i < FN; ++i) f[i] = OpB::frag(base + BM * 128, (wn * FN + i) * 16, ks, lane);
    };
    // one half of the n fragments with one half of the m fragments
    const auto multiply = [&](int half, const i32x4* a, const i32x4* b, int part) {
#pragma unroll
        for (int i = part * FN / 2; i < (part + 1) * FN / 2; ++i)
#pragma unroll
            for (int j = 0; j < H; ++j) acc[i][half * H + j] = mma16<E>(b[i], a[j], acc[i][half * H + j]);
    };
    const unsigned lda = (unsigned)g.lda, ldb = (unsigned)g.ldb;
    constexpr int AHEAD = (RING - 2) * (OpA::PER_WAVE + OpB::PER_WAVE);
    if (left < STEP) {
        oa.mask_tail();
        ob.mask_tail();
    }
    int ahead = left;                      // what is left of the contraction where the next load starts
    unsigned into = 0, from = 0;           // stages the next load fills and the next step reads
    const auto load_a = [&]() { oa.load(pa, lda, ahead, rows_m, lds0 + into, wave); };
    const auto load_b = [&]() { ob.load(pb, ldb, ahead, rows_n, lds0 + into + BM * 128, wave); };
    const auto advance = [&]() {
        ahead -= STEP;
        pa += step_a;
        pb += step_b;
        into = into == (RING - 1) * STAGE ? 0 : into + STAGE;
        if (ahead < STEP) {
            oa.mask_tail();
            ob.mask_tail();
        }
    };
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) {
        load_a();
        load_b();
        advance();
    }
    // before the first step the carried part is zeros
#pragma unroll
    for (int j = 0; j < H; ++j) fa[1][j] = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < FN; ++i) fb[1][i] = i32x4{0, 0, 0, 0};
    stage_wait<AHEAD>();
    do {
        // this step's tiles are in LDS, and every wave is done reading the stage before it, which the next load fills
        const char* sa = smem + from;
        from = from == (RING - 1) * STAGE ? 0 : from + STAGE;
        left -= STEP;
        read_b(sa, 0, fb[0]);
        read_a(sa, 0, 0, fa[0]);
        fence();
        multiply(1, fa[1], fb[1], 0);
        fence();
        load_a();
        fence();
        multiply(1, fa[1], fb[1], 1);
        fence();
        read_a(sa, 0, 1, fa[1]);
        fence();
        multiply(0, fa[0], fb[0], 0);
        fence();
        load_b();
        fence();
        multiply(0, fa[0], fb[0], 1);
        fence();
        read_b(sa, 1, fb[1]);
        read_a(sa, 1, 0, fa[0]);
        fence();
        multiply(1, fa[1], fb[0], 0);
        multiply(1, fa[1], fb[0], 1);
        fence();
        read_a(sa, 1, 1, fa[1]);
        fence();
        multiply(0, fa[0], fb[1], 0);
        multiply(0, fa[0], fb[1], 1);
        advance();
        fence();
        stage_wait<AHEAD>();
    } while (left > 0);
    multiply(1, fa[1], fb[1], 0);
    multiply(1, fa[1], fb[1], 1);
    // zeros still on their way into LDS must not meet what the epilogue puts there
    if (AHEAD > 0) asm volatile("s_waitcnt vmcnt(0)" : : : "memory");

    const int t = lane & 15, q = lane >> 4;
    if (KIND != TILE_STATS || g.partial) {
        // The sums go through LDS, as many rows as it holds at a time, and come back as 8 neighbouring columns a thread: whole
        // lines of memory for the epilogue's loads and stores.  16-byte chunk c of staged row r at slot c ^ (r & 15).
        constexpr int HOLD = RING * STAGE / (BN * 4), ROWS = HOLD < BM ? HOLD : BM, PASSES = BM / ROWS, JP = FM / PASSES;
        constexpr int MIX = (BN / 4 < 16 ? BN / 4 : 16) - 1, GROUPS = BN / 8;
        constexpr int RSTEP = WAVES * 64 / GROUPS, BATCH = ROWS / RSTEP < 4 ? ROWS / RSTEP : 4;
        static_assert(ROWS * PASSES == BM && JP * PASSES == FM && (WAVES * 64) % GROUPS == 0 && ROWS % (RSTEP * BATCH) == 0, "rows of a pass");
        const int c = (threadIdx.x % GROUPS) * 2;
        const int64_t n = n0 + c * 4, have = (KIND == TILE_DZ ? g.e.ld_out : g.N) - n;
        const int valid = (int)(have < 0 ? 0 : have < 8 ? have : 8);
        const Columns col = load_columns<E, KIND>(g.e, g.N, n);
        Eight sums = {};
#pragma unroll
        for (int pass = 0; pass < PASSES; ++pass) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < JP; ++j) {
                const int r = (wm * JP + j) * 16 + t;
#pragma unroll
                for (int i = 0; i < FN; ++i) {
                    const int c = (wn * FN + i) * 4 + q;
                    *(f32x4*)(smem + r * (BN * 4) + (c ^ (r & MIX)) * 16) = acc[i][pass * JP + j];
                }
            }
            __syncthreads();
            // a thread keeps its columns; its rows are THREADS / GROUPS apart
#pragma unroll 1
            for (int r0 = threadIdx.x / GROUPS; r0 < ROWS; r0 += RSTEP * BATCH) {
                Ahead ahead[BATCH];
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                    const int r = r0 + k * RSTEP, in = r / (JP * 16);      // which wave row staged it
                    const int64_t m = m0 + (in * FM + pass * JP) * 16 + (r - in * JP * 16);
                    if (r < ROWS && m < g.M && valid > 0) ahead[k] = load_ahead<E, KIND>(g.e, g.N, m, n, valid);
                }
#pragma unroll
                for (int k = 0; k < BATCH; ++k) {
                    const int r = r0 + k * RSTEP, in = r / (JP * 16);
                    const int64_t m = m0 + (in * FM + pass * JP) * 16 + (r - in * JP * 16);
                    if (r >= ROWS || m >= g.M || valid <= 0) continue;
                    const f32x4 lo = *(const f32x4*)(smem + r * (BN * 4) + (c ^ (r & MIX)) * 16);
                    const f32x4 hi = *(const f32x4*)(smem + r * (BN * 4) + ((c + 1) ^ (r & MIX)) * 16);
                    Eight a = {{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}};
                    if constexpr (KIND == TILE_PARTIAL || KIND == TILE_STATS) store8(g.partial + ((int64_t)split * g.M + m) * head_partial_ld(g.N) + n, a, valid);
                    else finish8<E, KIND>(g.e, g.N, m, n, valid, col, ahead[k], a);
                    if constexpr (KIND == TILE_DZ) {
                        if (g.e.col_part) add8(sums, a);
                    }
                }
            }
        }
        if constexpr (KIND == TILE_DZ) {
            // the tile's column sums: the threads of a column in order
            if (g.e.col_part) {
                __syncthreads();
                float* share = (float*)smem;      // [RSTEP][BN]
#pragma unroll
                for (int i = 0; i < 8; ++i) share[threadIdx.x / GROUPS * BN + c * 4 + i] = sums.v[i];
                __syncthreads();
                for (int k = threadIdx.x; k < BN && n0 + k < g.N; k += WAVES * 64) {
                    float v = 0.f;
                    for (int r = 0; r < RSTEP; ++r) v += share[r * BN + k];
                    g.e.col_part[(int64_t)tm * g.N + n0 + k] = v;
                }
            }
        }
    }
    if constexpr (KIND == TILE_STATS) {
        // a row's maximum, sum and target over this tile's columns: lane, then the 4 lanes of the row, then the waves
        __syncthreads();
        float4* share = (float4*)smem;      // [WN][BM]
        const int first_n = wn * FN * 16 + 4 * q;
        if (g.e.bias) {
#pragma unroll
            for (int i = 0; i < FN; ++i) {
                const int64_t n = n0 + first_n + i * 16;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float b = n + c < g.N ? (float)((const E*)g.e.bias)[n + c] : 0.f;
#pragma unroll
                    for (int j = 0; j < FM; ++j) acc[i][j][c] += b;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < FM; ++j) {
            const int r = (wm * FM + j) * 16 + t;
            const int64_t m = m0 + r;
            float zs = 0.f;
            if (g.e.want_logit_sum) {
#pragma unroll
                for (int i = 0; i < FN; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) zs += first_n + i * 16 + c < rows_n ? acc[i][j][c] : 0.f;
                zs += __shfl_xor(zs, 16);
                zs += __shfl_xor(zs, 32);
            }
            // the label's logit: one lane of the row holds it, if this tile does
            const int64_t y = m < g.M ? g.e.target[m] - n0 - first_n : -1;
            if (y >= 0 && y < FN * 16 && (y & 15) < 4 && first_n + y < rows_n) {
                float z = 0.f;
#pragma unroll
                for (int i = 0; i < FN; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) z = y == i * 16 + c ? acc[i][j][c] : z;
                g.e.target_logit[m] = z;
            }
            if (rows_n < BN) {
#pragma unroll
                for (int i = 0; i < FN; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[i][j][c] = first_n + i * 16 + c < rows_n ? acc[i][j][c] : -__builtin_inff();
            }
            float mx = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) mx = __builtin_fmaxf(mx, acc[i][j][c]);
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16));
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32));
            // exp(z - mx); where nothing is finite the terms are exp(-inf) = 0, not exp(-inf + inf)
            const float base = mx == -__builtin_inff() ? 0.f : mx;
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < FN; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) s += exp_of(acc[i][j][c], base);
            s += __shfl_xor(s, 16);
            s += __shfl_xor(s, 32);
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
    }
}

template <typename E, int BM, int BN, int WM, int WN, bool AK, bool BK, int KIND, int RING>
__global__ __launch_bounds__(WM * WN * 64, 2) void product_tile_kernel(TileArgs g) {
    product_tile<E, BM, BN, WM, WN, AK, BK, KIND, RING>(g, blockIdx.x);
}

// Both gradients of a product in one launch, 64 x 64 tiles: the first `first` workgroups are x's (or the weight's, where
// `weight_first`).  A launch less, and the second product's tiles run while the first one's last ones do: training 1024 x 1024 ->
// 1024 takes 33 us instead of 38 in bfloat16, 77 instead of 85 in float32.
template <typename E, int KIND_X, int KIND_W>
__global__ __launch_bounds__(256, 2) void gradient_pair_kernel(TileArgs x, TileArgs w, int first, bool weight_first) {
    const int block = blockIdx.x;
    const bool early = block < first;
    if (early != weight_first) product_tile<E, 64, 64, 2, 2, true, false, KIND_X, 3>(x, early ? block : block - first);
    else product_tile<E, 64, 64, 2, 2, false, false, KIND_W, 3>(w, early ? block : block - first);
}

// ---- launch -----------------------------------------------------------------------------------------------------------------

// tile shapes: 256 x 256 by 8 waves, 128 x 128, 64 x 64, 32 x 128 (few rows) and 128 x 32 (few columns) by 4
enum { SHAPE_256 = 0, SHAPE_128 = 1, SHAPE_64 = 2, SHAPE_FEW_ROWS = 3, SHAPE_FEW_COLS = 4 };
inline void shape_size(int shape, int* bm, int* bn) {
    *bm = shape == SHAPE_256 ? 256 : shape == SHAPE_64 ? 64 : shape == SHAPE_FEW_ROWS ? 32 : 128;
    *bn = shape == SHAPE_256 ? 256 : shape == SHAPE_64 ? 64 : shape == SHAPE_FEW_COLS ? 32 : 128;
}

template <typename E, int BM, int BN, int WM, int WN, bool AK, bool BK, int KIND, int RING>
hipError_t launch_one(const TileArgs& g, hipStream_t s) {
    constexpr int lds = RING * (BM + BN) * 128;
    const auto kern = product_tile_kernel<E, BM, BN, WM, WN, AK, BK, KIND, RING>;
    if (lds > 65536) {
        const hipError_t e = set_max_lds_once((const void*)kern, lds);
        if (e != hipSuccess) return e;
    }
    kern<<<(unsigned)(g.tiles_m * g.tiles_n * g.splits), WM * WN * 64, lds, s>>>(g);
    return hipGetLastError();
}

template <typename E, bool AK, bool BK, int KIND>
hipError_t launch_shape(int shape, const TileArgs& g, hipStream_t s) {
    switch (shape) {
        case SHAPE_256:
            // floats need no larger tile than 128: their matrix instructions take eight times as long over what LDS delivers
            if constexpr (sizeof(E) == 2) return launch_one<E, 256, 256, 2, 4, AK, BK, KIND, 2>(g, s);
            return hipErrorInvalidValue;
        case SHAPE_128:
            // alone on its compute unit a tile waits for its loads: one more stage (0.65 instead of 0.90 us a step); two to a
            // unit cover each other and would not fit with three stages
            if (sizeof(E) == 2 && g.tiles_m * g.tiles_n * g.splits <= 256) return launch_one<E, 128, 128, 2, 2, AK, BK, KIND, 3>(g, s);
            return launch_one<E, 128, 128, 2, 2, AK, BK, KIND, 2>(g, s);
        case SHAPE_64: return launch_one<E, 64, 64, 2, 2, AK, BK, KIND, 3>(g, s);
        case SHAPE_FEW_ROWS: return launch_one<E, 32, 128, 1, 4, AK, BK, KIND, 3>(g, s);
        default: return launch_one<E, 128, 32, 4, 1, AK, BK, KIND, 3>(g, s);
    }
}

// forward products and logits: both operands dense in the contraction; dx: the second one transposed; dW: both
template <typename E>
hipError_t launch_tile(int shape, int kind, bool ak, bool bk, const TileArgs& g, hipStream_t s) {
    if (ak && bk) {
        switch (kind) {
            case TILE_LINEAR: return launch_shape<E, true, true, TILE_LINEAR>(shape, g, s);
            case TILE_DZ: return launch_shape<E, true, true, TILE_DZ>(shape, g, s);
            case TILE_STATS: return launch_shape<E, true, true, TILE_STATS>(shape, g, s);
            case TILE_PARTIAL: return launch_shape<E, true, true, TILE_PARTIAL>(shape, g, s);
        }
    } else if (ak && !bk) {
        switch (kind) {
            case TILE_SCALED: return launch_shape<E, true, false, TILE_SCALED>(shape, g, s);
            case TILE_PARTIAL: return launch_shape<E, true, false, TILE_PARTIAL>(shape, g, s);
        }
    } else if (!ak && !bk) {
        switch (kind) {
            case TILE_SCALED: return launch_shape<E, false, false, TILE_SCALED>(shape, g, s);
            case TILE_PARTIAL: return launch_shape<E, false, false, TILE_PARTIAL>(shape, g, s);
        }
    }
    return hipErrorInvalidValue;
}

// x's and the weight's gradient, both in 64 x 64 tiles; the one whose tiles take more steps first
template <typename E>
hipError_t launch_pair(const TileArgs& x, const TileArgs& w, hipStream_t s) {
    constexpr int lds = 3 * 128 * 128;
    const int nx = x.tiles_m * x.tiles_n * x.splits, nw = w.tiles_m * w.tiles_n * w.splits;
    const bool weight_first = w.k_split > x.k_split;
    const int first = weight_first ? nw : nx;
#define PNGPD_PAIR(KX, KW) gradient_pair_kernel<E, KX, KW><<<(unsigned)(nx + nw), 256, lds, s>>>(x, w, first, weight_first)
    if (x.splits > 1) {
        if (w.splits > 1) PNGPD_PAIR(TILE_PARTIAL, TILE_PARTIAL);
        else PNGPD_PAIR(TILE_PARTIAL, TILE_SCALED);
    } else {
        if (w.splits > 1) PNGPD_PAIR(TILE_SCALED, TILE_PARTIAL);
        else PNGPD_PAIR(TILE_SCALED, TILE_SCALED);
    }
#undef PNGPD_PAIR
    return hipGetLastError();
}

hipError_t launch_pair_f32(const TileArgs& x, const TileArgs& w, hipStream_t s);
hipError_t launch_pair_bf16(const TileArgs& x, const TileArgs& w, hipStream_t s);
hipError_t launch_pair_f16(const TileArgs& x, const TileArgs& w, hipStream_t s);
hipError_t launch_tile_f32(int shape, int kind, bool ak, bool bk, const TileArgs& g, hipStream_t s);
hipError_t launch_tile_bf16(int shape, int kind, bool ak, bool bk, const TileArgs& g, hipStream_t s);
hipError_t launch_tile_f16(int shape, int kind, bool ak, bool bk, const TileArgs& g, hipStream_t s);

}  // namespace pngpd
