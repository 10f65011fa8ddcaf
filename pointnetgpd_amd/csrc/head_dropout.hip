// Dropout whose mask is a function of (seed, offset, position) and is never stored.
//
//   key = mix64(seed ^ mix64(offset)),  word(j) = mix64(key + j),  draw(i) = 32-bit half (i & 1) of word(i >> 1)
//   y[i] = residual[i] + (draw(i) >= round(p 2^32) ? x[i] / (1 - p) : 0),  i = position in row-major order
//
// The hash is the one the point selection uses (crop_select.h), one evaluation for two elements.  A dropped element is
// selected away, not multiplied: infinities and NaN in dropped places do not reach the result.
//
// Bound by memory, with eight neighbouring elements a thread: their four hashes hide behind its 16-byte accesses (an element
// a thread: 294 us).  16384 x 4096 in bfloat16: forward with its residual (403 MB) 73 us, backward without one (268 MB)
// 47 us, together 5.6 TB/s; 51 us for the latter where the input changes from call to call.
#include "crop_select.h"
#include "head.h"
#include "head_math.h"

namespace pngpd {
namespace {

constexpr int PER_THREAD = 8;      // neighbouring elements: 4 hashes, 16 bytes of a 16-bit type

template <typename T>
struct Eight {
    static constexpr int C = 16 / sizeof(T);
    typedef __attribute__((ext_vector_type(16 / sizeof(T)))) T chunk;
    T v[PER_THREAD];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int k = 0; k < PER_THREAD / C; ++k) {
            chunk c;
            __builtin_memcpy(&c, p + k * C, 16);      // at any element: the hardware takes it
#pragma unroll
            for (int i = 0; i < C; ++i) v[k * C + i] = c[i];
        }
    }
    __device__ __forceinline__ void store(T* p) const {
#pragma unroll
        for (int k = 0; k < PER_THREAD / C; ++k) {
            chunk c;
#pragma unroll
            for (int i = 0; i < C; ++i) c[i] = v[k * C + i];
            __builtin_memcpy(p + k * C, &c, 16);
        }
    }
};

// DENSE: x and the residual are one run of memory as y is
template <typename T, bool DENSE, bool RESIDUAL>
__device__ __forceinline__ void dropout_eight(int64_t i0, int64_t total, int64_t cols, const T* x, int64_t ldx, const T* r, int64_t ldr,
                                              T* y, unsigned long long border, float scale, unsigned long long key) {
    Eight<T> a, b;
    int64_t m = DENSE ? 0 : i0 / cols, n = i0 - m * cols;
    const bool whole = i0 + PER_THREAD <= total;
    if (whole && (DENSE || n + PER_THREAD <= cols)) {
        a.load(x + m * ldx + n);
        if (RESIDUAL) b.load(r + m * ldr + n);
    } else {
#pragma unroll
        for (int k = 0; k < PER_THREAD; ++k) {
            const bool there = i0 + k < total;
            a.v[k] = there ? x[DENSE ? i0 + k : m * ldx + n] : (T)0.f;
            if (RESIDUAL) b.v[k] = there ? r[DENSE ? i0 + k : m * ldr + n] : (T)0.f;
            if (++n == cols && !DENSE) {
                n = 0;
                ++m;
            }
        }
    }
    const unsigned long long first = key + (unsigned long long)(i0 >> 1);
#pragma unroll
    for (int k = 0; k < PER_THREAD; k += 2) {
        const unsigned long long w = mix64(first + (k >> 1));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const unsigned draw = h ? (unsigned)(w >> 32) : (unsigned)w;
            float v = (unsigned long long)draw >= border ? to_f32(a.v[k + h]) * scale : 0.f;
            if (RESIDUAL) v += to_f32(b.v[k + h]);
            a.v[k + h] = from_f32<T>(v);
        }
    }
    if (whole) {
        a.store(y + i0);
    } else {
#pragma unroll
        for (int k = 0; k < PER_THREAD; ++k)
            if (i0 + k < total) y[i0 + k] = a.v[k];
    }
}

template <typename T, bool DENSE, bool RESIDUAL>
__global__ __launch_bounds__(256) void dropout_kernel(int64_t total, int64_t cols, const T* x, int64_t ldx, const T* r, int64_t ldr,
                                                      T* y, unsigned long long border, float scale, unsigned long long seed,
                                                      unsigned long long offset, const int64_t* rng) {
    if (rng) {
        seed = (unsigned long long)rng[0];
        offset = (unsigned long long)rng[1];
    }
    const unsigned long long key = mix64(seed ^ mix64(offset));
    // one turn, unless the grid's 2^31 threads are not enough
    for (int64_t i0 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * PER_THREAD; i0 < total;
         i0 += (int64_t)gridDim.x * 256 * PER_THREAD)
        dropout_eight<T, DENSE, RESIDUAL>(i0, total, cols, x, ldx, r, ldr, y, border, scale, key);
}

template <typename T>
hipError_t launch(int64_t rows, int64_t cols, const void* x, int64_t ldx, const void* r, int64_t ldr, void* y, double p,
                  uint64_t seed, uint64_t offset, const int64_t* rng, hipStream_t s) {
    const int64_t total = rows * cols;
    const int64_t blocks = (total + 256 * PER_THREAD - 1) / (256 * PER_THREAD);
    const unsigned grid = (unsigned)(blocks < (1 << 23) ? blocks : 1 << 23);
    const unsigned long long border = (unsigned long long)__builtin_rint(p * 4294967296.0);
    const float scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f;
    auto run_of = [&](int64_t ld) { return ld == cols || rows == 1; };
    const bool dense = run_of(ldx) && (!r || run_of(ldr));
#define PNGPD_DROPOUT(D, R) \
    dropout_kernel<T, D, R><<<grid, 256, 0, s>>>(total, cols, (const T*)x, ldx, (const T*)r, ldr, (T*)y, border, scale, seed, offset, rng)
    if (dense && r) PNGPD_DROPOUT(true, true);
    else if (dense) PNGPD_DROPOUT(true, false);
    else if (r) PNGPD_DROPOUT(false, true);
    else PNGPD_DROPOUT(false, false);
#undef PNGPD_DROPOUT
    return hipGetLastError();
}

}  // namespace

hipError_t head_dropout(int type, int64_t rows, int64_t cols, const void* x, int64_t ldx, const void* r, int64_t ldr, void* y,
                        double p, uint64_t seed, uint64_t offset, const int64_t* rng, hipStream_t s) {
    switch (type) {
        case PNGPD_TYPE_F32: return launch<float>(rows, cols, x, ldx, r, ldr, y, p, seed, offset, rng, s);
        case PNGPD_TYPE_BF16: return launch<bf16_t>(rows, cols, x, ldx, r, ldr, y, p, seed, offset, rng, s);
        case PNGPD_TYPE_F16: return launch<f16_t>(rows, cols, x, ldx, r, ldr, y, p, seed, offset, rng, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace pngpd
