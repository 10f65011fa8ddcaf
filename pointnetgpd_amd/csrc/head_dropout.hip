// Dropout whose mask is a function of (seed, offset, position) and is never stored.
//
//   key = mix64(seed ^ mix64(offset)),  word(j) = mix64(key + j),  draw(i) = 32-bit half (i & 1) of word(i >> 1)
//   y[i] = residual[i] + (draw(i) >= round(p 2^32) ? x[i] / (1 - p) : 0),  i = position in row-major order
//
// The hash is the one the point selection uses (crop_select.h), one evaluation for two elements.  A dropped element is
// selected away, not multiplied: infinities and NaN in dropped places do not reach the result.
#include "crop_select.h"
#include "head.h"
#include "head_math.h"

namespace pngpd {
namespace {

template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(int64_t rows, int64_t cols, const T* x, int64_t ldx, const T* r, int64_t ldr,
                                                      T* y, unsigned long long border, float scale, unsigned long long seed,
                                                      unsigned long long offset, const int64_t* rng) {
    if (rng) {
        seed = (unsigned long long)rng[0];
        offset = (unsigned long long)rng[1];
    }
    const unsigned long long key = mix64(seed ^ mix64(offset));
    const int64_t total = rows * cols, pairs = (total + 1) / 2;
    for (int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x; j < pairs; j += (int64_t)gridDim.x * 256) {
        const unsigned long long w = mix64(key + (unsigned long long)j);
        for (int h = 0; h < 2; ++h) {
            const int64_t i = 2 * j + h;
            if (i >= total) break;
            const int64_t m = i / cols, n = i - m * cols;
            const bool keep = (h ? w >> 32 : w & 0xffffffffull) >= border;
            float v = keep ? to_f32(x[m * ldx + n]) * scale : 0.f;
            if (r) v += to_f32(r[m * ldr + n]);
            y[i] = from_f32<T>(v);
        }
    }
}

template <typename T>
hipError_t launch(int64_t rows, int64_t cols, const void* x, int64_t ldx, const void* r, int64_t ldr, void* y, double p,
                  uint64_t seed, uint64_t offset, const int64_t* rng, hipStream_t s) {
    const int64_t blocks = (rows * cols + 511) / 512;
    const unsigned grid = (unsigned)(blocks < 16384 ? blocks : 16384);
    const unsigned long long border = (unsigned long long)__builtin_rint(p * 4294967296.0);
    const float scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f;
    dropout_kernel<T><<<grid, 256, 0, s>>>(rows, cols, (const T*)x, ldx, (const T*)r, ldr, (T*)y, border, scale, seed, offset, rng);
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
