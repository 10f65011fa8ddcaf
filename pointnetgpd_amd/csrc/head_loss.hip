// Row statistics, loss and gradient weights of linear_cross_entropy (the products are head_product.hip's).
//
// A row's statistics run over the pieces of the vocabulary: maximum m, sum s of exp(z - m), the target's logit and, for
// label smoothing, the sum of the logits.  A piece joins them with  s <- s exp(m - m') + s_piece exp(m_piece - m').
#include "head.h"
#include "head_math.h"

namespace pngpd {
namespace {

// exp(v - m) for a running maximum that may be -inf (nothing finite seen yet): -inf - -inf counts as "no term"
__device__ __forceinline__ float exp_under(float v, float m) { return v == -__builtin_inff() ? 0.f : expf(v - m); }

// one wave a row
__global__ __launch_bounds__(256) void stats_piece_kernel(int64_t T, int64_t n, const float* logits, int64_t ld, int64_t first_n,
                                                          const int64_t* target, HeadRowStats st, bool first) {
    const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= T) return;
    const int lane = threadIdx.x & 63;
    const float* z = logits + t * ld;
    float m = -__builtin_inff(), zs = 0.f;
    for (int64_t i = lane; i < n; i += 64) {
        m = __builtin_fmaxf(m, z[i]);
        zs += z[i];
    }
    m = wave_max(m);
    zs = wave_sum(zs);
    float s = 0.f;
    for (int64_t i = lane; i < n; i += 64) s += exp_under(z[i], m);
    s = wave_sum(s);
    if (lane == 0) {
        const int64_t y = target[t] - first_n;
        if (y >= 0 && y < n) st.target_logit[t] = z[y];
        else if (first) st.target_logit[t] = __builtin_nanf("");      // stays so if no piece holds the label
        if (first) {
            st.max[t] = m;
            st.sum[t] = s;
            st.logit_sum[t] = zs;
        } else {
            const float m0 = st.max[t], m1 = __builtin_fmaxf(m0, m);
            st.sum[t] = st.sum[t] * (m0 == m1 ? 1.f : exp_under(m0, m1)) + s * (m == m1 ? 1.f : exp_under(m, m1));
            st.max[t] = m1;
            st.logit_sum[t] += zs;
        }
    }
}

// loss of every row, and of the batch: one workgroup, sums over the rows in 64 bits
__global__ __launch_bounds__(1024) void loss_finish_kernel(int64_t T, int64_t V, const int64_t* target, int64_t ignore, float eps,
                                                           int reduction, HeadRowStats st, float* loss, float* lse) {
    __shared__ double part[16], count[16];
    double sum = 0, used = 0;
    for (int64_t t = threadIdx.x; t < T; t += 1024) {
        const float l = st.max[t] + logf(st.sum[t]);
        lse[t] = l;
        float v = 0.f;
        if (target[t] != ignore) {
            v = l - (1.f - eps) * st.target_logit[t];
            if (eps > 0.f) v -= eps / (float)V * st.logit_sum[t];
            used += 1;
        }
        if (reduction == PNGPD_REDUCE_NONE) loss[t] = v;
        sum += v;
    }
    if (reduction == PNGPD_REDUCE_NONE) return;
    for (int o = 32; o; o >>= 1) {
        sum += __shfl_xor(sum, o);
        used += __shfl_xor(used, o);
    }
    if ((threadIdx.x & 63) == 0) {
        part[threadIdx.x >> 6] = sum;
        count[threadIdx.x >> 6] = used;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) {
            sum += part[i];
            used += count[i];
        }
        loss[0] = (float)(reduction == PNGPD_REDUCE_MEAN ? sum / used : sum);
    }
}

__global__ __launch_bounds__(1024) void row_weights_kernel(bool scaled, int64_t T, int64_t V, const int64_t* target, int64_t ignore,
                                                           int reduction, const float* dloss, float* weight, float* out_scale) {
    __shared__ float count[16], top[16];
    float used = 0.f, g = 0.f;
    for (int64_t t = threadIdx.x; t < T; t += 1024) {
        if (target[t] == ignore) continue;
        used += 1.f;
        if (target[t] >= 0 && target[t] < V) g = __builtin_fmaxf(g, __builtin_fabsf(dloss[reduction == PNGPD_REDUCE_NONE ? t : 0]));
    }
    used = wave_sum(used);
    g = wave_max(g);
    if ((threadIdx.x & 63) == 0) {
        count[threadIdx.x >> 6] = used;
        top[threadIdx.x >> 6] = g;
    }
    __syncthreads();
    used = 0.f;
    g = 0.f;
    for (int i = 0; i < 16; ++i) {
        used += count[i];
        g = __builtin_fmaxf(g, top[i]);
    }
    const float share = reduction == PNGPD_REDUCE_MEAN ? 1.f / used : 1.f;
    float scale = 1.f;
    if (scaled && g * share > 0.f && g * share < __builtin_inff()) {
        // the largest weight becomes 2^13 .. 2^14: |dz| <= 2 times that, inside half precision's range, and a
        // probability of 2^-37 still is a number
        int e;
        (void)frexpf(g * share, &e);
        scale = ldexpf(1.f, e - 14);
    }
    for (int64_t t = threadIdx.x; t < T; t += 1024) {
        const bool live = target[t] != ignore && target[t] >= 0 && target[t] < V;
        weight[t] = live ? dloss[reduction == PNGPD_REDUCE_NONE ? t : 0] * share / scale : 0.f;
    }
    if (threadIdx.x == 0) out_scale[0] = scale;
}

template <typename T>
__global__ __launch_bounds__(256) void live_rows_kernel(int64_t rows, int64_t D, const T* x, int64_t ldx, const float* weight,
                                                        T* out) {
    const int64_t total = rows * D;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t t = i / D, d = i - t * D;
        out[i] = weight[t] != 0.f ? x[t * ldx + d] : (T)0.f;
    }
}

// bytes: an even number (every element type has at least two)
__global__ __launch_bounds__(256) void zero_kernel(unsigned short* p, size_t n) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) p[i] = 0;
}

}  // namespace

hipError_t head_zero(void* p, size_t bytes, hipStream_t s) {
    const size_t n = bytes / 2, blocks = (n + 255) / 256;
    zero_kernel<<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, s>>>((unsigned short*)p, n);
    return hipGetLastError();
}

hipError_t head_live_rows(int type, int64_t T, int64_t D, const void* x, int64_t ldx, const float* weight, void* out,
                          hipStream_t s) {
    const int64_t blocks = (T * D + 255) / 256;
    const unsigned grid = (unsigned)(blocks < 16384 ? blocks : 16384);
    if (type == PNGPD_TYPE_F32) live_rows_kernel<float><<<grid, 256, 0, s>>>(T, D, (const float*)x, ldx, weight, (float*)out);
    else live_rows_kernel<bf16_t><<<grid, 256, 0, s>>>(T, D, (const bf16_t*)x, ldx, weight, (bf16_t*)out);      // 16-bit copies
    return hipGetLastError();
}

hipError_t head_stats_piece(int64_t T, int64_t n, const float* logits, int64_t ld, int64_t first_n, const int64_t* target,
                            const HeadRowStats& st, bool first, hipStream_t s) {
    stats_piece_kernel<<<(unsigned)((T + 3) / 4), 256, 0, s>>>(T, n, logits, ld, first_n, target, st, first);
    return hipGetLastError();
}

hipError_t head_loss_finish(int64_t T, int64_t V, const int64_t* target, int64_t ignore, float eps, int reduction,
                            const HeadRowStats& st, float* loss, float* lse, hipStream_t s) {
    loss_finish_kernel<<<1, 1024, 0, s>>>(T, V, target, ignore, eps, reduction, st, loss, lse);
    return hipGetLastError();
}

hipError_t head_row_weights(int type, int64_t T, int64_t V, const int64_t* target, int64_t ignore, int reduction,
                            const float* dloss, float* weight, float* out_scale, hipStream_t s) {
    row_weights_kernel<<<1, 1024, 0, s>>>(type == PNGPD_TYPE_F16, T, V, target, ignore, reduction, dloss, weight, out_scale);
    return hipGetLastError();
}

}  // namespace pngpd
