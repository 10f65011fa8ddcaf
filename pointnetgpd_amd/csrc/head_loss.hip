// Loss and gradient weights of linear_cross_entropy from the rows' statistics (the products are head_product.hip's).
//
// A block of columns leaves a row's maximum m, sum s of exp(z - m) and sum of z; blocks join by
// s = s1 exp(m1 - m) + s2 exp(m2 - m) under m = max(m1, m2).
#include "head.h"
#include "head_math.h"

namespace pngpd {
namespace {

__device__ __forceinline__ void join_stats(float4& v, const float4& u) {
    const float m = __builtin_fmaxf(v.x, u.x);
    v.y = v.y * (v.x == m ? 1.f : __expf(v.x - m)) + u.y * (u.x == m ? 1.f : __expf(u.x - m));
    v.x = m;
    v.z += u.z;
}

// 2^lanes rows a workgroup, the other threads side by side over a row's blocks; then the threads of a row in order
__global__ __launch_bounds__(256) void row_loss_kernel(int64_t T, int64_t V, int blocks, const float4* stats, const float* target_logit,
                                                       const int64_t* target, int64_t ignore, float eps, int lanes, float* loss, float* lse) {
    __shared__ float4 share[256];
    const int rows = 1 << lanes, r = threadIdx.x & (rows - 1), part = threadIdx.x >> lanes, shares = 256 >> lanes;
    const int64_t t = (int64_t)blockIdx.x * rows + r;
    float4 v = make_float4(-__builtin_inff(), 0.f, 0.f, 0.f);
    if (t < T)
        for (int i = part; i < blocks; i += shares) join_stats(v, stats[(int64_t)i * T + t]);
    share[threadIdx.x] = v;
    __syncthreads();
    for (int step = shares / 2; step; step >>= 1) {
        if (part < step) join_stats(share[threadIdx.x], share[threadIdx.x + (step << lanes)]);
        __syncthreads();
    }
    if (part || t >= T) return;
    v = share[r];
    const float l = v.x + logf(v.y);
    lse[t] = l;
    const int64_t y = target[t];
    float x = 0.f;
    if (y != ignore) {
        x = y >= 0 && y < V ? l - (1.f - eps) * target_logit[t] : __builtin_nanf("");
        if (eps > 0.f) x -= eps / (float)V * v.z;
    }
    loss[t] = x;
}

// the batch's loss: one workgroup, sums over the rows in 64 bits
__global__ __launch_bounds__(1024) void batch_loss_kernel(int64_t T, const float* row_loss, const int64_t* target, int64_t ignore,
                                                          int reduction, float* loss) {
    __shared__ double part[16], count[16];
    double sum = 0, used = 0;
#pragma unroll 8
    for (int64_t t = threadIdx.x; t < T; t += 1024) {
        sum += row_loss[t];
        used += target[t] != ignore;
    }
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
#pragma unroll 8
    for (int64_t t = threadIdx.x; t < T; t += 1024) {
        const int64_t y = target[t];
        used += y != ignore ? 1.f : 0.f;
        if (reduction == PNGPD_REDUCE_NONE) g = __builtin_fmaxf(g, y != ignore && y >= 0 && y < V ? __builtin_fabsf(dloss[t]) : 0.f);
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
    // half precision: the largest weight becomes 2^13 .. 2^14, |dz| <= 2 times that is inside its range, and a probability of
    // 2^-37 still is a number
    if (reduction != PNGPD_REDUCE_NONE) {
        // One weight for all rows stays out of dz and goes into the products' 32-bit sums: p - 1 of the labels would be rounded
        // the same way in every row otherwise (off by up to 2^-9 in one direction in bfloat16).
        const float unit = scaled ? 16384.f : 1.f;
        for (int64_t t = threadIdx.x; t < T; t += 1024) weight[t] = target[t] != ignore && target[t] >= 0 && target[t] < V ? unit : 0.f;
        if (threadIdx.x == 0) out_scale[0] = dloss[0] * (reduction == PNGPD_REDUCE_MEAN ? 1.f / __builtin_fmaxf(used, 1.f) : 1.f) / unit;
        return;
    }
    float scale = 1.f;
    if (scaled && g > 0.f && g < __builtin_inff()) {
        int e;
        (void)frexpf(g, &e);
        scale = ldexpf(1.f, e - 14);
    }
    for (int64_t t = threadIdx.x; t < T; t += 1024) {
        const bool live = target[t] != ignore && target[t] >= 0 && target[t] < V;
        weight[t] = live ? dloss[t] / scale : 0.f;
    }
    if (threadIdx.x == 0) out_scale[0] = scale;
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

hipError_t head_row_loss(int64_t T, int64_t V, int blocks, const float4* stats, const float* target_logit, const int64_t* target,
                         int64_t ignore, float eps, float* row_loss, float* lse, hipStream_t s) {
    int lanes = 5;                                       // few rows: more threads a row
    while (lanes > 0 && (T >> lanes) < 64 && (256 >> lanes) < blocks) --lanes;
    const int rows = 1 << lanes;
    row_loss_kernel<<<(unsigned)((T + rows - 1) / rows), 256, 0, s>>>(T, V, blocks, stats, target_logit, target, ignore, eps, lanes,
                                                                       row_loss, lse);
    return hipGetLastError();
}

hipError_t head_batch_loss(int64_t T, const float* row_loss, const int64_t* target, int64_t ignore, int reduction, float* loss,
                           hipStream_t s) {
    batch_loss_kernel<<<1, 1024, 0, s>>>(T, row_loss, target, ignore, reduction, loss);
    return hipGetLastError();
}

hipError_t head_row_weights(int type, int64_t T, int64_t V, const int64_t* target, int64_t ignore, int reduction,
                            const float* dloss, float* weight, float* out_scale, hipStream_t s) {
    row_weights_kernel<<<1, 1024, 0, s>>>(type == PNGPD_TYPE_F16, T, V, target, ignore, reduction, dloss, weight, out_scale);
    return hipGetLastError();
}

}  // namespace pngpd
