// The loss of linear_cross_entropy from the rows' statistics (the products are head_product.hip's).
//
// A block of columns leaves a row's maximum m, sum s of exp(z - m) and sum of z; blocks join by
// s = s1 exp(m1 - m) + s2 exp(m2 - m) under m = max(m1, m2).  Bound by their launches: 4096 rows of 128 blocks (8 MB) take
// 12 us, the batch's sum over them 5 us.
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

__device__ __forceinline__ float loss_of_row(const float4& v, int64_t t, int64_t V, const float* target_logit, const int64_t* target,
                                             int64_t ignore, float eps, float* lse) {
    const float l = v.x + logf(v.y);
    lse[t] = l;
    const int64_t y = target[t];
    if (y == ignore) return 0.f;
    float x = y >= 0 && y < V ? l - (1.f - eps) * target_logit[t] : __builtin_nanf("");
    if (eps > 0.f) x -= eps / (float)V * v.z;
    return x;
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
    loss[t] = loss_of_row(share[r], t, V, target_logit, target, ignore, eps, lse);
}

// the batch's loss: one workgroup, sums over the rows in 64 bits
__device__ __forceinline__ void batch_sum(double sum, double used, int reduction, float* loss, float* count_out) {
    __shared__ double part[16], count[16];
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
        if (count_out) count_out[0] = (float)used;
    }
}

__global__ __launch_bounds__(1024) void batch_loss_kernel(int64_t T, const float* row_loss, const int64_t* target, int64_t ignore,
                                                          int reduction, float* loss, float* count) {
    double sum = 0, used = 0;
#pragma unroll 8
    for (int64_t t = threadIdx.x; t < T; t += 1024) {
        sum += row_loss[t];
        used += target[t] != ignore;
    }
    batch_sum(sum, used, reduction, loss, count);
}

// Many rows: runs of them by a workgroup each, then their sums by one (65536 x 64 -> 3 training in bfloat16 44 -> 38 us, scoring
// 2^20 x 16 -> 3 280 -> 129 us).
constexpr int64_t BATCH_ALONE = 16384, BATCH_PARTS = 256;
inline int64_t rows_of_part(int64_t T) { return T <= 4096 * BATCH_PARTS ? 4096 : (T + BATCH_PARTS - 1) / BATCH_PARTS; }

__global__ __launch_bounds__(256) void loss_parts_kernel(int64_t T, int64_t rows, const float* row_loss, const int64_t* target,
                                                         int64_t ignore, double2* parts) {
    __shared__ double2 share[4];
    const int64_t first = blockIdx.x * rows, last = first + rows < T ? first + rows : T;
    double sum = 0, used = 0;
#pragma unroll 8
    for (int64_t t = first + threadIdx.x; t < last; t += 256) {
        sum += row_loss[t];
        used += target[t] != ignore;
    }
    for (int o = 32; o; o >>= 1) {
        sum += __shfl_xor(sum, o);
        used += __shfl_xor(used, o);
    }
    if ((threadIdx.x & 63) == 0) share[threadIdx.x >> 6] = make_double2(sum, used);
    __syncthreads();
    if (threadIdx.x == 0)
        parts[blockIdx.x] = make_double2(share[0].x + share[1].x + share[2].x + share[3].x, share[0].y + share[1].y + share[2].y + share[3].y);
}
__global__ __launch_bounds__(1024) void join_loss_kernel(int n, const double2* parts, int reduction, float* loss, float* count) {
    const double2 v = (int)threadIdx.x < n ? parts[threadIdx.x] : make_double2(0, 0);
    batch_sum(v.x, v.y, reduction, loss, count);
}

// rows' losses and the batch's for a small batch: a thread a row
__global__ __launch_bounds__(1024) void small_loss_kernel(int T, int64_t V, int blocks, const float4* stats, const float* target_logit,
                                                          const int64_t* target, int64_t ignore, float eps, int reduction, float* loss,
                                                          float* lse) {
    const int t = threadIdx.x;
    double sum = 0, used = 0;
    if (t < T) {
        float4 v = stats[t];
        for (int i = 1; i < blocks; ++i) join_stats(v, stats[(int64_t)i * T + t]);
        sum = loss_of_row(v, t, V, target_logit, target, ignore, eps, lse);
        used = target[t] != ignore;
    }
    batch_sum(sum, used, reduction, loss, nullptr);
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

bool head_loss_at_once(int64_t T, int blocks) { return T <= 1024 && blocks <= 8; }

hipError_t head_row_loss(int64_t T, int64_t V, int blocks, const float4* stats, const float* target_logit, const int64_t* target,
                         int64_t ignore, float eps, float* row_loss, float* lse, int reduction, float* batch, hipStream_t s) {
    if (batch && head_loss_at_once(T, blocks)) {
        small_loss_kernel<<<1, 1024, 0, s>>>((int)T, V, blocks, stats, target_logit, target, ignore, eps, reduction, batch, lse);
        return hipGetLastError();
    }
    int lanes = 5;                                       // few rows: more threads a row
    while (lanes > 0 && (T >> lanes) < 64 && (256 >> lanes) < blocks) --lanes;
    const int rows = 1 << lanes;
    row_loss_kernel<<<(unsigned)((T + rows - 1) / rows), 256, 0, s>>>(T, V, blocks, stats, target_logit, target, ignore, eps, lanes,
                                                                       row_loss, lse);
    return hipGetLastError();
}

int64_t head_batch_parts(int64_t T) { return T <= BATCH_ALONE ? 0 : (T + rows_of_part(T) - 1) / rows_of_part(T); }

hipError_t head_batch_loss(int64_t T, const float* row_loss, const int64_t* target, int64_t ignore, int reduction, float* loss,
                           float* used, double2* parts, hipStream_t s) {
    if (const int64_t n = head_batch_parts(T)) {
        loss_parts_kernel<<<(unsigned)n, 256, 0, s>>>(T, rows_of_part(T), row_loss, target, ignore, parts);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        join_loss_kernel<<<1, 1024, 0, s>>>((int)n, parts, reduction, loss, used);
        return hipGetLastError();
    }
    batch_loss_kernel<<<1, 1024, 0, s>>>(T, row_loss, target, ignore, reduction, loss, used);
    return hipGetLastError();
}

}  // namespace pngpd
