// Products of the classification head: out[m][n] = epilogue(sum_k A(m,k) B(n,k)).
//
// One tile of 64 x 64 outputs per workgroup of 256 threads, 4 x 4 outputs a thread, the contraction in steps of 16
// through LDS, sums as 32-bit fma chains.  Any stride, any alignment, both operand orders.
#include "head.h"
#include "head_math.h"

namespace pngpd {
namespace {

constexpr int TM = 64, TN = 64, TK = 16;

template <typename T, int ACT>
__device__ __forceinline__ void store_out(const HeadEpilogue& e, int64_t N, int64_t m, int64_t n, float acc) {
    float v;
    if (e.kind == HEAD_EPI_LINEAR) {
        const float z = acc + (e.bias ? to_f32(((const T*)e.bias)[n]) : 0.f);
        if (e.z) ((T*)e.z)[m * N + n] = keep_z<T, ACT>(z);
        v = act_f<ACT>(z);
        if (e.residual) v += to_f32(((const T*)e.residual)[m * e.ld_residual + n]);
    } else if (e.kind == HEAD_EPI_DZ) {
        const float w = e.row_weight[m];
        const float z = acc + (e.bias ? to_f32(((const T*)e.bias)[n]) : 0.f);
        const float p = expf(z - e.lse[m]) - e.smooth;
        v = w == 0.f ? 0.f : (p - (e.target[m] == n + e.first_n ? e.one_minus_eps : 0.f)) * w;
    } else {
        v = (acc + (e.add ? e.add[m * N + n] : 0.f)) * (e.scale ? e.scale[0] : 1.f);
    }
    if (e.out_f32) ((float*)e.out)[m * e.ld_out + n] = e.kind == HEAD_EPI_SCALED ? v : acc + (e.bias ? to_f32(((const T*)e.bias)[n]) : 0.f);
    else ((T*)e.out)[m * e.ld_out + n] = from_f32<T>(v);
}

template <typename T, int ACT>
__global__ __launch_bounds__(256) void product_simple_kernel(int64_t M, int64_t N, int64_t K, HeadOperand a, HeadOperand b,
                                                             HeadEpilogue e) {
    __shared__ float sa[TK][TM + 1], sb[TK][TN + 1];
    const int64_t m0 = (int64_t)blockIdx.y * TM, n0 = (int64_t)blockIdx.x * TN;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < K; k0 += TK) {
        for (int i = threadIdx.x; i < TM * TK; i += 256) {
            int r = a.k_contiguous ? i / TK : i % TM, k = a.k_contiguous ? i % TK : i / TM;
            const int64_t gm = m0 + r, gk = k0 + k;
            sa[k][r] = gm < M && gk < K ? to_f32(((const T*)a.p)[a.k_contiguous ? gm * a.ld + gk : gk * a.ld + gm]) : 0.f;
            r = b.k_contiguous ? i / TK : i % TN, k = b.k_contiguous ? i % TK : i / TN;
            const int64_t gn = n0 + r, hk = k0 + k;
            sb[k][r] = gn < N && hk < K ? to_f32(((const T*)b.p)[b.k_contiguous ? gn * b.ld + hk : hk * b.ld + gn]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < TK; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_fmaf(sa[k][ty + 16 * i], sb[k][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
            if (m < M && n < N) store_out<T, ACT>(e, N, m, n, acc[i][j]);
        }
}

template <typename T>
hipError_t launch(int64_t M, int64_t N, int64_t K, const HeadOperand& a, const HeadOperand& b, const HeadEpilogue& e,
                  hipStream_t s) {
    // at most 65535 tiles of rows in one launch
    const int64_t rows = (int64_t)65535 * TM;
    for (int64_t m = 0; m < M; m += rows) {
        const int64_t part = M - m < rows ? M - m : rows;
        HeadOperand ap = a;
        ap.p = (const T*)a.p + (a.k_contiguous ? m * a.ld : m);
        HeadEpilogue ep = e;
        ep.out = e.out_f32 ? (void*)((float*)e.out + m * e.ld_out) : (void*)((T*)e.out + m * e.ld_out);
        if (e.residual) ep.residual = (const T*)e.residual + m * e.ld_residual;
        if (e.z) ep.z = (T*)e.z + m * N;
        if (e.lse) ep.lse = e.lse + m;
        if (e.row_weight) ep.row_weight = e.row_weight + m;
        if (e.target) ep.target = e.target + m;
        if (e.add) ep.add = e.add + m * N;
        const dim3 grid((unsigned)((N + TN - 1) / TN), (unsigned)((part + TM - 1) / TM));
        switch (e.kind == HEAD_EPI_LINEAR ? e.act : PNGPD_ACT_NONE) {
            case PNGPD_ACT_RELU: product_simple_kernel<T, PNGPD_ACT_RELU><<<grid, 256, 0, s>>>(part, N, K, ap, b, ep); break;
            case PNGPD_ACT_GELU: product_simple_kernel<T, PNGPD_ACT_GELU><<<grid, 256, 0, s>>>(part, N, K, ap, b, ep); break;
            case PNGPD_ACT_GELU_TANH:
                product_simple_kernel<T, PNGPD_ACT_GELU_TANH><<<grid, 256, 0, s>>>(part, N, K, ap, b, ep);
                break;
            case PNGPD_ACT_SILU: product_simple_kernel<T, PNGPD_ACT_SILU><<<grid, 256, 0, s>>>(part, N, K, ap, b, ep); break;
            default: product_simple_kernel<T, PNGPD_ACT_NONE><<<grid, 256, 0, s>>>(part, N, K, ap, b, ep);
        }
        hipError_t err = hipGetLastError();
        if (err != hipSuccess) return err;
    }
    return hipSuccess;
}

template <typename T, int ACT>
__global__ __launch_bounds__(256) void act_backward_kernel(int64_t M, int64_t N, const T* dy, int64_t ld, const T* z, T* dz) {
    const int64_t total = M * N;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t m = i / N, n = i - m * N;
        dz[i] = from_f32<T>(to_f32(dy[m * ld + n]) * act_slope<ACT>(to_f32(z[i])));
    }
}

template <typename T>
hipError_t act_backward(int64_t M, int64_t N, const void* dy, int64_t ld, const void* z, int act, void* dz, hipStream_t s) {
    const int64_t blocks = (M * N + 255) / 256;
    const unsigned grid = (unsigned)(blocks < 16384 ? blocks : 16384);
#define PNGPD_ACT_CASE(A) \
    case A: act_backward_kernel<T, A><<<grid, 256, 0, s>>>(M, N, (const T*)dy, ld, (const T*)z, (T*)dz); break;
    switch (act) {
        PNGPD_ACT_CASE(PNGPD_ACT_RELU)
        PNGPD_ACT_CASE(PNGPD_ACT_GELU)
        PNGPD_ACT_CASE(PNGPD_ACT_GELU_TANH)
        PNGPD_ACT_CASE(PNGPD_ACT_SILU)
        default: return hipErrorInvalidValue;
    }
#undef PNGPD_ACT_CASE
    return hipGetLastError();
}

template <typename T>
__global__ __launch_bounds__(256) void col_sum_part_kernel(int64_t M, int64_t N, const T* a, int64_t ld, int64_t rows, float* part) {
    const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (n >= N) return;
    const int64_t m0 = (int64_t)blockIdx.y * rows, m1 = m0 + rows < M ? m0 + rows : M;
    float s = 0.f;
    for (int64_t m = m0; m < m1; ++m) s += to_f32(a[m * ld + n]);
    part[(int64_t)blockIdx.y * N + n] = s;
}

template <typename T>
__global__ __launch_bounds__(256) void col_sum_join_kernel(int parts, int64_t N, const float* part, const float* scale, T* out) {
    const int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (n >= N) return;
    float s = 0.f;
    for (int i = 0; i < parts; ++i) s += part[(int64_t)i * N + n];
    out[n] = from_f32<T>(scale ? s * scale[0] : s);
}

template <typename T>
hipError_t col_sum(int64_t M, int64_t N, const void* a, int64_t ld, float* part, const float* scale, void* out, hipStream_t s) {
    const int64_t parts = head_col_sum_parts(M), rows = (M + parts - 1) / parts;
    const unsigned gx = (unsigned)((N + 255) / 256);
    col_sum_part_kernel<T><<<dim3(gx, (unsigned)parts), 256, 0, s>>>(M, N, (const T*)a, ld, rows, part);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    col_sum_join_kernel<T><<<gx, 256, 0, s>>>((int)parts, N, part, scale, (T*)out);
    return hipGetLastError();
}

}  // namespace

int64_t head_col_sum_parts(int64_t M) {
    const int64_t p = (M + 63) / 64;
    return p < 1 ? 1 : p > 64 ? 64 : p;
}

#define PNGPD_BY_TYPE(call)                                  \
    switch (type) {                                          \
        case PNGPD_TYPE_F32: { typedef float T; return call; }   \
        case PNGPD_TYPE_BF16: { typedef bf16_t T; return call; } \
        case PNGPD_TYPE_F16: { typedef f16_t T; return call; }   \
        default: return hipErrorInvalidValue;                \
    }

hipError_t head_product(int type, int64_t M, int64_t N, int64_t K, const HeadOperand& a, const HeadOperand& b,
                        const HeadEpilogue& e, hipStream_t s) {
    PNGPD_BY_TYPE((launch<T>(M, N, K, a, b, e, s)))
}
hipError_t head_act_backward(int type, int64_t M, int64_t N, const void* dy, int64_t ld, const void* z, int act, void* dz,
                             hipStream_t s) {
    PNGPD_BY_TYPE((act_backward<T>(M, N, dy, ld, z, act, dz, s)))
}
hipError_t head_col_sum(int type, int64_t M, int64_t N, const void* a, int64_t ld, float* part, const float* scale, void* out,
                        hipStream_t s) {
    PNGPD_BY_TYPE((col_sum<T>(M, N, a, ld, part, scale, out, s)))
}

}  // namespace pngpd
