// The residual's addition, RMSNorm and 8-bit rows in one pass: a block a row, its elements kept in registers
// between the sum of squares and the result.
#include "../common.cuh"
#include "batch_ops.h"

namespace cb {
namespace batch {

namespace {

constexpr int kThreads = 1024, kKeep = kNormMaxDims / kThreads;

template <typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, T* red, F f) {
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int i = 1; i < (int)(blockDim.x >> 5); ++i) v = f(v, red[i]);
    return v;
}

// larger of the two; a NaN stays
__device__ __forceinline__ float max_nan(float a, float b) { return a != a || a > b ? a : b; }

__global__ void __launch_bounds__(kThreads) norm_q8_kernel(NormCall c) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ double red_sum[32];
    __shared__ float red_max[32];
    const long long row = blockIdx.x;
    __half s[kKeep];
    double sq = 0.0;
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
        const int k = i * kThreads + threadIdx.x;
        if (k >= c.dims) break;
        s[i] = c.x[row * c.x_stride + k];
        if (c.residual) s[i] = __hadd(s[i], c.residual[row * c.residual_stride + k]);
        if (c.sum) c.sum[row * c.sum_stride + k] = s[i];
        const double v = (double)h2f(s[i]);
        sq = fma(v, v, sq);
    }
    sq = block_reduce(sq, red_sum, [](double a, double b) { return a + b; });
    const float inv = (float)(1.0 / sqrt(sq / (double)c.dims + (double)c.eps));
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
        const int k = i * kThreads + threadIdx.x;
        if (k >= c.dims) break;
        const float y = __fmul_rn(__fmul_rn(h2f(s[i]), inv), h2f(c.weight[k]));
        if (c.normed) c.normed[row * c.dims + k] = f2h(y);
        top = max_nan(top, fabsf(y));
    }
    if (!c.q) return;
    top = block_reduce(top, red_max, [](float a, float b) { return max_nan(a, b); });
    const bool bad = !(top < INFINITY);
    const float scale = fmaxf(__fdiv_rn(top, 127.0f), 1e-10f), per = __fdiv_rn(1.0f, scale);
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
        const int k = i * kThreads + threadIdx.x;
        if (k >= c.dims) break;
        const float y = __fmul_rn(__fmul_rn(h2f(s[i]), inv), h2f(c.weight[k]));
        c.q[row * c.dims + k] = bad ? 0 : (int8_t)cvt_rne_sat(__fmul_rn(y, per));
    }
    if (threadIdx.x == 0) c.scales[row] = bad ? __int_as_float(0x7fc00000) : scale;
}

}  // namespace

int launch_norm_q8(const NormCall& c, cudaStream_t st) {
    return launch_k(norm_q8_kernel, dim3((unsigned)c.rows), dim3(kThreads), 0, st, c) == cudaSuccess ? 0 : -1;
}

}  // namespace batch
}  // namespace cb
