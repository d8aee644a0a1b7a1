// The residual's addition, RMSNorm and 8-bit rows in one pass: a row's elements are loaded once, wait in
// registers for the sum of squares and the largest result, and leave as codes (and fp16). HBM bounds it, and close
// behind its instructions: 16384 rows of 4096 take 85 us, 5.5 TB/s, with 80 % of the issue slots used. Two passes
// over elements kept as scalars took 664 us.
#include "../common.cuh"
#include "batch_ops.h"

namespace cb {
namespace batch {

namespace {

constexpr int kMostThreads = 1024, kWarpRows = 8;  // rows of a block where a warp takes a row

// larger of the two; a NaN stays
__device__ __forceinline__ float max_nan(float a, float b) { return a != a || a > b ? a : b; }
__device__ __forceinline__ double add(double a, double b) { return a + b; }

// Over the threads of a row: a warp's, or a block's through `red`.
template <bool WARP, typename T, T (*F)(T, T)>
__device__ __forceinline__ T reduce(T v, T* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = F(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (WARP) return v;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int i = 1; i < (int)(blockDim.x >> 5); ++i) v = F(v, red[i]);
    return v;
}

// V pieces of 8 elements a thread: with VEC a piece is 16 consecutive bytes, else elements a stride of the
// row's threads apart.
template <int V, bool VEC>
struct Row {
    int threads, at, dims;
    __device__ __forceinline__ int index(int i, int j) const {
        return VEC ? 8 * (i * threads + at) + j : (8 * i + j) * threads + at;
    }
    __device__ __forceinline__ bool live(int i, int j) const { return index(i, VEC ? 0 : j) < dims; }
    __device__ __forceinline__ uint4 load(const __half* p, int i) const {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (VEC) {
            if (live(i, 0)) v = *reinterpret_cast<const uint4*>(p + index(i, 0));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (live(i, j)) reinterpret_cast<__half*>(&v)[j] = p[index(i, j)];
        }
        return v;
    }
    __device__ __forceinline__ void store(__half* p, int i, const uint4& v) const {
        if (VEC) {
            if (live(i, 0)) *reinterpret_cast<uint4*>(p + index(i, 0)) = v;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (live(i, j)) p[index(i, j)] = reinterpret_cast<const __half*>(&v)[j];
        }
    }
    __device__ __forceinline__ void store8(int8_t* p, int i, const uint2& v) const {
        if (VEC) {
            if (live(i, 0)) *reinterpret_cast<uint2*>(p + index(i, 0)) = v;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (live(i, j)) p[index(i, j)] = reinterpret_cast<const int8_t*>(&v)[j];
        }
    }
};

// Two elements' results: the same two products wherever they are needed.
__device__ __forceinline__ float2 result(const uint4& s, const uint4& w, int j, float inv) {
    const float2 a = __half22float2(reinterpret_cast<const __half2*>(&s)[j]);
    const float2 b = __half22float2(reinterpret_cast<const __half2*>(&w)[j]);
    return make_float2(__fmul_rn(__fmul_rn(a.x, inv), b.x), __fmul_rn(__fmul_rn(a.y, inv), b.y));
}

template <int V, bool VEC, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kWarpRows : kMostThreads) norm_q8_kernel(NormCall c) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ double red_sum[32];
    __shared__ float red_max[32];
    const long long row = WARP ? (long long)blockIdx.x * kWarpRows + threadIdx.y : blockIdx.x;
    if (WARP && row >= c.rows) return;
    const Row<V, VEC> at = {(int)blockDim.x, (int)threadIdx.x, c.dims};
    uint4 s[V], w[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = at.load(c.x + row * c.x_stride, i);
    if (c.residual) {
        uint4 r[V];
#pragma unroll
        for (int i = 0; i < V; ++i) r[i] = at.load(c.residual + row * c.residual_stride, i);
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                reinterpret_cast<__half2*>(&s[i])[j] =
                    __hadd2(reinterpret_cast<const __half2*>(&s[i])[j], reinterpret_cast<const __half2*>(&r[i])[j]);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = at.load(c.weight, i);
    // Squares of fp16 numbers are added in 64 bits: their sum rounded to fp32 does not depend on its order
    // (but for one row in a hundred million), and so neither do the codes.
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (c.sum) at.store(c.sum + row * c.sum_stride, i, s[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double v = (double)__half2float(reinterpret_cast<const __half*>(&s[i])[j]);
            sum = fma(v, v, sum);
        }
    }
    sum = reduce<WARP, double, add>(sum, red_sum);
    const float inv = (float)(1.0 / sqrt(sum / (double)c.dims + (double)c.eps));
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        uint4 n;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 y = result(s[i], w[i], j, inv);
            reinterpret_cast<__half2*>(&n)[j] = __floats2half2_rn(y.x, y.y);
            if (at.live(i, 2 * j)) top = max_nan(top, fabsf(y.x));
            if (at.live(i, 2 * j + 1)) top = max_nan(top, fabsf(y.y));
        }
        if (c.normed) at.store(c.normed + row * c.dims, i, n);
    }
    if (!c.q) return;
    top = reduce<WARP, float, max_nan>(top, red_max);
    const bool bad = !(top < INFINITY);
    const float scale = fmaxf(__fdiv_rn(top, 127.0f), 1e-10f), per = bad ? 0.0f : __fdiv_rn(1.0f, scale);
    const float magic = 12582912.0f;  // 1.5 * 2^23: a sum with it is rounded half to even and has the code in its low bits
#pragma unroll
    for (int i = 0; i < V; ++i) {
        uint32_t b[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 y = result(s[i], w[i], j, inv);
            b[2 * j] = __float_as_uint(__fadd_rn(__fmul_rn(y.x, per), magic));
            b[2 * j + 1] = __float_as_uint(__fadd_rn(__fmul_rn(y.y, per), magic));
        }
        uint2 code;
        code.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
        code.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
        at.store8(c.q + row * c.dims, i, bad ? make_uint2(0, 0) : code);
    }
    if (at.at == 0) c.scales[row] = bad ? __int_as_float(0x7fc00000) : scale;
}

template <bool VEC>
cudaError_t launch(const NormCall& c, cudaStream_t st) {
    const int pieces = (c.dims + 7) / 8;
    // Many rows: four pieces a thread, so that a block's loads are in flight together and its reductions are short.
    // Few: one piece a thread, for the fewest steps. Few / many, us: 64 rows of 2048 3.1 / 3.7, 256 rows of 2048 3.6 / 4.2,
    // of 4096 4.7 / 4.6, 592 rows of 1024 3.6 / 3.7, of 4096 8.3 / 5.8, 64 rows of 8192 5.7 / 4.7; 1200 rows of 128
    // 3.1 / 3.1, 4000 rows of 128 5.7 / 3.7.
    const bool many = c.rows >= 2048 || (long long)c.rows * c.dims >= 1 << 20 || c.dims > 4096;
    if (many && pieces <= (VEC ? 128 : 32)) {  // short rows: a warp each, no barriers (4000 rows of 512 4.7 us, a block each 6.7)
        const dim3 grid((unsigned)((c.rows + kWarpRows - 1) / kWarpRows)), block(32, kWarpRows);
        auto kernel = norm_q8_kernel<1, VEC, true>;
        if constexpr (VEC)
            if (pieces > 32) kernel = pieces <= 64 ? norm_q8_kernel<2, VEC, true> : norm_q8_kernel<4, VEC, true>;
        return launch_k(kernel, grid, block, 0, st, c);
    }
    const int v = (many && VEC) || pieces > 2 * kMostThreads ? 4 : pieces > kMostThreads ? 2 : 1;
    const unsigned threads = (unsigned)(((pieces + v - 1) / v + 31) / 32 * 32);
    auto kernel = v == 4 ? norm_q8_kernel<4, VEC, false> : v == 2 ? norm_q8_kernel<2, VEC, false> : norm_q8_kernel<1, VEC, false>;
    return launch_k(kernel, dim3((unsigned)c.rows), dim3(threads), 0, st, c);
}

}  // namespace

int launch_norm_q8(const NormCall& c, cudaStream_t st) {
    auto wide = [](const void* p, long long stride) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0; };
    const bool vec = c.dims % 8 == 0 && wide(c.x, c.x_stride) && (!c.residual || wide(c.residual, c.residual_stride)) &&
                     (!c.sum || wide(c.sum, c.sum_stride)) && wide(c.weight, 0) && wide(c.normed, 0) &&
                     (reinterpret_cast<uintptr_t>(c.q) & 7) == 0;
    return (vec ? launch<true>(c, st) : launch<false>(c, st)) == cudaSuccess ? 0 : -1;
}

}  // namespace batch
}  // namespace cb
