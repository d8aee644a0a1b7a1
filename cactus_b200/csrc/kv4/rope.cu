// The append of the 4-bit paged KV cache that normalises and rotates on the way, and the table of turns
// that it reads. D / 8 lanes share a head's row (8 elements, one 16-byte load each): shuffles add up the
// squares of the norm, fetch the other element of each rotated pair and reduce a group's ends for the
// quantisation.
#include "kv4.cuh"
#include "kv4_ops.h"
#include "quantise.cuh"

namespace cb {
namespace kv4 {

namespace {

constexpr int kRopeTokens = 32, kRopeThreads = 256;

// (cos, sin) of position p's angles: p * theta^(-2 i / R), in 64 bits up to the last rounding.
__global__ void rope_table_kernel(double theta, int half, long long n, float2* __restrict__ table) {
    pdl_launch_dependents();
    pdl_wait();
    const long long at = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (at >= n) return;
    const int i = (int)(at % half);
    double s, c;
    sincos((double)(at / half) * pow(theta, -(double)i / (double)half), &s, &c);
    table[at] = make_float2((float)c, (float)s);
}

// Eight elements of a row of D, normalised (where there is a weight) and turned, as fp16.
template <int D>
__device__ __forceinline__ uint4 norm_and_turn(const uint4& in, const __half* __restrict__ weight, float eps,
                                               const float2* __restrict__ turns, int rotary, int lane) {
    constexpr int kLanes = D / 8;
    const unsigned full = 0xffffffffu;
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 p = __half22float2(reinterpret_cast<const __half2*>(&in)[j]);
        v[2 * j] = p.x;
        v[2 * j + 1] = p.y;
    }
    if (weight) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fmaf(v[j], v[j], sum);
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) sum += __shfl_xor_sync(full, sum, o);
        const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fmul_rn(sum, 1.0f / D), eps)));
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(weight) + lane);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 p = __half22float2(reinterpret_cast<const __half2*>(&w)[j]);
            v[2 * j] = __fmul_rn(__fmul_rn(v[2 * j], inv), p.x);
            v[2 * j + 1] = __fmul_rn(__fmul_rn(v[2 * j + 1], inv), p.y);
        }
    }
    if (rotary) {
        const int part = rotary >> 4;  // lanes of each half of the rotated elements
        const bool first = lane < part, turned = lane < 2 * part;
        const int other = first ? lane + part : lane - part, row = (threadIdx.x & 31) - lane;
        float2 t[8];
        if (turned) {
            const float4* at = reinterpret_cast<const float4*>(turns) + (first ? lane : other) * 4;
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<float4*>(&t[2 * j]) = __ldg(at + j);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float u = __shfl_sync(full, v[j], row + (turned ? other : lane));
            if (turned) {
                const float a = __fmul_rn(v[j], t[j].x), b = __fmul_rn(u, t[j].y);
                v[j] = first ? __fsub_rn(a, b) : __fadd_rn(a, b);
            }
        }
    }
    uint4 out;
#pragma unroll
    for (int j = 0; j < 4; ++j) reinterpret_cast<__half2*>(&out)[j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
    return out;
}

template <int D>
__global__ void __launch_bounds__(kRopeThreads) kv4_rope_append_kernel(RopeCall c, Pages pg, Geom ge) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ long long s_page[kRopeTokens];  // byte offset of the page, -1: nothing to append
    __shared__ int s_pos[kRopeTokens];         // -1: no position to turn to, -2: a row of no sequence
    constexpr int kLanes = D / 8, kRows = kRopeThreads / kLanes;
    const int t0 = blockIdx.x * kRopeTokens, lane = threadIdx.x % kLanes;
    const int per_group = ge.g >> 3, group = lane >> (__ffs(per_group) - 1);
    const int head = blockIdx.y;
    const bool query = head < c.hq, value = head >= c.hq + ge.hkv;
    const int kv_head = query ? 0 : (head - c.hq) - (value ? ge.hkv : 0);
    if (threadIdx.x < kRopeTokens) {
        const int t = t0 + threadIdx.x;
        const int b = t < c.num_tokens ? find_seq(c.offsets, c.num_seqs, t) : -1;
        long long page = -1;
        int at = -2;
        if (b >= 0) {
            const long long pos = (long long)c.lens[b] - c.offsets[b + 1] + t;
            at = -1;
            if (pos >= 0 && c.rotary && pos >= c.num_positions) {
                report_dev_error(kDevBadPage);
            } else if (pos >= 0) {
                at = (int)pos;
                if (!query) page = page_offset(pg, b, pos, ge.page_shift);
            }
        }
        s_page[threadIdx.x] = page;
        s_pos[threadIdx.x] = at;
    }
    __syncthreads();
    const __half* from = query ? c.q + (long long)head * D : (value ? c.v : c.k) + (long long)kv_head * D;
    const long long stride = query ? c.q_stride : c.row_stride;
    const unsigned full = 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kRopeTokens / kRows; ++i) {
        const int r = threadIdx.x / kLanes + i * kRows, t = min(t0 + r, c.num_tokens - 1);
        const int pos = s_pos[r];
        uint4 x = __ldg(reinterpret_cast<const uint4*>(from + t * stride) + lane);
        if (!value)
            x = norm_and_turn<D>(x, query ? c.q_weight : c.k_weight, c.eps,
                                 c.turns + (long long)max(pos, 0) * (c.rotary / 2), c.rotary, lane);
        if (query) {
            if (pos == -1) x = make_uint4(0, 0, 0, 0);
            if (pos != -2) reinterpret_cast<uint4*>(c.out + t * c.out_stride + (long long)head * D)[lane] = x;
            continue;
        }
        const __half2* h = reinterpret_cast<const __half2*>(&x);
        // (largest, -smallest): exact in fp16, and a NaN stays one
        const __half2 hi2 = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
        const __half2 lo2 = __hmin2_nan(__hmin2_nan(h[0], h[1]), __hmin2_nan(h[2], h[3]));
        __half2 ends = __hmax2_nan(__lows2half2(hi2, __hneg2(lo2)), __highs2half2(hi2, __hneg2(lo2)));
        for (int o = 1; o < per_group; o <<= 1) ends = __hmax2_nan(ends, __shfl_xor_sync(full, ends, o));
        const float hi = __low2float(ends), lo = -__high2float(ends);
        const __half step = step_of(hi, lo);
        const float fs = __half2float(step);
        const bool bad = !(__fsub_rn(hi, lo) < INFINITY);  // an infinity or a NaN in the group
        uint32_t w = 0;
        if (!bad && fs > 0.0f) w = quant_codes(h, lo, fs);
        if (s_page[r] >= 0) {
            uint8_t* block = pg.pool + s_page[r] + (long long)kv_head * ge.block_bytes() + (value ? ge.v_codes() : 0);
            const int row = pos & (ge.page() - 1);
            *reinterpret_cast<uint32_t*>(block + row * (D / 2) + lane * 4) = w;
            if ((lane & (per_group - 1)) == 0) {
                const __half nan = __ushort_as_half(0x7FFF);
                *reinterpret_cast<__half2*>(block + ge.k_params() + (row * ge.ng() + group) * 4) =
                    bad ? __halves2half2(nan, nan) : __halves2half2(step, __float2half_rn(lo));
            }
        }
    }
}

}  // namespace

int launch_rope_table(float theta, int half, long long positions, float* table, cudaStream_t st) {
    const long long n = positions * half;
    return launch_k(rope_table_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, (double)theta, half, n,
                    reinterpret_cast<float2*>(table)) == cudaSuccess
               ? 0
               : -1;
}

int launch_rope_append(const RopeCall& c, const Pages& pg, const Geom& ge, cudaStream_t st) {
    const dim3 grid((unsigned)((c.num_tokens + kRopeTokens - 1) / kRopeTokens), (unsigned)(c.hq + 2 * ge.hkv));
    auto kernel = ge.d == 64    ? kv4_rope_append_kernel<64>
                  : ge.d == 128 ? kv4_rope_append_kernel<128>
                                : kv4_rope_append_kernel<256>;
    return launch_k(kernel, grid, dim3(kRopeThreads), 0, st, c, pg, ge) == cudaSuccess ? 0 : -1;
}

}  // namespace kv4
}  // namespace cb
