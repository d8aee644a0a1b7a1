// Attention over the 4-bit paged KV cache.
//
// One warp per (token, q head): lane i scores key i of each 32-key block in fp32, the block's
// weights join the running maximum and sum, and lane l accumulates the output dims l, l + 32, ...
#include "kv4.cuh"
#include "kv4_ops.h"

namespace cb {
namespace kv4 {

namespace {

constexpr int kWarps = 4;

__device__ __forceinline__ float code_value(const uint8_t* codes, const uint8_t* params, int row, int d, int g, int i) {
    const int b = codes[row * (d / 2) + i / 2], c = (i & 1) ? b >> 4 : b & 15;
    const __half2 par = *reinterpret_cast<const __half2*>(params + (row * (d / g) + i / g) * 4);
    return __half2float(__hfma(__int2half_rn(c), __low2half(par), __high2half(par)));
}

template <int D>
__global__ void __launch_bounds__(kWarps * 32) kv4_attn_simple_kernel(AttnCall c, Pages pg, Geom ge) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ float s_q[kWarps][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * kWarps + warp;
    const int t = (int)(item / c.hq), h = (int)(item % c.hq);
    if (t >= c.num_tokens) return;
    const int b = find_seq(c.offsets, c.num_seqs, t);
    if (b < 0) return;
    if (t - c.offsets[b] >= c.max_q) {
        report_dev_error(kDevBadPage);
        return;
    }
    const int len = max(c.lens[b], 0), head = h / (c.hq / ge.hkv);
    const long long pos = (long long)c.lens[b] - c.offsets[b + 1] + t;
    const long long end = c.causal ? min((long long)len, pos + 1) : len;
    const long long start = c.window > 0 ? max(0LL, pos - c.window + 1) : 0;
    const __half* q = c.q + (long long)t * c.q_stride + (long long)h * D;
    for (int i = lane; i < D; i += 32) s_q[warp][i] = __half2float(q[i]);
    __syncwarp();
    float m = -INFINITY, l = 0.0f, acc[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = 0.0f;
    for (long long k0 = start; k0 < end; k0 += 32) {
        const long long k = k0 + lane;
        const uint8_t* block = nullptr;
        const int row = (int)(k & (ge.page() - 1));
        float s = -INFINITY;
        if (k < end) {
            const long long off = page_offset(pg, b, k, ge.page_shift);
            if (off >= 0) {
                block = pg.pool + off + (long long)head * ge.block_bytes();
                float sum = 0.0f;
                for (int i = 0; i < D; ++i)
                    sum = fmaf(s_q[warp][i], code_value(block, block + ge.k_params(), row, D, ge.g, i), sum);
                s = sum * c.scale;
            }
        }
        const float top = warp_max(s), m2 = fmaxf(m, top);
        if (m2 == -INFINITY) continue;
        const float p = expf(s - m2), fix = expf(m - m2);
        float sum = p;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l = fmaf(l, fix, sum);
        m = m2;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] *= fix;
        for (int j = 0; j < 32; ++j) {
            const float pj = __shfl_sync(0xffffffffu, p, j);
            const uint8_t* bj = reinterpret_cast<const uint8_t*>(
                __shfl_sync(0xffffffffu, (unsigned long long)(uintptr_t)block, j));
            const int rj = __shfl_sync(0xffffffffu, row, j);
            if (!bj) continue;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
                acc[i] = fmaf(pj, code_value(bj + ge.v_codes(), bj + ge.v_params(), rj, D, ge.g, lane + 32 * i), acc[i]);
        }
    }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    __half* o = c.out + ((long long)t * c.hq + h) * D;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[lane + 32 * i] = __float2half_rn(acc[i] * inv);
    if (c.lse && lane == 0) c.lse[(long long)t * c.hq + h] = m + logf(l);
}

}  // namespace

size_t attention_workspace(int, int, int, int, int) { return 16; }

int launch_attention(const AttnCall& c, const Pages& pg, const Geom& ge, cudaStream_t st) {
    const long long items = (long long)c.num_tokens * c.hq;
    const dim3 grid((unsigned)((items + kWarps - 1) / kWarps));
    auto kernel =
        ge.d == 64 ? kv4_attn_simple_kernel<64> : ge.d == 128 ? kv4_attn_simple_kernel<128> : kv4_attn_simple_kernel<256>;
    return launch_k(kernel, grid, dim3(kWarps * 32), 0, st, c, pg, ge) == cudaSuccess ? 0 : -1;
}

}  // namespace kv4
}  // namespace cb
