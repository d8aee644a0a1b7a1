// Attention of one query row over the 4-bit paged KV cache by one warp: the plain form, which the
// tiled kernels fall back to for rows whose result is not a number.
#pragma once
#include "kv4.cuh"
#include "kv4_ops.h"

namespace cb {
namespace kv4 {

__device__ __forceinline__ float code_value(const uint8_t* codes, const uint8_t* params, int row, int d, int g, int i) {
    const int b = codes[row * (d / 2) + i / 2], c = (i & 1) ? b >> 4 : b & 15;
    const __half2 par = *reinterpret_cast<const __half2*>(params + (row * (d / g) + i / g) * 4);
    return __half2float(__hfma(__int2half_rn(c), __low2half(par), __high2half(par)));
}

// Lane i scores key i of each 32-key block in fp32, the block's weights join the running maximum
// and sum, and lane l accumulates the output dims l, l + 32, ...; only keys that the row sees are
// read. Writes the row's output and log-sum-exp.
template <int D>
__device__ __forceinline__ void attention_row(const AttnCall& c, const Pages& pg, const Geom& ge, int b, int t, int h,
                                           int lane) {
    const long long room = pg.table_stride << ge.page_shift;
    const long long len = max(0LL, min((long long)c.lens[b], room));
    const int head = h / (c.hq / ge.hkv);
    const long long pos = (long long)c.lens[b] - c.offsets[b + 1] + t;
    const long long end = c.causal ? min(len, pos + 1) : len;
    const long long start = c.window > 0 ? max(0LL, pos - c.window + 1) : 0;
    const __half* q = c.q + (long long)t * c.q_stride + (long long)h * D;
    float m = -INFINITY, l = 0.0f, acc[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = 0.0f;
#pragma unroll 1
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
#pragma unroll 1
                for (int i = 0; i < D; ++i)
                    sum = fmaf(__half2float(q[i]), code_value(block, block + ge.k_params(), row, D, ge.g, i), sum);
                s = sum * c.scale;
            }
        }
        const float m2 = fmaxf(m, warp_max(s)), base = m2 == -INFINITY ? 0.0f : m2;
        const float p = expf(s - base), fix = m == -INFINITY ? 1.0f : expf(m - base);
        float sum = p;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l = fmaf(l, fix, sum);
        m = m2;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] *= fix;
#pragma unroll 1
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
    if (c.lse && lane == 0) c.lse[(long long)t * c.hq + h] = l == 0.0f ? -INFINITY : m + logf(l);
}

}  // namespace kv4
}  // namespace cb
