// The adapters' plan, as its kernel writes it and the products' kernels read it.
#pragma once
#include "../common.cuh"
#include "batch_ops.h"

namespace cb {
namespace batch {

// ints: header [16] | tiles [most_tiles(64)][4] (adapter, first place, rows, 0) | wide tiles, of up to 128 rows, the same
// | starts [A + 1] | tile starts, wide ones [A + 2 each] | cursors [A + 1] | rows [num_tokens]: the batch's rows in order
// of their adapters, the batch's order kept among those of one; rows without an adapter stand last.
constexpr int kTileRows = 64, kWideRows = 128;
enum { kHeadSeqs, kHeadTokens, kHeadAdapters, kHeadRows, kHeadTiles, kHeadBare, kHeadWide, kHeadInts = 16 };

// every adapter that has rows can have one tile that is not full
__host__ __device__ inline long long most_tiles(long long seqs, long long tokens, long long adapters, int rows = kTileRows) {
    return tokens / rows + (seqs < adapters ? seqs : adapters);
}
// where the parts begin, in ints
struct PlanLayout {
    long long tiles, wide, starts, tile_starts, wide_starts, cursors, rows;
    __host__ __device__ PlanLayout(long long seqs, long long tokens, long long adapters) {
        tiles = kHeadInts;
        wide = tiles + 4 * most_tiles(seqs, tokens, adapters);
        starts = wide + 4 * most_tiles(seqs, tokens, adapters, kWideRows);
        tile_starts = starts + adapters + 1;
        wide_starts = tile_starts + adapters + 2;
        cursors = wide_starts + adapters + 2;
        rows = cursors + adapters + 1;
    }
};

// Few tiles' first products are split over K, so that there is about a block for each SM; each part leaves its
// fp32 sums in the workspace [part][place][max_rank], and the second product's kernel adds them up in order.
constexpr int kTargetBlocks = kNumSMs, kMostParts = 32, kLeastK = 256;

__host__ __device__ inline int parts_of(int tiles, int k) {
    int p = kTargetBlocks / (tiles > 0 ? tiles : 1);
    p = p < k / kLeastK ? p : k / kLeastK;
    p = p < kMostParts ? p : kMostParts;
    return p > 1 ? p : 1;
}

struct Plan {
    int tiles, rows, bare, wide_tiles;
    const int4 *tile, *wide;
    const int* row;
};
// false where the plan is of other numbers
__device__ __forceinline__ bool read_plan(const LoraCall& c, Plan* p) {
    const int4 head = __ldg(reinterpret_cast<const int4*>(c.plan)), more = __ldg(reinterpret_cast<const int4*>(c.plan) + 1);
    if (head.x != c.num_seqs || head.y != c.num_tokens || head.z != c.num_adapters) return false;
    const PlanLayout at(c.num_seqs, c.num_tokens, c.num_adapters);
    p->rows = head.w;
    p->tiles = more.x;
    p->bare = more.y;
    p->wide_tiles = more.z;
    p->tile = reinterpret_cast<const int4*>(c.plan + at.tiles);
    p->wide = reinterpret_cast<const int4*>(c.plan + at.wide);
    p->row = c.plan + at.rows;
    return true;
}

// 2^e with a row's largest finite element, `top`, below 2^12 of it (an infinity or a NaN beside it is one at any power,
// but what is finite must not become one); rows without such an element or with nothing but zeros stay as they are
__device__ __forceinline__ int exponent_of(float top) {
    return top > 0.0f ? max((int)(__float_as_uint(top) >> 23) - 127 - 11, -125) : 0;
}
__device__ __forceinline__ float two_to(int e) { return __int_as_float((127 + e) << 23); }
// x as two fp16 numbers; an infinity or a NaN is the first one
__device__ __forceinline__ void two_halves(float x, __half* high, __half* low) {
    *high = __float2half_rn(x);
    const float rest = x - __half2float(*high);
    *low = __float2half_rn(fabsf(x) < INFINITY ? rest : 0.0f);
}

// N fours of a row of the first product, 16 elements apart, as far as `left` goes: the sums of the parts, which lie
// `step` apart. The loads of a part do not wait for one another.
template <int N>
__device__ __forceinline__ void sum_parts(const float* from, long long step, int parts, int left, float4 (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
        v[i] = left > 16 * i ? __ldcg(reinterpret_cast<const float4*>(from + 16 * i)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 2
    for (int part = 1; part < parts; ++part) {
        from += step;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (left > 16 * i) {
                const float4 h = __ldcg(reinterpret_cast<const float4*>(from + 16 * i));
                v[i].x += h.x, v[i].y += h.y, v[i].z += h.z, v[i].w += h.w;
            }
    }
}
__device__ __forceinline__ float size_if_finite(float v) { return fabsf(v) < INFINITY ? fabsf(v) : 0.0f; }
__device__ __forceinline__ float largest_finite(const float4& v) {
    return fmaxf(fmaxf(size_if_finite(v.x), size_if_finite(v.y)), fmaxf(size_if_finite(v.z), size_if_finite(v.w)));
}

// the first `bytes` of 16 bytes global -> shared, and zeros behind them (nothing is read where there are none)
__device__ __forceinline__ void copy_or_zero(uint32_t to, const void* from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

}  // namespace batch
}  // namespace cb
