// Low-rank adapters of many requests: a plan that groups a batch's rows by adapter, then two products a
// row with its adapter's matrices, the low-rank one in fp32 in the workspace between them.
#include "../common.cuh"
#include "batch_ops.h"

namespace cb {
namespace batch {

namespace {

// ---------------------------------------------------------------- plan
// ints: header [16] | tiles [max_tiles][4] (adapter, first place, rows, 0) | starts [A + 1] | tile starts [A + 2]
// | cursors [A + 1] | rows [num_tokens]: the batch's rows in order of their adapters, the batch's order
// kept among those of one; rows without an adapter stand last.
constexpr int kTileRows = 64;
enum { kHeadSeqs, kHeadTokens, kHeadAdapters, kHeadRows, kHeadTiles, kHeadBare, kHeadInts = 16 };

__host__ __device__ inline long long most_tiles(long long seqs, long long tokens, long long adapters) {
    return tokens / kTileRows + (seqs < adapters ? seqs : adapters);
}
struct PlanView {
    int4* tiles;
    int *starts, *tile_starts, *cursors, *rows;
    __host__ __device__ PlanView(int* p, long long seqs, long long tokens, long long adapters) {
        tiles = reinterpret_cast<int4*>(p + kHeadInts);
        starts = p + kHeadInts + 4 * most_tiles(seqs, tokens, adapters);
        tile_starts = starts + adapters + 1;
        cursors = tile_starts + adapters + 2;
        rows = cursors + adapters + 1;
    }
};

constexpr int kPlanThreads = 1024;

// exclusive sum over the block, and the total
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int s = v;
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += u;
    }
    __syncthreads();  // the last call's sums are read
    if (lane == 31) warp_sums[w] = s;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < kPlanThreads / 32; ++i) {
        before += i < w ? warp_sums[i] : 0;
        all += warp_sums[i];
    }
    *total = all;
    return before + s - v;
}

__global__ void __launch_bounds__(kPlanThreads)
    lora_plan_kernel(const int* __restrict__ offsets, const int* __restrict__ ids, int num_seqs, int num_tokens,
                     int num_adapters, int* plan) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ int warp_sums[kPlanThreads / 32], s_id[kPlanThreads], s_len[kPlanThreads], s_place[kPlanThreads];
    const int t = threadIdx.x;
    const PlanView v(plan, num_seqs, num_tokens, num_adapters);
    int bad = 0;
    for (int b = t; b < num_seqs; b += kPlanThreads) bad |= offsets[b] < 0 || offsets[b] > offsets[b + 1];
    if (t == 0) bad |= offsets[num_seqs] > num_tokens;
    bad = __syncthreads_or(bad);
    if (bad) {
        if (t == 0) report_dev_error(kDevBadList);
        if (t < kHeadInts)
            plan[t] = t == kHeadSeqs ? num_seqs : t == kHeadTokens ? num_tokens : t == kHeadAdapters ? num_adapters : 0;
        return;
    }
    // adapter of a sequence; the rows of none count as those of one more adapter
    auto adapter_of = [&](int b) {
        const int a = ids[b];
        if (a >= -1 && a < num_adapters) return a < 0 ? num_adapters : a;
        report_dev_error(kDevBadList);
        return num_adapters;
    };
    for (int a = t; a <= num_adapters; a += kPlanThreads) v.cursors[a] = 0;
    __syncthreads();
    for (int b = t; b < num_seqs; b += kPlanThreads) atomicAdd(&v.cursors[adapter_of(b)], offsets[b + 1] - offsets[b]);
    __syncthreads();
    int row0 = 0, tile0 = 0;
    for (int a0 = 0; a0 <= num_adapters; a0 += kPlanThreads) {
        const int a = a0 + t, n = a <= num_adapters ? v.cursors[a] : 0;
        int total = 0;
        const int start = row0 + block_scan(n, warp_sums, &total);
        row0 += total;
        const int tile = tile0 + block_scan(a < num_adapters ? (n + kTileRows - 1) / kTileRows : 0, warp_sums, &total);
        tile0 += total;
        if (a <= num_adapters) {
            v.starts[a] = start;
            v.tile_starts[a] = tile;
            v.cursors[a] = start;
        }
    }
    if (t == 0) v.tile_starts[num_adapters + 1] = tile0;
    __syncthreads();
    if (t < kHeadInts) {
        const int rows = v.starts[num_adapters];
        const int head[kHeadInts] = {num_seqs, num_tokens, num_adapters, rows, tile0, row0 - rows};
        plan[t] = head[t];
    }
    for (int i = t; i < tile0; i += kPlanThreads) {
        int lo = 0, hi = num_adapters;  // the last adapter whose tiles begin at or before i and that has any
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (v.tile_starts[mid] <= i) lo = mid; else hi = mid;
        }
        const int first = v.starts[lo] + (i - v.tile_starts[lo]) * kTileRows;
        v.tiles[i] = make_int4(lo, first, min(kTileRows, v.starts[lo + 1] - first), 0);
    }
    for (int b0 = 0; b0 < num_seqs; b0 += kPlanThreads) {
        const int b = b0 + t, n = min(kPlanThreads, num_seqs - b0);
        int id = -1, len = 0, place = 0;
        if (t < n) {
            id = adapter_of(b);
            len = offsets[b + 1] - offsets[b];
        }
        s_id[t] = id;
        s_len[t] = len;
        __syncthreads();
        if (t < n) {
            place = v.cursors[id];
            for (int j = 0; j < t; ++j) place += s_id[j] == id ? s_len[j] : 0;
            s_place[t] = place;
        }
        __syncthreads();
        if (t < n) atomicAdd(&v.cursors[id], len);
        for (int j = t >> 5; j < n; j += kPlanThreads / 32)
            for (int i = t & 31; i < s_len[j]; i += 32) v.rows[s_place[j] + i] = offsets[b0 + j] + i;
        __syncthreads();
    }
}

// ---------------------------------------------------------------- products
__device__ __forceinline__ bool plan_fits(const LoraCall& c) {
    return c.plan[kHeadSeqs] == c.num_seqs && c.plan[kHeadTokens] == c.num_tokens &&
           c.plan[kHeadAdapters] == c.num_adapters;
}
__device__ __forceinline__ int rank_of(const LoraCall& c, int adapter) {
    const int r = c.ranks ? c.ranks[adapter] : c.max_rank;
    if (r >= 0 && r <= c.max_rank) return r;
    report_dev_error(kDevBadList);
    return 0;
}
__device__ __forceinline__ int adapter_at(const LoraCall& c, const PlanView& v, int place) {
    int lo = 0, hi = c.num_adapters;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (v.starts[mid] <= place) lo = mid; else hi = mid;
    }
    return lo;
}

// A block a row: each warp the dot products of every eighth row of A.
__global__ void __launch_bounds__(256) lora_shrink_kernel(LoraCall c) {
    pdl_launch_dependents();
    pdl_wait();
    if (!plan_fits(c)) {
        report_dev_error(kDevBadList);
        return;
    }
    const PlanView v(const_cast<int*>(c.plan), c.num_seqs, c.num_tokens, c.num_adapters);
    const int place = blockIdx.x, lane = threadIdx.x & 31;
    if (place >= c.plan[kHeadRows]) return;
    const int adapter = adapter_at(c, v, place), rank = rank_of(c, adapter);
    const __half* x = c.x + v.rows[place] * c.x_stride;
    for (int r = threadIdx.x >> 5; r < rank; r += 8) {
        const __half* a = c.a + ((long long)adapter * c.max_rank + r) * c.k;
        float sum = 0.0f;
        for (int k = lane; k < c.k; k += 32) sum = fmaf(h2f(x[k]), h2f(a[k]), sum);
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) c.ws[(long long)place * c.max_rank + r] = sum;
    }
}

// A thread an output of a row.
__global__ void __launch_bounds__(256) lora_expand_kernel(LoraCall c) {
    pdl_launch_dependents();
    pdl_wait();
    if (!plan_fits(c)) return;
    const PlanView v(const_cast<int*>(c.plan), c.num_seqs, c.num_tokens, c.num_adapters);
    const int place = blockIdx.x, n = blockIdx.y * 256 + threadIdx.x, rows = c.plan[kHeadRows];
    if (place >= rows + c.plan[kHeadBare] || n >= c.n) return;
    const long long row = v.rows[place];
    float y = c.base ? h2f(c.base[row * c.base_stride + n]) : 0.0f;
    if (place < rows) {
        const int adapter = adapter_at(c, v, place), rank = rank_of(c, adapter);
        const __half* b = c.b + ((long long)adapter * c.n + n) * c.max_rank;
        const float* h = c.ws + (long long)place * c.max_rank;
        float sum = 0.0f;
        for (int r = 0; r < rank; ++r) sum = fmaf(h[r], h2f(b[r]), sum);
        y = fmaf(c.scales ? c.scales[adapter] : 1.0f, sum, y);
    }
    c.out[row * c.out_stride + n] = f2h(y);
}

}  // namespace

size_t lora_plan_bytes(long long seqs, long long tokens, long long adapters) {
    const PlanView v(nullptr, seqs, tokens, adapters);
    const size_t ints = (size_t)(reinterpret_cast<uintptr_t>(v.rows) / 4) + (size_t)tokens;
    return (ints * 4 + 15) / 16 * 16;
}

// rows of the low-rank product, times the parts that a product over few tiles has
constexpr int kTargetBlocks = 2 * kNumSMs, kMostParts = 32;
size_t lora_workspace(long long tokens, int max_rank) {
    const long long split = tokens * kMostParts < (long long)kTargetBlocks * kTileRows ? tokens * kMostParts
                                                                                      : (long long)kTargetBlocks * kTileRows;
    return ((size_t)(tokens > split ? tokens : split) * (size_t)max_rank * 4 + 15) / 16 * 16 + 16;
}

int launch_lora_plan(const int* offsets, const int* ids, int num_seqs, int num_tokens, int num_adapters, void* plan,
                     cudaStream_t st) {
    return launch_k(lora_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, offsets, ids, num_seqs, num_tokens,
                    num_adapters, static_cast<int*>(plan)) == cudaSuccess
               ? 0
               : -1;
}

int launch_lora(const LoraCall& c, cudaStream_t st) {
    if (launch_k(lora_shrink_kernel, dim3((unsigned)c.num_tokens), dim3(256), 0, st, c) != cudaSuccess) return -1;
    const dim3 grid((unsigned)c.num_tokens, (unsigned)((c.n + 255) / 256));
    return launch_k(lora_expand_kernel, grid, dim3(256), 0, st, c) == cudaSuccess ? 0 : -1;
}

}  // namespace batch
}  // namespace cb
