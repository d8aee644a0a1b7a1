// Low-rank adapters of many requests: a plan that groups a batch's rows by adapter, then two products with each
// tile's adapter, the low-rank one in fp32 between them. Three ways, by the measurements at the end of this file:
// one kernel, a cluster of blocks a tile (lora_few_kernel); two kernels with the sums in the workspace (lora_shrink_kernel,
// lora_expand_kernel); and for much work the second product, or both, by lora_tc.cu. What a call has to move is x, the base and
// the result once and the adapters it uses, 2 bytes each; of that 9288 rows of 2048 into 8192 reach 4.0 TB/s (85 us).
#include <algorithm>
#include <atomic>

#include "../common.cuh"
#include "batch_ops.h"
#include "lora_plan.cuh"

namespace cb {
namespace batch {

namespace {

// ---------------------------------------------------------------- plan
// One block, latency: one sequence 8 us, 64 or 128 of them 11.5, 300 14, 1024 37, 4096 of 16 rows 123 (each thread adds up the
// lengths before its own among 1024); a warp writes a sequence's rows, one of 9000 10 us, of 65536 25.
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
    const PlanLayout at(num_seqs, num_tokens, num_adapters);
    int *starts = plan + at.starts, *tile_starts = plan + at.tile_starts, *wide_starts = plan + at.wide_starts;
    int* cursors = plan + at.cursors;
    int* rows = plan + at.rows;
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
    for (int a = t; a <= num_adapters; a += kPlanThreads) cursors[a] = 0;
    __syncthreads();
    for (int b = t; b < num_seqs; b += kPlanThreads) atomicAdd(&cursors[adapter_of(b)], offsets[b + 1] - offsets[b]);
    __syncthreads();
    int row0 = 0, tile0 = 0, wide0 = 0;
    for (int a0 = 0; a0 <= num_adapters; a0 += kPlanThreads) {
        const int a = a0 + t, n = a <= num_adapters ? cursors[a] : 0;
        int total = 0;
        const int start = row0 + block_scan(n, warp_sums, &total);
        row0 += total;
        const int tile = tile0 + block_scan(a < num_adapters ? (n + kTileRows - 1) / kTileRows : 0, warp_sums, &total);
        tile0 += total;
        const int wide = wide0 + block_scan(a < num_adapters ? (n + kWideRows - 1) / kWideRows : 0, warp_sums, &total);
        wide0 += total;
        if (a <= num_adapters) {
            starts[a] = start;
            tile_starts[a] = tile;
            wide_starts[a] = wide;
            cursors[a] = start;
        }
    }
    __syncthreads();
    if (t < kHeadInts) {
        const int some = starts[num_adapters];
        const int head[kHeadInts] = {num_seqs, num_tokens, num_adapters, some, tile0, row0 - some, wide0};
        plan[t] = head[t];
    }
    auto list = [&](int4* tiles, const int* first_of, int n, int height) {
        for (int i = t; i < n; i += kPlanThreads) {
            int lo = 0, hi = num_adapters;  // the last adapter whose tiles begin at or before i and that has any
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (first_of[mid] <= i) lo = mid; else hi = mid;
            }
            const int first = starts[lo] + (i - first_of[lo]) * height;
            tiles[i] = make_int4(lo, first, min(height, starts[lo + 1] - first), 0);
        }
    };
    list(reinterpret_cast<int4*>(plan + at.tiles), tile_starts, tile0, kTileRows);
    list(reinterpret_cast<int4*>(plan + at.wide), wide_starts, wide0, kWideRows);
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
            place = cursors[id];
            for (int j = 0; j < t; ++j) place += s_id[j] == id ? s_len[j] : 0;
            s_place[t] = place;
        }
        __syncthreads();
        if (t < n) atomicAdd(&cursors[id], len);
        for (int j = t >> 5; j < n; j += kPlanThreads / 32)
            for (int i = t & 31; i < s_len[j]; i += 32) rows[s_place[j] + i] = offsets[b0 + j] + i;
        __syncthreads();
    }
}

// ---------------------------------------------------------------- products
// Both products go tile by tile: up to 64 rows of one adapter. The first one's work is (tile, part of K).
__device__ __forceinline__ bool open_plan(const LoraCall& c, Plan* p) {
    if (read_plan(c, p)) return true;
    report_dev_error(kDevBadList);
    return false;
}
__device__ __forceinline__ int rank_of(const LoraCall& c, int adapter) {
    const int r = c.ranks ? __ldg(c.ranks + adapter) : c.max_rank;
    if (r >= 0 && r <= c.max_rank) return r;
    report_dev_error(kDevBadList);
    return 0;
}

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void copy16_or_zero(uint32_t to, const void* from, bool live) {
    copy_or_zero(to, from, live ? 16 : 0);
}
// 16 bytes that are read once
__device__ __forceinline__ uint4 ldg_nc(const __half* p) {
    const int4 v = ldg_nc_v4(p);
    return make_uint4((unsigned)v.x, (unsigned)v.y, (unsigned)v.z, (unsigned)v.w);
}

__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// ---- x A^T
constexpr int kThreads = 256, kWarps = kThreads / 32, kChunk = 128;  // K elements a stage
// stages of the ring for a padded rank: 80 to 160 KB
__host__ __device__ constexpr int stages_of(int rp) { return rp <= 64 ? 4 : rp <= 128 ? 3 : 2; }
__host__ __device__ constexpr int ring_bytes(int rp) { return stages_of(rp) * (kTileRows + rp) * 2 * kChunk; }

// Few rows (8 at most): the adapter's rows are the 16 rows of the product, the batch's its 8 columns. K is
// free to be dealt out in any order, so a lane takes 8 consecutive elements of its row, one 16-byte load, as
// its share of two steps; nothing passes through shared memory but the warps' sums.
__device__ void shrink_few(const LoraCall& c, const Plan& p, const int4& tile, int rank, int k0, int k1, float* out) {
    __shared__ float s_sum[kWarps][16 * 8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int blocks = (rank + 15) / 16;  // of 16 rows
    int split = 1;                        // warps that share one over K
    while (split * 2 * blocks <= kWarps) split *= 2;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const __half* x = g < tile.z ? c.x + (long long)__ldg(p.row + tile.y + g) * c.x_stride : nullptr;
    for (int u0 = 0; u0 < blocks * split; u0 += kWarps) {
        const int u = u0 + warp, block = u / split, part = u % split;
        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (u < blocks * split) {
            const int r = block * 16 + g, steps = (k1 - k0 + 31) / 32;
            const __half* a = c.a + ((long long)tile.x * c.max_rank + r) * c.k;
            const int from = k0 + steps * part / split * 32, to = min(k1, k0 + steps * (part + 1) / split * 32);
#pragma unroll 4
            for (int k = from; k < to; k += 32) {
                const int at = k + 8 * t;
                const bool in = at < to;
                const uint4 lo = in && r < rank ? ldg_nc(a + at) : zero;
                const uint4 hi = in && r + 8 < rank ? ldg_nc(a + 8LL * c.k + at) : zero;
                const uint4 v = in && x ? __ldg(reinterpret_cast<const uint4*>(x + at)) : zero;
                mma_16816(d, lo.x, hi.x, lo.y, hi.y, v.x, v.y);
                mma_16816(d, lo.z, hi.z, lo.w, hi.w, v.z, v.w);
            }
        }
        if (split > 1) {
            __syncthreads();
            if (u < blocks * split) *reinterpret_cast<float4*>(&s_sum[warp][4 * lane]) = make_float4(d[0], d[1], d[2], d[3]);
            __syncthreads();
            if (u >= blocks * split || part) continue;
            for (int i = 1; i < split; ++i) {
                const float4 o = *reinterpret_cast<const float4*>(&s_sum[warp + i][4 * lane]);
                d[0] += o.x, d[1] += o.y, d[2] += o.z, d[3] += o.w;
            }
        } else if (u >= blocks) {
            continue;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = block * 16 + g + 8 * (i >> 1), row = 2 * t + (i & 1);
            // an infinity of x makes a NaN of the zeros that stand for rows past the rank
            if (row < tile.z && r < c.max_rank) out[(long long)row * c.max_rank + r] = r < rank ? d[i] : 0.0f;
        }
    }
}

// Many rows: both operands pass through a ring of shared-memory stages of 128 elements of K (two blocks of 128-byte rows, whose
// 16-byte pieces are swapped about by the row's low bits). What the matrix loads move bounds it, so a warp has 32 of
// the tile's rows and up to 64 of the adapter's, and warps share the steps of a stage before they share those: 16 x 32
// a warp read twice as much, and 9000 rows of 2048 took 19 us where this takes 16.5 (its bytes 6).
template <int RP>
__device__ void shrink_many(const LoraCall& c, const Plan& p, const int4& tile, int rank, int k0, int k1, float* out,
                            uint8_t* smem) {
    constexpr int kStages = stages_of(RP), kBlockBytes = (kTileRows + RP) * 128, kBlocks = kChunk / 64, kStageBytes = kBlocks * kBlockBytes;
    constexpr int kSplitK = RP <= 64 ? 4 : RP <= 128 ? 2 : 1, kSplitN = kWarps / 2 / kSplitK;
    constexpr int kCols = RP / kSplitN, kTilesN = kCols / 8, kSteps = kChunk / 16 / kSplitK;  // of a warp
    static_assert(kWarps * 2 * kTilesN * 512 <= kStages * kStageBytes, "the warps' sums fit into the ring");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, m = warp & 1, n = warp >> 1 & (kSplitN - 1), part = warp / (2 * kSplitN);
    const uint32_t base = smem_u32(smem);
    const int piece = threadIdx.x & 7, row = threadIdx.x >> 3;  // a thread copies one piece of every 32nd row
    const __half* xp[kTileRows / 32];
#pragma unroll
    for (int i = 0; i < kTileRows / 32; ++i)
        xp[i] = row + 32 * i < tile.z ? c.x + (long long)__ldg(p.row + tile.y + row + 32 * i) * c.x_stride : nullptr;
    const __half* ap = c.a + ((long long)tile.x * c.max_rank + row) * c.k;
    const uint32_t to = base + row * 128 + ((piece ^ (row & 7)) << 4);
    auto load = [&](int chunk, int stage) {
#pragma unroll
        for (int block = 0; block < kBlocks; ++block) {
            const int k = k0 + chunk * kChunk + block * 64 + piece * 8;
            const uint32_t at = to + stage * kStageBytes + block * kBlockBytes;
#pragma unroll
            for (int i = 0; i < kTileRows / 32; ++i) copy16_or_zero(at + i * 32 * 128, xp[i] ? xp[i] + k : c.x, xp[i] && k < k1);
#pragma unroll
            for (int i = 0; i < (RP + 31) / 32; ++i)
                if (RP >= 32 || row < RP) {
                    const bool live = row + 32 * i < rank && k < k1;
                    copy16_or_zero(at + (kTileRows + i * 32) * 128, live ? ap + (long long)i * 32 * c.k + k : c.a, live);
                }
        }
    };
    float d[2][kTilesN][4];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < kTilesN; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) d[u][j][i] = 0.0f;
    const int chunks = (k1 - k0 + kChunk - 1) / kChunk;
    __syncthreads();  // the stages of the tile before are read
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
        if (i < chunks) load(i, i);
        cp_async_commit();
    }
    const int xr = m * 32 + (lane & 15), br = kTileRows + n * kCols + (lane & 7) + ((lane >> 4) << 3);
    for (int chunk = 0; chunk < chunks; ++chunk) {
        cp_async_wait<kStages - 2>();
        __syncthreads();
        if (chunk + kStages - 1 < chunks) load(chunk + kStages - 1, (chunk + kStages - 1) % kStages);
        cp_async_commit();
        const uint32_t stage = base + (chunk % kStages) * kStageBytes;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int step = part * kSteps + i, s = step & 3;
            const uint32_t at = stage + (step >> 2) * kBlockBytes;
            uint32_t a[2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) ldmatrix_x4(a[u], at + (xr + u * 16) * 128 + (((2 * s + (lane >> 4)) ^ (xr & 7)) << 4));
#pragma unroll
            for (int j = 0; j < kTilesN; j += 2) {
                uint32_t b[4];  // two blocks of 8 rows, both halves of the step
                const int r = br + j * 8;
                ldmatrix_x4(b, at + r * 128 + (((2 * s + ((lane >> 3) & 1)) ^ (r & 7)) << 4));
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    mma_16816(d[u][j], a[u][0], a[u][1], a[u][2], a[u][3], b[0], b[1]);
                    mma_16816(d[u][j + 1], a[u][0], a[u][1], a[u][2], a[u][3], b[2], b[3]);
                }
            }
        }
    }
    cp_async_wait<0>();
    if (kSplitK > 1) {  // the sums of the warps that had the first steps, and after them those of the others
        __syncthreads();  // all stages are read
        float4* sums = reinterpret_cast<float4*>(smem) + lane;
        if (part)
#pragma unroll
            for (int j = 0; j < 2 * kTilesN; ++j) {
                const float* v = d[j / kTilesN][j % kTilesN];
                sums[(warp * 2 * kTilesN + j) * 32] = make_float4(v[0], v[1], v[2], v[3]);
            }
        __syncthreads();
        if (part) return;
#pragma unroll
        for (int other = 1; other < kSplitK; ++other)
#pragma unroll
            for (int j = 0; j < 2 * kTilesN; ++j) {
                const float4 o = sums[((warp + other * 2 * kSplitN) * 2 * kTilesN + j) * 32];
                float* v = d[j / kTilesN][j % kTilesN];
                v[0] += o.x, v[1] += o.y, v[2] += o.z, v[3] += o.w;
            }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < kTilesN; ++j) {
            const int r = n * kCols + j * 8 + 2 * (lane & 3);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = m * 32 + u * 16 + (lane >> 2) + 8 * i;
                if (at < tile.z && r < c.max_rank)
                    *reinterpret_cast<float2*>(out + (long long)at * c.max_rank + r) =
                        make_float2(r < rank ? d[u][j][2 * i] : 0.0f, r + 1 < rank ? d[u][j][2 * i + 1] : 0.0f);  // as shrink_few
            }
        }
}

constexpr int kFewRows = 8;

__global__ void __launch_bounds__(kThreads, 1) lora_shrink_kernel(LoraCall c) {
    extern __shared__ __align__(128) uint8_t smem[];
    pdl_launch_dependents();
    pdl_wait();
    Plan p;
    if (!open_plan(c, &p)) return;
    const int parts = parts_of(p.tiles, c.k);
    const int chunks = (c.k + kChunk - 1) / kChunk;
    for (int item = blockIdx.x; item < p.tiles * parts; item += gridDim.x) {
        const int part = item % parts;
        const int4 tile = __ldg(p.tile + item / parts);
        const int rank = rank_of(c, tile.x);
        const int k0 = (int)((long long)chunks * part / parts) * kChunk;
        const int k1 = min(c.k, (int)((long long)chunks * (part + 1) / parts) * kChunk);
        float* out = c.ws + ((long long)part * p.rows + tile.y) * c.max_rank;
        if (rank == 0) continue;
        if (tile.z <= kFewRows) shrink_few(c, p, tile, rank, k0, k1, out);
        else if (rank <= 16) shrink_many<16>(c, p, tile, rank, k0, k1, out, smem);
        else if (rank <= 32) shrink_many<32>(c, p, tile, rank, k0, k1, out, smem);
        else if (rank <= 64) shrink_many<64>(c, p, tile, rank, k0, k1, out, smem);
        else if (rank <= 128) shrink_many<128>(c, p, tile, rank, k0, k1, out, smem);
        else shrink_many<256>(c, p, tile, rank, k0, k1, out, smem);
    }
}

// ---- base + scale * h B^T
// A tile's low-rank rows h go to shared memory once, as two fp16 numbers an element (h = 2^e (high + low), e by the
// row's largest finite element, so that neither overflows and 22 bits are kept), and the block's warps take 32 outputs of
// all 64 rows at a time. The columns of the products are dealt out so that a lane's are 8 consecutive outputs (one
// 16-byte load and store a row), the steps over the rank so that a lane's elements of B are 4 consecutive ones.
constexpr int kWarpCols = 32, kBlockCols = kWarps * kWarpCols;

__host__ __device__ inline int padded_rank(int r) { return r <= 16 ? 16 : r <= 32 ? 32 : r <= 64 ? 64 : r <= 128 ? 128 : 256; }
__host__ __device__ inline int h_stride(int rp) { return 2 * rp + 16; }  // fp16 elements: high, low, padding against bank conflicts

// A tile's h into shared memory: four threads a row, each with every fourth four of its elements.
template <int RP>
__device__ __forceinline__ void store_h(const LoraCall& c, const int4& tile, const float4 (&v)[RP / 16], __half* s_h, float* s_scale) {
    const int row = threadIdx.x >> 2, q = threadIdx.x & 3;
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < RP / 16; ++i) top = fmaxf(top, largest_finite(v[i]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = exponent_of(top);
    const float down = two_to(-e);
    __half* to = s_h + row * h_stride(RP);
#pragma unroll
    for (int i = 0; i < RP / 16; ++i) {
        __half hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) two_halves((&v[i].x)[j] * down, &hi[j], &lo[j]);
        const int r = 16 * i + 4 * q;
        *reinterpret_cast<uint2*>(to + r) = *reinterpret_cast<const uint2*>(hi);
        *reinterpret_cast<uint2*>(to + RP + r) = *reinterpret_cast<const uint2*>(lo);
    }
    if (q == 0) s_scale[row] = (c.scales ? __ldg(c.scales + tile.x) : 1.0f) * two_to(e);
}
template <int RP>
__device__ void load_h(const LoraCall& c, const Plan& p, const int4& tile, int rank, int parts, __half* s_h, float* s_scale) {
    const int row = threadIdx.x >> 2, q = threadIdx.x & 3;
    float4 v[RP / 16];
    sum_parts<RP / 16>(c.ws + (long long)(tile.y + row) * c.max_rank + 4 * q, (long long)p.rows * c.max_rank, parts,
                       row < tile.z ? rank - 4 * q : 0, v);
    store_h<RP>(c, tile, v, s_h, s_scale);
}

// 32 outputs of up to 16 * MT rows, a warp.
template <int RP, int MT>
__device__ __forceinline__ void expand_warp(const LoraCall& c, const int4& tile, int rank, int n0, int row0,
                                            const __half* s_h, const float* s_scale, const int* s_row) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, col = n0 + 8 * t;
    uint4 y[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = row0 + m * 16 + g + 8 * i;
            y[m][i] = make_uint4(0, 0, 0, 0);
            if (c.base && row < tile.z && col < c.n)
                y[m][i] = *reinterpret_cast<const uint4*>(c.base + (long long)s_row[row] * c.base_stride + col);
        }
    float d[MT][4][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) d[m][j][i] = 0.0f;
    if (RP) {
        const int steps = (rank + 15) / 16;
        const __half* b = c.b + ((long long)tile.x * c.n + n0 + (g >> 1) * 8 + (g & 1)) * c.max_rank + 4 * t;
        const bool live = n0 + (g >> 1) * 8 < c.n;  // its 8 outputs exist or do not
#pragma unroll 4
        for (int s = 0; s < steps; ++s) {
            uint2 bv[4];
            const int r = 16 * s + 4 * t, left = rank - r;  // elements that this lane has of the rank
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                bv[j] = make_uint2(0, 0);
                if (live && left > 0) bv[j] = __ldg(reinterpret_cast<const uint2*>(b + (long long)2 * j * c.max_rank + 16 * s));
                if (left < 4) {  // what follows the rank may hold anything
                    bv[j].x = left >= 2 ? bv[j].x : left == 1 ? bv[j].x & 0xffffu : 0u;
                    bv[j].y = left == 3 ? bv[j].y & 0xffffu : 0u;
                }
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const __half* h = s_h + (row0 + m * 16 + g) * h_stride(RP) + r;
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    const uint2 lo = *reinterpret_cast<const uint2*>(h + part * RP);
                    const uint2 hi = *reinterpret_cast<const uint2*>(h + part * RP + 8 * h_stride(RP));
#pragma unroll
                    for (int j = 0; j < 4; ++j) mma_16816(d[m][j], lo.x, hi.x, lo.y, hi.y, bv[j].x, bv[j].y);
                }
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = row0 + m * 16 + g + 8 * i;
            if (row >= tile.z || col >= c.n) continue;
            uint4 out = y[m][i];
            if (RP) {
                const float scale = s_scale[row];
                __half2* o = reinterpret_cast<__half2*>(&out);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 v = __half22float2(o[j]);
                    o[j] = __floats2half2_rn(fmaf(scale, d[m][j][2 * i], v.x), fmaf(scale, d[m][j][2 * i + 1], v.y));
                }
            }
            *reinterpret_cast<uint4*>(c.out + (long long)s_row[row] * c.out_stride + col) = out;
        }
}

template <int RP>
__device__ __forceinline__ void expand_rows(const LoraCall& c, const int4& tile, int rank, int n0, const __half* s_h,
                                            const float* s_scale, const int* s_row) {
    if (tile.z <= 16) expand_warp<RP, 1>(c, tile, rank, n0, 0, s_h, s_scale, s_row);
    else
        for (int row0 = 0; row0 < tile.z; row0 += 32) expand_warp<RP, 2>(c, tile, rank, n0, row0, s_h, s_scale, s_row);
}

__global__ void __launch_bounds__(kThreads, 2) lora_expand_kernel(LoraCall c) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float s_scale[kTileRows];
    __shared__ int s_row[kTileRows];
    pdl_launch_dependents();
    __half* s_h = reinterpret_cast<__half*>(smem);
    Plan p;
    if (!open_plan(c, &p)) {
        pdl_wait();
        return;
    }
    const int parts = parts_of(p.tiles, c.k), across = (c.n + kBlockCols - 1) / kBlockCols;
    // rows without an adapter follow as tiles of rank 0, where they have to be copied
    const int bare = c.base == c.out ? 0 : (p.bare + kTileRows - 1) / kTileRows;
    const long long items = (long long)(p.tiles + bare) * across;
    const long long first = items * blockIdx.x / gridDim.x, end = items * (blockIdx.x + 1) / gridDim.x;
    pdl_wait();
    int have = -1, rank = 0;
    int4 tile = make_int4(0, 0, 0, 0);
    for (long long item = first; item < end; ++item) {
        const int at = (int)(item / across), n0 = (int)(item % across) * kBlockCols + (threadIdx.x >> 5) * kWarpCols;
        if (at != have) {
            have = at;
            __syncthreads();  // the tile before is done with
            if (at < p.tiles) {
                tile = __ldg(p.tile + at);
                rank = rank_of(c, tile.x);
            } else {
                const int i = (at - p.tiles) * kTileRows;
                tile = make_int4(0, p.rows + i, min(kTileRows, p.bare - i), 0);
                rank = 0;
            }
            if (threadIdx.x < tile.z) s_row[threadIdx.x] = __ldg(p.row + tile.y + threadIdx.x);
            if (rank > 128) load_h<256>(c, p, tile, rank, parts, s_h, s_scale);
            else if (rank > 64) load_h<128>(c, p, tile, rank, parts, s_h, s_scale);
            else if (rank > 32) load_h<64>(c, p, tile, rank, parts, s_h, s_scale);
            else if (rank > 16) load_h<32>(c, p, tile, rank, parts, s_h, s_scale);
            else if (rank > 0) load_h<16>(c, p, tile, rank, parts, s_h, s_scale);
            __syncthreads();
        }
        if (n0 >= c.n || (rank == 0 && c.base == c.out)) continue;
        if (rank > 128) expand_rows<256>(c, tile, rank, n0, s_h, s_scale, s_row);
        else if (rank > 64) expand_rows<128>(c, tile, rank, n0, s_h, s_scale, s_row);
        else if (rank > 32) expand_rows<64>(c, tile, rank, n0, s_h, s_scale, s_row);
        else if (rank > 16) expand_rows<32>(c, tile, rank, n0, s_h, s_scale, s_row);
        else if (rank > 0) expand_rows<16>(c, tile, rank, n0, s_h, s_scale, s_row);
        else expand_rows<0>(c, tile, rank, n0, s_h, s_scale, s_row);
    }
}

// ---- both products of few rows in one kernel
// A cluster of blocks has a tile: each block the low-rank product of its share of K, in its shared memory, then, with
// the sums of all of them, its share of the outputs. One launch, and h never leaves the SMs; but a tile's rows have one
// cluster alone.
constexpr int kClusterRank = 64;

// Where it is the faster one: up to 8 rows for each group that there can be (a block's warps take 8 at a time), and no
// more of B for a cluster than 2^18 elements unless clusters are many. Whole calls, two kernels / this one, us: K and outputs
// 2048, rank 16, one sequence of 8 tokens 8.3 / 6.3, of 32 9.4 / 10.4, 64 sequences of 8 adapters 9.6 / 8.3, 64 of 64 adapters
// 12.3 / 8.3; rank 64, 64 of 64 16.5 / 12.4, 256 of 256 49 / 37; 8192 outputs, rank 64, 4 of 4 10.4 / 14.4, 16 of 16 15.7 / 14.4.
// Those are adapters that are all used. The rule knows how many there are, not how many the batch uses: where 64 tokens are all of
// one of 64 adapters, one cluster has them, and this kernel is the slower one: 2048 outputs, rank 16 10.4 / 18.6, rank 64 14.5 /
// 28.8; 14336 outputs, rank 64 16.5 / 73.8; K 14336, 4096 outputs, rank 64 20.5 / 83.6. Three quarters of them of one adapter: 10.6
// / 18.5, 16.5 / 26.7, 30.8 / 70.3, 28.8 / 96.6.
inline bool cluster_pays(const LoraCall& c, long long tiles) {
    const long long groups = c.num_seqs < c.num_adapters ? c.num_seqs : c.num_adapters;
    return c.max_rank <= kClusterRank && c.num_tokens <= kFewRows * groups && ((long long)c.n * c.max_rank <= 1 << 18 || tiles >= 16);
}
// Blocks of a cluster: 8 while two blocks a SM are enough for them, else 4 (64 sequences of 64 adapters, rank 64, K and
// outputs 2048: 17.6 and 12.4 us).
inline int cluster_blocks(long long tiles) { return tiles * 8 <= 2 * kNumSMs ? 8 : 4; }

__device__ __forceinline__ unsigned cluster_size() {
    unsigned n;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
    return n;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// 16 bytes of another block's shared memory at the place that `at` is in this one's
__device__ __forceinline__ float4 load_of_block(const float* at, unsigned block) {
    uint32_t there;
    float4 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(smem_u32(at)), "r"(block));
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(there) : "memory");
    return v;
}

template <int RP>
__device__ void gather_h(const LoraCall& c, const int4& tile, int rank, const float* s_sum, __half* s_h, float* s_scale) {
    const int row = threadIdx.x >> 2, q = threadIdx.x & 3;
    const unsigned blocks = cluster_size();
    float4 v[RP / 16];
#pragma unroll
    for (int i = 0; i < RP / 16; ++i) {
        v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (row < tile.z && 16 * i + 4 * q < rank)
#pragma unroll 4
            for (unsigned block = 0; block < blocks; ++block) {
                const float4 h = load_of_block(s_sum + row * c.max_rank + 16 * i + 4 * q, block);
                v[i].x += h.x, v[i].y += h.y, v[i].z += h.z, v[i].w += h.w;
            }
    }
    store_h<RP>(c, tile, v, s_h, s_scale);
}

__global__ void __launch_bounds__(kThreads, 2) lora_few_kernel(LoraCall c) {
    extern __shared__ __align__(128) uint8_t smem[];  // the block's sums [64][max_rank], then h
    __shared__ float s_scale[kTileRows];
    __shared__ int s_row[kTileRows];
    pdl_launch_dependents();
    pdl_wait();
    Plan p;
    if (!open_plan(c, &p)) return;
    const int blocks = (int)cluster_size(), tile_no = blockIdx.x / blocks, me = blockIdx.x % blocks;
    const int bare = c.base == c.out ? 0 : (p.bare + kTileRows - 1) / kTileRows;
    if (tile_no >= p.tiles + bare) return;  // and so do the cluster's others
    float* s_sum = reinterpret_cast<float*>(smem);
    __half* s_h = reinterpret_cast<__half*>(smem + kTileRows * c.max_rank * 4);
    const int i0 = (tile_no - p.tiles) * kTileRows;
    const int4 tile = tile_no < p.tiles ? __ldg(p.tile + tile_no) : make_int4(-1, p.rows + i0, min(kTileRows, p.bare - i0), 0);
    const int rank = tile.x < 0 ? 0 : rank_of(c, tile.x);
    const int columns = (c.n + 31) / 32, from = columns * me / blocks, to = columns * (me + 1) / blocks;  // blocks of 32 outputs
    if (threadIdx.x < tile.z) s_row[threadIdx.x] = __ldg(p.row + tile.y + threadIdx.x);
    if (rank) {
        // the block's rows of B on their way to L2 meanwhile
        const char* b = reinterpret_cast<const char*>(c.b + ((long long)tile.x * c.n + from * 32) * c.max_rank);
        const long long bytes = (long long)(min(to * 32, c.n) - from * 32) * c.max_rank * 2;
        for (long long at = threadIdx.x * 128LL; at < bytes; at += kThreads * 128LL) prefetch_l2(b + at);
        const int steps = (c.k + 31) / 32, k0 = min(c.k, steps * me / blocks * 32), k1 = min(c.k, steps * (me + 1) / blocks * 32);
        for (int r0 = 0; r0 < tile.z; r0 += kFewRows) {
            const int4 some = make_int4(tile.x, tile.y + r0, min(kFewRows, tile.z - r0), 0);
            shrink_few(c, p, some, rank, k0, k1, s_sum + r0 * c.max_rank);
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();  // all sums are there
        if (rank > 32) gather_h<64>(c, tile, rank, s_sum, s_h, s_scale);
        else if (rank > 16) gather_h<32>(c, tile, rank, s_sum, s_h, s_scale);
        else gather_h<16>(c, tile, rank, s_sum, s_h, s_scale);
        __syncwarp();
        cluster_arrive();  // this block has read the others' sums
    }
    __syncthreads();
    if (rank || c.base != c.out)
        for (int column = from + (threadIdx.x >> 5); column < to; column += kWarps) {
            if (rank > 32) expand_rows<64>(c, tile, rank, column * 32, s_h, s_scale, s_row);
            else if (rank > 16) expand_rows<32>(c, tile, rank, column * 32, s_h, s_scale, s_row);
            else if (rank > 0) expand_rows<16>(c, tile, rank, column * 32, s_h, s_scale, s_row);
            else expand_rows<0>(c, tile, rank, column * 32, s_h, s_scale, s_row);
        }
    if (rank) {
        __syncwarp();
        cluster_wait();  // no block leaves while its sums are read
    }
}

int launch_few(const LoraCall& c, long long tiles, int blocks, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * blocks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kTileRows * c.max_rank * 4 + kTileRows * h_stride(padded_rank(c.max_rank)) * 2;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, lora_few_kernel, c) == cudaSuccess ? 0 : -1;
}

}  // namespace

size_t lora_plan_bytes(long long seqs, long long tokens, long long adapters) {
    const size_t ints = (size_t)(PlanLayout(seqs, tokens, adapters).rows + tokens);
    return (ints * 4 + 15) / 16 * 16;
}

// parts * rows is at most kMostParts * tokens, and where there is more than one part at most a wide tile's rows a block
size_t lora_workspace(long long tokens, int max_rank) {
    const long long many = tokens * kMostParts, few = (long long)kTargetBlocks * kWideRows, split = many < few ? many : few;
    return ((size_t)(tokens > split ? tokens : split) * (size_t)max_rank * 4 + 15) / 16 * 16 + 16;
}

int launch_lora_plan(const int* offsets, const int* ids, int num_seqs, int num_tokens, int num_adapters, void* plan,
                     cudaStream_t st) {
    return launch_k(lora_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, offsets, ids, num_seqs, num_tokens,
                    num_adapters, static_cast<int*>(plan)) == cudaSuccess
               ? 0
               : -1;
}

// The device error word's address on the current device, for the kernel that is compiled by itself.
unsigned* error_word(int dev) {
    static std::atomic<unsigned*> known[64];
    unsigned* p = known[dev & 63].load();
    void* at = nullptr;
    if (!p && cudaGetSymbolAddress(&at, g_dev_error) == cudaSuccess) known[dev & 63].store(p = static_cast<unsigned*>(at));
    return p;
}

// Which products lora_tc.cu's kernels have, from 64 tokens on, by the work (tokens * outputs * rank). Whole calls, us.
// Both from 2^25 on where the rank is above 32; both by mma.sync / tcgen05: rank 64, K and outputs 2048, 128 tokens 14.4 / 14.5, 256 14.4 /
// 14.4, 512 18.5 / 16.5, 1024 20.6 / 16.5; K 2048, 8192 outputs 64 tokens 14.5 / 14.4, 128 of 8 adapters 16.5 / 18.6, 512 22.6 / 18.5;
// rank 128, K 14336, 4096 outputs 64 tokens 26.8 / 23.1, 256 47.7 / 28.7. With a rank up to 32 mma.sync keeps up, and starts
// sooner: both from 2^27 on and 2^25 elements of x (rank 16, 1024 / 4096 tokens of 8 adapters, mma.sync first / tcgen05 both: K
// 2048, 8192 outputs 26.7 / 28.7 and 42.2 / 44.1, 16384 of them 125 / 121; K 14336 28.7 / 32.9 and 52.9 / 54.9, 8192 90 / 85), only the
// second below that (K 2048, 8192 outputs, both by mma.sync / it alone: 1024 tokens 22.4 / 20.6, 2048 34.2 / 27.5).
constexpr int kWideTokens = 64, kSmallRank = 32;
constexpr long long kWideWork = 1LL << 25, kWideWorkSmallRank = 1LL << 27, kWideElements = 1LL << 25;

int launch_lora(const LoraCall& c, cudaStream_t st) {
    const int rp = padded_rank(c.max_rank);
    const int shrink_smem = ring_bytes(rp), expand_smem = kTileRows * h_stride(rp) * 2;
    static std::atomic<unsigned long long> set{0};  // a bit a device
    int dev = 0;
    cudaGetDevice(&dev);
    if (!(set.load() >> (dev & 63) & 1)) {
        if (cudaFuncSetAttribute(lora_shrink_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 ring_bytes(kLoraMaxRank)) != cudaSuccess ||
            cudaFuncSetAttribute(lora_expand_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kTileRows * h_stride(kLoraMaxRank) * 2) != cudaSuccess)
            return -1;
        set.fetch_or(1ull << (dev & 63));
    }
    const long long all_tiles = most_tiles(c.num_seqs, c.num_tokens, c.num_adapters) + (c.num_tokens + kTileRows - 1) / kTileRows;
    if (cluster_pays(c, all_tiles)) return launch_few(c, all_tiles, cluster_blocks(all_tiles), st);
    // The second kernel reads the plan and the base before it waits for the first one, so that one starts behind all
    // that wrote them, whatever the caller's thread has switched on.
    pdl_scope behind(false);
    const long long work = (long long)c.num_tokens * c.n * c.max_rank;
    const bool wide = c.num_tokens >= kWideTokens && c.max_rank <= kLoraWideRank && c.num_adapters > 0 &&
                      work >= (c.max_rank > kSmallRank ? kWideWork : kWideWorkSmallRank);
    if (wide && (c.max_rank > kSmallRank || (long long)c.num_tokens * c.k >= kWideElements)) {
        if (launch_lora_shrink_wide(c, error_word(dev), st)) return -1;
        pdl_scope beside(true);  // as below
        return launch_lora_expand_wide(c, true, error_word(dev), st);
    }
    // as many blocks as the most tiles that there can be need, one or two for each SM at most
    const long long tiles = most_tiles(c.num_seqs, c.num_tokens, c.num_adapters);
    const long long shrink = std::min<long long>(kTargetBlocks, tiles * parts_of(1, c.k));
    if (shrink > 0 && launch_k(lora_shrink_kernel, dim3((unsigned)shrink), dim3(kThreads), shrink_smem, st, c) != cudaSuccess)
        return -1;
    const long long across = (c.n + kBlockCols - 1) / kBlockCols;
    const long long expand = std::min<long long>(kTargetBlocks, (tiles + (c.num_tokens + kTileRows - 1) / kTileRows) * across);
    pdl_scope beside(shrink > 0);  // the second kernel starts while the first one ends, and waits for it
    if (wide) return launch_lora_expand_wide(c, false, error_word(dev), st);
    return launch_k(lora_expand_kernel, dim3((unsigned)expand), dim3(kThreads), expand_smem, st, c) == cudaSuccess ? 0 : -1;
}

}  // namespace batch
}  // namespace cb
