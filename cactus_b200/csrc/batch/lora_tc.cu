// Low-rank adapters, many rows, on tcgen05. First x A^T (lora_shrink_wide_kernel): tiles of rows of one adapter, cut over
// K; 8 warps copy both operands into a ring of stages, one issues the products, and the 8 store the sums from TMEM.
// Against mma.sync (lora.cu), whose few warps wait for their matrix loads, whole calls with the same second product, us:
// rank 64, 9288 rows of 2048, 8192 outputs 86 / 85; 16384 rows of 14336, rank 128, 4096 outputs 296 / 169.
// Then base + scale * h B^T, h being those sums. What an output costs is the base's element in and its own out, 4 bytes for 2 *
// rank operations, so all is built to keep those moving: a persistent block for each SM goes over items of 128 rows of one
// adapter and 128 outputs.
//   loaders   (8 warps) B's rows and the base's rows into a ring of stages, 16 bytes a copy, items ahead; for each new
//             tile h as two fp16 numbers an element (h = 2^e (high + low), e by the row's largest finite element, so that
//             neither overflows and 22 bits are kept), in the operands' swizzled layout;
//   epilogue  (8 warps) sums from TMEM, a thread a row's 64 outputs; the results replace the base's elements in
//             shared memory and leave from there in whole rows;
//   issuer    (1 warp) the products: steps of 16 over the rank, first with the high parts, then with the low ones.
// 9288 rows of 8192 outputs, ranks 16 to 64: 70 us behind the first product, 4.2 TB/s (copying the base alone takes 60); by
// mma.sync with operands through shared memory 100, straight from and to memory 140. What is left over the copy: a tile's
// first h, which nothing hides at a block's start, and the copies of B (16 KB an item).
// This file is compiled as whole-program device code (build.py WHOLE_PROGRAM).
#include <algorithm>
#include <atomic>

#include "lora_plan.cuh"

namespace cb {
namespace batch {

namespace {

constexpr int kCols = 128;
constexpr int kLoaders = 8, kEpilogue = 8, kIssuer = kLoaders + kEpilogue, kThreads = (kIssuer + 1) * 32;
constexpr int kLoadThreads = 32 * kLoaders;
constexpr int kRowLists = 4;  // tiles whose rows' places are kept: more than the ring has items

template <int RP>
struct Cfg {
    static constexpr int kStages = RP == 64 ? 3 : 2, kTilesH = RP == 64 ? 2 : 1;
    static constexpr int kLag = kStages - 2;  // items whose copies may be under way when an item is handed on
    static constexpr int kBytesH = 2 * kWideRows * RP * 2, kBytesB = kCols * RP * 2;
    static constexpr int kPitch = kCols * 2 + 16, kBytesY = kWideRows * kPitch;  // rows begin on other banks
    static constexpr int kB = kTilesH * kBytesH, kY = kB + kStages * kBytesB;
    static constexpr int smem = kY + kStages * kBytesY + 1024;
};

struct Args {
    LoraCall c;
    unsigned* err;
    bool split;  // the first product is lora_shrink_wide_kernel's, cut as split_of() says
};

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Shared-memory matrix descriptor, K-major with the 128-byte swizzle: 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
// kind::f16: D fp32, A and B fp16, M = 128, N = 128
constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(kCols >> 3) << 17) | ((128u >> 4) << 24);

__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t acc, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc),
        "r"(leader));
}
__device__ __forceinline__ void commit(uint32_t leader, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar)),
        "r"(leader)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
          "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr)
        : "memory");
}
template <int ID, int N>
__device__ __forceinline__ void named_barrier() { asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N) : "memory"); }

// Bounded; one wait that gives up makes all others give up too.
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, unsigned parity, volatile int* abort) {
    for (uint32_t i = 0; i < (1u << 24); ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 255) == 255 && *abort) return false;
    }
    *abort = 1;
    return false;
}

// ---- x A^T
// Which tiles this kernel goes over, and how many parts of K: what takes less, counted in elements of a row of either
// operand that a block goes through, one wave after another, and kPartCost of them for each part, which the second product's
// kernel has to add up. Whole calls with as many parts as there are SMs for / as many as here, us: rank 64, K 2048, 8192
// outputs, 1024 tokens 30.8 / 22.6; K 14336, 4096 outputs, 512 tokens 34.9 / 25.5. Tiles of 64 / 128 rows: rank 64, K 8192, 2048
// outputs, 16384 tokens 106 / 96; 18000 tokens of 40 adapters 115 / 129.
// Both products' kernels evaluate it and have to find the same: the same IEEE steps on the same numbers, none of which the
// compiler may join into another (kPartCost is a power of two, so that its products are exact besides).
constexpr float kPartCost = 65536.0f;
struct Split {
    int rows, tiles, parts;
};
__device__ __forceinline__ Split split_of(const LoraCall& c, const Plan& p) {
    auto cut = [&](int rows, int tiles) {
        const int best = (int)(sqrtf((float)c.k * (float)(rows + c.max_rank) / kPartCost) + 0.5f);
        return Split{rows, tiles, max(1, min(parts_of(tiles, c.k), best))};
    };
    auto cost = [&](const Split& s) {
        const float waves = (float)((s.tiles * s.parts + kTargetBlocks - 1) / kTargetBlocks);
        return waves * (float)c.k * (float)(s.rows + c.max_rank) / (float)s.parts + kPartCost * (float)s.parts;
    };
    const Split wide = cut(kWideRows, p.wide_tiles), narrow = cut(kTileRows, p.tiles);
    return cost(wide) < cost(narrow) ? wide : narrow;
}

// stages of the ring, in 192 KB (tiles of 64 rows, four stages instead of six: 18000 rows of 14336 of 40 adapters, rank 128, 246
// us for 234)
__host__ __device__ constexpr int shrink_stages(int rp, int rows) { return 192 * 1024 / (256 * (rp + rows)); }
template <int RP, int ROWS>
struct ShrinkCfg {
    static constexpr int kStages = shrink_stages(RP, ROWS), kLag = kStages - 2;
    static constexpr int kBlockX = ROWS * 128, kBlockA = RP * 128, kBlocks = 2, kChunk = 64 * kBlocks;  // rows of 64 elements of K
    static constexpr int kA = kBlocks * kBlockX, kStage = kA + kBlocks * kBlockA;
    static constexpr int smem = kStages * kStage + 1024;
};

template <int STAGES>
struct ShrinkBars {
    uint64_t full[STAGES], empty[STAGES], acc_full, acc_empty, drain;
};

template <int RP, int ROWS>
__device__ __forceinline__ void shrink_items(const Args& a, const Plan& p, int tiles, int parts, uint8_t* smem,
                                             ShrinkBars<shrink_stages(RP, kTileRows)>& b, uint32_t tmem, volatile int* abort) {
    using C = ShrinkCfg<RP, ROWS>;
    const int4* const list = ROWS == kWideRows ? p.wide : p.tile;
    const LoraCall& c = a.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int chunks = (c.k + C::kChunk - 1) / C::kChunk;
    int n = 0, product = 0;  // chunks and items with a product so far
    bool ok = true;
    for (int item = blockIdx.x; item < tiles * parts && ok; item += gridDim.x) {
        const int part = item % parts;
        const int4 tile = __ldg(list + item / parts);
        int rank = c.ranks ? __ldg(c.ranks + tile.x) : c.max_rank;
        if (rank < 0 || rank > c.max_rank) {
            if (tid == 0) atomicCAS(a.err, 0u, (unsigned)kDevBadList);
            rank = 0;
        }
        if (rank == 0) continue;
        const int from = (int)((long long)chunks * part / parts), count = (int)((long long)chunks * (part + 1) / parts) - from;
        const int padded = (rank + 15) / 16 * 16, live_cols = count ? rank : 0;  // without a K nothing is multiplied
        if (warp < kLoaders) {
            const int piece = tid & 7, row = tid >> 3;  // a thread copies one piece of every 32nd row
            const int k1 = min(c.k, (from + count) * C::kChunk);
            const __half* xp[ROWS / 32];
#pragma unroll
            for (int i = 0; i < ROWS / 32; ++i)
                xp[i] = row + 32 * i < tile.z ? c.x + (long long)__ldg(p.row + tile.y + row + 32 * i) * c.x_stride : nullptr;
            const __half* ap = c.a + ((long long)tile.x * c.max_rank + row) * c.k;
            const uint32_t to = smem_u32(smem) + row * 128 + ((piece ^ (row & 7)) << 4);
            auto hand_on = [&](int i) {  // chunk i's copies of this thread are there
                fence_proxy_async_shared();
                mbar_arrive(&b.full[(n + i) % C::kStages]);
            };
            for (int i = 0; i < count; ++i) {
                const int stage = (n + i) % C::kStages;
                if (n + i >= C::kStages) {
                    ok = __all_sync(0xffffffffu, wait_or_abort(&b.empty[stage], ((n + i) / C::kStages - 1) & 1, abort));
                    if (!ok) break;
                }
#pragma unroll
                for (int block = 0; block < C::kBlocks; ++block) {
                    const int k = (from + i) * C::kChunk + block * 64 + piece * 8;
                    const uint32_t at = to + stage * C::kStage;
#pragma unroll
                    for (int j = 0; j < ROWS / 32; ++j) {
                        const bool live = xp[j] && k < k1;
                        copy_or_zero(at + block * C::kBlockX + j * 32 * 128, live ? xp[j] + k : c.x, live ? 16 : 0);
                    }
#pragma unroll
                    for (int j = 0; j < RP / 32; ++j)
                        if (row + 32 * j < padded) {
                            const bool live = row + 32 * j < rank && k < k1;
                            copy_or_zero(at + C::kA + block * C::kBlockA + j * 32 * 128, live ? ap + (long long)j * 32 * c.k + k : c.a,
                                         live ? 16 : 0);
                        }
                }
                cp_async_commit();
                if (i >= C::kLag) {
                    cp_async_wait<C::kLag>();
                    hand_on(i - C::kLag);
                }
            }
            if (!ok) break;
            cp_async_wait<0>();
            for (int i = max(0, count - C::kLag); i < count; ++i) hand_on(i);
            ok = __all_sync(0xffffffffu, wait_or_abort(&b.acc_full, product & 1, abort));
            if (!ok) break;
            tc_fence_after();
            const int quarter = warp & 3, half = warp >> 2, at = quarter * 32 + lane;
            float* out = c.ws + ((long long)part * p.rows + tile.y + at) * c.max_rank;
#pragma unroll
            for (int j = 0; j < RP / 64; ++j) {
                const int col = half * (RP / 2) + j * 32;
                float d[32];
                tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + col, d);
#pragma unroll
                for (int i = 0; i < 32; i += 4)
                    if (at < tile.z && col + i < c.max_rank)
                        *reinterpret_cast<float4*>(out + col + i) =
                            make_float4(col + i < live_cols ? d[i] : 0.0f, col + i + 1 < live_cols ? d[i + 1] : 0.0f,
                                        col + i + 2 < live_cols ? d[i + 2] : 0.0f, col + i + 3 < live_cols ? d[i + 3] : 0.0f);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.acc_empty);
        } else {
            const uint32_t leader = elect_one(), tm = __shfl_sync(0xffffffffu, tmem, 0);
            const uint32_t idesc = (1u << 4) | ((uint32_t)(padded >> 3) << 17) | ((128u >> 4) << 24);
            if (product) ok = __all_sync(0xffffffffu, wait_or_abort(&b.acc_empty, (product - 1) & 1, abort));
            for (int i = 0; i < count && ok; ++i) {
                const int stage = (n + i) % C::kStages;
                ok = __all_sync(0xffffffffu, wait_or_abort(&b.full[stage], ((n + i) / C::kStages) & 1, abort));
                if (!ok) break;
                tc_fence_after();
                const uint64_t xd = desc(smem_u32(smem + stage * C::kStage)), ad = desc(smem_u32(smem + stage * C::kStage + C::kA));
#pragma unroll
                for (int k = 0; k < C::kChunk / 16; ++k)
                    mma_ss(leader, tm, xd + ((k >> 2) * C::kBlockX + (k & 3) * 32) / 16, ad + ((k >> 2) * C::kBlockA + (k & 3) * 32) / 16,
                           i > 0 || k > 0, idesc);
                commit(leader, &b.empty[stage]);
            }
            if (!ok) break;
            commit(leader, &b.acc_full);
        }
        n += count;
        ++product;
    }
}

// An item is a part of a tile. RP: rows of A that a stage has room for (the products have the rank, rounded up to 16). Rows
// 64 to 127 of the products of a tile of 64 are of what follows in shared memory, and not stored.
template <int RP>
__global__ void __launch_bounds__(kLoadThreads + 32, 1) lora_shrink_wide_kernel(const __grid_constant__ Args a) {
    constexpr int kStages = shrink_stages(RP, kTileRows);  // at the most
    extern __shared__ uint8_t raw_smem[];
    __shared__ __align__(8) ShrinkBars<kStages> b;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    const LoraCall& c = a.c;
    uint8_t* smem = raw_smem + (1024 - (smem_u32(raw_smem) & 1023) & 1023);
    const int tid = threadIdx.x, warp = tid >> 5;
    pdl_launch_dependents();
    pdl_wait();
    Plan p;
    if (!read_plan(c, &p)) {
        if (tid == 0) atomicCAS(a.err, 0u, (unsigned)kDevBadList);
        return;
    }
    if (warp == kLoaders) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(128)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&b.full[i], kLoadThreads);
            mbar_init(&b.empty[i], 1);
        }
        mbar_init(&b.acc_full, 1);
        mbar_init(&b.acc_empty, kLoaders);
        mbar_init(&b.drain, 1);
        fence_mbar_init();
        s_abort = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const Split split = split_of(c, p);
    if (split.rows == kWideRows) shrink_items<RP, kWideRows>(a, p, split.tiles, split.parts, smem, b, s_tmem, &s_abort);
    else shrink_items<RP, kTileRows>(a, p, split.tiles, split.parts, smem, b, s_tmem, &s_abort);
    if (warp == kLoaders) {
        commit(elect_one(), &b.drain);  // no product may run on when the block leaves
        mbar_wait_bounded(&b.drain, 0);
    }
    cp_async_wait<0>();
    tc_fence_before();
    __syncwarp();
    __syncthreads();
    if (tid == 0 && s_abort) atomicCAS(a.err, 0u, (unsigned)kDevTmaTimeout);
    if (warp == kLoaders) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s_tmem), "r"(128) : "memory");
    }
}

// ---- base + scale * h B^T
// The block's items in order: tiles, and for each its blocks of outputs. Rows without an adapter follow as tiles of
// rank 0, where they have to be copied.
struct Walk {
    const LoraCall& c;
    const Plan& p;
    int across, left, at, block;
    int4 tile;  // adapter (-1: none), first place, rows
    int rank;
    bool fresh;  // the tile's first item here
    __device__ Walk(const LoraCall& c, const Plan& p) : c(c), p(p) {
        across = (c.n + kCols - 1) / kCols;
        const int bare = c.base == c.out ? 0 : (p.bare + kWideRows - 1) / kWideRows;
        const long long items = (long long)(p.wide_tiles + bare) * across, first = items * blockIdx.x / gridDim.x;
        left = (int)(items * (blockIdx.x + 1) / gridDim.x - first);
        at = (int)(first / across);
        block = (int)(first % across);
        open();
    }
    __device__ void open() {
        fresh = true;
        if (left <= 0) return;
        if (at < p.wide_tiles) {
            tile = __ldg(p.wide + at);
            rank = c.ranks ? __ldg(c.ranks + tile.x) : c.max_rank;
            if (rank < 0 || rank > c.max_rank) rank = 0;  // the first product's kernel has said so
        } else {
            const int i = (at - p.wide_tiles) * kWideRows;
            tile = make_int4(-1, p.rows + i, min(kWideRows, p.bare - i), 0);
            rank = 0;
        }
    }
    __device__ bool more() const { return left > 0; }
    __device__ bool last_of_tile() const { return left == 1 || block + 1 == across; }
    __device__ int n0() const { return block * kCols; }
    __device__ void next() {
        --left;
        fresh = false;
        if (++block == across) {
            block = 0;
            ++at;
            open();
        }
    }
};

template <int RP>
__global__ void __launch_bounds__(kThreads, 1) lora_expand_wide_kernel(const __grid_constant__ Args a) {
    using C = Cfg<RP>;
    extern __shared__ uint8_t raw_smem[];
    __shared__ __align__(8) uint64_t full[C::kStages], empty[C::kStages], h_full[C::kTilesH], h_empty[C::kTilesH], acc_full[2],
        acc_empty[2], drain;
    __shared__ long long s_from[kRowLists][kWideRows], s_to[kRowLists][kWideRows];  // where a tile's rows begin
    __shared__ float s_scale[kRowLists][kWideRows];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    const LoraCall& c = a.c;
    uint8_t* smem = raw_smem + (1024 - (smem_u32(raw_smem) & 1023) & 1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_launch_dependents();
    Plan p;
    if (!read_plan(c, &p)) {
        if (tid == 0) atomicCAS(a.err, 0u, (unsigned)kDevBadList);
        pdl_wait();
        return;
    }
    if (warp == kIssuer) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(256)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(&full[i], kLoadThreads);
            mbar_init(&empty[i], 1 + kEpilogue);
        }
        for (int i = 0; i < C::kTilesH; ++i) {
            mbar_init(&h_full[i], kLoadThreads);
            mbar_init(&h_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], kEpilogue);
        }
        mbar_init(&drain, 1);
        fence_mbar_init();
        s_abort = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    volatile int* const abort = &s_abort;
    Walk w(c, p);

    if (warp < kLoaders) {
        const uint32_t at_smem = smem_u32(smem);
        const int parts = a.split ? split_of(c, p).parts : parts_of(p.tiles, c.k);
        int list = -1, tiles_h = 0, item = 0;
        bool waited = false, ok = true;  // once a wait has given up, only the barriers that warps share are met
        auto hand_on = [&](int i) {  // item i's copies of this thread are there
            fence_proxy_async_shared();
            mbar_arrive(&full[i % C::kStages]);
        };
        for (; w.more(); w.next(), ++item) {
            const int stage = item % C::kStages, n0 = w.n0(), rank = w.rank;
            if (ok && item >= C::kStages)
                ok = __all_sync(0xffffffffu, wait_or_abort(&empty[stage], (item / C::kStages - 1) & 1, abort));
            if (w.fresh) {
                list = (list + 1) % kRowLists;
                if (tid < kWideRows) {
                    const long long row = tid < w.tile.z ? __ldg(p.row + w.tile.y + tid) : 0;
                    s_from[list][tid] = row * c.base_stride;
                    s_to[list][tid] = row * c.out_stride;
                }
                named_barrier<2, kLoadThreads>();
            }
            if (!ok) continue;
            if (c.base) {  // 16 lanes a row
                const int col = tid % 16 * 8, row0 = tid / 16;
                const __half* base = c.base + n0 + col;
                uint32_t to = at_smem + C::kY + stage * C::kBytesY + row0 * C::kPitch + col * 2;
                if (n0 + col < c.n)
#pragma unroll
                    for (int row = 0; row < kWideRows; row += kLoadThreads / 16)
                        if (row + row0 < w.tile.z) copy_or_zero(to + row * C::kPitch, base + s_from[list][row + row0], 16);
            }
            if (rank) {  // a thread copies one piece of every kStep-th row; what follows the rank is zeros
                constexpr int kPieces = RP / 8, kStep = kLoadThreads / kPieces;
                const int n = tid / kPieces, piece = tid % kPieces;
                if (piece < (rank + 15) / 16 * 2) {
                    const int bytes = max(0, min(8, rank - 8 * piece)) * 2, left = c.n - n0 - n;
                    const __half* b = c.b + ((long long)w.tile.x * c.n + n0 + n) * c.max_rank + (bytes ? 8 * piece : 0);
                    const uint32_t to = at_smem + C::kB + stage * C::kBytesB + (piece >> 3) * (kCols * 128) + n * 128;
#pragma unroll
                    for (int i = 0; i < kCols / kStep; ++i, b += (long long)kStep * c.max_rank)
                        copy_or_zero(to + i * kStep * 128 + (((piece & 7) ^ ((n + i * kStep) & 7)) << 4),
                                     left > i * kStep ? b : c.b, left > i * kStep ? bytes : 0);
                }
            }
            cp_async_commit();
            if (w.fresh && rank) {
                const int slot = tiles_h % C::kTilesH;
                if (tiles_h >= C::kTilesH) ok = __all_sync(0xffffffffu, wait_or_abort(&h_empty[slot], (tiles_h / C::kTilesH - 1) & 1, abort));
                if (!ok) continue;
                if (!waited) pdl_wait();  // for the first product
                waited = true;
                // four threads a row, each every fourth four of its elements
                uint8_t* h0 = smem + slot * C::kBytesH;
                const long long step = (long long)p.rows * c.max_rank;
#pragma unroll 1
                for (int pass = 0; pass < kWideRows * 4 / kLoadThreads; ++pass) {
                    const int row = pass * (kLoadThreads / 4) + (tid >> 2), q = tid & 3;
                    float4 v[RP / 16];
                    sum_parts<RP / 16>(c.ws + (long long)(w.tile.y + row) * c.max_rank + 4 * q, step, parts,
                                       row < w.tile.z ? rank - 4 * q : 0, v);
                    float top = 0.0f;
#pragma unroll
                    for (int i = 0; i < RP / 16; ++i) top = fmaxf(top, largest_finite(v[i]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const int e = exponent_of(top);
                    const float down = two_to(-e);
#pragma unroll
                    for (int i = 0; i < RP / 16; ++i) {
                        __half hi[4], lo[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) two_halves((&v[i].x)[j] * down, &hi[j], &lo[j]);
                        const int piece = 2 * i + (q >> 1);
                        uint8_t* to = h0 + (piece >> 3) * (kWideRows * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4) + 8 * (q & 1);
                        *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(hi);
                        *reinterpret_cast<uint2*>(to + C::kBytesH / 2) = *reinterpret_cast<const uint2*>(lo);
                    }
                    if (q == 0) s_scale[list][row] = (c.scales ? __ldg(c.scales + w.tile.x) : 1.0f) * two_to(e);
                }
                fence_proxy_async_shared();
                mbar_arrive(&h_full[slot]);
                ++tiles_h;
            }
            if (item >= C::kLag) {
                cp_async_wait<C::kLag>();
                hand_on(item - C::kLag);
            }
        }
        cp_async_wait<0>();
        if (ok)
            for (int i = max(0, item - C::kLag); i < item; ++i) hand_on(i);
        if (!waited) pdl_wait();
    } else if (warp == kIssuer) {
        pdl_wait();
        const uint32_t leader = elect_one(), tm = __shfl_sync(0xffffffffu, s_tmem, 0);
        const uint64_t h_desc = desc(smem_u32(smem)), b_desc = desc(smem_u32(smem + C::kB));
        int item = 0, products = 0, tiles_h = 0;
        bool ok = true;
        for (; w.more() && ok; w.next(), ++item) {
            const int stage = item % C::kStages, acc = products & 1, slot = tiles_h % C::kTilesH;
            ok = __all_sync(0xffffffffu, wait_or_abort(&full[stage], (item / C::kStages) & 1, abort));
            if (!w.rank) {  // nothing to multiply: the stage is the epilogue's alone
                if (lane == 0) mbar_arrive(&empty[stage]);
                continue;
            }
            if (ok && w.fresh) ok = __all_sync(0xffffffffu, wait_or_abort(&h_full[slot], (tiles_h / C::kTilesH) & 1, abort));
            if (ok && products >= 2) ok = __all_sync(0xffffffffu, wait_or_abort(&acc_empty[acc], (products / 2 - 1) & 1, abort));
            if (!ok) break;
            tc_fence_after();
            const int steps = __shfl_sync(0xffffffffu, (w.rank + 15) / 16, 0);
            const uint64_t hd = h_desc + (uint64_t)(slot * (C::kBytesH / 16)), bd = b_desc + (uint64_t)(stage * (C::kBytesB / 16));
#pragma unroll
            for (int part = 0; part < 2; ++part)
#pragma unroll
                for (int k = 0; k < RP / 16; ++k) {
                    if (k >= steps) break;
                    const uint64_t in = ((k >> 2) * (128 * 128) + (k & 3) * 32) / 16;  // both operands have 128 rows
                    mma_ss(leader, tm + acc * kCols, hd + part * (C::kBytesH / 32) + in, bd + in, part > 0 || k > 0, kIdesc);
                }
            commit(leader, &acc_full[acc]);
            commit(leader, &empty[stage]);
            if (w.last_of_tile()) {
                commit(leader, &h_empty[slot]);
                ++tiles_h;
            }
            ++products;
        }
        commit(leader, &drain);  // no product may run on when the block leaves
        mbar_wait_bounded(&drain, 0);
    } else {
        pdl_wait();
        const int quarter = warp & 3, half = (warp - kLoaders) >> 2, row = quarter * 32 + lane;
        const int out_col = lane % 16 * 8, out_row = (warp - kLoaders) * 2 + lane / 16;
        const uint32_t tm = s_tmem + ((uint32_t)(quarter * 32) << 16) + half * 64;
        int item = 0, products = 0, list = -1;
        bool ok = true;
        for (; w.more(); w.next(), ++item) {
            const int stage = item % C::kStages, acc = products & 1;
            if (w.fresh) list = (list + 1) % kRowLists;
            ok = ok && wait_or_abort(&full[stage], (item / C::kStages) & 1, abort);
            if (ok && w.rank) ok = wait_or_abort(&acc_full[acc], (products / 2) & 1, abort);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {  // once a wait has given up, only the barrier that warps share is met
                named_barrier<1, 32 * kEpilogue>();
                continue;
            }
            uint8_t* y0 = smem + C::kY + stage * C::kBytesY;
            if (w.rank) {
                tc_fence_after();
                const float scale = s_scale[list][row];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float d[32];
                    tmem_ld32(tm + acc * kCols + 32 * j, d);
                    if (j == 1) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&acc_empty[acc]);
                    }
                    uint4* y = reinterpret_cast<uint4*>(y0 + row * C::kPitch + (half * 64 + 32 * j) * 2);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        uint4 v = c.base ? y[i] : make_uint4(0, 0, 0, 0);
                        __half2* o = reinterpret_cast<__half2*>(&v);
#pragma unroll
                        for (int u = 0; u < 4; ++u) {
                            const float2 f = __half22float2(o[u]);
                            o[u] = __floats2half2_rn(fmaf(scale, d[8 * i + 2 * u], f.x), fmaf(scale, d[8 * i + 2 * u + 1], f.y));
                        }
                        y[i] = v;
                    }
                }
                ++products;
            } else if (!c.base) {
                uint4* y = reinterpret_cast<uint4*>(y0 + row * C::kPitch + half * 128);
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = make_uint4(0, 0, 0, 0);
            }
            named_barrier<1, 32 * kEpilogue>();
            if (w.n0() + out_col < c.n) {
                __half* out = c.out + w.n0() + out_col;
                const uint8_t* y = y0 + out_col * 2;
#pragma unroll
                for (int r = 0; r < kWideRows; r += 2 * kEpilogue)
                    if (r + out_row < w.tile.z)
                        *reinterpret_cast<uint4*>(out + s_to[list][r + out_row]) =
                            *reinterpret_cast<const uint4*>(y + (r + out_row) * C::kPitch);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[stage]);
        }
    }
    tc_fence_before();
    __syncwarp();
    __syncthreads();
    if (tid == 0 && *abort) atomicCAS(a.err, 0u, (unsigned)kDevTmaTimeout);
    if (warp == kIssuer) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(s_tmem), "r"(256) : "memory");
    }
}

template <int RP>
int launch_shrink(const LoraCall& c, unsigned* error_word, cudaStream_t st) {
    constexpr int smem = ShrinkCfg<RP, kWideRows>::smem;
    static std::atomic<unsigned long long> set{0};  // a bit a device
    int dev = 0;
    cudaGetDevice(&dev);
    if (!(set.load() >> (dev & 63) & 1)) {
        if (cudaFuncSetAttribute(lora_shrink_wide_kernel<RP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
            return -1;
        set.fetch_or(1ull << (dev & 63));
    }
    Args a = {c, error_word, true};
    if (!a.err) return -1;
    const long long tiles = most_tiles(c.num_seqs, c.num_tokens, c.num_adapters);
    const long long items = std::min<long long>(kNumSMs, tiles * parts_of(1, c.k));
    return launch_k(lora_shrink_wide_kernel<RP>, dim3((unsigned)items), dim3(kLoadThreads + 32), smem, st, a) == cudaSuccess ? 0 : -1;
}

template <int RP>
int launch(const LoraCall& c, bool split, unsigned* error_word, cudaStream_t st) {
    using C = Cfg<RP>;
    static std::atomic<unsigned long long> set{0};  // a bit a device
    int dev = 0;
    cudaGetDevice(&dev);
    if (!(set.load() >> (dev & 63) & 1)) {
        if (cudaFuncSetAttribute(lora_expand_wide_kernel<RP>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem) != cudaSuccess)
            return -1;
        set.fetch_or(1ull << (dev & 63));
    }
    Args a = {c, error_word, split};
    if (!a.err) return -1;
    const long long tiles = most_tiles(c.num_seqs, c.num_tokens, c.num_adapters, kWideRows) + (c.num_tokens + kWideRows - 1) / kWideRows;
    const long long items = tiles * ((c.n + kCols - 1) / kCols);
    return launch_k(lora_expand_wide_kernel<RP>, dim3((unsigned)std::min<long long>(kNumSMs, items)), dim3(kThreads), C::smem, st,
                    a) == cudaSuccess
               ? 0
               : -1;
}

}  // namespace

int launch_lora_shrink_wide(const LoraCall& c, unsigned* error_word, cudaStream_t st) {
    return c.max_rank <= 64 ? launch_shrink<64>(c, error_word, st) : launch_shrink<128>(c, error_word, st);
}
int launch_lora_expand_wide(const LoraCall& c, bool split, unsigned* error_word, cudaStream_t st) {
    return c.max_rank <= 64 ? launch<64>(c, split, error_word, st) : launch<128>(c, split, error_word, st);
}

}  // namespace batch
}  // namespace cb
