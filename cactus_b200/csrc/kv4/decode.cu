// Attention over the 4-bit paged KV cache for few queries a sequence (decode, drafted tokens). Its
// floor is the cache's bytes, read once; what bounds it is the instructions that turn codes into
// operands, and that they wait for one another: of about 419 a warp for 16 keys of 128, 208 unpack and
// scale 1024 elements (13 for 8), groups of 128 (0.53 bytes an element) take as long as groups of 32
// (0.63), and with under three warps a scheduler 59 % of the issue slots are used. On B200: 64 sequences
// of 16 to 32 thousand rows, 8 kv heads of 128, 518 us, 3.9 TB/s of the cache (floor 314 us); 256 short
// conversations in pages of 16, heads of 64, 78 us (floor 14 us: the starts and ends of 2048 items
// and the 16-key overheads at half the elements weigh most there); 12 sequences of 5 drafted tokens over 8
// thousand rows, 62 us (floor 14 us: 10 q rows take two column tiles of 8, each with two products a weight).
//
// Work. A sequence's q rows of one kv head (its tokens times the heads that share it, in tiles of
// 4, 8 or 16 rows) over its visible keys is an item; items are cut into tiles of 64 or 128 keys, and the
// tiles of all items, in one list, are dealt in equal contiguous ranges to as many CTAs as the GPU
// holds at once, whatever the sequences' lengths. Every CTA finds its range itself from the lengths
// in device memory. An item inside one range is finished there; the parts of one that spans several
// go to the workspace, and the CTA that brings the last part joins them in range order, so the
// result does not depend on which one that is.
//
// CTA. Four warps; each takes 16 or 32 keys of every tile through its own ring in shared memory and
// keeps its own softmax state, so the loop has no barrier and no registers go to a producer. The ring
// is filled by 16-byte asynchronous copies, whose addresses differ by constants within a page; page
// ids are fetched a step ahead. (Bulk copies by lanes of the warp run one after another and took 60
// instructions for 32 keys.) The four states are joined at the item's end, in the rings' memory.
//
// Tensor cores. S^T = K Q^T and O^T = V^T P^T, m16n8k16 with keys (and value dims) on the 16 side
// and q rows on the 8 side: 8 rows waste nothing, and the operand that comes from the cache is the
// A fragment, built in registers from the codes. The k index is permuted freely: lane t of a quad
// takes a contiguous quarter of the head for the keys (the q fragments use the same order), and a
// quarter of the 16 keys for the values, where the codes of two keys are interleaved by bytes first
// so that one mask gives the same dim of both. Key i of the fragment is row kappa(i) of the 16,
// which spreads the lanes' shared-memory reads over the banks. The weights go into O as two fp16
// numbers, p = hi + lo (22 bits, what is below 2^-31 of the largest weight left out); up to 4 rows have lo
// in the columns that they leave empty. The tensor core cuts its fp32 sums instead of rounding them, so a
// result is low by what 16 keys at a time lose: 8e-6 of it over 32768 rows, 4e-7 over 2000.
//
// Softmax. Weights are relative to 2^-kHead of the running maximum, which is raised only when a score
// exceeds it by more than 2^kLazy: until then they grow past 2^kHead (at most 2^15, inside fp16), which
// is exact up to rounding and saves the reduction over the lanes for almost every tile. At the other end
// fp16's last bit is 2^-24: small weights keep what is above 2^-31 of the largest.
#include <algorithm>
#include <atomic>

#include "attention.cuh"
#include "kv4.cuh"
#include "kv4_ops.h"

namespace cb {
namespace kv4 {

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr float kLazy = 8.0f, kHead = 7.0f;  // base-2 exponents

// row of the 16 that key i of the fragments is
__device__ __forceinline__ int kappa(int i) { return (i & 8) + (((i & 7) >> 1) ^ ((i & 1) * 5)); }

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_t(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cp_async16_at(uint32_t smem, const void* gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(gmem) : "memory");
}

// What one sequence asks for, in tiles. Positions fit 31 bits (the entry point checks the table's
// width), byte offsets do not.
struct Seq {
    int tokens, row_tiles;  // queries, tiles of q rows per kv head
    int pos0;               // position of token 0
    int start, end;         // keys that any of its queries sees
    int base, ntiles;       // tiles of keys from base (1 for none: the item still has to write)
};

template <int ROWS, int TILE>
__device__ __forceinline__ Seq seq_of(const AttnCall& c, const Pages& pg, const Geom& ge, int max_rows, int b, bool report) {
    Seq s;
    const int from = c.offsets[b], to = c.offsets[b + 1], len = max(c.lens[b], 0);
    const bool good = from >= 0 && from <= to && to <= c.num_tokens;  // else the sequence is left out
    const int count = good ? to - from : 0;
    const int room = (int)(pg.table_stride << ge.page_shift);
    s.tokens = max(0, min(count, c.max_q));
    if (report && (!good || count > c.max_q || (len > room && count > 0))) report_dev_error(kDevBadPage);
    const int rows = s.tokens * (c.hq / ge.hkv);
    s.row_tiles = rows > max_rows ? 0 : (rows + ROWS - 1) / ROWS;
    s.pos0 = len - count;
    const int n = min(len, room);
    s.end = c.causal ? min(n, s.pos0 + s.tokens) : n;
    s.start = c.window > 0 ? (int)max(0LL, s.pos0 - c.window + 1) : 0;
    if (s.start >= s.end) s.start = s.end = 0;
    s.base = s.start & ~(TILE - 1);
    s.ntiles = max(1, (s.end - s.base + TILE - 1) / TILE);
    return s;
}

// ROWS q rows are a tile: 16 or 8, which fill the columns of one or two fragments, or 4, which leave
// columns 4-7 of one to the low parts of the weights.
template <int ROWS>
constexpr int columns() { return ROWS < 8 ? 8 : ROWS; }
// Blocks of 16 keys that a warp takes at a time: two where the registers hold them (64 sequences of 4
// to 8 thousand rows at head_dim 128: 137 us with two, 152 with one; 256 short conversations at 64: 79
// and 73, 64 of 8000 rows: 100 and 114), one at 16 rows of 128 (12 sequences of 5 tokens over 8000 rows: 63 us with one, 62 with two). CTAs a
// multiprocessor holds: by the registers, 168 a thread (three) or 128 (four, at 64); four at 128 take
// 137 us too. Stages of a ring: what shared memory then holds.
template <int D, int ROWS>
constexpr int blocks() { return D == 64 || (D == 128 && ROWS <= 8) ? 2 : 1; }
template <int D, int ROWS>
constexpr int ctas_per_sm() { return D == 64 && ROWS <= 8 ? 4 : 3; }
template <int D, int ROWS>
constexpr int stages() { return D == 64 ? 4 : D == 128 && ROWS == 16 ? 5 : 3; }

template <int D, int ROWS>
struct Smem {
    static constexpr int kCols = columns<ROWS>();
    uint4 q[kCols / 8][D / 32][32];
    float m[kWarps][kCols], l[kWarps][kCols];
    int scan[kWarps], scan_items[kWarps];
    int base, item0, b0;  // the sequence that this CTA starts with: its first tile, its first item
    int last, nan;
};

template <int D, int ROWS>
__global__ void __launch_bounds__(kThreads, ctas_per_sm<D, ROWS>())
    kv4_decode_kernel(const __grid_constant__ AttnCall c, const __grid_constant__ Pages pg, const __grid_constant__ Geom ge,
                      int max_rows, int max_items) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int kCols = columns<ROWS>(), NT = kCols / 8, KB = blocks<D, ROWS>(), kTile = 16 * KB * kWarps, kStages = stages<D, ROWS>(), kPad = D + 4;
    constexpr bool kPaired = ROWS < 8;  // columns 4-7 repeat 0-3 and take the weights' low parts
    constexpr int kNoKeys = 0x7fffff00; // past every position
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ Smem<D, ROWS> sm;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int share = c.hq / ge.hkv, ng = ge.ng();

    // ---- the list of tiles, and this CTA's part of it
    const int per = (c.num_seqs + kThreads - 1) / kThreads, first_b = tid * per;
    int mine = 0, items = 0;
    for (int b = first_b; b < min(first_b + per, c.num_seqs); ++b) {
        const Seq s = seq_of<ROWS, kTile>(c, pg, ge, max_rows, b, blockIdx.x == 0);
        mine += s.row_tiles * ge.hkv * s.ntiles;
        items += s.row_tiles * ge.hkv;
    }
    int upto = mine, items_upto = items;  // sums over this thread and those before it
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, upto, o), i = __shfl_up_sync(0xffffffffu, items_upto, o);
        if (lane >= o) {
            upto += a;
            items_upto += i;
        }
    }
    if (lane == 31) {
        sm.scan[warp] = upto;
        sm.scan_items[warp] = items_upto;
    }
    if (tid == 0) sm.nan = 0;
    __syncthreads();
    int total = 0, all_items = 0;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) {
        all_items += sm.scan_items[x];
        if (x < warp) {
            upto += sm.scan[x];
            items_upto += sm.scan_items[x];
        }
        total += sm.scan[x];
    }
    // CTA x of n has the tiles first_tile(x) .. first_tile(x + 1) - 1: as many as the others, or one more
    const int n = min((int)gridDim.x, total);
    if ((int)blockIdx.x >= n) return;
    if (all_items > max_items) {  // token rows named by several sequences: there are not so many counters
        if (tid == 0) report_dev_error(kDevBadPage);
        return;
    }
    const int each = total / n, more = total - each * n;
    auto first_tile = [&](int x) { return x * each + min(x, more); };
    auto owner = [&](int tile) {
        const int lead = more * (each + 1);
        return tile < lead ? tile / (each + 1) : more + (tile - lead) / each;
    };
    const int w0 = first_tile(blockIdx.x), w1 = first_tile(blockIdx.x + 1);
    if (w0 >= upto - mine && w0 < upto) {
        int at = upto - mine, it = items_upto - items;
        for (int b = first_b;; ++b) {
            const Seq s = seq_of<ROWS, kTile>(c, pg, ge, max_rows, b, false);
            const int k = s.row_tiles * ge.hkv;
            if (w0 < at + k * s.ntiles) {
                sm.b0 = b;
                sm.base = at;
                sm.item0 = it;
                break;
            }
            at += k * s.ntiles;
            it += k;
        }
    }
    __syncthreads();
    // walks the items of [w0, w1): item `it` of sequence b (kv head it / row_tiles), tiles t .. t + k - 1
    struct Walk {
        int b, base, item0;
        Seq s;
    } wk;
    wk.b = sm.b0;
    wk.base = sm.base;
    wk.item0 = sm.item0;
    wk.s = seq_of<ROWS, kTile>(c, pg, ge, max_rows, wk.b, false);
    auto next_seq = [&](int w) {  // moves to the sequence that tile w belongs to
        while (w >= wk.base + wk.s.row_tiles * ge.hkv * wk.s.ntiles) {
            wk.base += wk.s.row_tiles * ge.hkv * wk.s.ntiles;
            wk.item0 += wk.s.row_tiles * ge.hkv;
            ++wk.b;
            wk.s = seq_of<ROWS, kTile>(c, pg, ge, max_rows, wk.b, false);
        }
    };

    const int g = lane >> 2, t = lane & 3;
    const float sc = c.scale * 1.4426950408889634f;
    float* const parts = reinterpret_cast<float*>(c.ws);
    unsigned* const counters = reinterpret_cast<unsigned*>(c.ws + kPartBytes);
    // A stage is the parts of one page (KB = 2 and a page of 16 rows: of two pages) one after the
    // other, R rows each: codes | parameters | the values' codes | parameters
    const int R = min(ge.page(), 16 * KB), row_p = 4 * ng, chunk_bytes = R * (D + 2 * row_p);
    const int stage_bytes = 16 * KB * (D + 2 * row_p);
    uint8_t* const mine_ring = ring + warp * kStages * stage_bytes;
    float* const s_o = reinterpret_cast<float*>(ring);  // [warp][row][kPad], at an item's end
    // byte offsets in a stage of this lane's parts of the first block: key kappa(g) (and 8 rows on), two
    // groups of parameters at most; value rows kappa(2 t), kappa(2 t + 1) (and 8 on), one group; and
    // how far the second block's are on
    const int kg = kappa(g), vk0 = kappa(2 * t), vk1 = kappa(2 * t + 1);
    const int p0 = R * (D / 2), v0 = p0 + R * row_p, q0 = v0 + R * (D / 2);
    const int k_codes = kg * (D / 2) + t * (D / 8);
    const int k_par0 = p0 + kg * row_p + t * (D / 4) / ge.g * 4;
    const int k_par1 = p0 + kg * row_p + (t * (D / 4) + 32) / ge.g * 4;
    const int v_codes0 = v0 + vk0 * (D / 2) + g * (D / 16), v_codes1 = v_codes0 + (vk1 - vk0) * (D / 2);
    const int v_par0 = q0 + vk0 * row_p + g * (D / 8) / ge.g * 4, v_par1 = v_par0 + (vk1 - vk0) * row_p;
    const int step_codes = R == 16 ? chunk_bytes : 8 * D, step_par = R == 16 ? chunk_bytes : 16 * row_p;
    const uint32_t ring_at = smem_u32(mine_ring) + lane * 16;
    const bool copies_par = lane < R * ng / 4;  // 16-byte pieces of R rows' parameters: at most 32

    for (int w = w0; w < w1;) {
        next_seq(w);
        const Seq s = wk.s;
        const int it = (w - wk.base) / s.ntiles, tile0 = w - wk.base - it * s.ntiles;
        const int head = s.row_tiles == 1 ? it : it / s.row_tiles, row0 = (it - head * s.row_tiles) * ROWS;
        const int ntile = min(s.ntiles - tile0, w1 - w);
        const int tok0 = c.offsets[wk.b], rows = min(ROWS, s.tokens * share - row0);
        const int qhead0 = head * share;

        // ---- q, in flight beside the page ids: column g of n-tile j is row row0 + 8 j + g (paired: row0 + g % 4)
        constexpr int kQ = (NT * (D / 32) + kWarps - 1) / kWarps;
        uint4 qv[kQ];
#pragma unroll
        for (int u = 0; u < kQ; ++u) {
            const int i = warp + u * kWarps, j = i / (D / 32), x = i % (D / 32);
            const int col = kPaired ? g & 3 : 8 * j + g, r = row0 + col;
            qv[u] = uint4{0, 0, 0, 0};
            if (i < NT * (D / 32) && col < rows)
                qv[u] = __ldg(reinterpret_cast<const uint4*>(c.q + (long long)(tok0 + r / share) * c.q_stride +
                                                             (long long)(qhead0 + r % share) * D + t * (D / 4)) + x);
        }

        // ---- the ring: stage i of this warp is the keys first + i * kTile .. + 16 KB - 1
        const int first = s.base + tile0 * kTile + warp * 16 * KB, stop = min(s.end, first + ntile * kTile);
        const int* const table = pg.table + (long long)wk.b * pg.table_stride;
        const uint8_t* const pool = pg.pool + (long long)head * ge.block_bytes() + lane * 16;
        unsigned have = 0;  // bits KB * slot ..: the blocks of the slot that were loaded
        auto page_of = [&](int k0) -> int {  // id of the page with the R keys from k0; -1: nothing to load
            if (k0 >= stop || k0 + R <= s.start) return -1;
            const int p = __ldg(table + (k0 >> ge.page_shift));
            if ((unsigned)p < (unsigned)pg.num_pages) return p;
            report_dev_error(kDevBadPage);
            return -1;
        };
        auto copy = [&](int page, int k0, uint32_t dst) {  // R keys
            const int r = k0 & (ge.page() - 1);
            const uint8_t* src = pool + (long long)page * pg.page_stride;
            const uint8_t* codes = src + r * (D / 2);
            const uint8_t* par = src + ge.k_params() + r * row_p;
            if (R == 16) {
#pragma unroll
                for (int x = 0; x < D / 64; ++x) cp_async16_at(dst + x * 512, codes + x * 512);
#pragma unroll
                for (int x = 0; x < D / 64; ++x) cp_async16_at(dst + v0 + x * 512, codes + ge.v_codes() + x * 512);
            } else {
#pragma unroll
                for (int x = 0; x < D / 32; ++x) cp_async16_at(dst + x * 512, codes + x * 512);
#pragma unroll
                for (int x = 0; x < D / 32; ++x) cp_async16_at(dst + v0 + x * 512, codes + ge.v_codes() + x * 512);
            }
            if (copies_par) {
                cp_async16_at(dst + p0, par);
                cp_async16_at(dst + q0, par + ge.v_codes());
            }
        };
        int page[KB];  // of the next stage; with R = 16 KB only the first counts
        auto pages_of = [&](int k0) {
            page[0] = page_of(k0);
            if (KB > 1 && R == 16) page[KB - 1] = page_of(k0 + 16);
        };
        auto advance = [&](int i, int slot) {  // stage i into the slot, and the ids for the next one
            const int k0 = first + i * kTile;
            const uint32_t dst = ring_at + slot * stage_bytes;
            unsigned got = 0;
            if (page[0] >= 0) {
                copy(page[0], k0, dst);
                got = R == 16 ? 1 : (1u << KB) - 1;
            }
            if (KB > 1 && R == 16 && page[KB - 1] >= 0) {
                copy(page[KB - 1], k0 + 16, dst + chunk_bytes);
                got |= 2;
            }
            have = (have & ~(((1u << KB) - 1) << KB * slot)) | got << KB * slot;
            cp_async_commit();
            pages_of(k0 + kTile);
        };
        pages_of(first);
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) advance(i, i);

        // q fragments for all warps
#pragma unroll
        for (int u = 0; u < kQ; ++u) {
            const int i = warp + u * kWarps;
            if (i < NT * (D / 32))
                sm.q[i / (D / 32)][i % (D / 32)][lane] =
                    uint4{__byte_perm(qv[u].x, qv[u].z, 0x5410), __byte_perm(qv[u].x, qv[u].z, 0x7632),
                          __byte_perm(qv[u].y, qv[u].w, 0x5410), __byte_perm(qv[u].y, qv[u].w, 0x7632)};
        }
        __syncthreads();
        // keys that every row of the tile sees
        const int tok_a = row0 / share, tok_b = min((row0 + ROWS - 1) / share, s.tokens - 1);
        const int all_from = c.window > 0 ? (int)max((long long)s.start, s.pos0 + tok_b - c.window + 1) : s.start;
        const int all_to = c.causal ? min(s.end, s.pos0 + tok_a + 1) : s.end;
        float o[NT][D / 16][4], l[NT][2];
        float base[NT][2], limit[NT][2];  // base-2 exponent that the state is relative to (0 at first); the
                                          // largest score that keeps it (-inf at first)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][i][e] = 0.0f;
            limit[j][0] = limit[j][1] = -INFINITY;
            base[j][0] = base[j][1] = 0.0f;
            l[j][0] = l[j][1] = 0.0f;
        }

        int slot = 0;
#pragma unroll 1
        for (int i = 0; i < ntile; ++i) {
            __syncwarp();  // every lane is done with the stage that is filled next
            advance(i + kStages - 1, slot == 0 ? kStages - 1 : slot - 1);
            cp_async_wait<kStages - 1>();
            __syncwarp();
            const uint8_t* const blk0 = mine_ring + slot * stage_bytes;
            const unsigned got = have >> KB * slot & ((1u << KB) - 1);
            slot = slot + 1 == kStages ? 0 : slot + 1;
            if (!got) continue;
            int k0[KB];  // first key of each block; a block that was not loaded counts as past the end
            bool whole = true;
#pragma unroll
            for (int k = 0; k < KB; ++k) {
                k0[k] = got >> k & 1 ? first + i * kTile + k * 16 : kNoKeys;
                whole &= k0[k] >= all_from && k0[k] + 16 <= all_to;
            }
            // ---- S^T
            float acc[KB][NT][4];
            constexpr int kWords = D / 32;  // words of codes of one key in a lane's quarter
#pragma unroll
            for (int k = 0; k < KB; ++k) {
            const uint8_t* const blk = blk0 + k * step_codes;
            const uint8_t* const pars = blk0 + k * step_par;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[k][j][e] = 0.0f;
            uint32_t wa[kWords], wb[kWords];
            if constexpr (kWords >= 4) {
#pragma unroll
                for (int x = 0; x < kWords / 4; ++x) {
                    *reinterpret_cast<uint4*>(wa + 4 * x) = *reinterpret_cast<const uint4*>(blk + k_codes + 16 * x);
                    *reinterpret_cast<uint4*>(wb + 4 * x) = *reinterpret_cast<const uint4*>(blk + k_codes + 16 * x + 4 * D);
                }
            } else {
                *reinterpret_cast<uint2*>(wa) = *reinterpret_cast<const uint2*>(blk + k_codes);
                *reinterpret_cast<uint2*>(wb) = *reinterpret_cast<const uint2*>(blk + k_codes + 4 * D);
            }
            __half2 sa, la, sb, lb;
#pragma unroll
            for (int x = 0; x < kWords; ++x) {
                if (x == 0 || (D == 256 && x == 4)) {  // at most two groups in a lane's quarter
                    const int par = x == 0 ? k_par0 : k_par1;
                    const __half2 pa = *reinterpret_cast<const __half2*>(pars + par);
                    const __half2 pb = *reinterpret_cast<const __half2*>(pars + par + 8 * row_p);
                    sa = __low2half2(pa);
                    la = __high2half2(pa);
                    sb = __low2half2(pb);
                    lb = __high2half2(pb);
                }
                __half2 ha[4], hb[4];
                codes_to_half(wa[x], ha);
                codes_to_half(wb[x], hb);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    ha[e] = __hfma2(ha[e], sa, la);
                    hb[e] = __hfma2(hb[e], sb, lb);
                }
                const uint32_t a0[4] = {h2u(ha[0]), h2u(hb[0]), h2u(ha[1]), h2u(hb[1])};
                const uint32_t a1[4] = {h2u(ha[2]), h2u(hb[2]), h2u(ha[3]), h2u(hb[3])};
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const uint4 q = sm.q[j][x][lane];
                    mma16816(acc[k][j], a0, q.x, q.y);
                    mma16816(acc[k][j], a1, q.z, q.w);
                }
            }
            }
            // ---- weights
            bool rise = false;
#pragma unroll
            for (int k = 0; k < KB; ++k)
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = acc[k][j][e] * sc;
                        if (!whole) {
                            const int key = k0[k] + kg + (e & 2 ? 8 : 0), col = 8 * j + 2 * t + (e & 1);
                            const int tok = (row0 + (kPaired ? col & 3 : col)) / share;
                            const int pos = s.pos0 + tok;
                            if (key >= s.end || (c.causal && key > pos) || (c.window > 0 && pos - key >= c.window))
                                x = -INFINITY;
                        }
                        acc[k][j][e] = x;
                        rise |= x > limit[j][e & 1];
                    }
            if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = fmaxf(acc[0][j][e], acc[0][j][e + 2]);
                        if (KB > 1) top = fmaxf(top, fmaxf(acc[KB - 1][j][e], acc[KB - 1][j][e + 2]));
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                        top -= kHead;
                        if (limit[j][e] != -INFINITY) top = fmaxf(top, base[j][e]);
                        if (top != -INFINITY) {
                            const float fix = limit[j][e] == -INFINITY ? 0.0f : ex2(base[j][e] - top);
                            base[j][e] = top;
                            limit[j][e] = __fadd_rd(top, kHead + kLazy);
                            l[j][e] *= fix;
#pragma unroll
                            for (int x = 0; x < D / 16; ++x) {
                                o[j][x][e] *= fix;
                                o[j][x][e + 2] *= fix;
                            }
                        }
                    }
                }
            }
            uint32_t hi[KB][NT][2], lo[KB][NT][2];
#pragma unroll
            for (int k = 0; k < KB; ++k)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] = ex2(acc[k][j][e] - base[j][e & 1]);
                    l[j][0] += p[0] + p[2];
                    l[j][1] += p[1] + p[3];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const __half2 h = __floats2half2_rn(p[2 * e], p[2 * e + 1]);
                        const float2 f = __half22float2(h);
                        const __half2 rest = __floats2half2_rn(p[2 * e] - f.x, p[2 * e + 1] - f.y);
                        hi[k][j][e] = movmatrix_t(h2u(kPaired && t >= 2 ? rest : h));
                        if (!kPaired) lo[k][j][e] = movmatrix_t(h2u(rest));
                    }
                }
            // ---- O^T
#pragma unroll
            for (int k = 0; k < KB; ++k) {
            const uint8_t* const blk = blk0 + k * step_codes;
            const uint8_t* const pars = blk0 + k * step_par;
            uint32_t vw[4][D / 64], par[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint8_t* src = blk + (e & 1 ? v_codes1 : v_codes0) + (e & 2 ? 4 * D : 0);
                if constexpr (D == 64) vw[e][0] = *reinterpret_cast<const uint32_t*>(src);
                if constexpr (D == 128) *reinterpret_cast<uint2*>(vw[e]) = *reinterpret_cast<const uint2*>(src);
                if constexpr (D == 256) *reinterpret_cast<uint4*>(vw[e]) = *reinterpret_cast<const uint4*>(src);
                par[e] = *reinterpret_cast<const uint32_t*>(pars + (e & 1 ? v_par1 : v_par0) + (e & 2 ? 8 * row_p : 0));
            }
            if (!whole) {  // rows that nobody sees may hold anything: they count as zeros
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = k0[k] + (e & 1 ? vk1 : vk0) + (e & 2 ? 8 : 0);
                    if (key < s.start || key >= s.end) par[e] = 0;
                }
            }
            const __half2 s01 = u2h(__byte_perm(par[0], par[1], 0x5410)), l01 = u2h(__byte_perm(par[0], par[1], 0x7632));
            const __half2 s23 = u2h(__byte_perm(par[2], par[3], 0x5410)), l23 = u2h(__byte_perm(par[2], par[3], 0x7632));
#pragma unroll
            for (int x = 0; x < D / 64; ++x) {
#pragma unroll
                for (int y = 0; y < 2; ++y) {  // dims 8 x + 4 y .. + 3 of the lane's D / 8
                    const unsigned sel = y ? 0x7632 : 0x5410;
                    __half2 a[4], b[4];
                    codes_to_half(__byte_perm(vw[0][x], vw[1][x], sel), a);
                    codes_to_half(__byte_perm(vw[2][x], vw[3][x], sel), b);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        a[e] = __hfma2(a[e], s01, l01);
                        b[e] = __hfma2(b[e], s23, l23);
                    }
                    const uint32_t f0[4] = {h2u(a[0]), h2u(a[1]), h2u(b[0]), h2u(b[1])};
                    const uint32_t f1[4] = {h2u(a[2]), h2u(a[3]), h2u(b[2]), h2u(b[3])};
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        mma16816(o[j][4 * x + 2 * y], f0, hi[k][j][0], hi[k][j][1]);
                        mma16816(o[j][4 * x + 2 * y + 1], f1, hi[k][j][0], hi[k][j][1]);
                        if (kPaired) continue;
                        mma16816(o[j][4 * x + 2 * y], f0, lo[k][j][0], lo[k][j][1]);
                        mma16816(o[j][4 * x + 2 * y + 1], f1, lo[k][j][0], lo[k][j][1]);
                    }
                }
            }
            }
        }
        cp_async_wait<0>();
        __syncthreads();

        // ---- the four warps' states -> one; fragment row g of step x is dim 2 x (row g + 8: 2 x + 1)
        // of lane g's D / 8, kept at column dim * 8 + g
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float sum = l[j][e];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                const int r = 8 * j + 2 * t + e;
                if (g == 0) {
                    sm.m[warp][r] = limit[j][e] == -INFINITY ? -INFINITY : base[j][e];
                    sm.l[warp][r] = sum;
                }
#pragma unroll
                for (int x = 0; x < D / 16; ++x) {
                    s_o[(warp * kCols + r) * kPad + (2 * x) * 8 + g] = o[j][x][e];
                    s_o[(warp * kCols + r) * kPad + (2 * x + 1) * 8 + g] = o[j][x][e + 2];
                }
            }
        __syncthreads();
        constexpr int kPer = D / 8, kPasses = ROWS * kPer > 128 ? ROWS * kPer / 128 : 1;  // 8 dims a thread
        const int item = wk.item0 + it, item_tile = wk.base + it * s.ntiles;
        const bool alone = ntile == s.ntiles;
        float* part = parts + ((size_t)blockIdx.x * 2 + (item_tile < w0 ? 0 : 1)) * kDecodePartFloats;
        float mm[kPasses], ll[kPasses], v[kPasses][8];
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            // threads past the last row repeat it (no divergence up to the barriers) and store nothing
            const int mine_r = tid / kPer + p * (128 / kPer), r = min(mine_r, rows - 1), d8 = tid % kPer;
            mm[p] = -INFINITY;
#pragma unroll
            for (int x = 0; x < kWarps; ++x) mm[p] = fmaxf(mm[p], sm.m[x][r]);
            ll[p] = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[p][e] = 0.0f;
#pragma unroll
            for (int x = 0; x < kWarps; ++x) {
                const float f = sm.m[x][r] == -INFINITY ? (sm.l[x][r] != sm.l[x][r] ? 1.0f : 0.0f) : ex2(sm.m[x][r] - mm[p]);
                ll[p] = fmaf(sm.l[x][r], f, ll[p]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int d = d8 * 8 + e;
                    const float* at = s_o + (x * kCols + r) * kPad + (d % (D / 8)) * 8 + d / (D / 8);
                    v[p][e] = fmaf(kPaired ? at[0] + at[4 * kPad] : at[0], f, v[p][e]);
                }
            }
            if (!alone && mine_r == r) {
                float4* dst = reinterpret_cast<float4*>(part + r * D + d8 * 8);
                dst[0] = make_float4(v[p][0], v[p][1], v[p][2], v[p][3]);
                dst[1] = make_float4(v[p][4], v[p][5], v[p][6], v[p][7]);
                if (d8 == 0) {
                    part[ROWS * D + r] = mm[p];
                    part[ROWS * D + ROWS + r] = ll[p];
                }
            }
        }
        bool last = alone;
        __syncwarp();
        if (!alone) {
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const unsigned before = atomicAdd(&counters[item], (unsigned)ntile);
                sm.last = before + (unsigned)ntile == (unsigned)s.ntiles;
                if (sm.last) counters[item] = 0;
            }
            __syncthreads();
            last = sm.last != 0;
            if (last) {
                __threadfence();
                const int c0 = owner(item_tile), c1 = owner(item_tile + s.ntiles - 1);
#pragma unroll
                for (int p = 0; p < kPasses; ++p) {
                    const int r = min(tid / kPer + p * (128 / kPer), rows - 1), d8 = tid % kPer;
                    mm[p] = -INFINITY;
                    ll[p] = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[p][e] = 0.0f;
#pragma unroll 8
                    for (int x = c0; x <= c1; ++x) {
                        const float* src = parts + ((size_t)x * 2 + (item_tile < first_tile(x) ? 0 : 1)) * kDecodePartFloats;
                        const float pm = __ldcg(src + ROWS * D + r), pl = __ldcg(src + ROWS * D + ROWS + r);
                        const float4 a = __ldcg(reinterpret_cast<const float4*>(src + r * D + d8 * 8));
                        const float4 b = __ldcg(reinterpret_cast<const float4*>(src + r * D + d8 * 8) + 1);
                        const float now = fmaxf(mm[p], pm);
                        const float f0 = mm[p] == -INFINITY ? (ll[p] != ll[p] ? 1.0f : 0.0f) : ex2(mm[p] - now);
                        const float f1 = pm == -INFINITY ? (pl != pl ? 1.0f : 0.0f) : ex2(pm - now);
                        mm[p] = now;
                        ll[p] = ll[p] * f0 + pl * f1;
                        const float u[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[p][e] = v[p][e] * f0 + u[e] * f1;
                    }
                }
            }
        }
        if (last) {
#pragma unroll
            for (int p = 0; p < kPasses; ++p) {
                const int mine_r = tid / kPer + p * (128 / kPer), r = min(mine_r, rows - 1), d8 = tid % kPer;
                const int tok = tok0 + (row0 + r) / share, h = qhead0 + (row0 + r) % share;
                const float inv = ll[p] > 0.0f ? 1.0f / ll[p] : 0.0f;
                bool nan = ll[p] != ll[p];
                __half2 out[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float a = v[p][2 * e] * inv, b = v[p][2 * e + 1] * inv;
                    nan |= a != a || b != b;
                    out[e] = __floats2half2_rn(a, b);
                }
                const long long at = (long long)tok * c.hq + h;
                if (mine_r == r) *reinterpret_cast<uint4*>(c.out + at * D + d8 * 8) = *reinterpret_cast<const uint4*>(out);
                if (mine_r == r && d8 == 0 && c.lse)
                    c.lse[at] = ll[p] > 0.0f ? (mm[p] + kHead + log2f(ll[p] * exp2f(-kHead))) * 0.6931471805599453f : -INFINITY;
                if (nan) atomicOr(&sm.nan, 1 << r);
            }
        }
        __syncwarp();
        __syncthreads();
        // A NaN among the values of a row that some of these queries see reaches all of them through
        // the products with weight zero: such rows are computed again one by one.
        const int nan = sm.nan;
        if (nan) {
            for (int r = warp; r < rows; r += kWarps)
                if (nan >> r & 1)
                    attention_row<D>(c, pg, ge, wk.b, tok0 + (row0 + r) / share, qhead0 + (row0 + r) % share, lane);
            __syncthreads();
            if (tid == 0) sm.nan = 0;
        }
        w += ntile;
    }
}

template <int D, int ROWS>
int launch(const AttnCall& c, const Pages& pg, const Geom& ge, int max_rows, cudaStream_t st) {
    auto kernel = kv4_decode_kernel<D, ROWS>;
    constexpr int kPerSm = ctas_per_sm<D, ROWS>(), kBlocks = kWarps * stages<D, ROWS>() * blocks<D, ROWS>() * 16, kMost = kBlocks * (D + 8 * (D / 32));
    const int smem = kBlocks * (D + 8 * ge.ng());
    if (kMost > 48 * 1024) {
        static std::atomic<unsigned long long> set{0};  // a bit a device
        int dev = 0;
        cudaGetDevice(&dev);
        if (!(set.load() >> (dev & 63) & 1)) {
            if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost) != cudaSuccess) return -1;
            set.fetch_or(1ull << (dev & 63));
        }
    }
    // no more CTAs than the tables have room for tiles
    const int share = c.hq / ge.hkv;
    const long long rows_most = std::min<long long>((long long)c.max_q * share, max_rows), tiles = pg.table_stride * ge.page() / (16 * blocks<D, ROWS>() * kWarps) + 2;
    const double bound = (double)c.num_seqs * ge.hkv * ((rows_most + ROWS - 1) / ROWS) * tiles;
    if (bound > 2147483647.0) return -2;  // tiles are counted in 31 bits
    const unsigned grid = (unsigned)(bound < kNumSMs * kPerSm ? bound : kNumSMs * kPerSm);
    return launch_k(kernel, dim3(grid), dim3(kThreads), (size_t)smem, st, c, pg, ge, max_rows,
                    (int)std::min<size_t>(decode_counters(c.num_seqs, c.num_tokens, c.hq, ge.hkv), 0x7fffffff)) == cudaSuccess ? 0 : -1;
}

}  // namespace

size_t decode_counters(int num_seqs, int num_tokens, int hq, int hkv) {
    // one an item: at most a row tile of 8 per 8 rows, and one more a sequence, per kv head
    return ((size_t)num_tokens * (size_t)(hq / hkv) / 8 + (size_t)num_seqs) * (size_t)hkv;
}

int launch_decode(const AttnCall& c, const Pages& pg, const Geom& ge, int max_rows, int usual_rows, cudaStream_t st) {
    // every kernel takes any number of rows, in tiles; the counters allow for tiles of 8 and more, and of 4
    // where no sequence has more rows
    const long long most = std::min<long long>((long long)c.max_q * (c.hq / ge.hkv), max_rows);
    const int rows = most <= 4 ? (int)most : (int)std::min<long long>(most, std::max(usual_rows, 8));
    switch (ge.d) {
        case 64:
            return rows <= 4   ? launch<64, 4>(c, pg, ge, max_rows, st)
                   : rows <= 8 ? launch<64, 8>(c, pg, ge, max_rows, st)
                               : launch<64, 16>(c, pg, ge, max_rows, st);
        case 128:
            return rows <= 4   ? launch<128, 4>(c, pg, ge, max_rows, st)
                   : rows <= 8 ? launch<128, 8>(c, pg, ge, max_rows, st)
                               : launch<128, 16>(c, pg, ge, max_rows, st);
        default: return rows <= 4 ? launch<256, 4>(c, pg, ge, max_rows, st) : launch<256, 8>(c, pg, ge, max_rows, st);
    }
}

}  // namespace kv4
}  // namespace cb
