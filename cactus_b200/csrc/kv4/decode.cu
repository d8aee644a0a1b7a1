// Attention over the 4-bit paged KV cache for few queries a sequence (decode, drafted tokens):
// bound by the cache's bytes.
//
// Work. A sequence's q rows of one kv head (its tokens times the heads that share it, in tiles of
// 8 or 16 rows) over its visible keys is an item; items are cut into tiles of 64 keys, and the
// tiles of all items, in one list, are dealt in equal contiguous ranges to as many CTAs as the GPU
// holds at once, whatever the sequences' lengths. Every CTA finds its range itself from the lengths
// in device memory. An item inside one range is finished there; the parts of one that spans several
// go to the workspace, and the CTA that brings the last part joins them in range order, so the
// result does not depend on which one that is.
//
// CTA. Warp 4 streams tiles into a ring in shared memory with 1-D bulk copies: 16 keys of one head
// are four contiguous pieces (codes and parameters of keys and values) of one page, whatever the
// page size. Warps 0-3 take 16 keys each and keep their own softmax state, so the loop has no
// barrier; the four states are joined at the item's end.
//
// Tensor cores. S^T = K Q^T and O^T = V^T P^T, m16n8k16 with keys (and value dims) on the 16 side
// and q rows on the 8 side: 8 rows waste nothing, and the operand that comes from the cache is the
// A fragment, built in registers from the codes. The k index is permuted freely: lane t of a quad
// takes a contiguous quarter of the head for the keys (the q fragments use the same order), and a
// quarter of the 16 keys for the values, where the codes of two keys are interleaved by bytes first
// so that one mask gives the same dim of both. Key i of the fragment is row kappa(i) of the 16,
// which spreads the lanes' shared-memory reads over the banks. The weights go into O as two fp16
// numbers, p = hi + lo (22 bits): the matrix instructions for lo are idle otherwise, and the result
// is then as good as fp32 weights'.
//
// Softmax. The running maximum is raised only when a score exceeds it by more than 2^kLazy; until
// then weights grow past 1 (at most 2^kLazy, far inside fp16), which is exact up to rounding and
// saves the reduction over the lanes for almost every tile.
#include "attention.cuh"
#include "kv4.cuh"
#include "kv4_ops.h"

namespace cb {
namespace kv4 {

namespace {

constexpr int kConsumers = 4, kThreads = (kConsumers + 1) * 32, kTile = 16 * kConsumers;
constexpr float kLazy = 8.0f;  // base-2 exponent
constexpr int kMaxCtas = kNumSMs * 4;
constexpr int kMaxPartFloats = 16 * (128 + 2);  // rows * (D + 2): 16 x 128 or 8 x 256 (2064) at most
constexpr size_t kPartBytes = (size_t)kMaxCtas * 2 * kMaxPartFloats * 4;

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
__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, unsigned parity, volatile int* abort) {
    if (mbar_try_wait(bar, parity)) return true;
    for (uint32_t i = 0; i < (1u << 24); ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 255) == 255 && *abort) return false;
    }
    *abort = 1;
    return false;
}

// What one sequence asks for, in tiles. Positions fit 31 bits (the entry point checks the table's
// width), byte offsets do not.
struct Seq {
    int tokens, row_tiles;  // queries, tiles of q rows per kv head
    int pos0;               // position of token 0
    int start, end;         // keys that any of its queries sees
    int base, ntiles;       // tiles of 64 keys from base (1 for none: the item still has to write)
};

template <int ROWS>
__device__ __forceinline__ Seq seq_of(const AttnCall& c, const Pages& pg, const Geom& ge, int b, bool report) {
    Seq s;
    const int count = c.offsets[b + 1] - c.offsets[b], len = max(c.lens[b], 0);
    const int room = (int)(pg.table_stride << ge.page_shift);
    s.tokens = max(0, min(count, c.max_q));
    if (report && (count > c.max_q || (len > room && count > 0))) report_dev_error(kDevBadPage);
    s.row_tiles = (s.tokens * (c.hq / ge.hkv) + ROWS - 1) / ROWS;
    s.pos0 = len - count;
    const int n = min(len, room);
    s.end = c.causal ? min(n, s.pos0 + s.tokens) : n;
    s.start = c.window > 0 ? (int)max(0LL, s.pos0 - c.window + 1) : 0;
    if (s.start >= s.end) s.start = s.end = 0;
    s.base = s.start & ~15;
    s.ntiles = max(1, (s.end - s.base + kTile - 1) / kTile);
    return s;
}

template <int D, int NT>
struct Smem {
    static constexpr int kRows = 8 * NT, kPad = D + 4;
    float o[kConsumers][kRows][kPad];
    float m[kConsumers][kRows], l[kConsumers][kRows];
    long long scan[kThreads], scan_items[kThreads];
    long long w0, w1, base, total;  // this CTA's tiles, the first one's sequence's first tile, all tiles
    long long item0;                // that sequence's first item
    int b0, n, last, nan, abort;
};

template <int D>
constexpr int stage_bytes(int ng) { return kTile * (D + 8 * ng); }

template <int D, int NT>
__global__ void __launch_bounds__(kThreads, D * NT <= 128 ? 4 : 2)
    kv4_decode_kernel(const __grid_constant__ AttnCall c, const __grid_constant__ Pages pg, const __grid_constant__ Geom ge,
                      int stages) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int kRows = 8 * NT;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ Smem<D, NT> sm;
    __shared__ uint64_t full[8], empty[8];
    __shared__ int s_ok[8 * kConsumers];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int share = c.hq / ge.hkv, ng = ge.ng();

    // ---- the list of tiles, and this CTA's part of it
    const int per = (c.num_seqs + kThreads - 1) / kThreads, first_b = tid * per;
    long long mine = 0, items = 0;
    for (int b = first_b; b < min(first_b + per, c.num_seqs); ++b) {
        const Seq s = seq_of<kRows>(c, pg, ge, b, blockIdx.x == 0);
        mine += (long long)s.row_tiles * ge.hkv * s.ntiles;
        items += (long long)s.row_tiles * ge.hkv;
    }
    sm.scan[tid] = mine;
    sm.scan_items[tid] = items;
    if (tid == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], kConsumers);
        }
        fence_mbar_init();
        sm.abort = 0;
        sm.nan = 0;
    }
    __syncthreads();
    for (int o = 1; o < kThreads; o <<= 1) {
        const long long a = tid >= o ? sm.scan[tid - o] : 0, i = tid >= o ? sm.scan_items[tid - o] : 0;
        __syncthreads();
        sm.scan[tid] += a;
        sm.scan_items[tid] += i;
        __syncthreads();
    }
    const long long total = sm.scan[kThreads - 1];
    const int n = (int)min((long long)gridDim.x, total);
    if ((int)blockIdx.x >= n) return;
    const long long w0 = total * blockIdx.x / n, w1 = total * (blockIdx.x + 1) / n;
    if (w0 >= sm.scan[tid] - mine && w0 < sm.scan[tid]) {
        long long at = sm.scan[tid] - mine, it = sm.scan_items[tid] - items;
        for (int b = first_b;; ++b) {
            const Seq s = seq_of<kRows>(c, pg, ge, b, false);
            const long long k = (long long)s.row_tiles * ge.hkv;
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
    const int bytes_block = 16 * (D + 8 * ng), bytes_stage = kConsumers * bytes_block;
    volatile int* const abort = &sm.abort;

    // walks the items of [w0, w1): item `it` of sequence b (kv head it / row_tiles), tiles t .. t + k - 1
    struct Walk {
        int b;
        long long base, item0;
        Seq s;
    } wk;
    wk.b = sm.b0;
    wk.base = sm.base;
    wk.item0 = sm.item0;
    wk.s = seq_of<kRows>(c, pg, ge, wk.b, false);
    auto next_seq = [&](long long w) {  // moves to the sequence that tile w belongs to
        while (w >= wk.base + (long long)wk.s.row_tiles * ge.hkv * wk.s.ntiles) {
            wk.base += (long long)wk.s.row_tiles * ge.hkv * wk.s.ntiles;
            wk.item0 += (long long)wk.s.row_tiles * ge.hkv;
            ++wk.b;
            wk.s = seq_of<kRows>(c, pg, ge, wk.b, false);
        }
    };

    if (warp == kConsumers) {
        // ---------------------------------------------------------------- producer
        int issued = 0;
        const int blk = lane >> 2, part = lane & 3;  // lanes 0-15: a 16-key block's four pieces
        const int cb = 16 * (D / 2), pb = 64 * ng;
        const int in_block = (part & 2 ? ge.v_codes() : 0) + (part & 1 ? ge.k_params() : 0);
        const int row_bytes = part & 1 ? 4 * ng : D / 2, piece = part & 1 ? pb : cb;
        const int in_stage = blk * bytes_block + (part & 2 ? cb + pb : 0) + (part & 1 ? cb : 0);
        bool ok = true;
        for (long long w = w0; w < w1 && ok;) {
            next_seq(w);
            const int it = (int)((w - wk.base) / wk.s.ntiles), tile0 = (int)((w - wk.base) % wk.s.ntiles);
            const int head = it / wk.s.row_tiles, ntile = (int)min((long long)(wk.s.ntiles - tile0), w1 - w);
            for (int i = 0; i < ntile; ++i) {
                const int k0 = wk.s.base + (tile0 + i) * kTile + blk * 16;
                long long off = -1;
                if (lane < 16 && k0 < wk.s.end) off = page_offset(pg, wk.b, k0, ge.page_shift);
                const int slot = issued % stages;
                if (issued >= stages && !wait_or_abort(&empty[slot], ((issued / stages) - 1) & 1, abort)) {
                    ok = false;
                    break;
                }
                const unsigned valid = __ballot_sync(0xffffffffu, off >= 0) & 0x1111u;
                if (lane < 16 && part == 0) s_ok[slot * kConsumers + blk] = off >= 0;
                __syncwarp();
                if (lane == 0) {
                    fence_proxy_async_shared();
                    mbar_arrive_expect_tx(&full[slot], (unsigned)(__popc(valid) * bytes_block));
                }
                __syncwarp();
                if (off >= 0) {
                    const int row = k0 & (ge.page() - 1);
                    const uint8_t* src = pg.pool + off + (long long)head * ge.block_bytes() + in_block + row * row_bytes;
                    tma_load_1d(ring + slot * bytes_stage + in_stage, src, (unsigned)piece, &full[slot]);
                }
                ++issued;
            }
            w += ntile;
        }
        // no copy may land after the block leaves
        if (*abort && lane == 0)
            for (int i = issued > stages ? issued - stages : 0; i < issued; ++i)
                mbar_wait_bounded(&full[i % stages], (i / stages) & 1);
        __syncwarp();
        if (lane == 0 && *abort) report_dev_error(kDevTmaTimeout);
        return;
    }

    // ---------------------------------------------------------------- consumers
    const int g = lane >> 2, t = lane & 3;
    const int kg = kappa(g);
    const float sc = c.scale * 1.4426950408889634f;
    float* const parts = reinterpret_cast<float*>(c.ws);
    unsigned* const counters = reinterpret_cast<unsigned*>(c.ws + kPartBytes);
    int used = 0;
    for (long long w = w0; w < w1;) {
        next_seq(w);
        const Seq s = wk.s;
        const long long rel = w - wk.base;
        const int it = (int)(rel / s.ntiles), tile0 = (int)(rel % s.ntiles);
        const int head = it / s.row_tiles, row0 = (it % s.row_tiles) * kRows;
        const int ntile = (int)min((long long)(s.ntiles - tile0), w1 - w);
        const int tok0 = c.offsets[wk.b], rows = min(kRows, s.tokens * share - row0);
        const int qhead0 = head * share;

        // ---- q fragments: column g of n-tile j is row row0 + 8 j + g
        uint32_t q[NT][D / 16][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int r = row0 + 8 * j + g;
            const bool on = 8 * j + g < rows;
            const __half* src = c.q + (long long)(tok0 + (on ? r / share : 0)) * c.q_stride +
                                (long long)(qhead0 + (on ? r % share : 0)) * D + t * (D / 4);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                const uint4 v = on ? __ldg(reinterpret_cast<const uint4*>(src) + i) : uint4{0, 0, 0, 0};
                q[j][2 * i][0] = __byte_perm(v.x, v.z, 0x5410);
                q[j][2 * i][1] = __byte_perm(v.x, v.z, 0x7632);
                q[j][2 * i + 1][0] = __byte_perm(v.y, v.w, 0x5410);
                q[j][2 * i + 1][1] = __byte_perm(v.y, v.w, 0x7632);
            }
        }
        // keys that the two columns of this thread (rows 2 t, 2 t + 1 of each n-tile) see
        int from[NT][2], to[NT][2];
        bool edge_cols = c.window > 0 || (c.causal && s.tokens > 1) || rows < kRows;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = row0 + 8 * j + 2 * t + e;
                const int pos = s.pos0 + r / share;
                from[j][e] = c.window > 0 ? (int)max(0LL, pos - c.window + 1) : 0;
                to[j][e] = c.causal ? min(s.end, pos + 1) : s.end;
                if (8 * j + 2 * t + e >= rows) to[j][e] = 0;
            }
        float o[NT][D / 16][4], m[NT][2], l[NT][2];  // m: base-2 exponent that the state is relative to
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][i][e] = 0.0f;
            m[j][0] = m[j][1] = -INFINITY;
            l[j][0] = l[j][1] = 0.0f;
        }

#pragma unroll 1
        for (int i = 0; i < ntile; ++i, ++used) {
            const int slot = used % stages;
            const bool got = wait_or_abort(&full[slot], (used / stages) & 1, abort);
            const int k0 = s.base + (tile0 + i) * kTile + warp * 16;
            if (got && s_ok[slot * kConsumers + warp]) {
                const uint8_t* blk = ring + slot * bytes_stage + warp * bytes_block;
                const uint8_t* kp = blk + 16 * (D / 2);
                const uint8_t* vc = kp + 64 * ng;
                const uint8_t* vp = vc + 16 * (D / 2);
                const bool whole = k0 >= s.start && k0 + 16 <= s.end;
                // ---- S^T
                float acc[NT][4];
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[j][e] = 0.0f;
                constexpr int kWords = D / 32;  // words of codes of one key in a lane's quarter
                const uint32_t* ka = reinterpret_cast<const uint32_t*>(blk + kg * (D / 2) + t * (D / 8));
                const uint32_t* kb = reinterpret_cast<const uint32_t*>(blk + (kg + 8) * (D / 2) + t * (D / 8));
                uint32_t wa[kWords], wb[kWords];
                if constexpr (kWords >= 4) {
#pragma unroll
                    for (int x = 0; x < kWords / 4; ++x) {
                        *reinterpret_cast<uint4*>(wa + 4 * x) = *reinterpret_cast<const uint4*>(ka + 4 * x);
                        *reinterpret_cast<uint4*>(wb + 4 * x) = *reinterpret_cast<const uint4*>(kb + 4 * x);
                    }
                } else {
                    *reinterpret_cast<uint2*>(wa) = *reinterpret_cast<const uint2*>(ka);
                    *reinterpret_cast<uint2*>(wb) = *reinterpret_cast<const uint2*>(kb);
                }
                __half2 sa, la, sb, lb;
#pragma unroll
                for (int x = 0; x < kWords; ++x) {
                    if (x == 0 || (D == 256 && x == 4)) {  // at most two groups in a lane's quarter
                        const int grp = (t * (D / 4) + x * 8) / ge.g;
                        const __half2 pa = *reinterpret_cast<const __half2*>(kp + (kg * ng + grp) * 4);
                        const __half2 pb = *reinterpret_cast<const __half2*>(kp + ((kg + 8) * ng + grp) * 4);
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
                        mma16816(acc[j], a0, q[j][2 * x][0], q[j][2 * x][1]);
                        mma16816(acc[j], a1, q[j][2 * x + 1][0], q[j][2 * x + 1][1]);
                    }
                }
                // ---- weights
                bool rise = false;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = acc[j][e] * sc;
                        if (!whole || edge_cols) {
                            const int k = k0 + kg + (e & 2 ? 8 : 0);
                            if (k < from[j][e & 1] || k >= to[j][e & 1]) x = -INFINITY;
                        }
                        acc[j][e] = x;
                        rise |= x > m[j][e & 1] + kLazy;
                    }
                }
                if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float top = fmaxf(acc[j][e], acc[j][e + 2]);
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                            const float now = fmaxf(m[j][e], top);
                            const float fix = now > m[j][e] ? ex2(m[j][e] - now) : 1.0f;
                            m[j][e] = now;
                            l[j][e] *= fix;
#pragma unroll
                            for (int x = 0; x < D / 16; ++x) {
                                o[j][x][e] *= fix;
                                o[j][x][e + 2] *= fix;
                            }
                        }
                    }
                }
                uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const float m0 = m[j][0] == -INFINITY ? 0.0f : m[j][0], m1 = m[j][1] == -INFINITY ? 0.0f : m[j][1];
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] = ex2(acc[j][e] - ((e & 1) ? m1 : m0));
                    l[j][0] += p[0] + p[2];
                    l[j][1] += p[1] + p[3];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const __half2 h = __floats2half2_rn(p[2 * e], p[2 * e + 1]);
                        const float2 f = __half22float2(h);
                        hi[j][e] = movmatrix_t(h2u(h));
                        lo[j][e] = movmatrix_t(h2u(__floats2half2_rn(p[2 * e] - f.x, p[2 * e + 1] - f.y)));
                    }
                }
                // ---- O^T
                int vk[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) vk[e] = kappa(2 * t + (e & 1) + (e & 2 ? 8 : 0));
                uint32_t vw[4][D / 64], par[4];
                const int grp = g * (D / 8) / ge.g;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint8_t* src = vc + vk[e] * (D / 2) + g * (D / 16);
                    if constexpr (D == 64) vw[e][0] = *reinterpret_cast<const uint32_t*>(src);
                    if constexpr (D == 128) *reinterpret_cast<uint2*>(vw[e]) = *reinterpret_cast<const uint2*>(src);
                    if constexpr (D == 256) *reinterpret_cast<uint4*>(vw[e]) = *reinterpret_cast<const uint4*>(src);
                    par[e] = *reinterpret_cast<const uint32_t*>(vp + (vk[e] * ng + grp) * 4);
                    // rows that nobody sees may hold anything: they count as zeros
                    if (!whole && (k0 + vk[e] < s.start || k0 + vk[e] >= s.end)) par[e] = 0;
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
                            mma16816(o[j][4 * x + 2 * y], f0, hi[j][0], hi[j][1]);
                            mma16816(o[j][4 * x + 2 * y + 1], f1, hi[j][0], hi[j][1]);
                            mma16816(o[j][4 * x + 2 * y], f0, lo[j][0], lo[j][1]);
                            mma16816(o[j][4 * x + 2 * y + 1], f1, lo[j][0], lo[j][1]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[slot]);
        }

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
                    sm.m[warp][r] = m[j][e];
                    sm.l[warp][r] = sum;
                }
#pragma unroll
                for (int x = 0; x < D / 16; ++x) {
                    sm.o[warp][r][(2 * x) * 8 + g] = o[j][x][e];
                    sm.o[warp][r][(2 * x + 1) * 8 + g] = o[j][x][e + 2];
                }
            }
        consumer_sync();
        constexpr int kPer = D / 8, kPasses = kRows * kPer / 128 ? kRows * kPer / 128 : 1;  // 8 dims a thread
        const long long item = wk.item0 + it, item_tile = wk.base + (long long)it * s.ntiles;
        const bool alone = ntile == s.ntiles;
        float* part = parts + ((size_t)blockIdx.x * 2 + (item_tile < w0 ? 0 : 1)) * kMaxPartFloats;
        float mm[kPasses], ll[kPasses], v[kPasses][8];
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            const int r = tid / kPer + p * (128 / kPer), d8 = tid % kPer;
            if (r >= rows) continue;
            mm[p] = -INFINITY;
#pragma unroll
            for (int x = 0; x < kConsumers; ++x) mm[p] = fmaxf(mm[p], sm.m[x][r]);
            ll[p] = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[p][e] = 0.0f;
#pragma unroll
            for (int x = 0; x < kConsumers; ++x) {
                const float f = sm.m[x][r] == -INFINITY ? (sm.l[x][r] != sm.l[x][r] ? 1.0f : 0.0f) : ex2(sm.m[x][r] - mm[p]);
                ll[p] = fmaf(sm.l[x][r], f, ll[p]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int d = d8 * 8 + e;
                    v[p][e] = fmaf(sm.o[x][r][(d % (D / 8)) * 8 + d / (D / 8)], f, v[p][e]);
                }
            }
            if (!alone) {
                float4* dst = reinterpret_cast<float4*>(part + r * D + d8 * 8);
                dst[0] = make_float4(v[p][0], v[p][1], v[p][2], v[p][3]);
                dst[1] = make_float4(v[p][4], v[p][5], v[p][6], v[p][7]);
                if (d8 == 0) {
                    part[kRows * D + r] = mm[p];
                    part[kRows * D + kRows + r] = ll[p];
                }
            }
        }
        bool last = alone;
        if (!alone) {
            __threadfence();
            consumer_sync();
            if (tid == 0) {
                const unsigned before = atomicAdd(&counters[item], (unsigned)ntile);
                sm.last = before + (unsigned)ntile == (unsigned)s.ntiles;
                if (sm.last) counters[item] = 0;
            }
            consumer_sync();
            last = sm.last != 0;
            if (last) {
                __threadfence();
                const int c0 = (int)(((item_tile + 1) * n - 1) / total);
                const int c1 = (int)(((item_tile + s.ntiles) * n - 1) / total);
#pragma unroll
                for (int p = 0; p < kPasses; ++p) {
                    const int r = tid / kPer + p * (128 / kPer), d8 = tid % kPer;
                    if (r >= rows) continue;
                    mm[p] = -INFINITY;
                    ll[p] = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[p][e] = 0.0f;
#pragma unroll 4
                    for (int x = c0; x <= c1; ++x) {
                        const float* src = parts + ((size_t)x * 2 + (item_tile < total * x / n ? 0 : 1)) * kMaxPartFloats;
                        const float pm = __ldcg(src + kRows * D + r), pl = __ldcg(src + kRows * D + kRows + r);
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
                const int r = tid / kPer + p * (128 / kPer), d8 = tid % kPer;
                if (r >= rows) continue;
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
                *reinterpret_cast<uint4*>(c.out + at * D + d8 * 8) = *reinterpret_cast<const uint4*>(out);
                if (d8 == 0 && c.lse) c.lse[at] = ll[p] > 0.0f ? (mm[p] + log2f(ll[p])) * 0.6931471805599453f : -INFINITY;
                if (nan) atomicOr(&sm.nan, 1 << r);
            }
        }
        consumer_sync();
        // A NaN among the values of a row that some of these queries see reaches all of them through
        // the products with weight zero: such rows are computed again one by one.
        const int nan = sm.nan;
        if (nan) {
            for (int r = warp; r < rows; r += kConsumers)
                if (nan >> r & 1)
                    attention_row<D>(c, pg, ge, wk.b, tok0 + (row0 + r) / share, qhead0 + (row0 + r) % share, lane);
            consumer_sync();
            if (tid == 0) sm.nan = 0;
        }
        w += ntile;
    }
}

template <int D, int NT>
int launch(const AttnCall& c, const Pages& pg, const Geom& ge, cudaStream_t st) {
    auto kernel = kv4_decode_kernel<D, NT>;
    constexpr int kPerSm = D * NT <= 128 ? 4 : 2;
    // as many stages as fit with the CTAs that the registers allow (1 KB of each is the system's)
    const int room = 227 * 1024 / kPerSm - 1024 - (int)sizeof(Smem<D, NT>) - 512;
    int stages = room / stage_bytes<D>(ge.ng());
    stages = stages > 8 ? 8 : stages < 2 ? 2 : stages;
    const int smem = stages * stage_bytes<D>(ge.ng());
    static int most = 0;
    if (smem > most) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -1;
        most = smem;
    }
    // no more CTAs than the tables have room for tiles
    const int share = c.hq / ge.hkv;
    const long long rows_most = (long long)c.max_q * share, tiles = (pg.table_stride * ge.page() + kTile - 1) / kTile + 1;
    const double bound = (double)c.num_seqs * ge.hkv * ((rows_most + 8 * NT - 1) / (8 * NT)) * tiles;
    const unsigned grid = (unsigned)(bound < kNumSMs * kPerSm ? bound : kNumSMs * kPerSm);
    return launch_k(kernel, dim3(grid), dim3(kThreads), (size_t)smem, st, c, pg, ge, stages) == cudaSuccess ? 0 : -1;
}

}  // namespace

size_t decode_workspace(int num_seqs, int num_tokens, int hq, int hkv) {
    // a counter an item: at most a row tile of 8 per 8 rows, and one more a sequence, per kv head
    const size_t items = ((size_t)num_tokens * (size_t)(hq / (hkv ? hkv : 1)) / 8 + (size_t)num_seqs) * (size_t)hkv;
    return kPartBytes + (items * 4 + 15) / 16 * 16;
}

int launch_decode(const AttnCall& c, const Pages& pg, const Geom& ge, cudaStream_t st) {
    const int rows = c.max_q * (c.hq / ge.hkv);
    switch (ge.d) {
        case 64: return rows <= 8 ? launch<64, 1>(c, pg, ge, st) : launch<64, 2>(c, pg, ge, st);
        case 128: return rows <= 8 ? launch<128, 1>(c, pg, ge, st) : launch<128, 2>(c, pg, ge, st);
        default: return launch<256, 1>(c, pg, ge, st);
    }
}

}  // namespace kv4
}  // namespace cb
