// Attention over the 4-bit paged KV cache for many queries a sequence (prompts, their chunks), on the
// 5th-generation tensor cores.
//
// Work. A CTA takes 256 q rows of one sequence and kv head (two tiles of 128; 128 rows at
// head_dim 256), row = token * heads that share the kv head + head, over a range of key tiles (128
// keys, 64 at head_dim 256). The row tiles that do not fill a round of the GPU (all, if they are few)
// have their keys split over several CTAs; the parts go to the workspace, and the CTA that brings the
// last one joins them in order.
//
// Warps (16, whose registers are dealt out by their need), handing over through mbarriers:
//   producer  raw codes and parameters of K and V half tiles into a ring (1-D bulk copies);
//   dequant   codes -> fp16 values in the swizzled operand layout, once for all 256 rows;
//   mma       one thread: S = Q K^T (operands in shared memory), O += P V (P in TMEM);
//   softmax   one thread a row: S from TMEM, weights as two fp16 parts back over S, O rescaled in TMEM when the
//             running maximum has risen by more than 2^kLazy, the result at the end.
// The two row tiles alternate on the tensor core, so one's products overlap the other's softmax; where
// there is one (always at head_dim 256) it has both buffers for S, and S of the next keys is computed
// during the softmax.
//
// Layout. K, V and Q tiles are blocks of 64 elements (128 bytes) by rows with the 128-byte swizzle.
// K and Q are read K-major; V with its rows as the contraction, MN-major, from the same layout. The
// 8 elements of a 16-byte piece stand in the order 0 4 1 5 2 6 3 7 that the unpacking gives: Q is
// permuted alike when it is loaded, and O when it is stored.
// Weights go to the tensor core as two fp16 numbers, p = hi + lo (22 bits), in the columns of the S that
// they come from: hi in its first half, lo in the other, each with a product of its own. They are
// relative to 2^-kHead of the running maximum, as in the kernel for few queries. The tensor core cuts its
// fp32 sums instead of rounding them, twice for 16 keys: a result is low by 4e-6 of it over 2300 rows, 1.9e-5
// over 8192, in proportion to the rows.
//
// What bounds it: a row's chain from S to the next S, of which the other row tile hides about half; it
// has all of the weights' work (the exponentials of two row tiles take 2048 cycles a key tile of 128)
// and both of their products, with which the tensor pipe is busy 67 % of the time. The unpacking of K
// and V takes 2700 cycles on its four warps beside them. On B200: 2048 queries after up to 6144 rows,
// 4 sequences, 16 / 8 heads of 128: 608 us, 726 TFLOP/s of the 4 D operations a pair of query and key
// (with weights of one fp16 number 493 us, but then their rounding is as large as the result's; floor
// 266 us at the measured peak). 256 queries with a window of 512, 4 heads of 256 on one, 16 sequences:
// 31 us, of which the start takes 6, the results 4 and 9 key tiles the rest.
//
// This file is compiled as whole-program device code (build.py WHOLE_PROGRAM).
#include <atomic>

#include "attention.cuh"
#include "kv4.cuh"
#include "kv4_ops.h"

namespace cb {
namespace kv4 {

namespace {

constexpr int kWarps = 16, kThreads = kWarps * 32, kMma = 12, kProducer = 13;  // warps 14 and 15 have no work
constexpr float kLazy = 8.0f, kHead = 7.0f;  // base-2 exponents

template <int D>
struct Cfg {
    static constexpr int kKeys = D == 256 ? 64 : 128;   // of a tile
    static constexpr int kTiles = D == 256 ? 1 : 2;     // row tiles
    static constexpr int kRows = 128 * kTiles;
    static constexpr int kBufBytes = kKeys * D * 2;     // a K or V tile in fp16
    static constexpr int kBufs = D == 64 ? 6 : 4;
    static constexpr int kRaw = D == 64 ? 6 : 3;         // raw half tiles
    static constexpr int kSoftmax = 4 * kTiles, kDequant = kMma - kSoftmax;  // warps
    // registers a thread: the block is launched with 128 each
    static constexpr int kSoftmaxRegs = 184, kDequantRegs = kTiles == 2 ? 88 : 96, kOtherRegs = 56;
    static constexpr int kRegs = 32 * (kSoftmax * kSoftmaxRegs + kDequant * kDequantRegs + 4 * kOtherRegs);
    static constexpr int kQBytes = kRows * D * 2;
    static constexpr int kO = 256;                      // TMEM column of O (S: kKeys columns a row tile from 0)
    __host__ __device__ static constexpr int raw_bytes(int ng) { return kKeys * (D / 2 + 4 * ng); }
    __host__ __device__ static constexpr int smem(int ng) { return kQBytes + kBufs * kBufBytes + kRaw * raw_bytes(ng) + 1024; }
};

struct Args {
    AttnCall c;
    Pages pg;
    Geom ge;
    unsigned* err;
    float* parts;
    unsigned* counters;
    int min_rows;    // sequences with fewer rows a kv head are another kernel's
    int most_parts;  // of a row tile's keys
};

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Shared-memory matrix descriptor with the 128-byte swizzle: 8-row groups 1024 bytes apart; LBO is
// the distance of 64-element blocks for the MN-major operand (not used for K-major).
__device__ __forceinline__ uint64_t desc(uint32_t addr, uint32_t lbo) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// kind::f16: D fp32, A and B fp16, M = 128; B MN-major where mn
constexpr uint32_t idesc(int n, bool mn) {
    return (1u << 4) | ((mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
// The issuing warp runs converged, one elected lane's predicate on the instructions themselves: their
// operands then stay in uniform registers (in a branch of one lane each product took 120 cycles to issue).
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(acc),
        "r"(leader));
}
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(acc),
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
// The same without the wait: the registers hold the values after tmem_wait_ld on them.
__device__ __forceinline__ void tmem_ld32_start(uint32_t taddr, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
          "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
          "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
          "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr)
        : "memory");
}
// Waits for every load of the thread; the operands keep uses of the registers behind it.
__device__ __forceinline__ void tmem_wait_ld(float (&v)[32]) {
    asm volatile(
        "tcgen05.wait::ld.sync.aligned;"
        : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
          "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]),
          "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]),
          "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
        :
        : "memory");
}
// Two fp32 operations in one instruction, each rounded as its own
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)),
          "l"(reinterpret_cast<unsigned long long&>(c)));
    return d;
}
// w - h in one instruction; with h converted to fp32 first the prompts above take 682 us
__device__ __forceinline__ float rest_of(__half h, float w) {
    float d;
    asm("fma.rn.f32.f16 %0, %1, %2, %3;" : "=f"(d) : "h"(__half_as_ushort(h)), "h"((unsigned short)0xBC00), "f"(w));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<unsigned long long&>(a)), "l"(reinterpret_cast<unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, unsigned parity, volatile int* abort) {
    if (mbar_try_wait(bar, parity)) return true;
    for (uint32_t i = 0; i < (1u << 24); ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 63) == 63 && *abort) return false;
    }
    *abort = 1;
    return false;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) kv4_prefill_kernel(const __grid_constant__ Args a) {
    pdl_launch_dependents();
    using C = Cfg<D>;
    constexpr int KT = C::kKeys, MT = C::kTiles;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* const s_q = smem;                       // [row tile][D / 64][128 rows][128 bytes]
    uint8_t* const s_buf = smem + C::kQBytes;        // ring of K, V tiles [D / 64][KT rows][128 bytes]
    uint8_t* const s_raw = s_buf + C::kBufs * C::kBufBytes;
    __shared__ uint64_t s_full[2], p_full[2][2], o_full[2], pv_done, buf_full[C::kBufs], buf_free[C::kBufs], raw_full[C::kRaw],
        raw_free[C::kRaw], q_full, drain;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort, s_item[4], s_scan[kWarps], s_last;
    __shared__ unsigned s_valid[8];  // a bit for each 16 keys of a tile that were loaded, tiles modulo 8
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const AttnCall& c = a.c;
    const Pages& pg = a.pg;
    const Geom& ge = a.ge;
    const int share = c.hq / ge.hkv, ng = ge.ng();
    pdl_wait();

    // ---- which sequence, rows, kv head and part of the keys: row tiles of a sequence from its last,
    // which sees the most
    const int per = (c.num_seqs + kThreads - 1) / kThreads;
    auto row_tiles = [&](int b) {
        const int from = c.offsets[b], to = c.offsets[b + 1];
        if (from < 0 || from > to || to > c.num_tokens) {  // the sequence is left out
            atomicCAS(a.err, 0u, (unsigned)kDevBadPage);
            return 0;
        }
        const int rows = min(to - from, c.max_q) * share;
        return rows < a.min_rows ? 0 : (rows + C::kRows - 1) / C::kRows;
    };
    int mine = 0;
    for (int b = tid * per; b < min((tid + 1) * per, c.num_seqs); ++b) mine += row_tiles(b);
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) s_scan[warp] = upto;
    if (tid == 0) {
        s_item[0] = -1;
        s_abort = 0;
    }
    __syncthreads();
    int items = 0;
    for (int x = 0; x < kWarps; ++x) {
        if (x < warp) upto += s_scan[x];
        items += s_scan[x] * ge.hkv;
    }
    // whole rounds of the GPU first; the rest in as many parts as a round has room for
    const int whole_items = items / kNumSMs * kNumSMs, rest = items - whole_items;
    const int parts = rest ? min(kNumSMs / rest, a.most_parts) : 1, unit = (int)blockIdx.x - whole_items;
    if (unit >= rest * parts) return;
    const int splits = unit < 0 ? 1 : parts, split = unit < 0 ? 0 : unit % parts;
    const int item = unit < 0 ? (int)blockIdx.x : whole_items + unit / parts;
    const int pair = item / ge.hkv, head = item % ge.hkv;
    if (pair >= upto - mine && pair < upto) {
        int at = upto - mine, b = tid * per;
        for (;; ++b) {
            const int k = row_tiles(b);
            if (pair < at + k) {
                s_item[0] = b;
                s_item[1] = k - 1 - (pair - at);
                break;
            }
            at += k;
        }
    }
    __syncwarp();
    __syncthreads();
    const int b = s_item[0];
    if (b < 0) return;
    const int count = c.offsets[b + 1] - c.offsets[b], tok0 = c.offsets[b], tokens = min(count, c.max_q);
    const int row0 = s_item[1] * C::kRows, rows = min(C::kRows, tokens * share - row0);
    const int len = max(c.lens[b], 0), room = (int)(pg.table_stride << ge.page_shift), n = min(len, room);
    const int pos0 = len - count;  // position of token 0
    if (tid == 0 && (count > c.max_q || len > room)) atomicCAS(a.err, 0u, (unsigned)kDevBadPage);
    // the keys that these rows see, and this part's tiles of them
    const int first_tok = row0 / share, last_tok = (row0 + rows - 1) / share;
    int end = c.causal ? min(n, pos0 + last_tok + 1) : n;
    int start = c.window > 0 ? (int)max(0LL, pos0 + first_tok - c.window + 1) : 0;
    if (start >= end) start = end = 0;
    const int base = start & ~(KT - 1), all = (end - base + KT - 1) / KT;
    const int t_from = (int)((long long)all * split / splits), t_to = (int)((long long)all * (split + 1) / splits);
    const int tiles = t_to - t_from, key0 = base + t_from * KT;
    const bool one = MT == 1 || rows <= 128;  // one row tile: it has both S buffers

    // ---- set-up: barriers, TMEM
    if (warp == kMma) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        mbar_init(&pv_done, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i][0], 128);
            mbar_init(&p_full[i][1], 128);
            mbar_init(&o_full[i], 1);
        }
        for (int i = 0; i < C::kBufs; ++i) {
            mbar_init(&buf_full[i], C::kDequant * 32);
            mbar_init(&buf_free[i], 1);
        }
        for (int i = 0; i < C::kRaw; ++i) {
            mbar_init(&raw_full[i], 1);
            mbar_init(&raw_free[i], C::kDequant);
        }
        mbar_init(&q_full, kMma * 32);
        mbar_init(&drain, 1);
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    volatile int* const abort = &s_abort;
    const int halves = 2 * tiles;  // K and V of each tile in turn
    const int R = min(ge.page(), KT), half_chunk = R * (D / 2 + 4 * ng), raw_bytes = C::raw_bytes(ng);

    auto load_q = [&] {  // by the softmax and dequantisation warps, while the first keys are on their way
        constexpr int kAll = C::kRows * (D / 8), kStep = kMma * 32,
                      kBatch = (kAll + kStep - 1) / kStep;  // all loads in flight at once
        const int i0 = tid;
        {
            uint4 v[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int i = i0 + u * kStep, r = i / (D / 8), row = row0 + r, token = row / share;
                v[u] = uint4{0, 0, 0, 0};
                if (i < kAll && r < rows)
                    v[u] = __ldg(reinterpret_cast<const uint4*>(c.q + (long long)(tok0 + token) * c.q_stride +
                                                                (long long)(head * share + row - token * share) * D) +
                                 i % (D / 8));
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int i = i0 + u * kStep, r = i / (D / 8), ch = i % (D / 8), rt = r & 127;
                if (i < kAll)
                    *reinterpret_cast<uint4*>(s_q + (r >> 7) * (128 * D * 2) + (ch >> 3) * (128 * 128) + rt * 128 +
                                              (((ch & 7) ^ (rt & 7)) << 4)) =
                        uint4{__byte_perm(v[u].x, v[u].z, 0x5410), __byte_perm(v[u].x, v[u].z, 0x7632),
                              __byte_perm(v[u].y, v[u].w, 0x5410), __byte_perm(v[u].y, v[u].w, 0x7632)};
            }
        }
        fence_proxy_async_shared();
        mbar_arrive(&q_full);
    };

    // each role starts with its share of the registers (a warpgroup asks for one number)
    if (warp >= kMma) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kOtherRegs));
    if (warp == kProducer) {
        // ------------------------------------------------------------ producer
        // lane 2 i + p: chunk i of a half tile (the rows of one page), codes (0) or parameters (1); a
        // chunk that is all of a page's rows is one piece
        const int chunk = lane >> 1, part = lane & 1;
        int issued = 0;
        for (int h = 0; h < halves; ++h) {
            const int slot = h % C::kRaw, tile = h >> 1, k0 = key0 + tile * KT + chunk * R;
            long long off = -1;
            if (chunk * R < KT && k0 < end && k0 + R > start) {
                off = page_offset(pg, b, k0, ge.page_shift);
                if (off < 0 && part == 0 && !(h & 1)) atomicCAS(a.err, 0u, (unsigned)kDevBadPage);
            }
            const int n_rows = min(R, (end - k0 + 15) & ~15);
            const int bytes = __reduce_add_sync(0xffffffffu, off >= 0 && part == 0 ? (R == ge.page() ? R : n_rows) * (D / 2 + 4 * ng) : 0);
            if (h >= C::kRaw && !wait_or_abort(&raw_free[slot], ((h / C::kRaw) - 1) & 1, abort)) break;
            if (!(h & 1)) {
                unsigned bits = 0;
                if (off >= 0 && part == 0) bits = ((1u << (R / 16)) - 1) << (chunk * R / 16);
                bits = __reduce_or_sync(0xffffffffu, bits);
                if (lane == 0) s_valid[tile & 7] = bits;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive_expect_tx(&raw_full[slot], (unsigned)bytes);
            __syncwarp();
            if (off >= 0 && !(R == ge.page() && part)) {
                const int row_bytes = part ? 4 * ng : D / 2, r = k0 & (ge.page() - 1);
                const uint8_t* src = pg.pool + off + (long long)head * ge.block_bytes() + (h & 1 ? ge.v_codes() : 0) +
                                     (part ? ge.k_params() : 0) + r * row_bytes;
                tma_load_1d(s_raw + slot * raw_bytes + chunk * half_chunk + (part ? R * (D / 2) : 0), src,
                            (unsigned)(R == ge.page() ? half_chunk : n_rows * row_bytes), &raw_full[slot]);
            }
            ++issued;
        }
        // no copy may land after the block leaves
        if (*abort && lane == 0)
            for (int h = max(0, issued - C::kRaw); h < issued; ++h) mbar_wait_bounded(&raw_full[h % C::kRaw], (h / C::kRaw) & 1);
    } else if (warp == kMma) {
        // ------------------------------------------------------------ tensor core
        {
            const uint32_t leader = elect_one();
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const int n_tiles = __shfl_sync(0xffffffffu, tiles, 0), alone = __shfl_sync(0xffffffffu, (int)one, 0);
            // descriptors differ from these by constants: a product must take less time to issue than to run
            const uint64_t q_desc = desc(smem_u32(s_q), 16), k_desc = desc(smem_u32(s_buf), 16),
                           v_desc = desc(smem_u32(s_buf), KT * 128);
            bool ok = true;
            auto need = [&](int h) -> int {  // waits for half tile h (K of tile h / 2, or its V) and returns its slot
                const int s = h % C::kBufs;
                ok = ok && __all_sync(0xffffffffu, wait_or_abort(&buf_full[s], (h / C::kBufs) & 1, abort));
                tc_fence_after();
                return s;
            };
            auto qk = [&](int t, int buf, int s) {
                const uint64_t qa = q_desc + (uint64_t)(t * (128 * D * 2 / 16)), kb = k_desc + (uint64_t)(s * (C::kBufBytes / 16));
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    mma_ss(leader, tm + buf * KT, qa + ((k >> 2) * (128 * 128) + (k & 3) * 32) / 16,
                           kb + ((k >> 2) * (KT * 128) + (k & 3) * 32) / 16, idesc(KT, false), k > 0);
                commit(leader, &s_full[buf]);
            };
            auto pv = [&](int t, int buf, int s, int parity, bool first) {
                const uint64_t vb = v_desc + (uint64_t)(s * (C::kBufBytes / 16));
#pragma unroll
                for (int half = 0; half < 2; ++half) {  // the weights come in two halves
                    ok = ok && __all_sync(0xffffffffu, wait_or_abort(&p_full[buf][half], parity, abort));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int k = half * (KT / 32); k < (half + 1) * (KT / 32); ++k) {
                        const uint32_t p = tm + buf * KT + k * 8;  // high parts, low parts
                        mma_ts(leader, tm + C::kO + t * D, p, vb + k * (2048 / 16), idesc(D, true), !first || k > 0);
                        mma_ts(leader, tm + C::kO + t * D, p + KT / 2, vb + k * (2048 / 16), idesc(D, true), 1);
                    }
                }
            };
            if (n_tiles > 0) {
                ok = __all_sync(0xffffffffu, wait_or_abort(&q_full, 0, abort));
                const int s = need(0);
                for (int t = 0; t < (alone ? 1 : MT) && ok; ++t) qk(t, t, s);
                if (ok) commit(leader, &buf_free[s]);
            }
            for (int j = 0; j < n_tiles && ok; ++j) {
                const bool more = j + 1 < n_tiles;
                if (alone) {  // S of the next tile into the other buffer, then this tile's values
                    if (more) {
                        const int s = need(2 * j + 2);
                        if (!ok) break;
                        qk(0, (j + 1) & 1, s);
                        commit(leader, &buf_free[s]);
                    }
                    const int s = need(2 * j + 1);
                    pv(0, j & 1, s, (j >> 1) & 1, j == 0);
                    if (!ok) break;
                    commit(leader, &buf_free[s]);
                    commit(leader, &pv_done);
                    if (!more) commit(leader, &o_full[0]);
                } else {
                    int vs = 0, ks = 0;
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        if (t == 0) vs = need(2 * j + 1);
                        pv(t, t, vs, j & 1, j == 0);
                        if (!ok) break;
                        if (t == MT - 1) commit(leader, &buf_free[vs]);
                        if (more) {
                            if (t == 0) ks = need(2 * j + 2);
                            if (!ok) break;
                            qk(t, t, ks);
                            if (t == MT - 1) commit(leader, &buf_free[ks]);
                        } else {
                            commit(leader, &o_full[t]);
                        }
                    }
                }
            }
            commit(leader, &drain);  // every product issued has completed before TMEM is released
            mbar_wait_bounded(&drain, 0);
        }
        __syncwarp();
    }
    } else if (warp >= C::kSoftmax) {
        // ------------------------------------------------------------ dequantisation
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kDequantRegs));
        load_q();
        // A task is 32 elements of a row: piece q of row r. Neighbouring lanes take 4 rows by 2 pieces, so
        // that their stores miss each other's banks; a thread keeps its piece and goes down the rows.
        constexpr int kTasks = KT * (D / 32), kStep = C::kDequant * 32 / (D / 32);  // rows from task to task
        static_assert(C::kDequant * 32 % (2 * D / 8) == 0 && kTasks % (2 * C::kDequant * 32) == 0, "a thread keeps its piece");
        const int dt = tid - C::kSoftmax * 32, q = ((dt >> 3) % (D / 64)) * 2 + (dt & 1);
        const int r0 = (dt >> 3) / (D / 64) * 4 + ((dt >> 1) & 3);
        const int shift = 31 - __clz(R), par_at = R * (D / 2) + (q * 32 / ge.g) * 4, row_p = 4 * ng;
        for (int h = 0; h < halves; ++h) {
            const int slot = h % C::kRaw, bslot = h % C::kBufs, k0 = key0 + (h >> 1) * KT;
            if (!wait_or_abort(&raw_full[slot], (h / C::kRaw) & 1, abort)) break;
            if (h >= C::kBufs && !wait_or_abort(&buf_free[bslot], ((h / C::kBufs) - 1) & 1, abort)) break;
            const uint8_t* raw = s_raw + slot * raw_bytes;
            uint8_t* out = s_buf + bslot * C::kBufBytes + (q >> 1) * (KT * 128);
            const unsigned valid = s_valid[(h >> 1) & 7];
            const bool whole = valid == (1u << (KT / 16)) - 1 && k0 >= start && k0 + KT <= end;
            constexpr int kMine = kTasks / (C::kDequant * 32);
#pragma unroll 1
            for (int i0 = 0; i0 < kMine; i0 += 2) {  // two tasks' loads first
                uint4 w[2];
                uint32_t par[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int r = r0 + (i0 + u) * kStep, rr = r & (R - 1);
                    const uint8_t* src = raw + (r >> shift) * half_chunk;
                    w[u] = *reinterpret_cast<const uint4*>(src + rr * (D / 2) + q * 16);
                    par[u] = *reinterpret_cast<const uint32_t*>(src + rr * row_p + par_at);
                    // rows that nobody sees may hold anything: they count as zeros
                    if (!whole && !((valid >> (r >> 4) & 1) && k0 + r >= start && k0 + r < end)) par[u] = 0;
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const __half2 step = __low2half2(as_half2(par[u])), low = __high2half2(as_half2(par[u]));
                    const uint32_t ww[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
                    uint8_t* dst = out + (r0 + (i0 + u) * kStep) * 128;
                    const int x7 = (r0 + (i0 + u) * kStep) & 7;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        __half2 f[4];
                        codes_to_half(ww[x], f);
#pragma unroll
                        for (int e = 0; e < 4; ++e) f[e] = __hfma2(f[e], step, low);
                        *reinterpret_cast<uint4*>(dst + ((((q & 1) * 4 + x) ^ x7) << 4)) = *reinterpret_cast<const uint4*>(f);
                    }
                }
            }
            fence_proxy_async_shared();
            mbar_arrive(&buf_full[bslot]);
            __syncwarp();
            if (lane == 0) mbar_arrive(&raw_free[slot]);
        }
    } else {
        // ------------------------------------------------------------ softmax: a thread a row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kSoftmaxRegs));
        load_q();
        const int t = warp >> 2, r = t * 128 + (warp & 3) * 32 + lane, row = row0 + r;
        const bool on = r < rows;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t o_at = tmem + lanes + C::kO + t * D;
        const int tok = tok0 + (on ? row / share : 0), qh = head * share + row % share;
        const int pos = pos0 + (on ? row / share : 0);
        // the row sees keys [lo, hi); rows past the last one see all, and nobody reads them
        const int lo = on && c.window > 0 ? (int)max(0LL, pos - c.window + 1) : 0;
        const int hi = !on ? INT_MAX : c.causal ? min(n, pos + 1) : n;
        const float sc = c.scale * 1.4426950408889634f;
        float m = 0.0f, limit = -INFINITY, l = 0.0f;  // as in the kernel for few queries
        bool ok = true;
        const int my_tiles = t == 0 || !one ? tiles : 0;
        for (int j = 0; j < my_tiles; ++j) {
            // its S buffer: its row tile's, or where there is one row tile the two in turn
            const int buf = one ? j & 1 : t;
            const uint32_t s_at = tmem + lanes + buf * KT;
            if (!(ok = wait_or_abort(&s_full[buf], (one ? j >> 1 : j) & 1, abort))) break;
            tc_fence_after();
            const int k0 = key0 + j * KT;
            const unsigned valid = s_valid[j & 7];
            const bool whole = lo <= k0 && hi >= k0 + KT && valid == (1u << (KT / 16)) - 1;
            const bool masked = __any_sync(0xffffffffu, !whole);
            float x[KT / 32][32], tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < KT / 32; ++i) tmem_ld32_start(s_at + i * 32, x[i]);
#pragma unroll
            for (int i = 0; i < KT / 32; ++i) tmem_wait_ld(x[i]);
            if (masked) {
#pragma unroll
                for (int i = 0; i < KT / 32; ++i) {
                    const int c0 = i * 32;
                    const int c_lo = min(max(lo - k0 - c0, 0), 32), c_hi = min(max(max(hi, k0) - k0 - c0, 0), 32);
                    unsigned bits = (c_hi == 32 ? ~0u : (1u << c_hi) - 1) & (c_lo == 32 ? 0u : ~0u << c_lo);
                    bits &= ((valid >> (c0 / 16) & 1) ? 0xFFFFu : 0u) | ((valid >> (c0 / 16) & 2) ? 0xFFFF0000u : 0u);
#pragma unroll
                    for (int e = 0; e < 32; ++e) x[i][e] = bits >> e & 1 ? x[i][e] : -INFINITY;
                }
            }
#pragma unroll
            for (int i = 0; i < KT / 32; ++i)
#pragma unroll
                for (int e = 0; e < 32; e += 8)
#pragma unroll
                    for (int k = 0; k < 4; ++k) tops[k] = fmaxf(tops[k], fmaxf(x[i][e + 2 * k], x[i][e + 2 * k + 1]));
            float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
            top *= sc;
            if (__any_sync(0xffffffffu, top > limit)) {
                float fix = 1.0f;
                if (top > limit) {
                    const float now = top - kHead;
                    fix = limit == -INFINITY ? 0.0f : ex2(m - now);
                    m = now;
                    limit = __fadd_rd(now, kHead + kLazy);
                    l *= fix;
                }
                if (j > 0) {  // with a row tile's own buffer its S was computed after the products before
                    if (one) ok = wait_or_abort(&pv_done, (j - 1) & 1, abort);
                    tc_fence_after();
#pragma unroll 1
                    for (int d = 0; d < D; d += 16) {
                        uint32_t v[16];
                        tmem_ld16(o_at + d, v);
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * fix);
                        tmem_st16(o_at + d, v);
                    }
                }
            }
            const float2 scale2 = make_float2(sc, sc), shift2 = make_float2(-m, -m);
            float2 sums[2] = {};
            auto hand_over = [&](int half) {
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&p_full[buf][half]);
            };
#pragma unroll
            for (int i = 0; i < KT / 16; ++i) {
                uint32_t p[8], rest[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float* const s2 = &x[i / 2][(i & 1) * 16 + 2 * e];
                    float2 w = fma2(make_float2(s2[0], s2[1]), scale2, shift2);
                    w = make_float2(ex2(w.x), ex2(w.y));
                    sums[e & 1] = add2(sums[e & 1], w);
                    const __half2 h = __floats2half2_rn(w.x, w.y);
                    const __half2 lo = __floats2half2_rn(rest_of(__low2half(h), w.x), rest_of(__high2half(h), w.y));
                    p[e] = *reinterpret_cast<const uint32_t*>(&h);
                    rest[e] = *reinterpret_cast<const uint32_t*>(&lo);
                }
                tmem_st8(s_at + i * 8, p);  // over S, which this thread has read
                tmem_st8(s_at + KT / 2 + i * 8, rest);
                if ((i + 1) % (KT / 32) == 0) hand_over(i / (KT / 32));
            }
            l += (sums[0].x + sums[0].y) + (sums[1].x + sums[1].y);
        }
        if (my_tiles > 0 && ok) ok = wait_or_abort(&o_full[t], 0, abort);
        // the result goes through Q's memory, which every warp has to be done filling: without key tiles no
        // product has waited for that
        if (ok) ok = wait_or_abort(&q_full, 0, abort);
        tc_fence_after();
        // ---- the result, or this part of it
        const float m_out = limit == -INFINITY ? -INFINITY : m;
        bool last = splits == 1;
        const int slot0 = unit - split;  // where there are parts
        constexpr int kSlot = C::kRows * (D + 2);  // floats: [D / 4][row][4], then m and l of the rows
        if (!last) {
            float* part = a.parts + (size_t)(slot0 + split) * kSlot;
            if (__any_sync(0xffffffffu, on)) {
#pragma unroll
                for (int d = 0; d < D; d += 32) {
                    float v[32];
                    tmem_ld32(o_at + d, v);
#pragma unroll
                    for (int i = 0; i < 32; i += 4)  // a part that saw nothing has zeros
                        *reinterpret_cast<float4*>(part + ((size_t)((d + i) / 4) * C::kRows + r) * 4) =
                            tiles > 0 ? make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
            }
            part[(size_t)C::kRows * D + r] = m_out;
            part[(size_t)C::kRows * D + C::kRows + r] = l;
            __threadfence();
            asm volatile("bar.sync 1, %0;" ::"n"(C::kSoftmax * 32) : "memory");
            if (tid == 0) {
                const unsigned before = atomicAdd(&a.counters[item - whole_items], 1u);
                s_last = before + 1 == (unsigned)splits;
                if (s_last) a.counters[item - whole_items] = 0;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(C::kSoftmax * 32) : "memory");
            last = s_last != 0;
            __threadfence();
        }
        if (last) {
            float mm = m_out, ll = l;
            if (splits > 1) {
                mm = -INFINITY;
                for (int x = 0; x < splits; ++x)
                    mm = fmaxf(mm, __ldcg(a.parts + (size_t)(slot0 + x) * kSlot + (size_t)C::kRows * D + r));
                ll = 0.0f;
                for (int x = 0; x < splits; ++x) {
                    const float* p = a.parts + (size_t)(slot0 + x) * kSlot + (size_t)C::kRows * D + r;
                    const float pl = __ldcg(p + C::kRows), pm = __ldcg(p);
                    ll += pl * (pm == -INFINITY ? (pl != pl ? 1.0f : 0.0f) : ex2(pm - mm));
                }
            }
            const float inv = ll > 0.0f ? 1.0f / ll : 0.0f;
            const float2 inv2 = make_float2(inv, inv), zero2 = {};
            float2 test = {};
            const long long at = (long long)tok * c.hq + qh;
            // this row tile's part of Q's memory, which no product reads any more
            uint8_t* const s_row = s_q + t * (128 * D * 2) + (warp & 3) * (32 * D * 2);
#pragma unroll
            for (int d = 0; d < D; d += 32) {
                float v[32];
                if (splits == 1) {
                    if (tiles > 0) {
                        tmem_ld32(o_at + d, v);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = 0.0f;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0.0f;
                    if (on) {
#pragma unroll 4
                        for (int x = 0; x < splits; ++x) {  // the parts' loads overlap
                            const float* p = a.parts + (size_t)(slot0 + x) * kSlot;
                            const float pm = __ldcg(p + (size_t)C::kRows * D + r), pl = __ldcg(p + (size_t)C::kRows * D + C::kRows + r);
                            const float f = pm == -INFINITY ? (pl != pl ? 1.0f : 0.0f) : ex2(pm - mm);
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                const float4 u = __ldcg(reinterpret_cast<const float4*>(p + ((size_t)((d + i) / 4) * C::kRows + r) * 4));
                                v[i] = fmaf(u.x, f, v[i]);
                                v[i + 1] = fmaf(u.y, f, v[i + 1]);
                                v[i + 2] = fmaf(u.z, f, v[i + 2]);
                                v[i + 3] = fmaf(u.w, f, v[i + 3]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < 32; e += 8) {  // column e + i is dim e + {0, 4, 1, 5, 2, 6, 3, 7}[i]
                    float2 f[4];  // dims k and k + 4
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        f[k] = fma2(make_float2(v[e + 2 * k], v[e + 2 * k + 1]), inv2, zero2);
                        test = fma2(f[k], zero2, test);  // not a number from here on if this is none
                    }
                    const __half2 h[4] = {__floats2half2_rn(f[0].x, f[1].x), __floats2half2_rn(f[2].x, f[3].x),
                                          __floats2half2_rn(f[0].y, f[1].y), __floats2half2_rn(f[2].y, f[3].y)};
                    *reinterpret_cast<uint4*>(s_row + lane * (D * 2) + ((((d + e) / 8) ^ (lane & 7)) << 4)) =
                        *reinterpret_cast<const uint4*>(h);
                }
            }
            // the warp's rows to memory, neighbouring lanes along a row
            __syncwarp();
#pragma unroll 4
            for (int i = lane; i < 32 * (D / 8); i += 32) {
                const int rr = i / (D / 8), ch = i % (D / 8);
                const long long to = __shfl_sync(0xffffffffu, on ? at : -1, rr);
                if (to >= 0)
                    *reinterpret_cast<uint4*>(c.out + to * D + ch * 8) =
                        *reinterpret_cast<const uint4*>(s_row + rr * (D * 2) + ((ch ^ (rr & 7)) << 4));
            }
            __syncwarp();
            if (on && c.lse) c.lse[at] = ll > 0.0f ? (mm + kHead + log2f(ll * exp2f(-kHead))) * 0.6931471805599453f : -INFINITY;
            // rows whose result is not a number are computed again one by one: a NaN among the values
            // reaches rows that do not see it through weights of zero
            unsigned again = __ballot_sync(0xffffffffu, on && !(ll == ll && test.x + test.y == 0.0f) && !*abort);
            while (again) {
                const int x = __ffs(again) - 1;
                again &= again - 1;
                attention_row<D>(c, pg, ge, b, __shfl_sync(0xffffffffu, tok, x), __shfl_sync(0xffffffffu, qh, x), lane);
            }
        }
    }
    tc_fence_before();
    __syncwarp();
    __syncthreads();
    if (tid == 0 && *abort) atomicCAS(a.err, 0u, (unsigned)kDevTmaTimeout);
    if (warp == kMma) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <int D>
int launch(const AttnCall& c, const Pages& pg, const Geom& ge, int min_rows, cudaStream_t st) {
    using C = Cfg<D>;
    auto kernel = kv4_prefill_kernel<D>;
    static std::atomic<unsigned long long> set{0};  // a bit a device
    int dev = 0;
    cudaGetDevice(&dev);
    if (!(set.load() >> (dev & 63) & 1)) {
        // the registers that the warps deal out among themselves have to be there
        cudaFuncAttributes attr;
        if (cudaFuncGetAttributes(&attr, kernel) != cudaSuccess || attr.numRegs * kThreads < C::kRegs) return -1;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::smem(D / 32)) != cudaSuccess)
            return -1;
        set.fetch_or(1ull << (dev & 63));
    }
    Args a = {};
    a.c = c;
    a.pg = pg;
    a.ge = ge;
    a.err = dev_error_ptr();
    if (!a.err) return -1;
    a.parts = reinterpret_cast<float*>(c.ws);
    a.counters = reinterpret_cast<unsigned*>(c.ws + kPartBytes);
    a.min_rows = min_rows;
    // row tiles: no more than the tokens fill, and one a sequence that they fill in part
    const int share = c.hq / ge.hkv;
    const long long rows = (long long)c.num_tokens * share, most = (long long)c.max_q * share;
    const long long tiles_most = c.num_seqs * ((most + C::kRows - 1) / C::kRows);
    const long long pairs = rows / C::kRows + c.num_seqs < tiles_most ? rows / C::kRows + c.num_seqs : tiles_most;
    const long long items = pairs * ge.hkv;
    long long keys = pg.table_stride << ge.page_shift;
    if (c.window > 0 && c.window + C::kRows / share + 1 < keys) keys = c.window + C::kRows / share + 1;
    // four tiles of keys a part at least: joining costs about as much
    const long long parts = (keys + C::kKeys - 1) / C::kKeys / 4;
    a.most_parts = parts < 1 ? 1 : parts > 32 ? 32 : (int)parts;
    const long long grid = (items / kNumSMs + 1) * kNumSMs;
    if (grid > 0x7fffffffLL) return -2;
    return launch_k(kernel, dim3((unsigned)grid), dim3(kThreads), (size_t)C::smem(ge.ng()), st, a) == cudaSuccess ? 0 : -1;
}

}  // namespace

int launch_prefill(const AttnCall& c, const Pages& pg, const Geom& ge, int min_rows, cudaStream_t st) {
    switch (ge.d) {
        case 64: return launch<64>(c, pg, ge, min_rows, st);
        case 128: return launch<128>(c, pg, ge, min_rows, st);
        default: return launch<256>(c, pg, ge, min_rows, st);
    }
}

}  // namespace kv4
}  // namespace cb
