// The 4-bit paged KV cache's writers and movers: append (quantise into pages), read (dequantise
// rows), copy of whole pages, compaction (rows into other pages). Each input byte is read once and each
// output byte written once, in 16-byte pieces where the row is long enough.
//
// On B200: append of 32 prompts (69 thousand rows, 8 heads of 128) about 129 us, bound by the
// instructions of the quantisation (196 a warp for 256 elements; its bytes take 57 us); their
// read-back 66 us (floor 57); copy of 640 pages in 16 layers 116 us, 7.2 TB/s (a quarter of the copies
// read one page); compaction of 2045 scattered rows of 16 sequences in 16 layers 251 us, 4.8 TB/s
// (floor 188 us; rows of 64 and 8 bytes do not fill the 64-byte units that DRAM reads).
#include "kv4.cuh"
#include "kv4_ops.h"
#include "quantise.cuh"

namespace cb {
namespace kv4 {

namespace {

// ---------------------------------------------------------------- append
// A block quantises 32 token rows of one kv head, keys and values. D / 8 lanes share a row (8
// elements, one 16-byte load each), the G / 8 lanes of a group reduce its smallest and largest
// element by shuffles, and each lane stores its 8 codes as one word.
constexpr int kAppendTokens = 32, kAppendThreads = 256;

template <int D>
__global__ void __launch_bounds__(kAppendThreads)
    kv4_append_kernel(const __half* __restrict__ keys, const __half* __restrict__ values, long long row_stride,
                      const int* __restrict__ offsets, const int* __restrict__ lens, Pages pg, int num_seqs,
                      int num_tokens, Geom ge) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ long long s_page[kAppendTokens];  // byte offset of the page, -1: nothing to write
    __shared__ int s_row[kAppendTokens];
    constexpr int kLanes = D / 8, kRows = kAppendThreads / kLanes;
    const int t0 = blockIdx.x * kAppendTokens, head = blockIdx.y;
    const int lane = threadIdx.x % kLanes, per_group = ge.g >> 3, group = lane >> (__ffs(per_group) - 1);
    const unsigned full = 0xffffffffu;
    constexpr int kPasses = kAppendTokens / kRows;
    static_assert(kAppendTokens % kRows == 0, "whole passes");
    uint4 x[2 * kPasses];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {  // in flight while the rows' pages are looked up
        const int t = min(t0 + threadIdx.x / kLanes + i * kRows, num_tokens - 1);
        const long long at = (long long)t * row_stride + head * D + lane * 8;
        x[2 * i] = __ldg(reinterpret_cast<const uint4*>(keys + at));
        x[2 * i + 1] = __ldg(reinterpret_cast<const uint4*>(values + at));
    }
    if (threadIdx.x < kAppendTokens) {
        const int t = t0 + threadIdx.x;
        const int b = t < num_tokens ? find_seq(offsets, num_seqs, t) : -1;
        long long page = -1;
        int row = 0;
        if (b >= 0) {
            const long long pos = (long long)lens[b] - offsets[b + 1] + t;
            if (pos >= 0) page = page_offset(pg, b, pos, ge.page_shift);
            row = (int)(pos & (ge.page() - 1));
        }
        s_page[threadIdx.x] = page;
        s_row[threadIdx.x] = row;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2 * kPasses; ++i) {
        const int r = threadIdx.x / kLanes + (i / 2) * kRows;
        const __half2* h = reinterpret_cast<const __half2*>(&x[i]);
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
            uint8_t* block = pg.pool + s_page[r] + (long long)head * ge.block_bytes() + ((i & 1) ? ge.v_codes() : 0);
            const int row = s_row[r];
            *reinterpret_cast<uint32_t*>(block + row * (D / 2) + lane * 4) = w;
            if ((lane & (per_group - 1)) == 0) {
                const __half nan = __ushort_as_half(0x7FFF);
                *reinterpret_cast<__half2*>(block + ge.k_params() + (row * ge.ng() + group) * 4) =
                    bad ? __halves2half2(nan, nan) : __halves2half2(step, __float2half_rn(lo));
            }
        }
    }
}

// ---------------------------------------------------------------- read
// A block reads 32 rows of one kv head back as fp16, 8 elements (one word of codes) a thread.
template <int D>
__global__ void __launch_bounds__(kAppendThreads)
    kv4_read_kernel(Pages pg, const int* __restrict__ offsets, const int* __restrict__ first, __half* keys,
                    __half* values, int num_seqs, int num_rows, Geom ge) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ long long s_page[kAppendTokens];
    __shared__ int s_row[kAppendTokens];
    constexpr int kLanes = D / 8, kRows = kAppendThreads / kLanes;
    const int t0 = blockIdx.x * kAppendTokens, head = blockIdx.y;
    if (threadIdx.x < kAppendTokens) {
        const int t = t0 + threadIdx.x;
        const int b = t < num_rows ? find_seq(offsets, num_seqs, t) : -1;
        long long page = -1;
        int row = 0;
        if (b >= 0) {
            const long long pos = (long long)(first ? first[b] : 0) + (t - offsets[b]);
            page = page_offset(pg, b, pos, ge.page_shift);
            row = (int)(pos & (ge.page() - 1));
        }
        s_page[threadIdx.x] = page;
        s_row[threadIdx.x] = row;
    }
    __syncthreads();
    const int lane = threadIdx.x % kLanes, group = lane * 8 >> (__ffs(ge.g) - 1);
    constexpr int kPasses = kAppendTokens / kRows;
    uint32_t w[2 * kPasses];
    __half2 par[2 * kPasses];
#pragma unroll
    for (int i = 0; i < 2 * kPasses; ++i) {
        const int r = threadIdx.x / kLanes + (i / 2) * kRows;
        if (s_page[r] < 0 || !((i & 1) ? values : keys)) continue;
        const uint8_t* part = pg.pool + s_page[r] + (long long)head * ge.block_bytes() + ((i & 1) ? ge.v_codes() : 0);
        w[i] = __ldg(reinterpret_cast<const uint32_t*>(part + s_row[r] * (D / 2) + lane * 4));
        par[i] = __ldg(reinterpret_cast<const __half2*>(part + ge.k_params() + (s_row[r] * ge.ng() + group) * 4));
    }
#pragma unroll
    for (int i = 0; i < 2 * kPasses; ++i) {
        const int r = threadIdx.x / kLanes + (i / 2) * kRows;
        __half* out = (i & 1) ? values : keys;
        if (s_page[r] < 0 || !out) continue;
        const __half2 step = __low2half2(par[i]), low = __high2half2(par[i]);
        __half2 c[4];
        codes_to_half(w[i], c);
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = __hfma2(c[j], step, low);
        const __half2 o[4] = {__lows2half2(c[0], c[1]), __lows2half2(c[2], c[3]), __highs2half2(c[0], c[1]),
                              __highs2half2(c[2], c[3])};
        *reinterpret_cast<uint4*>(out + ((long long)(t0 + r) * ge.hkv + head) * D + lane * 8) =
            *reinterpret_cast<const uint4*>(o);
    }
}

// ---------------------------------------------------------------- page copies
constexpr int kCopyThreads = 256, kCopyUnroll = 4;

__global__ void __launch_bounds__(kCopyThreads)
    kv_copy_pages_kernel(uint8_t* pool, long long num_pages, long long page_bytes, long long page_stride,
                         long long plane_stride, const int* __restrict__ src, const int* __restrict__ dst) {
    pdl_launch_dependents();
    pdl_wait();
    const int s = src[blockIdx.x], d = dst[blockIdx.x];
    if (s < 0 || s >= num_pages || d < 0 || d >= num_pages) {
        if (threadIdx.x == 0) report_dev_error(kDevBadPage);
        return;
    }
    const uint4* from = reinterpret_cast<const uint4*>(pool + blockIdx.z * plane_stride + s * page_stride);
    uint4* to = reinterpret_cast<uint4*>(pool + blockIdx.z * plane_stride + d * page_stride);
    const long long n = page_bytes / 16, base = (long long)blockIdx.y * kCopyThreads * kCopyUnroll + threadIdx.x;
    uint4 v[kCopyUnroll];
#pragma unroll
    for (int i = 0; i < kCopyUnroll; ++i)
        if (base + i * kCopyThreads < n) v[i] = from[base + i * kCopyThreads];
#pragma unroll
    for (int i = 0; i < kCopyUnroll; ++i)
        if (base + i * kCopyThreads < n) to[base + i * kCopyThreads] = v[i];
}

// ---------------------------------------------------------------- compaction
// A block moves 32 destination rows of one plane, all heads.
constexpr int kMoveRows = 32, kMoveThreads = 256;

__global__ void __launch_bounds__(kMoveThreads)
    kv4_compact_kernel(Pages src, const int* __restrict__ dst_table, long long plane_stride,
                       const int* __restrict__ kept, const int* __restrict__ offsets, int num_seqs, int num_kept,
                       Geom ge) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ long long s_from[kMoveRows], s_to[kMoveRows];  // page offsets; from < 0: nothing to move
    __shared__ int s_frow[kMoveRows], s_trow[kMoveRows];
    const int t0 = blockIdx.x * kMoveRows;
    if (threadIdx.x < kMoveRows) {
        const int t = t0 + threadIdx.x;
        const int b = t < num_kept ? find_seq(offsets, num_seqs, t) : -1;
        long long from = -1, to = -1;
        int frow = 0, trow = 0;
        if (b >= 0) {
            const int pos = kept[t], j = t - offsets[b];
            Pages dst = src;
            dst.table = dst_table;
            from = page_offset(src, b, pos, ge.page_shift);
            to = page_offset(dst, b, j, ge.page_shift);
            if (to < 0) from = -1;
            frow = pos & (ge.page() - 1);
            trow = j & (ge.page() - 1);
        }
        s_from[threadIdx.x] = from;
        s_to[threadIdx.x] = to;
        s_frow[threadIdx.x] = frow;
        s_trow[threadIdx.x] = trow;
    }
    __syncthreads();
    uint8_t* plane = src.pool + blockIdx.y * plane_stride;
    const int block = ge.block_bytes();
    // codes: a thread keeps one 16-byte piece of one row and goes through the heads, four at a time
    const int cw = ge.code_bytes() / 16, units = 2 * kMoveRows * cw;  // pieces of a row: 2, 4 or 8
    const int lanes = min(units, kMoveThreads), heads = kMoveThreads / lanes;
    for (int u = threadIdx.x % lanes; u < units; u += lanes) {
        const int piece = u % cw, r = u / cw % kMoveRows;
        if (s_from[r] < 0) continue;
        const long long at = (u >= kMoveRows * cw ? ge.v_codes() : 0) + piece * 16;
        const uint8_t* from = plane + s_from[r] + at + s_frow[r] * ge.code_bytes();
        uint8_t* to = plane + s_to[r] + at + s_trow[r] * ge.code_bytes();
        for (int h = threadIdx.x / lanes; h < ge.hkv; h += 4 * heads) {
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (h + i * heads < ge.hkv) v[i] = *reinterpret_cast<const uint4*>(from + (long long)(h + i * heads) * block);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (h + i * heads < ge.hkv) *reinterpret_cast<uint4*>(to + (long long)(h + i * heads) * block) = v[i];
        }
    }
    // parameters: a thread keeps those of one row, keys or values, and goes through every fourth head
    const int r = threadIdx.x % kMoveRows, ng = ge.ng();
    if (s_from[r] < 0) return;
    const long long at = (threadIdx.x & kMoveRows) ? ge.v_params() : ge.k_params();
    const uint8_t* from = plane + s_from[r] + at + s_frow[r] * ge.param_bytes();
    uint8_t* to = plane + s_to[r] + at + s_trow[r] * ge.param_bytes();
    constexpr int kStep = kMoveThreads / (2 * kMoveRows);
    auto move = [&](auto word) {
        using T = decltype(word);
        for (int h = threadIdx.x / (2 * kMoveRows); h < ge.hkv; h += 2 * kStep) {
            const bool two = h + kStep < ge.hkv;
            const long long x = (long long)h * block, y = x + (long long)kStep * block;
            const T a = *reinterpret_cast<const T*>(from + x), b = *reinterpret_cast<const T*>(from + (two ? y : x));
            *reinterpret_cast<T*>(to + x) = a;
            if (two) *reinterpret_cast<T*>(to + y) = b;
        }
    };
    struct alignas(16) Eight {
        uint4 a, b;
    };
    if (ng == 1) move(uint32_t{});
    else if (ng == 2) move(uint2{});
    else if (ng == 4) move(uint4{});
    else move(Eight{});
}

}  // namespace

int launch_append(const __half* k, const __half* v, long long row_stride, const int* offsets, const int* lens,
                  const Pages& pg, int num_seqs, int num_tokens, const Geom& ge, cudaStream_t st) {
    const dim3 grid((unsigned)((num_tokens + kAppendTokens - 1) / kAppendTokens), (unsigned)ge.hkv);
    auto kernel = ge.d == 64 ? kv4_append_kernel<64> : ge.d == 128 ? kv4_append_kernel<128> : kv4_append_kernel<256>;
    return launch_k(kernel, grid, dim3(kAppendThreads), 0, st, k, v, row_stride, offsets, lens, pg, num_seqs,
                    num_tokens, ge) == cudaSuccess
               ? 0
               : -1;
}

int launch_read(const Pages& pg, const int* offsets, const int* first, __half* k, __half* v, int num_seqs,
                int num_rows, const Geom& ge, cudaStream_t st) {
    const dim3 grid((unsigned)((num_rows + kAppendTokens - 1) / kAppendTokens), (unsigned)ge.hkv);
    auto kernel = ge.d == 64 ? kv4_read_kernel<64> : ge.d == 128 ? kv4_read_kernel<128> : kv4_read_kernel<256>;
    return launch_k(kernel, grid, dim3(kAppendThreads), 0, st, pg, offsets, first, k, v, num_seqs, num_rows, ge) ==
                   cudaSuccess
               ? 0
               : -1;
}

int launch_copy_pages(uint8_t* pool, long long num_pages, long long page_bytes, long long page_stride, int planes,
                      long long plane_stride, const int* src, const int* dst, int n, cudaStream_t st) {
    const long long per = 16LL * kCopyThreads * kCopyUnroll;
    const dim3 grid((unsigned)n, (unsigned)((page_bytes + per - 1) / per), (unsigned)planes);
    return launch_k(kv_copy_pages_kernel, grid, dim3(kCopyThreads), 0, st, pool, num_pages, page_bytes, page_stride,
                    plane_stride, src, dst) == cudaSuccess
               ? 0
               : -1;
}

int launch_compact(const Pages& src, const int* dst_table, int planes, long long plane_stride, const int* kept,
                   const int* offsets, int num_seqs, int num_kept, const Geom& ge, cudaStream_t st) {
    const dim3 grid((unsigned)((num_kept + kMoveRows - 1) / kMoveRows), (unsigned)planes);
    return launch_k(kv4_compact_kernel, grid, dim3(kMoveThreads), 0, st, src, dst_table, plane_stride, kept, offsets,
                    num_seqs, num_kept, ge) == cudaSuccess
               ? 0
               : -1;
}

}  // namespace kv4
}  // namespace cb
