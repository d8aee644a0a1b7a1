// The 4-bit paged KV cache's writers and movers: append (quantise into pages), read (dequantise
// rows), copy of whole pages, compaction (rows into other pages). All are bound by HBM: each input
// byte is read once and each output byte written once, in 16-byte pieces where the row is long
// enough.
#include "kv4.cuh"
#include "kv4_ops.h"

namespace cb {
namespace kv4 {

namespace {

// ---------------------------------------------------------------- append
// A block quantises 32 token rows of one kv head, keys and values. D / 8 lanes share a row (8
// elements, one 16-byte load each), the G / 8 lanes of a group reduce its smallest and largest
// element by shuffles, and each lane stores its 8 codes as one word.
constexpr int kAppendTokens = 32, kAppendThreads = 256;

// (x - low) / step rounded half to even, held in 0..15. Below 16 the product with the reciprocal is
// within 4e-6 of the quotient (two roundings of 2^-24 each), so only a result that near a half,
// where the rounding could differ, takes the true division.
__device__ __forceinline__ uint32_t quant_code(float x, float step, float inv) {
    float q = __fmul_rn(x, inv);
    if (fabsf(__fsub_rn(fabsf(__fsub_rn(q, rintf(q))), 0.5f)) < 1e-5f) q = __fdiv_rn(x, step);
    return (uint32_t)fminf(rintf(q), 15.0f);
}

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
    const int lane = threadIdx.x % kLanes, per_group = ge.g / 8;
    const unsigned full = 0xffffffffu;
    constexpr int kPasses = (kAppendTokens + kRows - 1) / kRows;
    uint4 x[2 * kPasses];
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
        const int r = threadIdx.x / kLanes + i * kRows;
        const bool on = s_page[r] >= 0;
        const long long at = (long long)(t0 + r) * row_stride + head * D + lane * 8;
        x[2 * i] = on ? __ldg(reinterpret_cast<const uint4*>(keys + at)) : uint4{0, 0, 0, 0};
        x[2 * i + 1] = on ? __ldg(reinterpret_cast<const uint4*>(values + at)) : uint4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < 2 * kPasses; ++i) {
        const int r = threadIdx.x / kLanes + (i / 2) * kRows;
        float f[8];
        const __half2* h = reinterpret_cast<const __half2*>(&x[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 p = __half22float2(h[j]);
            f[2 * j] = p.x;
            f[2 * j + 1] = p.y;
        }
        float lo = f[0], hi = f[0];
        bool bad = false;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            lo = fminf(lo, f[j]);
            hi = fmaxf(hi, f[j]);
            bad |= !(fabsf(f[j]) <= 65504.0f);  // an infinity or a NaN
        }
        for (int o = 1; o < per_group; o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(full, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(full, hi, o));
            bad |= __shfl_xor_sync(full, (int)bad, o) != 0;
        }
        const __half step = __float2half_rz(__fdiv_rn(__fsub_rn(hi, lo), 15.0f));
        const float fs = __half2float(step), inv = fs > 0.0f ? __frcp_rn(fs) : 0.0f;
        uint32_t w = 0;
        if (!bad && fs > 0.0f) {
#pragma unroll
            for (int j = 0; j < 8; ++j) w |= quant_code(__fsub_rn(f[j], lo), fs, inv) << (4 * j);
        }
        if (s_page[r] < 0) continue;
        uint8_t* block = pg.pool + s_page[r] + (long long)head * ge.block_bytes() + ((i & 1) ? ge.v_codes() : 0);
        const int row = s_row[r];
        *reinterpret_cast<uint32_t*>(block + row * (D / 2) + lane * 4) = w;
        if (lane % per_group == 0) {
            const __half nan = __ushort_as_half(0x7FFF);
            *reinterpret_cast<__half2*>(block + ge.k_params() + (row * ge.ng() + lane / per_group) * 4) =
                bad ? __halves2half2(nan, nan) : __halves2half2(step, __float2half_rn(lo));
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
    const int lane = threadIdx.x % kLanes, group = lane * 8 / ge.g;
    for (int r = threadIdx.x / kLanes; r < kAppendTokens; r += kRows) {
        if (s_page[r] < 0) continue;
        const uint8_t* block = pg.pool + s_page[r] + (long long)head * ge.block_bytes();
        const int row = s_row[r];
        const long long at = ((long long)(t0 + r) * ge.hkv + head) * D + lane * 8;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            __half* out = which ? values : keys;
            if (!out) continue;
            const uint8_t* part = block + (which ? ge.v_codes() : 0);
            const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(part + row * (D / 2) + lane * 4));
            const __half2 par =
                __ldg(reinterpret_cast<const __half2*>(part + ge.k_params() + (row * ge.ng() + group) * 4));
            const __half2 step = __low2half2(par), low = __high2half2(par);
            __half2 c[4];
            codes_to_half(w, c);
#pragma unroll
            for (int j = 0; j < 4; ++j) c[j] = __hfma2(c[j], step, low);
            __half2 o[4] = {__lows2half2(c[0], c[1]), __lows2half2(c[2], c[3]), __highs2half2(c[0], c[1]),
                            __highs2half2(c[2], c[3])};
            *reinterpret_cast<uint4*>(out + at) = *reinterpret_cast<const uint4*>(o);
        }
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
    const int cw = ge.code_bytes() / 16, block = ge.block_bytes();  // 16-byte pieces of a row's codes: 2, 4 or 8
    const int per_head = 2 * kMoveRows * cw;
    for (int i = threadIdx.x; i < per_head * ge.hkv; i += kMoveThreads) {
        const int head = i / per_head, k = i % per_head, piece = k % cw, r = (k / cw) % kMoveRows;
        if (s_from[r] < 0) continue;
        const long long at = (long long)head * block + (k >= kMoveRows * cw ? ge.v_codes() : 0) + piece * 16;
        *reinterpret_cast<uint4*>(plane + s_to[r] + at + s_trow[r] * ge.code_bytes()) =
            *reinterpret_cast<const uint4*>(plane + s_from[r] + at + s_frow[r] * ge.code_bytes());
    }
    const int ng = ge.ng(), words = 2 * kMoveRows * ng;
    for (int i = threadIdx.x; i < words * ge.hkv; i += kMoveThreads) {
        const int head = i / words, k = i % words, piece = k % ng, r = (k / ng) % kMoveRows;
        if (s_from[r] < 0) continue;
        const long long at =
            (long long)head * block + (k >= kMoveRows * ng ? ge.v_params() : ge.k_params()) + piece * 4;
        *reinterpret_cast<uint32_t*>(plane + s_to[r] + at + s_trow[r] * ge.param_bytes()) =
            *reinterpret_cast<const uint32_t*>(plane + s_from[r] + at + s_frow[r] * ge.param_bytes());
    }
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
