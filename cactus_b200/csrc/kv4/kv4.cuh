// The 4-bit paged KV cache: page layout and device helpers shared by its kernels.
//
// Page layout (include/cactus_b200_kv4.h): per kv head one block of bytes
//   key codes [P][D/2] | key parameters [P][D/G] (step, low) | value codes | value parameters.
// One head's part of a page is one contiguous range, so a tile of keys and values is one or a few
// long runs whatever the number of heads.
#pragma once
#include <limits.h>

#include "../common.cuh"

namespace cb {
namespace kv4 {

struct Geom {
    int page_shift, hkv, d, g, groups;  // groups: of a row
    __host__ __device__ int page() const { return 1 << page_shift; }
    __host__ __device__ int ng() const { return groups; }
    __host__ __device__ int code_bytes() const { return d / 2; }      // of one row
    __host__ __device__ int param_bytes() const { return 4 * ng(); }  // of one row
    // byte offsets inside a block
    __host__ __device__ int k_params() const { return (d / 2) << page_shift; }
    __host__ __device__ int v_codes() const { return (d / 2 + 4 * ng()) << page_shift; }
    __host__ __device__ int v_params() const { return (d + 4 * ng()) << page_shift; }
    __host__ __device__ int block_bytes() const { return (d + 8 * ng()) << page_shift; }
};

struct Pages {
    uint8_t* pool;
    long long num_pages, page_stride;
    const int* table;  // [sequences][table_stride]
    long long table_stride;
};

// Byte offset in the pool of the page that holds position `pos` of sequence b, or -1 (with the
// device error word raised) where the table has no such page.
__device__ __forceinline__ long long page_offset(const Pages& pg, int b, long long pos, int page_shift) {
    const long long i = pos >> page_shift;
    if (i >= 0 && i < pg.table_stride) {
        const int p = pg.table[(long long)b * pg.table_stride + i];
        if (p >= 0 && p < pg.num_pages) return (long long)p * pg.page_stride;
    }
#ifdef __CUDACC_RDC__
    report_dev_error(kDevBadPage);
#endif
    return -1;
}

// The sequence that token row t belongs to: the last b in [0, n) with offsets[b] <= t; -1 for rows
// at or past offsets[n].
__device__ __forceinline__ int find_seq(const int* offsets, int n, int t) {
    if (t >= offsets[n]) return -1;
    int lo = 0, hi = n;  // offsets[lo] <= t < offsets[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ __half2 as_half2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// (w & MASK) | 0x64006400 as one instruction (the compiler makes two of the expression)
template <uint32_t MASK>
__device__ __forceinline__ uint32_t mask_magic(uint32_t w) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "n"(MASK), "r"(0x64006400u));
    return r;
}

// Eight codes (element i in bits 4i..4i+3) as exact fp16 integers, in the order (0, 4), (1, 5),
// (2, 6), (3, 7): 0x6400 | c is the fp16 number 1024 + c, and 0x6400 | (c << 4) is 1024 + 16 c.
__device__ __forceinline__ void codes_to_half(uint32_t w, __half2 (&h)[4]) {
    const uint32_t n1024 = 0xE400E400u, r16 = 0x2C002C00u, n64 = 0xD400D400u;  // -1024, 1/16, -64
    const uint32_t w8 = w >> 8;
    h[0] = __hadd2(as_half2(mask_magic<0x000F000Fu>(w)), as_half2(n1024));
    h[1] = __hfma2(as_half2(mask_magic<0x00F000F0u>(w)), as_half2(r16), as_half2(n64));
    h[2] = __hadd2(as_half2(mask_magic<0x000F000Fu>(w8)), as_half2(n1024));
    h[3] = __hfma2(as_half2(mask_magic<0x00F000F0u>(w8)), as_half2(r16), as_half2(n64));
}

}  // namespace kv4
}  // namespace cb
