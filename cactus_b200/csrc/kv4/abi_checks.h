// What the kernel entry points of include/cactus_b200_kv4.h check of their arguments alike.
#pragma once
#include <string>

#include "../../../include/cactus_b200_kv4.h"
#include "../ops.h"
#include "kv4.cuh"

namespace cb {
namespace kv4 {
namespace abi {

using cb::abi_check_launch;
using cb::abi_fail;

constexpr size_t kIntMax = 0x7fffffff;
inline cudaStream_t S(void* s) { return reinterpret_cast<cudaStream_t>(s); }
inline const __half* H(const uint16_t* p) { return reinterpret_cast<const __half*>(p); }
inline __half* H(uint16_t* p) { return reinterpret_cast<__half*>(p); }
inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

inline const char* make_geom(size_t page_size, size_t hkv, size_t d, size_t g, Geom* ge) {
    int shift = 0;
    while (shift < 8 && (size_t(1) << shift) < page_size) ++shift;
    if (shift < 4 || (size_t(1) << shift) != page_size) return "page_size must be 16, 32, 64, 128 or 256";
    if (hkv == 0 || hkv > 1024) return "num_kv_heads must be 1 to 1024";
    if (d != 64 && d != 128 && d != 256) return "head_dim must be 64, 128 or 256";
    if ((g != 32 && g != 64 && g != 128) || d % g) return "group_size must be 32, 64 or 128 and divide head_dim";
    *ge = Geom{shift, (int)hkv, (int)d, (int)g, (int)(d / g)};
    return nullptr;
}

inline const char* make_pages(const void* pool, size_t num_pages, size_t page_stride, const int32_t* table,
                       size_t table_stride, const Geom& ge, Pages* pg) {
    if (!pool || !table) return "null pool or block table";
    if (num_pages == 0 || num_pages > kIntMax) return "num_pages must be 1 to 2^31 - 1";
    if (table_stride == 0 || table_stride > kIntMax) return "table_stride must be 1 to 2^31 - 1";
    if (table_stride * (size_t)ge.page() > kIntMax - 1024) return "a table row holds more than 2^31 - 1024 positions";
    if (!aligned(pool, 16) || page_stride % 16) return "pool and page_stride must be 16-byte aligned";
    if (page_stride < (size_t)ge.block_bytes() * (size_t)ge.hkv) return "page_stride is less than a page";
    if (page_stride > ((size_t)1 << 62) / num_pages) return "pool size overflows";
    if (!aligned(table, 4)) return "block table must be 4-byte aligned";
    *pg = Pages{static_cast<uint8_t*>(const_cast<void*>(pool)), (long long)num_pages, (long long)page_stride, table,
                (long long)table_stride};
    return nullptr;
}

inline int arg(const char* name, const char* why) { return abi_fail(CB_ERR_ARG, std::string(name) + ": " + why); }

// what a launcher's result means: a failure without an error of the runtime is one all the same
inline int launched(const char* name, int rc) {
    if (const int e = abi_check_launch(name)) return e;
    return rc ? abi_fail(CB_ERR_LAUNCH, std::string(name) + ": launch failed") : CB_OK;
}

}  // namespace abi
}  // namespace kv4
}  // namespace cb
