// extern "C" entry points of include/cactus_b200_kv4.h: argument checks, then the launchers of
// pages.cu and attention.cu. No entry point throws.
#include <string>

#include "../../../include/cactus_b200_kv4.h"
#include "abi_checks.h"
#include "kv4_ops.h"

namespace {

using namespace cb::kv4::abi;
using cb::kv4::Geom;
using cb::kv4::Pages;

// the planes of a pool of pages: [plane][page], or each page with all its planes
const char* planes_check(size_t num_planes, size_t plane_stride) {
    if (num_planes > 65535) return "num_planes must be at most 65535";
    if (plane_stride % 16) return "plane_stride must be 16-byte aligned";
    if (plane_stride && num_planes > ((size_t)1 << 62) / plane_stride) return "pool size overflows";
    return nullptr;
}

}  // namespace

extern "C" {

CB_API size_t cactus_cuda_kv4_page_bytes(size_t page_size, size_t num_kv_heads, size_t head_dim, size_t group_size) {
    Geom ge;
    if (make_geom(page_size, num_kv_heads, head_dim, group_size, &ge)) return 0;
    return (size_t)ge.block_bytes() * num_kv_heads;
}

CB_API int cactus_cuda_kv4_append(const uint16_t* keys, const uint16_t* values, size_t row_stride,
                                  const int32_t* token_offsets, const int32_t* context_lens,
                                  const int32_t* block_table, size_t table_stride, void* pool, size_t num_pages,
                                  size_t page_stride, size_t num_seqs, size_t num_tokens, size_t page_size,
                                  size_t num_kv_heads, size_t head_dim, size_t group_size, void* stream) {
    const char* name = "kv4_append";
    Geom ge;
    Pages pg;
    if (const char* why = make_geom(page_size, num_kv_heads, head_dim, group_size, &ge)) return arg(name, why);
    if (num_seqs == 0 || num_tokens == 0) return CB_OK;
    if (const char* why = make_pages(pool, num_pages, page_stride, block_table, table_stride, ge, &pg))
        return arg(name, why);
    if (!keys || !values || !token_offsets || !context_lens) return arg(name, "null argument");
    if (num_seqs > kIntMax - 1 || num_tokens > kIntMax - 64) return arg(name, "size too large");
    if (row_stride % 8 || !aligned(keys, 16) || !aligned(values, 16))
        return arg(name, "keys, values and row_stride must be 16-byte aligned");
    if (row_stride < num_kv_heads * head_dim || row_stride > ((size_t)1 << 40)) return arg(name, "bad row_stride");
    return launched(name, cb::kv4::launch_append(H(keys), H(values), (long long)row_stride, token_offsets, context_lens,
                                                 pg, (int)num_seqs, (int)num_tokens, ge, S(stream)));
}

CB_API int cactus_cuda_kv4_read(const void* pool, size_t num_pages, size_t page_stride, const int32_t* block_table,
                                size_t table_stride, const int32_t* row_offsets, const int32_t* first_rows,
                                uint16_t* keys, uint16_t* values, size_t num_seqs, size_t num_rows, size_t page_size,
                                size_t num_kv_heads, size_t head_dim, size_t group_size, void* stream) {
    const char* name = "kv4_read";
    Geom ge;
    Pages pg;
    if (const char* why = make_geom(page_size, num_kv_heads, head_dim, group_size, &ge)) return arg(name, why);
    if (num_seqs == 0 || num_rows == 0) return CB_OK;
    if (const char* why = make_pages(pool, num_pages, page_stride, block_table, table_stride, ge, &pg))
        return arg(name, why);
    if (!row_offsets || (!keys && !values)) return arg(name, "null argument");
    if (num_seqs > kIntMax - 1 || num_rows > kIntMax - 64) return arg(name, "size too large");
    if (!aligned(keys, 16) || !aligned(values, 16)) return arg(name, "keys and values must be 16-byte aligned");
    return launched(name, cb::kv4::launch_read(pg, row_offsets, first_rows, H(keys), H(values), (int)num_seqs,
                                               (int)num_rows, ge, S(stream)));
}

CB_API size_t cactus_cuda_kv4_attention_workspace(size_t num_seqs, size_t num_tokens, size_t num_q_heads,
                                                  size_t num_kv_heads, size_t head_dim) {
    if (num_seqs > kIntMax - 1 || num_tokens > kIntMax - 64 || num_q_heads > 65536 || num_kv_heads > 1024 ||
        num_kv_heads == 0 || num_q_heads < num_kv_heads || head_dim > 256)
        return 0;
    return cb::kv4::attention_workspace((int)num_seqs, (int)num_tokens, (int)num_q_heads, (int)num_kv_heads,
                                        (int)head_dim);
}

CB_API int cactus_cuda_kv4_attention(const uint16_t* queries, size_t query_stride, const int32_t* token_offsets,
                                     const int32_t* context_lens, const int32_t* block_table, size_t table_stride,
                                     const void* pool, size_t num_pages, size_t page_stride, uint16_t* output,
                                     float* lse, size_t num_seqs, size_t num_tokens, size_t max_query_len,
                                     size_t num_q_heads, size_t page_size, size_t num_kv_heads, size_t head_dim,
                                     size_t group_size, float scale, size_t window_size, int is_causal,
                                     void* workspace, size_t workspace_bytes, void* stream) {
    const char* name = "kv4_attention";
    Geom ge;
    Pages pg;
    if (const char* why = make_geom(page_size, num_kv_heads, head_dim, group_size, &ge)) return arg(name, why);
    if (num_q_heads == 0 || num_q_heads % num_kv_heads || num_q_heads > 65536)
        return arg(name, "num_q_heads must be a multiple of num_kv_heads");
    if (num_seqs == 0 || num_tokens == 0 || max_query_len == 0) return CB_OK;
    if (const char* why = make_pages(pool, num_pages, page_stride, block_table, table_stride, ge, &pg))
        return arg(name, why);
    if (!queries || !token_offsets || !context_lens || !output || !workspace) return arg(name, "null argument");
    if (num_seqs > kIntMax - 1 || num_tokens > kIntMax - 64) return arg(name, "size too large");
    if ((max_query_len < num_tokens ? max_query_len : num_tokens) * (num_q_heads / num_kv_heads) > kIntMax / 2)
        return arg(name, "too many query rows for one kv head");
    if (query_stride % 8 || !aligned(queries, 16) || !aligned(output, 16) || !aligned(workspace, 16))
        return arg(name, "queries, query_stride, output and workspace must be 16-byte aligned");
    if (query_stride < num_q_heads * head_dim || query_stride > ((size_t)1 << 40)) return arg(name, "bad query_stride");
    if (!aligned(lse, 4)) return arg(name, "lse must be 4-byte aligned");
    if (workspace_bytes <
        cactus_cuda_kv4_attention_workspace(num_seqs, num_tokens, num_q_heads, num_kv_heads, head_dim))
        return arg(name, "workspace too small");
    if (!(scale > 0.0f) || !(scale <= 3.0e38f)) return arg(name, "scale must be a positive number");
    cb::kv4::AttnCall c = {};
    c.q = H(queries);
    c.q_stride = (long long)query_stride;
    c.offsets = token_offsets;
    c.lens = context_lens;
    c.out = H(output);
    c.lse = lse;
    c.num_seqs = (int)num_seqs;
    c.num_tokens = (int)num_tokens;
    c.max_q = (int)(max_query_len < num_tokens ? max_query_len : num_tokens);
    c.hq = (int)num_q_heads;
    c.scale = scale;
    c.window = window_size > kIntMax ? 0 : (long long)window_size;
    c.causal = is_causal != 0;
    c.ws = static_cast<uint8_t*>(workspace);
    const int rc = cb::kv4::launch_attention(c, pg, ge, S(stream));
    if (rc == -2) return arg(name, "too many sequences of too wide a block table");
    return launched(name, rc);
}

CB_API int cactus_cuda_kv_copy_pages(void* pool, size_t num_pages, size_t page_bytes, size_t page_stride,
                                     size_t num_planes, size_t plane_stride, const int32_t* src_pages,
                                     const int32_t* dst_pages, size_t num_copies, void* stream) {
    const char* name = "kv_copy_pages";
    if (num_copies == 0 || num_planes == 0 || page_bytes == 0) return CB_OK;
    if (!pool || !src_pages || !dst_pages) return arg(name, "null argument");
    if (num_pages == 0 || num_pages > kIntMax || num_copies > kIntMax) return arg(name, "size too large");
    if (!aligned(pool, 16) || page_bytes % 16 || page_stride % 16)
        return arg(name, "pool, page_bytes and page_stride must be multiples of 16 bytes");
    if (page_bytes > page_stride || page_bytes > ((size_t)1 << 28)) return arg(name, "bad page_bytes");
    if (page_stride > ((size_t)1 << 62) / num_pages) return arg(name, "pool size overflows");
    if (const char* why = planes_check(num_planes, plane_stride)) return arg(name, why);
    return launched(name, cb::kv4::launch_copy_pages(static_cast<uint8_t*>(pool), (long long)num_pages,
                                                     (long long)page_bytes, (long long)page_stride, (int)num_planes,
                                                     (long long)plane_stride, src_pages, dst_pages, (int)num_copies,
                                                     S(stream)));
}

CB_API int cactus_cuda_kv4_compact(void* pool, size_t num_pages, size_t page_stride, size_t num_planes,
                                   size_t plane_stride, const int32_t* src_table, const int32_t* dst_table,
                                   size_t table_stride, const int32_t* kept_rows, const int32_t* kept_offsets,
                                   size_t num_seqs, size_t num_kept, size_t page_size, size_t num_kv_heads,
                                   size_t head_dim, size_t group_size, void* stream) {
    const char* name = "kv4_compact";
    Geom ge;
    Pages pg;
    if (const char* why = make_geom(page_size, num_kv_heads, head_dim, group_size, &ge)) return arg(name, why);
    if (num_seqs == 0 || num_kept == 0 || num_planes == 0) return CB_OK;
    if (const char* why = make_pages(pool, num_pages, page_stride, src_table, table_stride, ge, &pg))
        return arg(name, why);
    if (!dst_table || !kept_rows || !kept_offsets) return arg(name, "null argument");
    if (num_seqs > kIntMax - 1 || num_kept > kIntMax - 64) return arg(name, "size too large");
    if (const char* why = planes_check(num_planes, plane_stride)) return arg(name, why);
    return launched(name, cb::kv4::launch_compact(pg, dst_table, (int)num_planes, (long long)plane_stride, kept_rows,
                                                  kept_offsets, (int)num_seqs, (int)num_kept, ge, S(stream)));
}

}  // extern "C"
