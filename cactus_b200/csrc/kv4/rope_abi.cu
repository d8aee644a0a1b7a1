// extern "C" entry points of the rotating append (include/cactus_b200_kv4.h): argument checks, then the
// launchers of rope.cu. No entry point throws.
#include "abi_checks.h"
#include "kv4_ops.h"

using namespace cb::kv4::abi;
using cb::kv4::Geom;
using cb::kv4::Pages;

extern "C" {

CB_API int cactus_cuda_rope_table(float theta, size_t rotary_dim, size_t num_positions, float* table, void* stream) {
    const char* name = "rope_table";
    if (rotary_dim % 2) return arg(name, "rotary_dim must be even");
    if (rotary_dim == 0 || num_positions == 0) return CB_OK;
    if (!table) return arg(name, "null argument");
    if (!aligned(table, 16)) return arg(name, "table must be 16-byte aligned");
    if (rotary_dim > 65536 || num_positions > ((size_t)1 << 38) / rotary_dim) return arg(name, "size too large");
    if (!(theta > 0.0f) || !(theta <= 3.0e38f)) return arg(name, "theta must be a positive number");
    return launched(name, cb::kv4::launch_rope_table(theta, (int)(rotary_dim / 2), (long long)num_positions, table,
                                                     S(stream)));
}

CB_API int cactus_cuda_kv4_rope_append(const uint16_t* queries, size_t query_stride, uint16_t* rotated,
                                       size_t rotated_stride, const uint16_t* keys, const uint16_t* values,
                                       size_t row_stride, const float* rope_table, size_t num_positions,
                                       size_t rotary_dim, const uint16_t* q_weight, const uint16_t* k_weight,
                                       float eps, const int32_t* token_offsets, const int32_t* context_lens,
                                       const int32_t* block_table, size_t table_stride, void* pool, size_t num_pages,
                                       size_t page_stride, size_t num_seqs, size_t num_tokens, size_t num_q_heads,
                                       size_t page_size, size_t num_kv_heads, size_t head_dim, size_t group_size,
                                       void* stream) {
    const char* name = "kv4_rope_append";
    Geom ge;
    Pages pg;
    if (const char* why = make_geom(page_size, num_kv_heads, head_dim, group_size, &ge)) return arg(name, why);
    if (rotary_dim % 16 || rotary_dim > head_dim) return arg(name, "rotary_dim must be a multiple of 16, at most head_dim");
    if (!(eps >= 0.0f) || !(eps <= 3.0e38f)) return arg(name, "eps must be a number, not negative");
    if (queries && (num_q_heads == 0 || num_q_heads > 32768)) return arg(name, "num_q_heads must be 1 to 32768");
    if (num_seqs == 0 || num_tokens == 0) return CB_OK;
    if (const char* why = make_pages(pool, num_pages, page_stride, block_table, table_stride, ge, &pg))
        return arg(name, why);
    if (!keys || !values || !token_offsets || !context_lens || (rotary_dim && !rope_table) || (queries && !rotated))
        return arg(name, "null argument");
    if (rotary_dim && num_positions == 0) return arg(name, "rope_table has no positions");
    if (num_seqs > kIntMax - 1 || num_tokens > kIntMax - 64) return arg(name, "size too large");
    if (row_stride % 8 || !aligned(keys, 16) || !aligned(values, 16))
        return arg(name, "keys, values and row_stride must be 16-byte aligned");
    if (row_stride < num_kv_heads * head_dim || row_stride > ((size_t)1 << 40)) return arg(name, "bad row_stride");
    if (!aligned(rope_table, 16) || !aligned(q_weight, 16) || !aligned(k_weight, 16))
        return arg(name, "rope_table, q_weight and k_weight must be 16-byte aligned");
    if (queries) {
        if (query_stride % 8 || rotated_stride % 8 || !aligned(queries, 16) || !aligned(rotated, 16))
            return arg(name, "queries, rotated and their strides must be 16-byte aligned");
        if (query_stride < num_q_heads * head_dim || query_stride > ((size_t)1 << 40)) return arg(name, "bad query_stride");
        if (rotated_stride < num_q_heads * head_dim || rotated_stride > ((size_t)1 << 40))
            return arg(name, "bad rotated_stride");
        if (queries == rotated && query_stride != rotated_stride)
            return arg(name, "rotated overlaps queries at another stride");
    }
    cb::kv4::RopeCall c = {};
    c.q = H(queries);
    c.k = H(keys);
    c.v = H(values);
    c.q_stride = (long long)query_stride;
    c.out_stride = (long long)rotated_stride;
    c.row_stride = (long long)row_stride;
    c.out = H(rotated);
    c.turns = reinterpret_cast<const float2*>(rope_table);
    c.num_positions = num_positions > kIntMax ? (long long)kIntMax : (long long)num_positions;
    c.rotary = (int)rotary_dim;
    c.q_weight = H(q_weight);
    c.k_weight = H(k_weight);
    c.eps = eps;
    c.offsets = token_offsets;
    c.lens = context_lens;
    c.num_seqs = (int)num_seqs;
    c.num_tokens = (int)num_tokens;
    c.hq = queries ? (int)num_q_heads : 0;
    return launched(name, cb::kv4::launch_rope_append(c, pg, ge, S(stream)));
}

}  // extern "C"
