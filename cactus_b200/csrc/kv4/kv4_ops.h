// Launchers of the 4-bit paged KV cache's kernels (arguments checked by kv4_abi.cu).
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace cb {
namespace kv4 {

struct Geom;
struct Pages;

// pages.cu
int launch_append(const __half* k, const __half* v, long long row_stride, const int* offsets, const int* lens,
                  const Pages& pg, int num_seqs, int num_tokens, const Geom& ge, cudaStream_t st);
int launch_read(const Pages& pg, const int* offsets, const int* first, __half* k, __half* v, int num_seqs,
                int num_rows, const Geom& ge, cudaStream_t st);
int launch_copy_pages(uint8_t* pool, long long num_pages, long long page_bytes, long long page_stride, int planes,
                      long long plane_stride, const int* src, const int* dst, int n, cudaStream_t st);
int launch_compact(const Pages& src, const int* dst_table, int planes, long long plane_stride, const int* kept,
                   const int* offsets, int num_seqs, int num_kept, const Geom& ge, cudaStream_t st);

// rope.cu
struct RopeCall {
    const __half *q, *k, *v;  // q may be null where hq is 0
    long long q_stride, out_stride, row_stride;
    __half* out;
    const float2* turns;  // [num_positions][rotary / 2]
    long long num_positions;
    int rotary;
    const __half *q_weight, *k_weight;  // may be null
    float eps;
    const int *offsets, *lens;
    int num_seqs, num_tokens, hq;
};
int launch_rope_table(float theta, int half, long long positions, float* table, cudaStream_t st);
int launch_rope_append(const RopeCall& c, const Pages& pg, const Geom& ge, cudaStream_t st);

struct AttnCall {
    const __half* q;
    long long q_stride;
    const int *offsets, *lens;
    __half* out;
    float* lse;  // may be null
    int num_seqs, num_tokens, max_q, hq;
    float scale;
    long long window;
    int causal;
    uint8_t* ws;
};

// The workspace is two regions: the parts of results that several blocks share, at a fixed size, so
// that the counters after it, which have to be zero before every call, are at the same place for
// every shape.
constexpr int kDecodeCtas = 148 * 4, kDecodePartFloats = 16 * (128 + 2);  // 2 parts a block, 16 rows of 128 at most
constexpr int kPrefillParts = 148;                                        // of 256 rows of 128 (128 of 256) at most
constexpr size_t kPartBytes = (size_t)kPrefillParts * 256 * (128 + 2) * 4;
static_assert(kPartBytes >= (size_t)kDecodeCtas * 2 * kDecodePartFloats * 4, "workspace");

// decode.cu: sequences with at most max_rows q rows (tokens times the heads that share a kv head), of
// which most have at most usual_rows
size_t decode_counters(int num_seqs, int num_tokens, int hq, int hkv);
int launch_decode(const AttnCall& c, const Pages& pg, const Geom& ge, int max_rows, int usual_rows, cudaStream_t st);
// prefill_tc.cu: sequences with at least min_rows q rows
int launch_prefill(const AttnCall& c, const Pages& pg, const Geom& ge, int min_rows, cudaStream_t st);
// attention.cu
size_t attention_workspace(int num_seqs, int num_tokens, int hq, int hkv, int d);
int launch_attention(const AttnCall& c, const Pages& pg, const Geom& ge, cudaStream_t st);

}  // namespace kv4
}  // namespace cb
