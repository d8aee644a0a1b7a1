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
// decode.cu
size_t decode_workspace(int num_seqs, int num_tokens, int hq, int hkv);
int launch_decode(const AttnCall& c, const Pages& pg, const Geom& ge, cudaStream_t st);
// attention.cu
size_t attention_workspace(int num_seqs, int num_tokens, int hq, int hkv, int d);
int launch_attention(const AttnCall& c, const Pages& pg, const Geom& ge, cudaStream_t st);

}  // namespace kv4
}  // namespace cb
