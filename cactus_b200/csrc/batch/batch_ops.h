// Launchers of the ragged batch's operators (arguments checked by batch_abi.cu).
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace cb {
namespace batch {

// norm_q8.cu
constexpr int kNormMaxDims = 32768;
struct NormCall {
    const __half *x, *residual, *weight;  // residual may be null
    long long x_stride, residual_stride, sum_stride;
    __half *sum, *normed;  // may be null
    int8_t* q;             // may be null
    float* scales;
    int rows, dims;
    float eps;
};
int launch_norm_q8(const NormCall& c, cudaStream_t st);

// lora.cu
constexpr int kLoraMaxRank = 256;
size_t lora_plan_bytes(long long num_seqs, long long num_tokens, long long num_adapters);
size_t lora_workspace(long long num_tokens, int max_rank);
int launch_lora_plan(const int* offsets, const int* ids, int num_seqs, int num_tokens, int num_adapters, void* plan,
                     cudaStream_t st);
struct LoraCall {
    const __half *x, *a, *b, *base;  // base may be null
    const int* ranks;                // may be null
    const float* scales;             // may be null
    __half* out;
    long long x_stride, base_stride, out_stride;
    const int* plan;
    int num_seqs, num_tokens, num_adapters, max_rank, k, n;
    float* ws;
};
int launch_lora(const LoraCall& c, cudaStream_t st);
// lora_tc.cu: the products for batches of many rows, ranks up to kLoraWideRank; split: the first one was that file's
constexpr int kLoraWideRank = 128;
int launch_lora_shrink_wide(const LoraCall& c, unsigned* error_word, cudaStream_t st);
int launch_lora_expand_wide(const LoraCall& c, bool split, unsigned* error_word, cudaStream_t st);

// logits.cu
struct LogitsCall {
    const __half* in;
    __half* out;
    long long in_stride, out_stride;
    int rows, vocab;
    const float* penalties;  // may be null, as all lists below
    const uint32_t* history;
    const int *history_offsets, *prompt_lens;
    int num_history;
    const uint32_t* bias_ids;
    const float* bias_values;
    const int* bias_offsets;
    int num_biases;
    const uint32_t* masks;
    long long mask_stride;
    int num_masks;
    const int* mask_ids;
};
int launch_logits(const LogitsCall& c, cudaStream_t st);

}  // namespace batch
}  // namespace cb
