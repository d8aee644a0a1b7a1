/*
 * cactus_b200_batch.h — C ABI of the operators around the projections of a ragged batch: the residual's
 * addition with RMSNorm and 8-bit rows, low-rank adapters of many requests beside a shared projection,
 * and penalties, biases and grammar masks on the batch's logits. (Its 4-bit cache, with the append that
 * normalises and rotates on the way, is cactus_b200_kv4.h.) No counterparts in the reference; sums are
 * fp32 or wider and each result is rounded once.
 *
 * Conventions are those of cactus_b200.h: DEVICE pointers, fp16 as uint16_t bits, asynchronous calls on
 * `stream`, 0 or a negative code with a message in cactus_cuda_last_error(). Nothing here allocates, and
 * every call can be captured in a CUDA graph (after a first call of the same kind outside of it on that
 * device, which sets kernel attributes). Strides are in elements. Lists, lengths and ids are read on
 * the device; what they name outside the arguments is skipped and raises the device error word
 * (cactus_cuda_device_error() == 4). Calls with a size of zero do nothing.
 */
#ifndef CACTUS_B200_BATCH_H
#define CACTUS_B200_BATCH_H

#include "cactus_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* s = fp16(x + residual) of each row (s = x where residual is NULL), stored in `sum` where that is not
 * NULL; y = s / sqrt(mean(s^2) + eps) * weight. Where q is not NULL the row's scales[row] is
 * max(largest |y| / 127, 1e-10) and q[row][i] = round-half-even(y[i] * (1 / scale)): what
 * cactus_cuda_matmul_int8 and _int4 take. Where normed is not NULL, normed[row][i] = fp16(y[i]). One of q
 * (with scales) and normed at least is not NULL; q and normed are [rows][dims]. A row with an infinity or
 * a NaN among its y gets codes 0 and a NaN as its scale, so that it shows in what is computed from it.
 * The mean is a 64-bit sum. `sum` may be x or residual (with the same stride), rows otherwise do not
 * overlap. dims up to 32768. */
CB_API int cactus_cuda_add_rms_norm_q8(const uint16_t* x, size_t x_stride, const uint16_t* residual,
                                       size_t residual_stride, const uint16_t* weight, uint16_t* sum,
                                       size_t sum_stride, int8_t* q, float* scales, uint16_t* normed, size_t rows,
                                       size_t dims, float eps, void* stream);

/* ---- Low-rank adapters. Sequence b has the token rows token_offsets[b] .. token_offsets[b + 1] - 1
 * (token_offsets: [num_seqs + 1], rising from 0, at most num_tokens) and adapter adapter_ids[b], or none
 * where that is -1. The plan groups the rows by adapter; a step's batch has one, for all projections of all
 * layers, as long as neither array changes. A plan whose token_offsets fall or pass num_tokens has no rows. */
CB_API size_t cactus_cuda_lora_plan_bytes(size_t num_seqs, size_t num_tokens, size_t num_adapters);
CB_API int cactus_cuda_lora_plan(const int32_t* token_offsets, const int32_t* adapter_ids, size_t num_seqs,
                                 size_t num_tokens, size_t num_adapters, void* plan, size_t plan_bytes, void* stream);
/* output[t] = base[t] + scales[i] * (x[t] A_i^T) B_i^T for the rows t of sequences with adapter i, and
 * base[t] for rows of sequences without one; base NULL stands for zeros. Rows of no sequence stay as they are.
 * a [num_adapters][max_rank][in_features], b [num_adapters][out_features][max_rank]: adapter i has the first
 * ranks[i] rows of its a and columns of its b (ranks NULL: all; 0: none), and what the others hold does not
 * reach a result. Infinities of x and a go through as the formula has them; one in b may come out as a NaN.
 * scales NULL: 1. output may be base (with the same stride) and otherwise overlaps nothing.
 * in_features, out_features, max_rank (8 to 256) and the strides are multiples of 8, all pointers 16-byte
 * aligned. The middle product is fp32, and enters the second one as two fp16 numbers of a row's own power of
 * two (22 bits of the row's largest). plan: of cactus_cuda_lora_plan with the same num_seqs, num_tokens and
 * num_adapters (plans of other numbers raise the device error word, and nothing is written). workspace:
 * cactus_cuda_lora_workspace() bytes, 16-byte aligned, of any content; calls that may overlap in time need a
 * workspace each. */
CB_API size_t cactus_cuda_lora_workspace(size_t num_tokens, size_t max_rank);
CB_API int cactus_cuda_lora_f16(const uint16_t* x, size_t x_stride, const uint16_t* a, const uint16_t* b,
                                const int32_t* ranks, const float* scales, const uint16_t* base, size_t base_stride,
                                uint16_t* output, size_t output_stride, const void* plan, size_t plan_bytes,
                                size_t num_seqs, size_t num_tokens, size_t num_adapters, size_t max_rank,
                                size_t in_features, size_t out_features, void* workspace, size_t workspace_bytes,
                                void* stream);

/* Logits [rows][vocab] before sampling (output may be logits, with the same stride). For each row, in this order:
 *  - penalties [rows][3] (repetition, frequency, presence; NULL: none) for the tokens of its history,
 *    history[history_offsets[row]] .. history[history_offsets[row + 1] - 1], of which the first
 *    prompt_lens[row] (NULL: 0; all, where there are fewer) are the prompt: l / repetition where l > 0, else
 *    l * repetition, for a token that occurs; minus frequency * count and, where count is not 0, minus
 *    presence, with its count behind the prompt. A repetition penalty that is not positive and finite raises the device error word and
 *    counts as 1, a prompt's length below 0 raises it and counts as 0.
 *  - biases: bias_values[j] is added to token bias_ids[j], j from bias_offsets[row] to bias_offsets[row + 1] - 1.
 *    Of a token's several entries the last one counts. -inf bans a token.
 *  - a mask: -inf for tokens whose bit is 0 in masks[mask_ids[row]] (bit t % 32 of word t / 32; masks
 *    [num_masks][mask_stride]); mask_ids[row] == -1: none; mask_ids NULL: row i has mask i.
 * What is left of a row goes to cactus_cuda_argmax_f16 or cactus_cuda_sample_f16 (whose `uniform` has to be above
 * 0 then: with 0 it answers index 0, masked or not).
 * history, bias_ids and masks are NULL where there are none. Offsets rise from 0 and end at num_history and
 * num_biases at most; ids are below vocab. Arithmetic is fp32, each step rounded; a finite result past fp16's
 * range becomes its largest number of that sign. */
CB_API int cactus_cuda_logits_process_f16(const uint16_t* logits, size_t logits_stride, uint16_t* output,
                                          size_t output_stride, size_t rows, size_t vocab, const float* penalties,
                                          const uint32_t* history, const int32_t* history_offsets,
                                          const int32_t* prompt_lens, size_t num_history, const uint32_t* bias_ids,
                                          const float* bias_values, const int32_t* bias_offsets, size_t num_biases,
                                          const uint32_t* masks, size_t mask_stride, size_t num_masks,
                                          const int32_t* mask_ids, void* stream);

#ifdef __cplusplus
}
#endif
#endif
