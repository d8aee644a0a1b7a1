// extern "C" entry points of include/cactus_b200_batch.h: argument checks, then the launchers of
// norm_q8.cu, lora.cu and logits.cu. No entry point throws.
#include <math.h>

#include <string>

#include "../../../include/cactus_b200_batch.h"
#include "../ops.h"
#include "batch_ops.h"

namespace {

using cb::abi_check_launch;
using cb::abi_fail;

constexpr size_t kIntMax = 0x7fffffff, kStrideMax = (size_t)1 << 40;
inline cudaStream_t S(void* s) { return reinterpret_cast<cudaStream_t>(s); }
inline const __half* H(const uint16_t* p) { return reinterpret_cast<const __half*>(p); }
inline __half* H(uint16_t* p) { return reinterpret_cast<__half*>(p); }
inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int arg(const char* name, const char* why) { return abi_fail(CB_ERR_ARG, std::string(name) + ": " + why); }

// what a launcher's result means: a failure without an error of the runtime is one all the same
int launched(const char* name, int rc) {
    if (const int e = abi_check_launch(name)) return e;
    return rc ? abi_fail(CB_ERR_LAUNCH, std::string(name) + ": launch failed") : CB_OK;
}

const char* lora_sizes(size_t num_seqs, size_t num_tokens, size_t num_adapters) {
    if (num_seqs > kIntMax / 2 || num_tokens > kIntMax / 2) return "size too large";
    if (num_adapters > 65536) return "num_adapters must be at most 65536";
    return nullptr;
}

}  // namespace

extern "C" {

CB_API int cactus_cuda_add_rms_norm_q8(const uint16_t* x, size_t x_stride, const uint16_t* residual,
                                       size_t residual_stride, const uint16_t* weight, uint16_t* sum,
                                       size_t sum_stride, int8_t* q, float* scales, uint16_t* normed, size_t rows,
                                       size_t dims, float eps, void* stream) {
    const char* name = "add_rms_norm_q8";
    if (rows == 0 || dims == 0) return CB_OK;
    if (!x || !weight) return arg(name, "null argument");
    if (!q && !normed) return arg(name, "neither q nor normed is wanted");
    if (q && !scales) return arg(name, "q without scales");
    if (rows > kIntMax) return arg(name, "too many rows");
    if (dims > (size_t)cb::batch::kNormMaxDims) return arg(name, "dims must be at most 32768");
    if (x_stride < dims || (residual && residual_stride < dims) || (sum && sum_stride < dims))
        return arg(name, "a stride is less than dims");
    if (x_stride > kStrideMax || (residual && residual_stride > kStrideMax) || (sum && sum_stride > kStrideMax))
        return arg(name, "stride too large");
    if ((sum == x && sum_stride != x_stride) || (sum && sum == residual && sum_stride != residual_stride))
        return arg(name, "sum overlaps its input at another stride");
    if (!(eps >= 0.0f) || !(eps <= 3.0e38f)) return arg(name, "eps must be a number, not negative");
    if (!aligned(x, 2) || !aligned(residual, 2) || !aligned(weight, 2) || !aligned(sum, 2) || !aligned(normed, 2) ||
        !aligned(scales, 4))
        return arg(name, "misaligned argument");
    cb::batch::NormCall c = {};
    c.x = H(x);
    c.residual = H(residual);
    c.weight = H(weight);
    c.x_stride = (long long)x_stride;
    c.residual_stride = (long long)residual_stride;
    c.sum_stride = (long long)sum_stride;
    c.sum = H(sum);
    c.normed = H(normed);
    c.q = q;
    c.scales = scales;
    c.rows = (int)rows;
    c.dims = (int)dims;
    c.eps = eps;
    return launched(name, cb::batch::launch_norm_q8(c, S(stream)));
}

CB_API size_t cactus_cuda_lora_plan_bytes(size_t num_seqs, size_t num_tokens, size_t num_adapters) {
    if (lora_sizes(num_seqs, num_tokens, num_adapters)) return 0;
    return cb::batch::lora_plan_bytes((long long)num_seqs, (long long)num_tokens, (long long)num_adapters);
}

CB_API int cactus_cuda_lora_plan(const int32_t* token_offsets, const int32_t* adapter_ids, size_t num_seqs,
                                 size_t num_tokens, size_t num_adapters, void* plan, size_t plan_bytes, void* stream) {
    const char* name = "lora_plan";
    if (const char* why = lora_sizes(num_seqs, num_tokens, num_adapters)) return arg(name, why);
    if (num_seqs == 0 || num_tokens == 0) return CB_OK;
    if (!token_offsets || !adapter_ids || !plan) return arg(name, "null argument");
    if (!aligned(token_offsets, 4) || !aligned(adapter_ids, 4) || !aligned(plan, 16))
        return arg(name, "token_offsets and adapter_ids must be 4-byte, plan 16-byte aligned");
    if (plan_bytes < cactus_cuda_lora_plan_bytes(num_seqs, num_tokens, num_adapters))
        return arg(name, "plan too small");
    return launched(name, cb::batch::launch_lora_plan(token_offsets, adapter_ids, (int)num_seqs, (int)num_tokens,
                                                      (int)num_adapters, plan, S(stream)));
}

CB_API size_t cactus_cuda_lora_workspace(size_t num_tokens, size_t max_rank) {
    if (num_tokens > kIntMax / 2 || max_rank > (size_t)cb::batch::kLoraMaxRank) return 0;
    return cb::batch::lora_workspace((long long)num_tokens, (int)max_rank);
}

CB_API int cactus_cuda_lora_f16(const uint16_t* x, size_t x_stride, const uint16_t* a, const uint16_t* b,
                                const int32_t* ranks, const float* scales, const uint16_t* base, size_t base_stride,
                                uint16_t* output, size_t output_stride, const void* plan, size_t plan_bytes,
                                size_t num_seqs, size_t num_tokens, size_t num_adapters, size_t max_rank,
                                size_t in_features, size_t out_features, void* workspace, size_t workspace_bytes,
                                void* stream) {
    const char* name = "lora_f16";
    if (const char* why = lora_sizes(num_seqs, num_tokens, num_adapters)) return arg(name, why);
    if (num_adapters && (max_rank < 8 || max_rank > (size_t)cb::batch::kLoraMaxRank || max_rank % 8))
        return arg(name, "max_rank must be a multiple of 8, 8 to 256");
    if (in_features % 8 || out_features % 8) return arg(name, "in_features and out_features must be multiples of 8");
    if (in_features > ((size_t)1 << 20) || out_features > ((size_t)1 << 20)) return arg(name, "size too large");
    if (num_seqs == 0 || num_tokens == 0 || out_features == 0) return CB_OK;
    if (!output || !plan || !workspace || (num_adapters && out_features && (!b || (in_features && (!x || !a)))))
        return arg(name, "null argument");
    if (x_stride < in_features || output_stride < out_features || (base && base_stride < out_features))
        return arg(name, "a stride is less than its row");
    if (x_stride > kStrideMax || output_stride > kStrideMax || (base && base_stride > kStrideMax))
        return arg(name, "stride too large");
    if (x_stride % 8 || output_stride % 8 || (base && base_stride % 8) || !aligned(x, 16) || !aligned(a, 16) ||
        !aligned(b, 16) || !aligned(base, 16) || !aligned(output, 16) || !aligned(plan, 16) || !aligned(workspace, 16))
        return arg(name, "pointers must be 16-byte aligned and strides multiples of 8");
    if (!aligned(ranks, 4) || !aligned(scales, 4)) return arg(name, "ranks and scales must be 4-byte aligned");
    if (base == output && base_stride != output_stride) return arg(name, "output overlaps base at another stride");
    if (plan_bytes < cactus_cuda_lora_plan_bytes(num_seqs, num_tokens, num_adapters)) return arg(name, "plan too small");
    if (workspace_bytes < cactus_cuda_lora_workspace(num_tokens, max_rank)) return arg(name, "workspace too small");
    cb::batch::LoraCall c = {};
    c.x = H(x);
    c.a = H(a);
    c.b = H(b);
    c.base = H(base);
    c.ranks = ranks;
    c.scales = scales;
    c.out = H(output);
    c.x_stride = (long long)x_stride;
    c.base_stride = (long long)base_stride;
    c.out_stride = (long long)output_stride;
    c.plan = static_cast<const int*>(plan);
    c.num_seqs = (int)num_seqs;
    c.num_tokens = (int)num_tokens;
    c.num_adapters = (int)num_adapters;
    c.max_rank = (int)max_rank;
    c.k = (int)in_features;
    c.n = (int)out_features;
    c.ws = static_cast<float*>(workspace);
    return launched(name, cb::batch::launch_lora(c, S(stream)));
}

CB_API int cactus_cuda_logits_process_f16(const uint16_t* logits, size_t logits_stride, uint16_t* output,
                                          size_t output_stride, size_t rows, size_t vocab, const float* penalties,
                                          const uint32_t* history, const int32_t* history_offsets,
                                          const int32_t* prompt_lens, size_t num_history, const uint32_t* bias_ids,
                                          const float* bias_values, const int32_t* bias_offsets, size_t num_biases,
                                          const uint32_t* masks, size_t mask_stride, size_t num_masks,
                                          const int32_t* mask_ids, void* stream) {
    const char* name = "logits_process_f16";
    if (rows == 0 || vocab == 0) return CB_OK;
    if (!logits || !output) return arg(name, "null argument");
    if (rows > kIntMax || vocab > ((size_t)1 << 27)) return arg(name, "size too large");
    if (logits_stride < vocab || output_stride < vocab) return arg(name, "a stride is less than vocab");
    if (logits_stride > kStrideMax || output_stride > kStrideMax) return arg(name, "stride too large");
    if (logits == output && logits_stride != output_stride) return arg(name, "output overlaps logits at another stride");
    if (num_history > kIntMax || num_biases > kIntMax || num_masks > kIntMax) return arg(name, "size too large");
    if (penalties && history && !history_offsets) return arg(name, "history without history_offsets");
    if (bias_ids && (!bias_values || !bias_offsets)) return arg(name, "bias_ids without bias_values or bias_offsets");
    if (masks && (mask_stride > kStrideMax || mask_stride < (vocab + 31) / 32))
        return arg(name, "mask_stride must be at least the words of vocab");
    if (masks && !mask_ids && num_masks < rows) return arg(name, "fewer masks than rows");
    if (!aligned(logits, 2) || !aligned(output, 2) || !aligned(penalties, 4) || !aligned(history, 4) ||
        !aligned(history_offsets, 4) || !aligned(prompt_lens, 4) || !aligned(bias_ids, 4) || !aligned(bias_values, 4) ||
        !aligned(bias_offsets, 4) || !aligned(masks, 4) || !aligned(mask_ids, 4))
        return arg(name, "misaligned argument");
    cb::batch::LogitsCall c = {};
    c.in = H(logits);
    c.out = H(output);
    c.in_stride = (long long)logits_stride;
    c.out_stride = (long long)output_stride;
    c.rows = (int)rows;
    c.vocab = (int)vocab;
    if (penalties && history) {
        c.penalties = penalties;
        c.history = history;
        c.history_offsets = history_offsets;
        c.prompt_lens = prompt_lens;
        c.num_history = (int)num_history;
    }
    if (bias_ids) {
        c.bias_ids = bias_ids;
        c.bias_values = bias_values;
        c.bias_offsets = bias_offsets;
        c.num_biases = (int)num_biases;
    }
    if (masks) {
        c.masks = masks;
        c.mask_stride = (long long)mask_stride;
        c.num_masks = (int)num_masks;
        c.mask_ids = mask_ids;
    }
    return launched(name, cb::batch::launch_logits(c, S(stream)));
}

}  // extern "C"
