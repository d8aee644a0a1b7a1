// Penalties, biases and masks on a batch's logits. A block takes a slice of a row's vocabulary: it counts the
// tokens of the row's history and finds the row's biases that fall into the slice, in shared memory, then
// passes once over the slice.
#include "../common.cuh"
#include "batch_ops.h"

namespace cb {
namespace batch {

namespace {

constexpr int kThreads = 256, kSlice = 4096;
constexpr unsigned kSeen = 0x80000000u;  // the history has it; the other bits: how often behind the prompt

// first and count of a row's list, cut to what the call has
__device__ __forceinline__ void list_of(const int* offsets, int row, int most, int* first, int* count) {
    const int a = offsets[row], b = offsets[row + 1];
    *first = *count = 0;
    if (a >= 0 && a <= b && b <= most) {
        *first = a;
        *count = b - a;
    } else if (threadIdx.x == 0) {
        report_dev_error(kDevBadList);
    }
}

__global__ void __launch_bounds__(kThreads) logits_kernel(LogitsCall c) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ unsigned s_count[kSlice];
    __shared__ int s_bias[kSlice];  // place of a token's last bias + 1
    const int row = blockIdx.x, v0 = blockIdx.y * kSlice, size = min(kSlice, c.vocab - v0);
    for (int i = threadIdx.x; i < kSlice; i += kThreads) {
        s_count[i] = 0;
        s_bias[i] = 0;
    }
    __syncthreads();
    float repetition = 1.0f, frequency = 0.0f, presence = 0.0f;
    if (c.penalties) {
        repetition = c.penalties[3LL * row];
        frequency = c.penalties[3LL * row + 1];
        presence = c.penalties[3LL * row + 2];
        if (!(repetition > 0.0f && repetition < INFINITY)) {
            if (threadIdx.x == 0) report_dev_error(kDevBadList);
            repetition = 1.0f;
        }
        int first, count;
        list_of(c.history_offsets, row, c.num_history, &first, &count);
        const int prompt = c.prompt_lens ? c.prompt_lens[row] : 0;
        for (int i = threadIdx.x; i < count; i += kThreads) {
            const unsigned id = c.history[first + i];
            if (id >= (unsigned)c.vocab) report_dev_error(kDevBadList);
            else if (id - (unsigned)v0 < (unsigned)size) {
                atomicOr(&s_count[id - v0], kSeen);
                if (i >= prompt) atomicAdd(&s_count[id - v0], 1u);
            }
        }
    }
    int bias_first = 0;
    if (c.bias_ids) {
        int count;
        list_of(c.bias_offsets, row, c.num_biases, &bias_first, &count);
        for (int i = threadIdx.x; i < count; i += kThreads) {
            const unsigned id = c.bias_ids[bias_first + i];
            if (id >= (unsigned)c.vocab) report_dev_error(kDevBadList);
            else if (id - (unsigned)v0 < (unsigned)size) atomicMax(&s_bias[id - v0], i + 1);
        }
    }
    const uint32_t* mask = nullptr;
    if (c.masks) {
        const int m = c.mask_ids ? c.mask_ids[row] : row;
        if (m >= 0 && m < c.num_masks) mask = c.masks + m * c.mask_stride;
        else if (m != -1 && threadIdx.x == 0) report_dev_error(kDevBadList);
    }
    __syncthreads();
    const __half* in = c.in + row * c.in_stride + v0;
    __half* out = c.out + row * c.out_stride + v0;
    for (int i = threadIdx.x; i < size; i += kThreads) {
        const unsigned n = s_count[i];
        if (mask && !((mask[(v0 + i) >> 5] >> ((v0 + i) & 31)) & 1u)) {
            out[i] = __ushort_as_half(0xFC00);
            continue;
        }
        if (!n && !s_bias[i]) {
            out[i] = in[i];
            continue;
        }
        float l = h2f(in[i]);
        if (n) {
            l = l > 0.0f ? __fdiv_rn(l, repetition) : __fmul_rn(l, repetition);
            const unsigned made = n & ~kSeen;
            if (made) l = __fsub_rn(__fsub_rn(l, __fmul_rn(frequency, (float)made)), presence);
        }
        if (s_bias[i]) l = __fadd_rn(l, c.bias_values[bias_first + s_bias[i] - 1]);
        if (fabsf(l) < INFINITY) l = fminf(fmaxf(l, -65504.0f), 65504.0f);
        out[i] = f2h(l);
    }
}

}  // namespace

int launch_logits(const LogitsCall& c, cudaStream_t st) {
    const dim3 grid((unsigned)c.rows, (unsigned)((c.vocab + kSlice - 1) / kSlice));
    return launch_k(logits_kernel, grid, dim3(kThreads), 0, st, c) == cudaSuccess ? 0 : -1;
}

}  // namespace batch
}  // namespace cb
