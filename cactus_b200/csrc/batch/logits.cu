// Penalties, biases and masks on a batch's logits. A block takes a slice of a row's vocabulary. It lists the
// slice's tokens that the row's history or biases name (each once, with its count and its last bias, in shared
// memory), passes over the slice in 16-byte pieces for the mask, and then computes the listed tokens.
#include <atomic>

#include "../common.cuh"
#include "batch_ops.h"

namespace cb {
namespace batch {

namespace {

constexpr int kThreads = 256;
constexpr unsigned kSeen = 0x80000000u;  // the history has it; the other bits: how often behind the prompt

// shared memory of a slice of n tokens: counts, biases, list, bits
__host__ __device__ constexpr int slice_bytes(int n) { return n * 10 + n / 8; }

struct List {
    int first, count;
};
// a row's list, cut to nothing where its offsets are not the call's
__device__ __forceinline__ List list_of(const int* offsets, int row, int most) {
    const int a = __ldg(offsets + row), b = __ldg(offsets + row + 1);
    if (a >= 0 && a <= b && b <= most) return {a, b - a};
    if (threadIdx.x == 0) report_dev_error(kDevBadList);
    return {0, 0};
}

// the bits of tokens v .. v + 7 (v may be below 0; bits of tokens that are none are anything)
__device__ __forceinline__ unsigned mask8(const uint32_t* mask, int v, int words) {
    if (v < 0) return __ldg(mask) << -v & 0xffu;
    const int w = v >> 5, shift = v & 31;
    unsigned bits = __ldg(mask + w) >> shift;
    if (shift > 24 && w + 1 < words) bits |= __ldg(mask + w + 1) << (32 - shift);
    return bits & 0xffu;
}

// V pieces of 8 tokens a thread. Pieces begin where the input's 16-byte units do: piece i of a row has its tokens
// 8 i - skew to 8 i - skew + 7, as far as there are such.
template <int V>
__global__ void __launch_bounds__(kThreads) logits_kernel(LogitsCall c) {
    constexpr int kSlice = kThreads * 8 * V;
    extern __shared__ __align__(16) uint8_t smem[];
    unsigned* s_count = reinterpret_cast<unsigned*>(smem);
    int* s_bias = reinterpret_cast<int*>(smem + 4 * kSlice);  // place of a token's last bias + 1
    uint16_t* s_list = reinterpret_cast<uint16_t*>(smem + 8 * kSlice);
    unsigned* s_bits = reinterpret_cast<unsigned*>(smem + 10 * kSlice);
    __shared__ int s_listed;
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x;
    const __half* in = c.in + row * c.in_stride;
    __half* out = c.out + row * c.out_stride;
    const int skew = (int)(reinterpret_cast<uintptr_t>(in) >> 1 & 7);
    const bool in_place = in == out, same_skew = (int)(reinterpret_cast<uintptr_t>(out) >> 1 & 7) == skew;
    const int v0 = blockIdx.y * kSlice - skew;
    if (v0 >= c.vocab) return;
    const uint32_t* mask = nullptr;
    if (c.masks) {
        const int m = c.mask_ids ? __ldg(c.mask_ids + row) : row;
        if (m >= 0 && m < c.num_masks) mask = c.masks + m * c.mask_stride;
        else if (m != -1 && threadIdx.x == 0) report_dev_error(kDevBadList);
    }
    // the pieces: what a mask leaves nothing of is not read, and in place neither is what stays whole
    unsigned bits[V];
    uint4 x[V];
    const int words = (c.vocab + 31) >> 5;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int v = v0 + 8 * (i * kThreads + (int)threadIdx.x);
        bits[i] = v >= c.vocab ? 0u : mask ? mask8(mask, v, words) : 0xffu;
    }
    auto whole = [&](int v) { return v >= 0 && v + 8 <= c.vocab; };
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int v = v0 + 8 * (i * kThreads + (int)threadIdx.x);
        x[i] = make_uint4(0, 0, 0, 0);
        if (bits[i] == 0 || (in_place && bits[i] == 0xffu)) continue;
        if (whole(v)) {
            x[i] = *reinterpret_cast<const uint4*>(in + v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (v + j >= 0 && v + j < c.vocab) reinterpret_cast<__half*>(&x[i])[j] = in[v + j];
        }
    }
    // the listed tokens
    List history = {0, 0}, biases = {0, 0};
    float repetition = 1.0f, frequency = 0.0f, presence = 0.0f;
    int prompt = 0;
    if (c.penalties) {
        history = list_of(c.history_offsets, row, c.num_history);
        repetition = __ldg(c.penalties + 3LL * row);
        frequency = __ldg(c.penalties + 3LL * row + 1);
        presence = __ldg(c.penalties + 3LL * row + 2);
        if (!(repetition > 0.0f && repetition < INFINITY)) {
            if (threadIdx.x == 0) report_dev_error(kDevBadList);
            repetition = 1.0f;
        }
        prompt = c.prompt_lens ? __ldg(c.prompt_lens + row) : 0;
    }
    if (c.bias_ids) biases = list_of(c.bias_offsets, row, c.num_biases);
    const uint32_t *ids = c.history + history.first, *bias_ids = c.bias_ids + biases.first;
    const bool lists = history.count + biases.count > 0;
    if (lists) {
        for (int i = threadIdx.x; i < kSlice / 32; i += kThreads) s_bits[i] = 0;
        if (threadIdx.x == 0) s_listed = 0;
        __syncthreads();
        auto note = [&](unsigned id) {
            const unsigned at = id - (unsigned)v0;  // wraps around where id is before the slice
            if (id >= (unsigned)c.vocab) report_dev_error(kDevBadList);
            else if (at < (unsigned)kSlice && !(atomicOr(&s_bits[at >> 5], 1u << (at & 31)) >> (at & 31) & 1u)) {
                s_count[at] = 0;
                s_bias[at] = 0;
                s_list[atomicAdd(&s_listed, 1)] = (uint16_t)at;
            }
        };
#pragma unroll 4
        for (int i = threadIdx.x; i < history.count; i += kThreads) note(__ldg(ids + i));
#pragma unroll 4
        for (int i = threadIdx.x; i < biases.count; i += kThreads) note(__ldg(bias_ids + i));
        __syncthreads();
#pragma unroll 4
        for (int i = threadIdx.x; i < history.count; i += kThreads) {
            const unsigned at = __ldg(ids + i) - (unsigned)v0;
            if (at < (unsigned)kSlice && at + (unsigned)v0 < (unsigned)c.vocab) {
                atomicOr(&s_count[at], kSeen);
                if (i >= prompt) atomicAdd(&s_count[at], 1u);
            }
        }
#pragma unroll 4
        for (int i = threadIdx.x; i < biases.count; i += kThreads) {
            const unsigned at = __ldg(bias_ids + i) - (unsigned)v0;
            if (at < (unsigned)kSlice && at + (unsigned)v0 < (unsigned)c.vocab) atomicMax(&s_bias[at], i + 1);
        }
        __syncthreads();
    }
    // the listed tokens' results, before anything is written: in place their logits are still there
    constexpr int kHeld = 2;  // a thread's first listed tokens wait in registers, further ones for the barrier
    const int listed = lists ? s_listed : 0;
    auto result = [&](int at) {
        float l = h2f(in[v0 + at]);
        const unsigned n = s_count[at];
        const int bias = s_bias[at];
        if (n) {
            l = l > 0.0f ? __fdiv_rn(l, repetition) : __fmul_rn(l, repetition);
            const unsigned made = n & ~kSeen;
            if (made) l = __fsub_rn(__fsub_rn(l, __fmul_rn(frequency, (float)made)), presence);
        }
        if (bias) l = __fadd_rn(l, __ldg(c.bias_values + biases.first + bias - 1));
        if (fabsf(l) < INFINITY) l = fminf(fmaxf(l, -65504.0f), 65504.0f);
        return f2h(l);
    };
    auto hidden = [&](int at) { return mask && !(mask8(mask, v0 + at, words) & 1u); };
    __half held[kHeld];
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        const int i = k * kThreads + threadIdx.x;
        if (i < listed && !hidden(s_list[i])) held[k] = result(s_list[i]);
    }
    // the pass over the slice
    const __half none = __ushort_as_half(0xFC00);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int v = v0 + 8 * (i * kThreads + (int)threadIdx.x);
        if (v >= c.vocab || (in_place && bits[i] == 0xffu)) continue;
        __half* h = reinterpret_cast<__half*>(&x[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (!(bits[i] >> j & 1u)) h[j] = none;
        if (whole(v) && same_skew) {
            *reinterpret_cast<uint4*>(out + v) = x[i];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (v + j >= 0 && v + j < c.vocab) out[v + j] = h[j];
        }
    }
    if (!listed) return;
    __syncthreads();  // the pass has written what the listed tokens' results replace
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        const int i = k * kThreads + threadIdx.x;
        if (i < listed && !hidden(s_list[i])) out[v0 + s_list[i]] = held[k];
    }
    for (int i = kHeld * kThreads + threadIdx.x; i < listed; i += kThreads)
        if (!hidden(s_list[i])) out[v0 + s_list[i]] = result(s_list[i]);
}

template <int V>
cudaError_t launch(const LogitsCall& c, cudaStream_t st) {
    constexpr int kSlice = kThreads * 8 * V;
    const int smem = c.penalties || c.bias_ids ? slice_bytes(kSlice) : 0;
    if (slice_bytes(kSlice) > 48 * 1024) {
        static std::atomic<unsigned long long> set{0};  // a bit a device
        int dev = 0;
        cudaGetDevice(&dev);
        if (!(set.load() >> (dev & 63) & 1)) {
            const cudaError_t e = cudaFuncSetAttribute(logits_kernel<V>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                       slice_bytes(kSlice));
            if (e != cudaSuccess) return e;
            set.fetch_or(1ull << (dev & 63));
        }
    }
    const dim3 grid((unsigned)c.rows, (unsigned)((c.vocab + 7 + kSlice - 1) / kSlice));
    return launch_k(logits_kernel<V>, grid, dim3(kThreads), smem, st, c);
}

}  // namespace

int launch_logits(const LogitsCall& c, cudaStream_t st) {
    // The largest slices that leave two blocks for each SM: each block reads the row's lists, and with four
    // pieces a thread more loads are in flight.
    auto blocks = [&](int v) { return (long long)c.rows * ((c.vocab + 7) / (kThreads * 8 * v) + 1); };
    const cudaError_t e = blocks(4) >= 2 * kNumSMs   ? launch<4>(c, st)
                          : blocks(2) >= 2 * kNumSMs ? launch<2>(c, st)
                                                     : launch<1>(c, st);
    return e == cudaSuccess ? 0 : -1;
}

}  // namespace batch
}  // namespace cb
