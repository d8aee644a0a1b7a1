// Penalties, biases and masks on a batch's logits. A block takes a slice of a row's vocabulary: it notes which of the
// slice's tokens the row's history or biases name, and where, passes over the slice in 16-byte pieces for the mask, and then
// counts and computes the noted tokens. Each logit is read and written once, what a mask hides only written, and in
// place what stays is not touched. 256 rows of 128256 with histories of 750 to 1500 ids take 37 us, 3.6 TB/s of what that
// moves; the barriers between noting, passing and counting bound it (with counters for every token of a slice, which
// left room for two blocks a SM, it took 92; with the lists read once more for the count 39). Masks alone, in place: 48
// rows of 262144 9.0 us.
#include "../common.cuh"
#include "batch_ops.h"

namespace cb {
namespace batch {

namespace {

constexpr unsigned kSeen = 0x80000000u;  // the history has it; the other bits: how often behind the prompt
constexpr int kKept = 512;               // entries of the lists in a slice that are kept for the count
constexpr int kRound = 1024;             // noted tokens that are counted at a time

// T threads, V pieces of 8 tokens a thread. Shared memory: bits of the noted tokens, their numbers (in the order of
// their noting), of one round the counts, last biases and tokens, and the entries that are kept: place in the list and token.
template <int T, int V>
struct Slice {
    static constexpr int kTokens = T * 8 * V;
    static constexpr int kNumbers = kTokens / 8, kCounts = kNumbers + 2 * kTokens, kBiases = kCounts + 4 * kRound;
    static constexpr int kList = kBiases + 4 * kRound, kPlaces = kList + 2 * kRound, kAts = kPlaces + 4 * kKept;
    static constexpr int smem = kAts + 2 * kKept;
    static_assert(kTokens <= 65536, "16-bit numbers");
};

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

// Each id of a list, with its place there.
template <int T, typename F>
__device__ __forceinline__ void each(const uint32_t* ids, int count, F f) {
    constexpr int kAhead = 4;  // loads in flight
    for (int i0 = threadIdx.x; i0 < count; i0 += T * kAhead) {
        unsigned id[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) id[k] = i0 + k * T < count ? __ldg(ids + i0 + k * T) : 0xffffffffu;
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (i0 + k * T < count) f(id[k], i0 + k * T);
    }
}

// Pieces begin where the input's 16-byte units do: piece i of a row has its tokens 8 i - skew to 8 i - skew + 7, as
// far as there are such.
template <int T, int V>
__global__ void __launch_bounds__(T, T == 512 ? 3 : 1) logits_kernel(LogitsCall c) {
    using S = Slice<T, V>;
    extern __shared__ __align__(16) uint8_t smem[];
    unsigned* s_bits = reinterpret_cast<unsigned*>(smem);
    uint16_t* s_number = reinterpret_cast<uint16_t*>(smem + S::kNumbers);
    unsigned* s_count = reinterpret_cast<unsigned*>(smem + S::kCounts);
    int* s_bias = reinterpret_cast<int*>(smem + S::kBiases);  // place of a token's last bias + 1
    uint16_t* s_list = reinterpret_cast<uint16_t*>(smem + S::kList);
    int* s_place = reinterpret_cast<int*>(smem + S::kPlaces);
    uint16_t* s_at = reinterpret_cast<uint16_t*>(smem + S::kAts);
    __shared__ int s_noted, s_kept;
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.x;
    const __half* in = c.in + row * c.in_stride;
    __half* out = c.out + row * c.out_stride;
    const int skew = (int)(reinterpret_cast<uintptr_t>(in) >> 1 & 7);
    const bool in_place = in == out, same_skew = (int)(reinterpret_cast<uintptr_t>(out) >> 1 & 7) == skew;
    const int v0 = blockIdx.y * S::kTokens - skew;
    if (v0 >= c.vocab) return;
    List history = {0, 0}, biases = {0, 0};
    if (c.penalties) history = list_of(c.history_offsets, row, c.num_history);
    if (c.bias_ids) biases = list_of(c.bias_offsets, row, c.num_biases);
    const uint32_t *ids = c.history + history.first, *bias_ids = c.bias_ids + biases.first;
    const bool lists = history.count + biases.count > 0;
    const uint32_t* mask = nullptr;
    if (c.masks) {
        const int m = c.mask_ids ? __ldg(c.mask_ids + row) : row;
        if (m >= 0 && m < c.num_masks) mask = c.masks + m * c.mask_stride;
        else if (m != -1 && threadIdx.x == 0) report_dev_error(kDevBadList);
    }
    // the slice's tokens among the ids; one before the slice wraps around
    auto inside = [&](unsigned id) { return id - (unsigned)v0 < (unsigned)S::kTokens && id < (unsigned)c.vocab; };
    if (lists) {  // the tokens that they name get numbers
        for (int i = threadIdx.x; i < S::kTokens / 32; i += T) s_bits[i] = 0;
        for (int i = threadIdx.x; i < kRound; i += T) s_count[i] = 0, s_bias[i] = 0;
        if (threadIdx.x == 0) s_noted = s_kept = 0;
        __syncthreads();
        auto note = [&](unsigned id, int i) {
            const unsigned at = id - (unsigned)v0;
            if (inside(id)) {
                const int kept = atomicAdd(&s_kept, 1);
                if (kept < kKept) s_place[kept] = i, s_at[kept] = (uint16_t)at;
                if (!(atomicOr(&s_bits[at >> 5], 1u << (at & 31)) >> (at & 31) & 1u)) s_number[at] = (uint16_t)atomicAdd(&s_noted, 1);
            } else if (id >= (unsigned)c.vocab) {
                report_dev_error(kDevBadList);
            }
        };
        each<T>(ids, history.count, note);
        each<T>(bias_ids, biases.count, [&](unsigned id, int i) { note(id, i - biases.count); });
    }
    // the pieces: what a mask leaves nothing of is not read, and in place neither is what stays whole
    unsigned bits[V];
    uint4 x[V];
    const int words = (c.vocab + 31) >> 5;
    const bool inner = v0 >= 0 && v0 + S::kTokens <= c.vocab;  // all pieces are whole
    auto place = [&](int i) { return v0 + 8 * (i * T + (int)threadIdx.x); };
    auto whole = [&](int v) { return inner || (v >= 0 && v + 8 <= c.vocab); };
#pragma unroll
    for (int i = 0; i < V; ++i) bits[i] = !inner && place(i) >= c.vocab ? 0u : mask ? mask8(mask, place(i), words) : 0xffu;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int v = place(i);
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
    // the pass over the slice
    const __half none = __ushort_as_half(0xFC00);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int v = place(i);
        if ((!inner && v >= c.vocab) || (in_place && bits[i] == 0xffu)) continue;
        __half* h = reinterpret_cast<__half*>(&x[i]);
        if (bits[i] != 0xffu)
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
    float repetition = 1.0f, frequency = 0.0f, presence = 0.0f;
    int prompt = 0;
    // what is no factor or no length is said of a row without lists too, by one of its slices
    if (c.penalties && (lists || (blockIdx.y == 0 && threadIdx.x == 0))) {
        repetition = __ldg(c.penalties + 3LL * row);
        frequency = __ldg(c.penalties + 3LL * row + 1);
        presence = __ldg(c.penalties + 3LL * row + 2);
        prompt = c.prompt_lens ? __ldg(c.prompt_lens + row) : 0;
        const bool factor = repetition > 0.0f && repetition < INFINITY;
        if ((!factor || prompt < 0) && threadIdx.x == 0) report_dev_error(kDevBadList);
        if (!factor) repetition = 1.0f;
    }
    if (!lists) return;
    // The noted tokens, kRound numbers at a time (nearly always all of them). In place their logits are still there:
    // the pass wrote them as they were, but for hidden ones, which are left out here.
    for (int first = 0;; first += kRound) {
        __syncthreads();  // the pass has written what the results replace; numbers and zeros are there
        const int noted = min(s_noted - first, kRound);
        if (noted <= 0) break;
        // of the token at a place of the slice: place i of the history, or, with i below 0, i + their count of the biases
        auto count = [&](unsigned at, int i) {
            const unsigned n = (unsigned)s_number[at] - (unsigned)first;
            if (n >= (unsigned)kRound) return;
            s_list[n] = (uint16_t)at;
            if (i < 0) atomicMax(&s_bias[n], i + biases.count + 1);
            else if (i >= prompt) atomicAdd(&s_count[n], 1u);
            else atomicOr(&s_count[n], kSeen);
        };
        if (s_kept <= kKept) {  // else the lists once more
            for (int i = threadIdx.x; i < s_kept; i += T) count(s_at[i], s_place[i]);
        } else {
            each<T>(ids, history.count, [&](unsigned id, int i) {
                if (inside(id)) count(id - (unsigned)v0, i);
            });
            each<T>(bias_ids, biases.count, [&](unsigned id, int i) {
                if (inside(id)) count(id - (unsigned)v0, i - biases.count);
            });
        }
        __syncthreads();
        for (int i = threadIdx.x; i < noted; i += T) {
            const int v = v0 + s_list[i];
            const unsigned n = s_count[i];
            const int bias = s_bias[i];
            s_count[i] = 0, s_bias[i] = 0;  // for the next round
            if (mask && !(__ldg(mask + (v >> 5)) >> (v & 31) & 1u)) continue;
            float l = h2f(in[v]);
            if (n) {
                l = l > 0.0f ? __fdiv_rn(l, repetition) : __fmul_rn(l, repetition);
                const unsigned made = n & ~kSeen;
                if (made) l = __fsub_rn(__fsub_rn(l, __fmul_rn(frequency, (float)made)), presence);
            }
            if (bias) l = __fadd_rn(l, __ldg(c.bias_values + biases.first + bias - 1));
            if (fabsf(l) < INFINITY) l = fminf(fmaxf(l, -65504.0f), 65504.0f);
            out[v] = f2h(l);
        }
    }
}

template <int T, int V>
cudaError_t launch(const LogitsCall& c, cudaStream_t st) {
    using S = Slice<T, V>;
    static_assert(S::smem <= 48 * 1024, "no attribute needed");
    const dim3 grid((unsigned)c.rows, (unsigned)((c.vocab + 7 + S::kTokens - 1) / S::kTokens));
    return launch_k(logits_kernel<T, V>, grid, dim3(T), c.penalties || c.bias_ids ? S::smem : 0, st, c);
}

}  // namespace

int launch_logits(const LogitsCall& c, cudaStream_t st) {
    // Large slices, since each block goes through the row's lists (and once more where it has more than kKept of their
    // entries); small ones, for the shortest time, where those are no more than four blocks for each SM. Slices of 2048 /
    // 16384, histories of 750 to 1500, a graph's replay, us: 4 rows of 128256 6.3 / 8.3, of 262144 6.3 / 8.3, 16 rows of
    // 32000 7.5 / 8.3, 32 of 32000 8.3 / 8.3, 16 rows of 128256 10.4 / 8.3, 64 rows of 32000 12.4 / 8.3.
    const long long small = (long long)c.rows * ((c.vocab + 7) / 2048 + 1);
    const cudaError_t e = small <= 4 * kNumSMs ? launch<256, 1>(c, st) : launch<512, 4>(c, st);
    return e == cudaSuccess ? 0 : -1;
}

}  // namespace batch
}  // namespace cb
