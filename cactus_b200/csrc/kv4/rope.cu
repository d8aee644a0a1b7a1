// The append of the 4-bit paged KV cache that normalises and rotates on the way, and the table of turns
// that it reads. A warp takes a token's heads one group after another, 32 * 8 / D heads at a time: D / 8 lanes
// share a head's row (8 elements, one 16-byte load each), and the token's turns stay in registers for all of
// them. Shuffles add up the squares of the norm, fetch the other element of each rotated pair and reduce a
// group's ends for the quantisation.
#include <algorithm>
#include <type_traits>

#include "kv4.cuh"
#include "kv4_ops.h"
#include "quantise.cuh"

namespace cb {
namespace kv4 {

namespace {

constexpr int kRopeThreads = 256;

// (cos, sin) of position p's angles: p * theta^(-2 i / R), in 64 bits up to the last rounding.
__global__ void rope_table_kernel(double theta, int half, long long n, float2* __restrict__ table) {
    pdl_launch_dependents();
    pdl_wait();
    const long long at = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (at >= n) return;
    const int i = (int)(at % half);
    double s, c;
    sincos((double)(at / half) * pow(theta, -(double)i / (double)half), &s, &c);
    table[at] = make_float2((float)c, (float)s);
}

// The sequence of token row t as find_seq() finds it, 32 places at a time.
__device__ __forceinline__ int find_seq_warp(const int* offsets, int n, int t) {
    if (t >= __ldg(offsets + n)) return -1;
    int lo = 0, hi = n;  // offsets[lo] <= t < offsets[hi]
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + ((int)(threadIdx.x & 31) + 1) * step;
        lo += __popc(__ballot_sync(0xffffffffu, at < hi && __ldg(offsets + at) <= t)) * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

// The sum of a row's squares, eight of them a lane. The halves of the row are added to one another, element by
// element, then the halves of that (down to 32 sums of four neighbours for D >= 128): a fixed order of few steps,
// of which every lane has its share, as each exchange passes on the part that the lane does not keep.
template <int D>
__device__ __forceinline__ float sum_of_squares(const float (&v)[8], int lane) {
    const unsigned full = 0xffffffffu;
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = __fmul_rn(v[j], v[j]);
    // keeps N of 2 N values: the upper ones where `upper`
    auto halve = [&](auto n, bool upper, int o) {
        constexpr int N = decltype(n)::value;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float keep = upper ? q[N + j] : q[j], give = upper ? q[j] : q[N + j];
            q[j] = __fadd_rn(keep, __shfl_xor_sync(full, give, o));
        }
    };
    auto add = [&](int o) { q[0] = __fadd_rn(q[0], __shfl_xor_sync(full, q[0], o)); };
    auto four = [&](int j) { return __fadd_rn(__fadd_rn(__fadd_rn(q[j], q[j + 1]), q[j + 2]), q[j + 3]); };
    if constexpr (D == 64) {
        halve(std::integral_constant<int, 4>{}, lane & 4, 4);
        halve(std::integral_constant<int, 2>{}, lane & 2, 2);
        halve(std::integral_constant<int, 1>{}, lane & 1, 1);
        add(4), add(2), add(1);
    } else if constexpr (D == 128) {
        q[0] = four(0), q[1] = four(4);
        halve(std::integral_constant<int, 1>{}, lane & 8, 8);
        add(4), add(2), add(1), add(8);
    } else {
        halve(std::integral_constant<int, 4>{}, lane & 16, 16);
        q[0] = four(0);
        add(8), add(4), add(2), add(1), add(16);
    }
    return q[0];
}

// Eight elements of a row of D, normalised (where there is a weight) and turned, as fp16. turn: the lane's pairs
// (cos, sin); `part` lanes have each half of the rotated elements.
template <int D>
__device__ __forceinline__ uint4 norm_and_turn(const uint4& in, bool norm, const uint4& weight, float eps,
                                               const float2 (&turn)[8], int part, int lane) {
    const unsigned full = 0xffffffffu;
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 p = __half22float2(reinterpret_cast<const __half2*>(&in)[j]);
        v[2 * j] = p.x;
        v[2 * j + 1] = p.y;
    }
    if (norm) {
        const float inv = rsqrtf(__fadd_rn(__fmul_rn(sum_of_squares<D>(v, lane), 1.0f / D), eps));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 p = __half22float2(reinterpret_cast<const __half2*>(&weight)[j]);
            v[2 * j] = __fmul_rn(__fmul_rn(v[2 * j], inv), p.x);
            v[2 * j + 1] = __fmul_rn(__fmul_rn(v[2 * j + 1], inv), p.y);
        }
    }
    if (part) {
        const bool first = lane < part, turned = lane < 2 * part;
        const int from = (threadIdx.x & 31) + (first ? part : turned ? -part : 0);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float u = __shfl_sync(full, v[j], from);
            const float a = __fmul_rn(v[j], turn[j].x), b = __fmul_rn(u, turn[j].y);
            if (turned) v[j] = first ? __fsub_rn(a, b) : __fadd_rn(a, b);
        }
    }
    uint4 out;
#pragma unroll
    for (int j = 0; j < 4; ++j) reinterpret_cast<__half2*>(&out)[j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
    return out;
}

// Eight elements of a row into its block: codes, and the parameters of their group. All lanes take part.
template <int D>
__device__ __forceinline__ void quantise_row(const uint4& x, uint8_t* part, int row, int lane, const Geom& ge) {
    const __half2* h = reinterpret_cast<const __half2*>(&x);
    const int per_group = ge.g >> 3;
    // (largest, -smallest): exact in fp16, and a NaN stays one
    const __half2 hi2 = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    const __half2 lo2 = __hmin2_nan(__hmin2_nan(h[0], h[1]), __hmin2_nan(h[2], h[3]));
    __half2 ends = __hmax2_nan(__lows2half2(hi2, __hneg2(lo2)), __highs2half2(hi2, __hneg2(lo2)));
    for (int o = 1; o < per_group; o <<= 1) ends = __hmax2_nan(ends, __shfl_xor_sync(0xffffffffu, ends, o));
    const float hi = __low2float(ends), lo = -__high2float(ends);
    const __half step = step_of(hi, lo);
    const float fs = __half2float(step);
    const bool bad = !(__fsub_rn(hi, lo) < INFINITY);  // an infinity or a NaN in the group
    uint32_t w = 0;
    if (!bad && fs > 0.0f) w = quant_codes(h, lo, fs);
    if (!part) return;
    *reinterpret_cast<uint32_t*>(part + row * (D / 2) + lane * 4) = w;
    if ((lane & (per_group - 1)) == 0) {
        const __half nan = __ushort_as_half(0x7FFF);
        *reinterpret_cast<__half2*>(part + ge.k_params() + (row * ge.ng() + (lane >> (__ffs(per_group) - 1))) * 4) =
            bad ? __halves2half2(nan, nan) : __halves2half2(step, __float2half_rn(lo));
    }
}

// Block (x, y): tokens kWarps x .., one a warp, and the y-th share of the groups of heads: query heads, then key
// heads, then values.
constexpr int kWarps = kRopeThreads / 32, kBatch = 4;  // groups whose loads are in flight together

template <int D>
__global__ void __launch_bounds__(kRopeThreads) kv4_rope_append_kernel(RopeCall c, Pages pg, Geom ge) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int kLanes = D / 8, kHeads = 32 / kLanes;
    const int lane = threadIdx.x % kLanes, sub = (threadIdx.x & 31) / kLanes;
    const int t = blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (t >= c.num_tokens) return;
    const int q_groups = (c.hq + kHeads - 1) / kHeads, kv_groups = (ge.hkv + kHeads - 1) / kHeads;
    const int groups = q_groups + 2 * kv_groups, first = groups * blockIdx.y / gridDim.y, end = groups * (blockIdx.y + 1) / gridDim.y;
    uint4 x[kBatch];
    auto load = [&](int from) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int at = from + i;
            x[i] = make_uint4(0, 0, 0, 0);
            if (at >= end) continue;
            const bool query = at < q_groups, value = at >= q_groups + kv_groups;
            const int head = (query ? at : at - q_groups - (value ? kv_groups : 0)) * kHeads + sub;
            if (head >= (query ? c.hq : ge.hkv)) continue;
            const __half* p = query ? c.q + t * c.q_stride : (value ? c.v : c.k) + t * c.row_stride;
            x[i] = *(reinterpret_cast<const uint4*>(p + (long long)head * D) + lane);
        }
    };
    load(first);  // in flight while the token's place is looked up
    const int b = find_seq_warp(c.offsets, c.num_seqs, t);
    if (b < 0) return;
    const long long pos = (long long)__ldg(c.lens + b) - __ldg(c.offsets + b + 1) + t;
    const bool past = c.rotary && pos >= c.num_positions, placed = pos >= 0 && !past;
    if (past && threadIdx.x % 32 == 0) report_dev_error(kDevBadPage);
    const long long page = placed && end > q_groups ? page_offset(pg, b, pos, ge.page_shift) : -1;
    const int row = (int)(pos & (ge.page() - 1)), part = c.rotary >> 4;
    float2 turn[8];
    if (part && placed && lane < 2 * part) {
        const float4* at = reinterpret_cast<const float4*>(c.turns + pos * (c.rotary / 2)) + (lane < part ? lane : lane - part) * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) *reinterpret_cast<float4*>(&turn[2 * j]) = __ldg(at + j);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) turn[j] = make_float2(0.0f, 0.0f);
    }
    const uint4 none = make_uint4(0, 0, 0, 0);
    const uint4 q_weight = c.q_weight ? __ldg(reinterpret_cast<const uint4*>(c.q_weight) + lane) : none;
    const uint4 k_weight = c.k_weight ? __ldg(reinterpret_cast<const uint4*>(c.k_weight) + lane) : none;
    for (int from = first; from < end; from += kBatch) {
        if (from != first) load(from);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int at = from + i;
            if (at >= end) break;
            if (at < q_groups) {
                const int head = at * kHeads + sub;
                uint4 y = norm_and_turn<D>(x[i], c.q_weight != nullptr, q_weight, c.eps, turn, part, lane);
                if (!placed) y = none;
                if (head < c.hq) reinterpret_cast<uint4*>(c.out + t * c.out_stride + (long long)head * D)[lane] = y;
                continue;
            }
            const bool value = at >= q_groups + kv_groups;
            const int head = (at - q_groups - (value ? kv_groups : 0)) * kHeads + sub;
            uint4 y = x[i];
            if (!value) y = norm_and_turn<D>(y, c.k_weight != nullptr, k_weight, c.eps, turn, part, lane);
            uint8_t* block = page < 0 || head >= ge.hkv
                                 ? nullptr
                                 : pg.pool + page + (long long)head * ge.block_bytes() + (value ? ge.v_codes() : 0);
            quantise_row<D>(y, block, row, lane, ge);
        }
    }
}

}  // namespace

int launch_rope_table(float theta, int half, long long positions, float* table, cudaStream_t st) {
    const long long n = positions * half;
    return launch_k(rope_table_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, (double)theta, half, n,
                    reinterpret_cast<float2*>(table)) == cudaSuccess
               ? 0
               : -1;
}

int launch_rope_append(const RopeCall& c, const Pages& pg, const Geom& ge, cudaStream_t st) {
    // many tokens: a warp takes all heads of one; few: its heads are shared by several, down to one batch of loads
    // each, until there are about two blocks for each SM
    const int heads = 256 / ge.d, groups = (c.hq + heads - 1) / heads + 2 * ((ge.hkv + heads - 1) / heads);
    const long long blocks = ((long long)c.num_tokens + kWarps - 1) / kWarps;
    const long long shares = std::min<long long>((groups + kBatch - 1) / kBatch, std::max<long long>(1, 2 * kNumSMs / blocks));
    auto kernel = ge.d == 64    ? kv4_rope_append_kernel<64>
                  : ge.d == 128 ? kv4_rope_append_kernel<128>
                                : kv4_rope_append_kernel<256>;
    return launch_k(kernel, dim3((unsigned)blocks, (unsigned)shares), dim3(kRopeThreads), 0, st, c, pg, ge) == cudaSuccess ? 0 : -1;
}

}  // namespace kv4
}  // namespace cb
