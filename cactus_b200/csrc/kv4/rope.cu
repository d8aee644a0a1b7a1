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

// Eight elements of a row of D, normalised (where NORM) and turned, as fp16. turn: the lane's (cos, -sin) for elements of
// the first half and (cos, sin) for those of the second, so that both are v cos + u sin with the pair's other element
// u; `part` lanes have each half. ALL: the whole row turns.
template <int D, bool ALL, bool NORM>
__device__ __forceinline__ uint4 norm_and_turn(const uint4& in, const uint4& weight, float eps, const float2 (&turn)[8],
                                               int part, int lane) {
    const unsigned full = 0xffffffffu;
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 p = __half22float2(reinterpret_cast<const __half2*>(&in)[j]);
        v[2 * j] = p.x;
        v[2 * j + 1] = p.y;
    }
    if (NORM) {
        const float inv = rsqrtf(__fadd_rn(__fmul_rn(sum_of_squares<D>(v, lane), 1.0f / D), eps));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 p = __half22float2(reinterpret_cast<const __half2*>(&weight)[j]);
            v[2 * j] = __fmul_rn(__fmul_rn(v[2 * j], inv), p.x);
            v[2 * j + 1] = __fmul_rn(__fmul_rn(v[2 * j + 1], inv), p.y);
        }
    }
    if (ALL) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = __fadd_rn(__fmul_rn(v[j], turn[j].x), __fmul_rn(__shfl_xor_sync(full, v[j], D / 16), turn[j].y));
    } else if (part) {
        const bool turned = lane < 2 * part;
        const int from = (threadIdx.x & 31) + (lane < part ? part : turned ? -part : 0);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float w = __fadd_rn(__fmul_rn(v[j], turn[j].x), __fmul_rn(__shfl_sync(full, v[j], from), turn[j].y));
            if (turned) v[j] = w;
        }
    }
    uint4 out;
#pragma unroll
    for (int j = 0; j < 4; ++j) reinterpret_cast<__half2*>(&out)[j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
    return out;
}

// Eight elements of a row into its block: codes, and the parameters of their group. All lanes take part; `codes` and
// `pair` are where the lane's go, null where nothing does.
__device__ __forceinline__ void quantise_eight(const uint4& x, uint8_t* codes, uint8_t* pair, int per_group) {
    const unsigned full = 0xffffffffu;
    const __half2* h = reinterpret_cast<const __half2*>(&x);
    // (largest, -smallest): exact in fp16, and a NaN stays one
    const __half2 hi2 = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    const __half2 lo2 = __hmin2_nan(__hmin2_nan(h[0], h[1]), __hmin2_nan(h[2], h[3]));
    __half2 ends = __hmax2_nan(__lows2half2(hi2, __hneg2(lo2)), __highs2half2(hi2, __hneg2(lo2)));
    ends = __hmax2_nan(ends, __shfl_xor_sync(full, ends, 1));
    ends = __hmax2_nan(ends, __shfl_xor_sync(full, ends, 2));
    if (per_group > 4) ends = __hmax2_nan(ends, __shfl_xor_sync(full, ends, 4));
    if (per_group > 8) ends = __hmax2_nan(ends, __shfl_xor_sync(full, ends, 8));
    const float hi = __low2float(ends), lo = -__high2float(ends);
    const __half step = step_of(hi, lo);
    const float fs = __half2float(step);
    const bool bad = !(__fsub_rn(hi, lo) < INFINITY);  // an infinity or a NaN in the group
    uint32_t w = 0;
    if (!bad && fs > 0.0f) w = quant_codes(h, lo, fs);
    if (codes) *reinterpret_cast<uint32_t*>(codes) = w;
    if (pair) {
        const __half nan = __ushort_as_half(0x7FFF);
        *reinterpret_cast<__half2*>(pair) = bad ? __halves2half2(nan, nan) : __halves2half2(step, __float2half_rn(lo));
    }
}

// Block (x, y): tokens kWarps x .., one a warp, and the y-th share of its heads. Units of work, each with kBatch
// loads in flight: kBatch groups of query heads, or kBatch / 2 groups of key heads and their values.
constexpr int kWarps = kRopeThreads / 32, kBatch = 4;

__host__ __device__ inline int units_of(int heads, int a_group, int groups) { return (heads + a_group * groups - 1) / (a_group * groups); }

template <int D, bool ALL>
__global__ void __launch_bounds__(kRopeThreads, 3) kv4_rope_append_kernel(RopeCall c, Pages pg, Geom ge) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int kLanes = D / 8, kHeads = 32 / kLanes;
    const int lane = threadIdx.x % kLanes, sub = (threadIdx.x & 31) / kLanes;
    const int t = blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (t >= c.num_tokens) return;
    const int q_units = units_of(c.hq, kHeads, kBatch), units = q_units + units_of(ge.hkv, kHeads, kBatch / 2);
    const int first = units * blockIdx.y / gridDim.y, end = units * (blockIdx.y + 1) / gridDim.y;
    const __half* q = c.q + t * c.q_stride + sub * D + lane * 8;
    const __half* k = c.k + t * c.row_stride + sub * D + lane * 8;
    const __half* v = c.v + t * c.row_stride + sub * D + lane * 8;
    uint4 x[kBatch];
    auto load = [&](int unit) {
        if (unit < q_units) {
            const int head = unit * kBatch * kHeads;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                x[i] = make_uint4(0, 0, 0, 0);
                if (head + i * kHeads + sub < c.hq) x[i] = *reinterpret_cast<const uint4*>(q + (head + i * kHeads) * D);
            }
        } else {
            const int head = (unit - q_units) * (kBatch / 2) * kHeads;
#pragma unroll
            for (int i = 0; i < kBatch / 2; ++i) {
                x[2 * i] = x[2 * i + 1] = make_uint4(0, 0, 0, 0);
                if (head + i * kHeads + sub < ge.hkv) {
                    x[2 * i] = *reinterpret_cast<const uint4*>(k + (head + i * kHeads) * D);
                    x[2 * i + 1] = *reinterpret_cast<const uint4*>(v + (head + i * kHeads) * D);
                }
            }
        }
    };
    load(first);  // in flight while the token's place is looked up
    const int b = find_seq_warp(c.offsets, c.num_seqs, t);
    if (b < 0) return;
    const long long pos = (long long)__ldg(c.lens + b) - __ldg(c.offsets + b + 1) + t;
    const bool past = c.rotary && pos >= c.num_positions, placed = pos >= 0 && !past;
    if (past && threadIdx.x % 32 == 0) report_dev_error(kDevBadPage);
    const int part = c.rotary >> 4;
    float2 turn[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) turn[j] = make_float2(0.0f, 0.0f);
    if (part && placed && (ALL || lane < 2 * part)) {
        const bool upper = lane >= part;
        const float4* at = reinterpret_cast<const float4*>(c.turns + pos * (c.rotary / 2)) + (upper ? lane - part : lane) * 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            *reinterpret_cast<float4*>(&turn[2 * j]) = __ldg(at + j);
            if (!upper) turn[2 * j].y = -turn[2 * j].y, turn[2 * j + 1].y = -turn[2 * j + 1].y;
        }
    }
    const uint4 none = make_uint4(0, 0, 0, 0);
    int unit = first;
    if (unit < q_units) {
        const bool norm = c.q_weight != nullptr;
        const uint4 weight = norm ? __ldg(reinterpret_cast<const uint4*>(c.q_weight) + lane) : none;
        __half* out = c.out + t * c.out_stride + sub * D + lane * 8;
        for (; unit < min(end, q_units); ++unit) {
            if (unit != first) load(unit);
            const int head = unit * kBatch * kHeads;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                if (head + i * kHeads >= c.hq) break;
                uint4 y = norm ? norm_and_turn<D, ALL, true>(x[i], weight, c.eps, turn, part, lane)
                               : norm_and_turn<D, ALL, false>(x[i], weight, c.eps, turn, part, lane);
                if (!placed) y = none;
                if (head + i * kHeads + sub < c.hq) *reinterpret_cast<uint4*>(out + (head + i * kHeads) * D) = y;
            }
        }
    }
    if (unit >= end) return;
    const long long page = placed ? page_offset(pg, b, pos, ge.page_shift) : -1;
    if (page < 0) return;
    const bool norm = c.k_weight != nullptr;
    const uint4 weight = norm ? __ldg(reinterpret_cast<const uint4*>(c.k_weight) + lane) : none;
    const int row = (int)(pos & (ge.page() - 1)), per_group = ge.g >> 3;
    const bool leads = (lane & (per_group - 1)) == 0;
    // of the warp's first head: the lane's codes and, where it leads its group, its parameters
    uint8_t* codes = pg.pool + page + (long long)sub * ge.block_bytes() + row * (D / 2) + lane * 4;
    uint8_t* pair = pg.pool + page + (long long)sub * ge.block_bytes() + ge.k_params() +
                    (row * ge.ng() + (lane >> (__ffs(per_group) - 1))) * 4;
    for (; unit < end; ++unit) {
        if (unit != first) load(unit);
#pragma unroll
        for (int i = 0; i < kBatch / 2; ++i) {
            const int head = ((unit - q_units) * (kBatch / 2) + i) * kHeads;
            if (head >= ge.hkv) break;
            const bool live = head + sub < ge.hkv;
            const long long at = (long long)head * ge.block_bytes();
            const uint4 y = norm ? norm_and_turn<D, ALL, true>(x[2 * i], weight, c.eps, turn, part, lane)
                                 : norm_and_turn<D, ALL, false>(x[2 * i], weight, c.eps, turn, part, lane);
            quantise_eight(y, live ? codes + at : nullptr, live && leads ? pair + at : nullptr, per_group);
            quantise_eight(x[2 * i + 1], live ? codes + at + ge.v_codes() : nullptr,
                           live && leads ? pair + at + ge.v_codes() : nullptr, per_group);
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
    // many tokens: a warp takes all heads of one; few: its units are dealt out to several, until there are about two
    // blocks for each SM
    const int heads = 256 / ge.d, units = units_of(c.hq, heads, kBatch) + units_of(ge.hkv, heads, kBatch / 2);
    const long long blocks = ((long long)c.num_tokens + kWarps - 1) / kWarps;
    const long long shares = std::min<long long>(units, std::max<long long>(1, 2 * kNumSMs / blocks));
    const bool all = c.rotary == ge.d;
    auto kernel = ge.d == 64    ? (all ? kv4_rope_append_kernel<64, true> : kv4_rope_append_kernel<64, false>)
                  : ge.d == 128 ? (all ? kv4_rope_append_kernel<128, true> : kv4_rope_append_kernel<128, false>)
                                : (all ? kv4_rope_append_kernel<256, true> : kv4_rope_append_kernel<256, false>);
    return launch_k(kernel, dim3((unsigned)blocks, (unsigned)shares), dim3(kRopeThreads), 0, st, c, pg, ge) == cudaSuccess ? 0 : -1;
}

}  // namespace kv4
}  // namespace cb
