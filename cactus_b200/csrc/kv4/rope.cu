// The append of the 4-bit paged KV cache that normalises and rotates on the way, and the table of turns
// that it reads. A warp takes a token's heads one group after another, 32 * 8 / D heads at a time: D / 8 lanes
// share a head's row (8 elements, one 16-byte load each), and the token's turns stay in registers for all of
// them. Shuffles add up the squares of the norm, fetch the other element of each rotated pair and reduce a
// group's ends for the quantisation. Each element is read and written once. 65 thousand prompt rows of 24 query heads, 8 key
// heads and 8 of values, of 64, take 126 us, 4.5 TB/s (a block a head and 32 rows took 300). Neither HBM nor the issue slots
// (68 %) are full then: 24 warps a SM, of 80 registers and some words spilled, wait for their loads first.
#include <type_traits>

#include "kv4.cuh"
#include "kv4_ops.h"
#include "quantise.cuh"

namespace cb {
namespace kv4 {

namespace {

constexpr int kRopeThreads = 128;

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

// The sum of a row's squares, eight of them a lane: the halves of the row are added to one another, element by
// element, then the halves of that; at D = 128 after four neighbours each, at D = 256 after the first halves and four
// neighbours each. Any fixed order would be as close to the 64-bit sum. This one, another for each D, is that of the plain form's row means (PyTorch in fp32 on this GPU,
// found by trying orders out), and with rsqrtf as its root a normalised key has the plain form's bits: a code next to the
// border of two does not differ between the two. That equality is no evidence of exactness; the bound is against 64 bits.
// Every lane has its share, as each exchange passes on the part that the lane does not keep.
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

// Eight elements' codes, and step and low of their group (G / 8 lanes share one; all lanes take part): the
// parameters as they are stored.
template <int G>
__device__ __forceinline__ uint32_t quantise_eight(const uint4& x, __half2* pair) {
    const __half2* h = reinterpret_cast<const __half2*>(&x);
    // (largest, -smallest): exact in fp16, and a NaN stays one
    const __half2 hi2 = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    const __half2 lo2 = __hmin2_nan(__hmin2_nan(h[0], h[1]), __hmin2_nan(h[2], h[3]));
    __half2 ends = __hmax2_nan(__lows2half2(hi2, __hneg2(lo2)), __highs2half2(hi2, __hneg2(lo2)));
#pragma unroll
    for (int o = 1; o < G / 8; o <<= 1) ends = __hmax2_nan(ends, __shfl_xor_sync(0xffffffffu, ends, o));
    const float hi = __low2float(ends), lo = -__high2float(ends);
    const __half step = step_of(hi, lo);
    const float fs = __half2float(step);
    const bool bad = !(__fsub_rn(hi, lo) < INFINITY);  // an infinity or a NaN in the group
    uint32_t w = 0;
    if (!bad && fs > 0.0f) w = quant_codes(h, lo, fs);
    const __half nan = __ushort_as_half(0x7FFF);
    *pair = bad ? __halves2half2(nan, nan) : __halves2half2(step, __float2half_rn(lo));
    return w;
}

// Block (x, y): tokens kWarps x .., one a warp, and the y-th share of its heads. Units of work, each with kBatch
// loads in flight: kBatch groups of query heads, or kBatch / 2 groups of key heads and their values.
constexpr int kWarps = kRopeThreads / 32, kBatch = 4;

__host__ __device__ inline int units_of(int heads, int a_group, int groups) { return (heads + a_group * groups - 1) / (a_group * groups); }

template <int D, int G, bool ALL>
__global__ void __launch_bounds__(kRopeThreads, 6) kv4_rope_append_kernel(RopeCall c, Pages pg, Geom ge) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int kLanes = D / 8, kHeads = 32 / kLanes;
    const int lane = threadIdx.x % kLanes, sub = (threadIdx.x & 31) / kLanes;
    const int t = blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (t >= c.num_tokens) return;
    const int q_units = units_of(c.hq, kHeads, kBatch), units = q_units + units_of(ge.hkv, kHeads, kBatch / 2);
    const int first = units * blockIdx.y / gridDim.y, end = units * (blockIdx.y + 1) / gridDim.y;
    const int in_row = sub * D + lane * 8;
    const __half* q = c.q + t * c.q_stride + in_row;
    const __half* k = c.k + t * c.row_stride + in_row;
    const long long to_v = c.v - c.k;
    uint4 x[kBatch];
    auto load_q = [&](int unit) {
        const int head = unit * kBatch * kHeads;
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (head + i * kHeads + sub < c.hq) x[i] = *reinterpret_cast<const uint4*>(q + (head + i * kHeads) * D);
    };
    auto load_kv = [&](int unit) {
        const int head = (unit - q_units) * (kBatch / 2) * kHeads;
#pragma unroll
        for (int i = 0; i < kBatch / 2; ++i)
            if (head + i * kHeads + sub < ge.hkv) {
                const __half* at = k + (head + i * kHeads) * D;
                x[2 * i] = *reinterpret_cast<const uint4*>(at);
                x[2 * i + 1] = *reinterpret_cast<const uint4*>(at + to_v);
            }
    };
#pragma unroll
    for (int i = 0; i < kBatch; ++i) x[i] = make_uint4(0, 0, 0, 0);  // heads that are none are computed all the same
    if (first < q_units) load_q(first); else load_kv(first);  // in flight while the token's place is looked up
    const int b = find_seq_warp(c.offsets, c.num_seqs, t);
    if (b < 0) return;
    const long long pos = (long long)__ldg(c.lens + b) - __ldg(c.offsets + b + 1) + t;
    __half* out = c.out + t * c.out_stride + in_row;
    if (pos < 0 || (c.rotary && pos >= c.num_positions)) {  // no place to turn to
        if (pos >= 0 && threadIdx.x % 32 == 0) report_dev_error(kDevBadPage);
        for (int head = first * kBatch * kHeads; head < min(end, q_units) * kBatch * kHeads; head += kHeads)
            if (head + sub < c.hq) *reinterpret_cast<uint4*>(out + head * D) = make_uint4(0, 0, 0, 0);
        return;
    }
    const int part = c.rotary >> 4;
    float2 turn[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) turn[j] = make_float2(0.0f, 0.0f);
    if (ALL || lane < 2 * part) {
        const bool upper = lane >= part;
        const float4* at = reinterpret_cast<const float4*>(c.turns + pos * (c.rotary / 2)) + (upper ? lane - part : lane) * 4;
        const float sign = upper ? 1.0f : -1.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4 two = __ldg(at + j);
            turn[2 * j] = make_float2(two.x, sign * two.y);
            turn[2 * j + 1] = make_float2(two.z, sign * two.w);
        }
    }
    int unit = first;
    auto queries = [&](auto norm, const uint4& weight) {
        for (; unit < min(end, q_units); ++unit) {
            if (unit != first) load_q(unit);
            const int head = unit * kBatch * kHeads;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const uint4 y = norm_and_turn<D, ALL, decltype(norm)::value>(x[i], weight, c.eps, turn, part, lane);
                if (head + i * kHeads + sub < c.hq) *reinterpret_cast<uint4*>(out + (head + i * kHeads) * D) = y;
            }
        }
    };
    if (unit < q_units) {
        if (c.q_weight) queries(std::true_type{}, __ldg(reinterpret_cast<const uint4*>(c.q_weight) + lane));
        else queries(std::false_type{}, make_uint4(0, 0, 0, 0));
    }
    if (unit >= end) return;
    const long long page = page_offset(pg, b, pos, ge.page_shift);
    if (page < 0) return;
    constexpr int kPerGroup = G / 8, kGroups = D / G;
    const int row = (int)(pos & (ge.page() - 1));
    // of the warp's first head: the lane's codes and, where it leads its group, its parameters
    uint8_t* block = pg.pool + page + (long long)sub * ge.block_bytes();
    uint8_t* codes = block + row * (D / 2) + lane * 4;
    uint8_t* pair = block + ge.k_params() + (row * kGroups + lane / kPerGroup) * 4;
    const bool leads = lane % kPerGroup == 0;
    auto keys = [&](auto norm, const uint4& weight) {
        for (; unit < end; ++unit) {
            if (unit != first) load_kv(unit);
#pragma unroll
            for (int i = 0; i < kBatch / 2; ++i) {
                const int head = ((unit - q_units) * (kBatch / 2) + i) * kHeads;
                if (head >= ge.hkv) break;
                const bool live = head + sub < ge.hkv;
                const int at = head * ge.block_bytes();
                const uint4 y = norm_and_turn<D, ALL, decltype(norm)::value>(x[2 * i], weight, c.eps, turn, part, lane);
                __half2 kp, vp;
                const uint32_t kw = quantise_eight<G>(y, &kp), vw = quantise_eight<G>(x[2 * i + 1], &vp);
                if (live) {
                    *reinterpret_cast<uint32_t*>(codes + at) = kw;
                    *reinterpret_cast<uint32_t*>(codes + at + ge.v_codes()) = vw;
                    if (leads) {
                        *reinterpret_cast<__half2*>(pair + at) = kp;
                        *reinterpret_cast<__half2*>(pair + at + ge.v_codes()) = vp;
                    }
                }
            }
        }
    };
    if (c.k_weight) keys(std::true_type{}, __ldg(reinterpret_cast<const uint4*>(c.k_weight) + lane));
    else keys(std::false_type{}, make_uint4(0, 0, 0, 0));
}

template <int D, int G>
cudaError_t launch_group(const RopeCall& c, const Pages& pg, const Geom& ge, dim3 grid, cudaStream_t st) {
    auto kernel = c.rotary == D ? kv4_rope_append_kernel<D, G, true> : kv4_rope_append_kernel<D, G, false>;
    return launch_k(kernel, grid, dim3(kRopeThreads), 0, st, c, pg, ge);
}
template <int D>
cudaError_t launch_dim(const RopeCall& c, const Pages& pg, const Geom& ge, cudaStream_t st) {
    // Many tokens: a warp takes all heads of one. Few: each of its units is a warp's. A warp a token / a unit, us: heads of
    // 64, one token 6.7 / 4.1, 64 tokens 8.3 / 5.7, 1152 9.3 / 7.2, 2368 10.3 / 11.3; of 128 1152 11.3 / 10.0, 2368 12.9 / 14.9; of
    // 256 1152 6.7 / 5.8, 2368 7.7 / 8.8.
    constexpr int kHeads = 256 / D;
    const int units = units_of(c.hq, kHeads, kBatch) + units_of(ge.hkv, kHeads, kBatch / 2);
    const unsigned blocks = ((unsigned)c.num_tokens + kWarps - 1) / kWarps;
    const dim3 grid(blocks, blocks <= 2 * kNumSMs ? (unsigned)units : 1u);
    if (ge.g == 32) return launch_group<D, 32>(c, pg, ge, grid, st);
    if (ge.g == 64) return launch_group<D, 64>(c, pg, ge, grid, st);
    if constexpr (D >= 128) return launch_group<D, 128>(c, pg, ge, grid, st);
    return cudaErrorInvalidValue;
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
    const cudaError_t e = ge.d == 64    ? launch_dim<64>(c, pg, ge, st)
                          : ge.d == 128 ? launch_dim<128>(c, pg, ge, st)
                                        : launch_dim<256>(c, pg, ge, st);
    return e == cudaSuccess ? 0 : -1;
}

}  // namespace kv4
}  // namespace cb
