// Attention over the 4-bit paged KV cache: which kernel takes a call.
#include "attention.cuh"

namespace cb {
namespace kv4 {

namespace {

constexpr int kWarps = 4;

// One warp per (token, q head).
template <int D>
__global__ void __launch_bounds__(kWarps * 32) kv4_attn_rows_kernel(const __grid_constant__ AttnCall c, const __grid_constant__ Pages pg, const __grid_constant__ Geom ge) {
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * kWarps + warp;
    const int t = (int)(item / c.hq), h = (int)(item % c.hq);
    if (t >= c.num_tokens) return;
    const int b = find_seq(c.offsets, c.num_seqs, t);
    if (b < 0) return;
    if (t - c.offsets[b] >= c.max_q || c.lens[b] > (pg.table_stride << ge.page_shift)) report_dev_error(kDevBadPage);
    if (t - c.offsets[b] < c.max_q) attention_row<D>(c, pg, ge, b, t, h, lane);
}

}  // namespace

size_t attention_workspace(int num_seqs, int num_tokens, int hq, int hkv, int) {
    return decode_workspace(num_seqs, num_tokens, hq, hkv);
}

int launch_attention(const AttnCall& c, const Pages& pg, const Geom& ge, cudaStream_t st) {
    if (c.max_q * (c.hq / ge.hkv) <= 32) return launch_decode(c, pg, ge, st);
    const long long items = (long long)c.num_tokens * c.hq;
    const dim3 grid((unsigned)((items + kWarps - 1) / kWarps));
    auto kernel =
        ge.d == 64 ? kv4_attn_rows_kernel<64> : ge.d == 128 ? kv4_attn_rows_kernel<128> : kv4_attn_rows_kernel<256>;
    return launch_k(kernel, grid, dim3(kWarps * 32), 0, st, c, pg, ge) == cudaSuccess ? 0 : -1;
}

}  // namespace kv4
}  // namespace cb
