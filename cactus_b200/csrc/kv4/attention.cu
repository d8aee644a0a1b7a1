// Attention over the 4-bit paged KV cache: which kernel takes which sequences.
#include "kv4.cuh"
#include "kv4_ops.h"

namespace cb {
namespace kv4 {

namespace {
// Sequences with up to so many q rows a kv head (tokens times the heads that share it) go to the
// kernel for few queries, which unpacks the keys once for 16 rows (8 at head_dim 256), the others to the
// one for many, which does once for 256 (128). Measured over 8000 rows, times in us of the one for few
// and the one for many. 12 sequences, heads of 128, 8 kv heads: 16 rows 72 and 110, 32 rows 117 and 111,
// 48 rows 163 and 110 (one sequence 32 rows 31 and 39, 48 rows 35 and 44, 64 rows 40 and 40). Heads of 64,
// 8 kv heads: 32 rows 73 and 96, 48 rows 100 and 97, 64 rows 128 and 97. Heads of 256, 4 kv heads: 16 rows
// 89 and 89, 32 rows 149 and 91; but where there are few sequences and kv heads, which the one for many
// does not split so far: 1 kv head 24 rows 46 and 63, 32 rows 54 and 54.
int few_rows(const AttnCall& c, const Geom& ge) {
    if (ge.d == 64) return 48;
    if (ge.d == 128) return 32;
    return (long long)c.num_seqs * ge.hkv >= 32 ? 16 : 32;
}
}  // namespace

size_t attention_workspace(int num_seqs, int num_tokens, int hq, int hkv, int) {
    const size_t counters = decode_counters(num_seqs, num_tokens, hq, hkv);
    return kPartBytes + ((counters > (size_t)kPrefillParts ? counters : (size_t)kPrefillParts) * 4 + 15) / 16 * 16;
}

int launch_attention(const AttnCall& c, const Pages& pg, const Geom& ge, cudaStream_t st) {
    const int few = few_rows(c, ge);
    if ((long long)c.max_q * (c.hq / ge.hkv) <= few) return launch_decode(c, pg, ge, few, few, st);
    // The counts are on the device, and there may be fewer tokens than the call has room for. Where all
    // sequences may be as long as the longest, the kernel for many takes every one, also those that turn out
    // short, and a batch of equal prompts needs no launch that finds nothing to do.
    if ((long long)c.num_seqs * c.max_q <= c.num_tokens) return launch_prefill(c, pg, ge, 1, st);
    // sequences of both kinds may be there; a prompt's chunk among single tokens is the usual case, so the
    // others' mean says how large a tile of rows they need. 256 tokens among 63 single ones over 4096 rows, 2
    // heads of 128 to each of 8 kv heads: 148 us, 194 with the tile of 16 rows; among 127 over 1024 rows, 4
    // heads of 64 to each: 74 and 91
    const long long others = (long long)(c.num_tokens - c.max_q) * (c.hq / ge.hkv);
    const int rc = launch_decode(c, pg, ge, few, c.num_seqs > 1 && others <= 8LL * (c.num_seqs - 1) ? 8 : few, st);
    return rc ? rc : launch_prefill(c, pg, ge, few + 1, st);
}

}  // namespace kv4
}  // namespace cb
