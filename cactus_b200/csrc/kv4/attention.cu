// Attention over the 4-bit paged KV cache: which kernel takes which sequences.
#include "kv4.cuh"
#include "kv4_ops.h"

namespace cb {
namespace kv4 {

namespace {
// Sequences with up to so many q rows a kv head (tokens times the heads that share it) go to the
// kernel for few queries, which reads the keys once for 16 rows, the others to the one for many, which
// does for 256. Over 8000 rows, 16 / 8 heads of 128: 32 q rows of 12 sequences 123 us there and 139
// here, 48 rows 172 and 140; one sequence alone 32 rows 32 and 47, 64 rows 40 and 43.
constexpr int kFewRows = 32;
}  // namespace

size_t attention_workspace(int num_seqs, int num_tokens, int hq, int hkv, int) {
    const size_t counters = decode_counters(num_seqs, num_tokens, hq, hkv);
    return kPartBytes + ((counters > (size_t)kPrefillParts ? counters : (size_t)kPrefillParts) * 4 + 15) / 16 * 16;
}

int launch_attention(const AttnCall& c, const Pages& pg, const Geom& ge, cudaStream_t st) {
    if ((long long)c.max_q * (c.hq / ge.hkv) <= kFewRows) return launch_decode(c, pg, ge, kFewRows, st);
    // sequences of both kinds may be there unless all are as long as the longest
    if ((long long)c.num_seqs * c.max_q > c.num_tokens) {
        const int rc = launch_decode(c, pg, ge, kFewRows, st);
        if (rc) return rc;
    }
    return launch_prefill(c, pg, ge, kFewRows + 1, st);
}

}  // namespace kv4
}  // namespace cb
