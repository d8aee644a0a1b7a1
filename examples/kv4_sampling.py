"""Several samples of one prompt over the 4-bit paged KV cache (cactus_b200/kv4.py).

A small decoder with random weights prefills a prompt in chunks, forks it into samples that share its
pages, decodes them as one batch, drops half of them, lets the others slide to a window with a few
first rows kept, and goes on. It prints the pages in use at each stage and how far the attention over
4-bit keys and values is from fp16 attention on the same activations.

    python examples/kv4_sampling.py [--prompt 700] [--samples 4] [--steps 40]
"""
import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from cactus_b200.kv4 import KVCache4  # noqa: E402

LAYERS, HIDDEN, HQ, HKV, D, VOCAB, CHUNK = 4, 512, 8, 4, 64, 1000, 256


class Decoder:
    """Attention-only decoder layers: normalise, q k v, attention over the cache, output, residual."""

    def __init__(self, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        mat = lambda *s: (torch.randn(s, generator=g, device="cuda") / math.sqrt(s[0])).half()  # noqa: E731
        self.embed = torch.randn((VOCAB, HIDDEN), generator=g, device="cuda").half()
        self.qkv = [mat(HIDDEN, (HQ + 2 * HKV) * D) for _ in range(LAYERS)]
        self.out = [mat(HQ * D, HIDDEN) for _ in range(LAYERS)]

    def forward(self, cache, seqs, tokens, shadow=None):
        """tokens: a list of new token ids for each sequence. Returns the last logits of each and, where
        `shadow` (fp16 keys and values of each layer and sequence) is kept, the attention's error."""
        counts = [len(t) for t in tokens]
        cache.begin(seqs, counts)
        x = self.embed[torch.tensor(sum(tokens, []), device="cuda")]
        error = 0.0
        for layer in range(LAYERS):
            h = x.float()
            h = (h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6)).half()
            qkv = h @ self.qkv[layer]  # q | k | v of each token: the cache reads them where they are
            k, v = qkv[:, HQ * D:], qkv[:, (HQ + HKV) * D:]
            cache.append(layer, k.data_ptr(), v.data_ptr(), row_stride=qkv.shape[1])
            out = torch.empty((x.shape[0], HQ * D), dtype=torch.float16, device="cuda")
            cache.attention(layer, qkv, out, 1.0 / math.sqrt(D), query_stride=qkv.shape[1])
            if shadow is not None:
                error = max(error, self._check(shadow, layer, seqs, counts, qkv, out))
            x = x + out @ self.out[layer]
        ends = torch.tensor(counts, device="cuda").cumsum(0) - 1
        return (x[ends].float() @ self.embed.float().T) / math.sqrt(HIDDEN), error

    @staticmethod
    def _check(shadow, layer, seqs, counts, qkv, out):
        worst, at = 0.0, 0
        for s, n in zip(seqs, counts):
            rows = qkv[at:at + n].float()
            k, v = (rows[:, i:i + HKV * D].reshape(n, HKV, D) for i in (HQ * D, (HQ + HKV) * D))
            old = shadow.get((layer, s))
            k, v = (k, v) if old is None else (torch.cat([old[0], k]), torch.cat([old[1], v]))
            shadow[layer, s] = (k, v)
            q = rows[:, :HQ * D].reshape(n, HQ, D)
            score = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(HQ // HKV, 1)) / math.sqrt(D)
            pos = torch.arange(k.shape[0], device="cuda")
            score = score.masked_fill(pos > pos[-n:, None], -math.inf)
            ref = torch.einsum("hqk,khd->qhd", score.softmax(-1), v.repeat_interleave(HQ // HKV, 1)).reshape(n, -1)
            worst = max(worst, float((out[at:at + n].float() - ref).norm() / ref.norm()))
            at += n
        return worst


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--prompt", type=int, default=700)
    ap.add_argument("--samples", type=int, default=4)
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args(argv)
    torch.manual_seed(a.seed)
    model = Decoder(a.seed)
    cache = KVCache4(LAYERS, HQ, HKV, D, num_pages=256, max_seqs=a.samples, max_context=2048, max_tokens=CHUNK,
                     group_size=32, page_size=16)
    used = lambda: cache.info()["pages"] - cache.info()["free_pages"]  # noqa: E731

    prompt = torch.randint(VOCAB, (a.prompt,)).tolist()
    shadow, error = {}, 0.0
    for at in range(0, a.prompt, CHUNK):
        logits, e = model.forward(cache, [0], [prompt[at:at + CHUNK]], shadow)
        error = max(error, e)
    print(f"prompt of {a.prompt} rows: {used()} pages, attention within {error:.3f} of fp16 keys and values")

    samples = list(range(a.samples))
    cache.fork([0] * (a.samples - 1), samples[1:])
    for (layer, s) in list(shadow):
        for t in samples[1:]:
            shadow[layer, t] = shadow[layer, s]
    shared = used()
    logits = logits.expand(a.samples, -1)
    texts = [[] for _ in samples]
    for _ in range(a.steps):
        step = torch.multinomial(logits.softmax(-1), 1)[:, 0].tolist()
        for t, s in zip(step, samples):
            texts[s].append(t)
        logits, e = model.forward(cache, samples, [[t] for t in step], shadow)
        error = max(error, e)
    print(f"{a.samples} samples of {a.steps} tokens: {used()} pages ({shared} when forked), within {error:.3f}")

    kept = samples[: max(1, a.samples // 2)]
    cache.free([s for s in samples if s not in kept])
    cache.slide(kept, sink=4, window=128)
    print(f"{len(kept)} samples kept, their caches at 128 rows: {used()} pages")
    logits = logits[: len(kept)]
    for _ in range(8):
        step = torch.multinomial(logits.softmax(-1), 1)[:, 0].tolist()
        for t, s in zip(step, kept):
            texts[s].append(t)
        logits, _ = model.forward(cache, kept, [[t] for t in step])
    print(f"8 tokens more: lengths {[cache.length(s) for s in kept]}, {used()} pages; sample 0 ends {texts[0][-8:]}")
    cache.free(kept)
    torch.cuda.synchronize()
    assert used() == 0
    cache.close()
    return error


if __name__ == "__main__":
    main()
