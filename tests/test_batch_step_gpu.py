"""The operators of a ragged batch together, as a decoder's layers use them over the 4-bit cache: residual and
RMSNorm into 8 bits, the INT8 projection with each request's adapter beside it, the append that normalises and
turns, attention, and the penalties and masks on the last logits.

The statement in 64 bits takes the codes and the cached rows that the library made (each checked by its own tests),
so that what is compared is how the parts fit: rows, strides, positions, adapters, scales."""
import math

import numpy as np
import pytest

import cactus_b200 as cb
from cactus_b200 import batch, kv4
from tests import batch_util as B
from tests import kv4_util as U
from tests.gpu_util import dev, empty, host, torch

pytestmark = pytest.mark.gpu

HIDDEN, HQ, HKV, D, VOCAB, RANK, G = 256, 4, 2, 64, 1003, 16, 32
QKV = (HQ + 2 * HKV) * D


def _int8(rng, n, k):
    """INT8 weights [n, k] in groups of G, their fp16 scales, and what they stand for."""
    q = rng.integers(-127, 128, (n, k)).astype(np.int8)
    s = (rng.random((n, k // G)) * 0.5 / 127 / math.sqrt(k) + 0.2 / 127 / math.sqrt(k)).astype(np.float16)
    return dev(q), dev(s), q.astype(np.float64) * np.repeat(s.astype(np.float64), G, 1)


class Layer:
    def __init__(self, rng):
        self.norm = (1 + 0.2 * rng.standard_normal(HIDDEN)).astype(np.float16)
        self.qkv, self.out = _int8(rng, QKV, HIDDEN), _int8(rng, HIDDEN, HQ * D)
        self.qw, self.kw = ((1 + 0.2 * rng.standard_normal(D)).astype(np.float16) for _ in range(2))
        self.a = (rng.standard_normal((3, RANK, HIDDEN)) / math.sqrt(HIDDEN)).astype(np.float16)
        self.b = (rng.standard_normal((3, QKV, RANK)) * 0.1).astype(np.float16)
        self.dev = {n: dev(getattr(self, n)) for n in ("norm", "qw", "kw", "a", "b")}


@pytest.mark.parametrize("long", [False, True])
def test_layers_of_a_ragged_batch(long):
    rng = np.random.default_rng(5 + long)
    L, ranks, scales = cb.lib(), np.array([16, 5, 9], np.int32), np.array([0.5, 2.0, 1.0], np.float32)
    layers = [Layer(rng) for _ in range(2)]
    cache = kv4.KVCache4(2, HQ, HKV, D, 400, 4, 1200, 1200, G, 16)
    positions = 1200
    table = empty((positions, D // 2, 2), np.float32)
    kv4.rope_table(1e4, D, positions, table)
    turns = host(table, np.float32)
    d_ranks, d_scales = dev(ranks), dev(scales)
    done, ids = [0, 0, 0, 0], [0, -1, 2, 1]
    steps = ([600, 1, 333, 40], [1, 1, 1, 1], [1, 5, 1, 2]) if long else ([17, 1, 9, 3], [1, 1, 1, 1], [2, 0, 1, 1])
    embed = (rng.standard_normal((VOCAB, HIDDEN))).astype(np.float16)
    head = dev(embed)
    tokens = [rng.integers(0, VOCAB, n) for n in steps[0]]
    for counts in steps:
        t = sum(counts)
        tokens = [np.resize(x, n) for x, n in zip(tokens, counts)]
        offsets = np.cumsum([0] + counts).astype(np.int32)
        pos = np.concatenate([np.arange(d, d + n) for d, n in zip(done, counts)])
        d_off, d_ids = dev(offsets), dev(np.array(ids, np.int32))
        plan = empty((batch.lora_plan_bytes(4, t, 3),), np.uint8)
        batch.lora_plan(d_off, d_ids, 4, t, 3, plan, plan.numel())
        ws = empty((batch.lora_workspace(t, RANK),), np.uint8)
        cache.begin([0, 1, 2, 3], counts)
        x = dev(embed[np.concatenate(tokens)])  # the layer's input, and with what follows the next one's
        residual = None
        for n, layer in enumerate(layers):
            total, normed = empty((t, HIDDEN), np.float16), empty((t, HIDDEN), np.float16)
            codes, cs = empty((t, HIDDEN), np.int8), empty((t,), np.float32)
            before = host(x, np.float16).copy(), None if residual is None else host(residual, np.float16).copy()
            batch.add_rms_norm_q8(x, layer.dev["norm"], t, HIDDEN, codes, cs, normed, residual, total)
            qkv, turned, out = empty((t, QKV), np.float16), empty((t, HQ, D), np.float16), empty((t, HQ * D), np.float16)
            cb.check(L.cactus_cuda_matmul_int8(codes.data_ptr(), cs.data_ptr(), layer.qkv[0].data_ptr(), layer.qkv[1].data_ptr(),
                                               qkv.data_ptr(), t, HIDDEN, QKV, G, None))
            shared = host(qkv, np.float16).copy()
            batch.lora(normed, layer.dev["a"], layer.dev["b"], qkv, plan, plan.numel(), 4, t, 3, RANK, HIDDEN, QKV, ws,
                       ws.numel(), base=qkv, ranks=d_ranks, scales=d_scales)
            k = qkv.data_ptr() + 2 * HQ * D
            cache.rope_append(n, k, k + 2 * HKV * D, table, positions, D, qkv, turned, layer.dev["qw"], layer.dev["kw"],
                              row_stride=QKV, query_stride=QKV)
            cache.attention(n, turned, out, 1 / math.sqrt(D))
            # what it stands for, from the library's codes on
            s = before[0] if before[1] is None else B.add16(*before)
            assert np.array_equal(host(total, np.float16), s)
            y, tol = B.norm(s, layer.norm, 1e-6)
            B.within(host(normed, np.float16), y, tol + B.fp16_step(y))
            code = host(codes, np.int8).astype(np.float64) * host(cs, np.float32).astype(np.float64)[:, None]
            assert (np.abs(code - y) <= np.abs(y).max(-1, keepdims=True) / 127 * 0.51).all()
            ref, size = code @ layer.qkv[2].T, np.abs(code) @ np.abs(layer.qkv[2]).T
            B.within(shared, ref, B.fp16_step(ref) + (HIDDEN // G + 4) * B.U32 * size)
            seqs = list(zip(offsets[:-1], offsets[1:]))
            got = host(qkv, np.float16)
            B.within(got, *B.lora(host(normed, np.float16), layer.a, layer.b, ranks, scales, shared, seqs, ids))
            heads = got.reshape(t, -1, D)
            v, e = B.rotate(heads[:, :HQ], layer.qw, 1e-6, turns[pos], D)
            B.within(host(turned, np.float16), v, e + B.fp16_step(v))
            q, o = host(turned, np.float16), host(out, np.float16).reshape(t, HQ, D)
            for b, (t0, t1) in enumerate(seqs):
                rows = done[b] + counts[b]
                if t1 == t0:
                    continue
                keys, vals = empty((rows, HKV, D), np.float16), empty((rows, HKV, D), np.float16)
                cache.read(n, b, 0, rows, keys, vals)
                ref, _, tol, _ = U.attention(q[t0:t1], host(keys, np.float16), host(vals, np.float16), 1 / math.sqrt(D), True, 0)
                B.within(o[t0:t1], ref, tol)
                new = heads[t0:t1, HQ:].astype(np.float64)
                want, e = B.rotate(heads[t0:t1, HQ:HQ + HKV], layer.kw, 1e-6, turns[pos[t0:t1]], D)
                for cached, x64, e64 in ((keys, want, e), (vals, new[:, HKV:], 0.0)):
                    c = host(cached, np.float16)[done[b]:].astype(np.float64)
                    g = x64.reshape(*x64.shape[:-1], -1, G)
                    step = np.repeat((g.max(-1) - g.min(-1)) / 15, G, -1)
                    assert (np.abs(c - x64) <= step * 0.6 + 2 * (e64 + B.fp16_step(x64)) + B.fp16_step(c)).all()
            delta = empty((t, HIDDEN), np.float16)
            cb.check(L.cactus_cuda_linear_int8(out.data_ptr(), layer.out[0].data_ptr(), layer.out[1].data_ptr(), delta.data_ptr(),
                                               t, HQ * D, HIDDEN, G, None))
            x, residual = delta, total
        done = [d + n for d, n in zip(done, counts)]
        # the last rows' logits, with penalties, a ban and a grammar, and the greedy choice of each
        total, normed = empty((t, HIDDEN), np.float16), empty((t, HIDDEN), np.float16)
        batch.add_rms_norm_q8(x, layers[0].dev["norm"], t, HIDDEN, normed=normed, residual=residual, sum=total)
        live = [b for b in range(4) if counts[b]]
        last = normed[torch().tensor([int(offsets[b + 1]) - 1 for b in live], device="cuda")].contiguous()
        raw = empty((len(live), VOCAB), np.float16)
        cb.check(L.cactus_cuda_matmul_f16(last.data_ptr(), head.data_ptr(), raw.data_ptr(), len(live), HIDDEN, VOCAB, None))
        plain = host(raw, np.float16).copy()
        hist = [tokens[b] for b in live]
        pen = np.tile(np.float32([1.2, 0.3, 0.1]), (len(live), 1))
        bias = [[(int(plain[i].argmax()), -np.inf)] for i in range(len(live))]
        mask = [rng.random(VOCAB) < 0.5 if i % 2 else None for i in range(len(live))]
        have = [m for m in mask if m is not None] or [np.ones(VOCAB, bool)]
        index = np.cumsum([m is not None for m in mask]) - 1
        args = [dev(pen), dev(np.concatenate(hist).astype(np.uint32)),
                dev(np.cumsum([0] + [len(h) for h in hist]).astype(np.int32)), None, sum(len(h) for h in hist),
                dev(np.array([b[0][0] for b in bias], np.uint32)), dev(np.full(len(live), -np.inf, np.float32)),
                dev(np.arange(len(live) + 1, dtype=np.int32)), len(live), dev(np.stack([B.pack_bits(m) for m in have])), None,
                len(have), dev(np.where([m is None for m in mask], -1, index).astype(np.int32))]
        batch.logits_process(raw, raw, len(live), VOCAB, *args)
        ref, tol = B.logits(plain, pen, hist, [0] * len(live), bias, mask)
        got = host(raw, np.float16)
        B.within(got, ref, tol)
        choice = empty((len(live),), np.uint32)
        for i in range(len(live)):
            cb.check(L.cactus_cuda_argmax_f16(raw[i:i + 1].data_ptr(), 1, VOCAB, choice[i:].data_ptr(), None))
        assert host(choice, np.uint32).tolist() == [int(np.argmax(g.astype(np.float32))) for g in got]
        for i, b in enumerate(live):
            tokens[b] = np.append(tokens[b], host(choice, np.uint32)[i])[-1:]
    assert L.cactus_cuda_device_error(None) == 0
    cache.close()
