"""Calls of the 4-bit paged KV cache that a program may make and that tests/test_kv4_gpu.py does not:
queries that see nothing, padded token rows, offsets that change under a captured call, whole batches
moved at once. References are the 64-bit statements of tests/kv4_util.py."""
import math

import numpy as np
import pytest

import cactus_b200 as cb
from tests import kv4_util as U
from tests.gpu_util import dev, empty, host, ptr, torch
from tests.test_kv4_gpu import _check, _err, _filled, _offsets

pytestmark = pytest.mark.gpu


class Call:
    """An attention call on device copies of its arguments, its outputs filled with a value no result has."""

    def __init__(self, pool, table, q, counts, lens, hq, max_q=None, causal=True, window=0):
        ge, t = pool.ge, q.shape[0]
        self.n, self.causal, self.window, self.hq, self.pool, self.width = t, causal, window, hq, pool, table.shape[1]
        self.max_q, self.seqs = max_q or max(counts), len(counts)
        self.q, self.off, self.lens, self.table, self.bytes = (
            dev(a) for a in (q, _offsets(counts), np.array(lens, np.int32), table, pool.bytes))
        self.out, self.lse = empty((t, hq, ge.d), np.float16), empty((t, hq), np.float32)
        self.ws = empty((cb.lib().cactus_cuda_kv4_attention_workspace(len(lens), t, hq, ge.hkv, ge.d),), np.uint8)
        torch().cuda.synchronize()

    def clear(self):
        self.out.fill_(np.float16(123.0).view(np.int16).item())
        self.lse.fill_(123.0)

    def run(self, stream=None):
        ge = self.pool.ge
        cb.check(cb.lib().cactus_cuda_kv4_attention(
            ptr(self.q), self.hq * ge.d, ptr(self.off), ptr(self.lens), ptr(self.table), self.width, ptr(self.bytes),
            self.pool.pages, self.pool.stride, ptr(self.out), ptr(self.lse), self.seqs, self.n, self.max_q, self.hq,
            *ge.args(), 1.0 / math.sqrt(ge.d), self.window, int(self.causal), ptr(self.ws), self.ws.numel(), stream),
            "attention")

    def got(self):
        return host(self.out, np.float16), host(self.lse, np.float32)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_queries_that_see_nothing_give_zeros(d):
    """Whole row tiles of queries before position 0, or of an empty sequence: zeros and -inf every time."""
    ge = U.Geom(16, 2, d, 32)
    rng = np.random.default_rng(d)
    counts, lens, hq = [600, 150, 400, 300], [10, 0, 37, 300], 4
    pool, table = _filled(ge, lens, rng)
    q = np.full((sum(counts), hq, d), 7.0, np.float16) + rng.standard_normal((sum(counts), hq, d)).astype(np.float16)
    call = Call(pool, table, q, counts, lens, hq)
    call.clear()
    call.run()
    first, _ = call.got()
    _check(pool, table, q, counts, lens, hq, True, 0, *call.got())
    for _ in range(30):
        call.clear()
        call.run()
        out, lse = call.got()
        assert np.array_equal(out.view(np.uint16), first.view(np.uint16))
        assert np.isneginf(lse[:590]).all() and np.isneginf(lse[600:750]).all() and np.isneginf(lse[750:1113]).all()
    assert _err() == 0


@pytest.mark.parametrize("d", [64, 128, 256])
def test_parts_of_the_keys_that_are_empty(d):
    """A table far wider than what the first queries see: most parts of their keys hold none, in any order of arrival."""
    ge = U.Geom(16, 1, d, 32)
    rng = np.random.default_rng(d + 1)
    lens, counts, hq = [700, 2600], [700, 80], 2
    pool, table = _filled(ge, lens, rng)
    q = rng.standard_normal((sum(counts), hq, d)).astype(np.float16)
    call = Call(pool, table, q, counts, lens, hq)
    call.clear()
    call.run()
    first, _ = call.got()
    _check(pool, table, q, counts, lens, hq, True, 0, *call.got())
    for _ in range(30):
        call.clear()
        call.run()
        assert np.array_equal(call.got()[0].view(np.uint16), first.view(np.uint16))
    assert _err() == 0


PADDED = [
    # counts, rows of the call, max_query_len, lens, (page, hkv, d, g), hq, window
    ([10], 256, 256, [300], (16, 2, 64, 32), 4, 0),
    ([5], 256, 256, [5], (32, 1, 128, 32), 2, 0),
    ([100, 1], 200, 100, [900, 77], (16, 2, 128, 64), 4, 0),
    ([256, 1], 512, 256, [256, 1000], (16, 1, 64, 64), 2, 0),
    ([1, 90, 3], 300, 100, [400, 90, 12], (32, 1, 256, 32), 4, 50),
    ([1, 0, 2], 384, 128, [33, 0, 2], (16, 2, 128, 128), 2, 0),
    # room for fewer than all at their longest: both kernels
    ([100, 1], 150, 100, [100, 500], (16, 1, 128, 32), 2, 0),
    ([1, 3, 40], 64, 64, [9, 300, 41], (16, 1, 64, 32), 4, 0),
    # few queries, padded
    ([1, 2], 16, 4, [200, 2], (16, 2, 64, 32), 4, 0),
]


@pytest.mark.parametrize("counts,rows,max_q,lens,geom,hq,window", PADDED)
def test_padded_token_rows(counts, rows, max_q, lens, geom, hq, window):
    """Fewer tokens than the call has rows: every sequence is answered, and the rows past the last are left alone."""
    ge = U.Geom(*geom)
    rng = np.random.default_rng(rows + sum(lens))
    pool, table = _filled(ge, lens, rng)
    q = rng.standard_normal((rows, hq, ge.d)).astype(np.float16)
    call = Call(pool, table, q, counts, lens, hq, max_q=max_q, window=window)
    call.clear()
    call.run()
    n = sum(counts)
    out, lse = call.got()
    _check(pool, table, q[:n], counts, lens, hq, True, window, out[:n], lse[:n])
    assert (out[n:] == 123.0).all() and (lse[n:] == 123.0).all()
    assert _err() == 0


@pytest.mark.parametrize("rows,max_q", [(160, 80), (120, 80), (80, 80)])
def test_captured_call_follows_offsets_on_the_device(rows, max_q):
    """A captured call whose sequences cross, from replay to replay, from many queries to few and back."""
    t = torch()
    ge, hq = U.Geom(32, 2, 128, 32), 4
    rng = np.random.default_rng(rows)
    lens = [400, 150]
    pool, table = _filled(ge, lens, rng)
    q = rng.standard_normal((rows, hq, ge.d)).astype(np.float16)
    call = Call(pool, table, q, [rows // 2, rows // 2], lens, hq, max_q=max_q)
    call.run()  # sets the kernels' attributes
    t.cuda.synchronize()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        call.run(t.cuda.current_stream().cuda_stream)
    for counts, now in (([rows // 2, rows // 2], lens), ([1, 1], [399, 64]), ([rows // 2, 1], [120, 150]), ([2, 60 % rows], [17, 100]),
                        ([0, 5], [0, 5]), ([min(max_q, rows - 1), 1], lens)):
        call.clear()
        call.off.copy_(dev(_offsets(counts)))
        call.lens.copy_(dev(np.array(now, np.int32)))
        graph.replay()
        out, lse = call.got()
        n = sum(counts)
        _check(pool, table, q[:n], counts, now, hq, True, 0, out[:n], lse[:n])
        assert (out[n:] == 123.0).all() and (lse[n:] == 123.0).all()
    assert _err() == 0


def _batch_cache(ge, layers, lens, max_context, num_pages):
    """A cache whose sequences hold lens rows each, and the rows [layer][seq][keys, values] as the format stands for them."""
    from cactus_b200.kv4 import KVCache4
    rng = np.random.default_rng(sum(lens))
    cache = KVCache4(layers, 2 * ge.hkv, ge.hkv, ge.d, num_pages=num_pages, max_seqs=len(lens), max_context=max_context,
                     max_tokens=sum(lens), group_size=ge.g, page_size=ge.page)
    cache.begin(range(len(lens)), lens)
    off, rows = _offsets(lens), []
    for layer in range(layers):
        kv = rng.standard_normal((2, sum(lens), ge.hkv, ge.d)).astype(np.float16)
        d = [dev(x) for x in kv]
        cache.append(layer, ptr(d[0]), ptr(d[1]))
        want = [U.values(*U.quantise(x, ge.g), ge.g) for x in kv]
        rows.append([[x[off[s]:off[s + 1]] for x in want] for s in range(len(lens))])
    return cache, rows


def _holds(cache, ge, layer, seq, want):
    n = cache.length(seq)
    assert n == want[0].shape[0]
    got = [empty((n, ge.hkv, ge.d), np.float16) for _ in range(2)]
    cache.read(layer, seq, 0, n, *(ptr(g) for g in got))
    return all(np.array_equal(host(g, np.float16), w) for g, w in zip(got, want))


def test_a_whole_batch_is_compacted_in_one_call():
    """All sequences keep more rows together than one context holds, one of them all of its rows, one none."""
    ge, layers = U.Geom(16, 2, 64, 32), 2
    lens = [512, 400, 512, 17, 333, 512, 1, 480, 512, 256, 512, 90]
    cache, rows = _batch_cache(ge, layers, lens, 512, 600)
    rng = np.random.default_rng(4)
    kept = [np.sort(rng.choice(n, n // 2 + 1 if n > 1 else 1, replace=False)) for n in lens]
    kept[5], kept[7] = np.arange(512), np.arange(0)
    cache.compact(range(len(lens)), kept)
    for layer in range(layers):
        for s in range(len(lens)):
            rows[layer][s] = [x[kept[s]] for x in rows[layer][s]]
            assert _holds(cache, ge, layer, s, rows[layer][s])
    cache.slide(range(len(lens)), sink=3, window=200)
    for layer in range(layers):
        for s in range(len(lens)):
            n = len(kept[s])
            at = np.concatenate([np.arange(min(3, n)), np.arange(max(min(3, n), n - 197), n)])
            assert _holds(cache, ge, layer, s, [x[at] for x in rows[layer][s]])
    assert cache.info()["free_pages"] == 600 - sum(-(-cache.length(s) // 16) for s in range(len(lens)))
    cache.close()
    assert _err() == 0


def test_the_handle_refuses_to_be_captured():
    """The shapes of a batch's launches are the host's at the time of the call: a replay after the next begin would be wrong."""
    t = torch()
    ge = U.Geom(16, 1, 64, 32)
    cache, rows = _batch_cache(ge, 1, [20, 3], 64, 12)
    cache.begin([0, 1], [1, 1])
    x = dev(np.ones((2, 2, 64), np.float16))
    out = empty((2, 2, 64), np.float16)
    t.cuda.synchronize()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        t.zeros(1, device="cuda")
        s = t.cuda.current_stream().cuda_stream
        for call in (lambda: cache.append(0, ptr(x), ptr(x), stream=s),
                     lambda: cache.attention(0, ptr(x), ptr(out), 0.125, stream=s),
                     lambda: cache.read(0, 0, 0, 1, ptr(out), ptr(out), stream=s),
                     lambda: cache.begin([0], [1], stream=s), lambda: cache.compact([0], [[0, 1]], stream=s)):
            with pytest.raises(cb.CactusError, match="captured"):
                call()
    assert cache.length(0) == 21
    cache.append(0, ptr(x), ptr(x))  # the batch is still there, outside of a capture
    assert _holds(cache, ge, 0, 0, [np.concatenate([w, np.ones((1, 1, 64), np.float16)]) for w in rows[0][0]])
    cache.close()
    assert _err() == 0


@pytest.mark.parametrize("d,g", [(64, 32), (64, 64), (128, 128), (256, 32)])
def test_append_rounds_the_differences_as_they_are(d, g):
    """Groups whose range and elements differ from fifteen steps and from halves by less than fp32 resolves beside
    them: the format's step and codes are those of the exact differences."""
    L, ge = cb.lib(), U.Geom(16, 1, d, g)
    rng = np.random.default_rng(d + g)
    n = 160
    x = np.empty((n, d // g, g), np.float16)
    for i in range(n):
        for j in range(d // g):
            s = 2.0 ** rng.integers(-3, 4)
            row = s * (rng.integers(0, 15, g) + 0.5)     # halves of a step
            row[rng.integers(0, g, g // 4)] = s * 7.0
            row[0], row[1] = 15 * s, rng.choice([-1, 1, 1, 3]) * 2.0 ** -24 * 2.0 ** rng.integers(0, 6)
            x[i, j] = rng.permutation(row) * rng.choice([-1, 1])
    x = x.reshape(n, d)
    pool = U.Pool(ge, n // 16, rng)
    dpool, dx = dev(pool.bytes), dev(x)
    meta = [dev(np.array(a, np.int32)) for a in ([0, n], [n], [list(range(n // 16))])]
    cb.check(L.cactus_cuda_kv4_append(ptr(dx), ptr(dx), d, ptr(meta[0]), ptr(meta[1]), ptr(meta[2]), n // 16, ptr(dpool),
                                      n // 16, pool.stride, 1, n, *ge.args(), None))
    for i in range(n):
        for which in (0, 1):
            pool.write(which, i // 16, i % 16, x[i].reshape(1, d))
    assert np.array_equal(host(dpool, np.uint8), pool.bytes)
    assert _err() == 0
