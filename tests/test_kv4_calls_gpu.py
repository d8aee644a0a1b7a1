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
