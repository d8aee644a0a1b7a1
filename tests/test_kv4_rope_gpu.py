"""The rotating append of the 4-bit paged KV cache and its table against 64-bit statements (tests/batch_util.py,
tests/kv4_util.py)."""
import numpy as np
import pytest

import cactus_b200 as cb
from cactus_b200 import kv4
from tests import batch_util as B
from tests import kv4_util as U
from tests.gpu_util import dev, empty, host, torch

pytestmark = pytest.mark.gpu


def _err():
    return cb.lib().cactus_cuda_device_error(None)


class Call:
    """Queries, keys and values are slices of one projection's output; what no position reaches is kept to compare."""

    def __init__(self, ge, counts, lens, hq, rotary, rng, norm=False, eps=1e-6, positions=None, extra=0, scale=1.0, pad=0):
        self.ge, self.counts, self.lens, self.hq, self.rotary, self.eps = ge, counts, lens, hq, rotary, eps
        self.t = sum(counts) + extra
        self.width = (hq + 2 * ge.hkv) * ge.d + pad
        self.qkv = (rng.standard_normal((self.t, self.width)) * scale).astype(np.float16)
        self.q = self.qkv[:, :hq * ge.d].reshape(self.t, hq, ge.d)
        self.k, self.v = (self.qkv[:, i * ge.d:(i + ge.hkv) * ge.d].reshape(self.t, ge.hkv, ge.d) for i in (hq, hq + ge.hkv))
        table, pages, _ = U.tables(lens, ge.page, rng)
        self.table, self.pool = table, U.Pool(ge, pages, rng)
        self.n_pos = max(max(lens), 1) if positions is None else positions
        self.turns = B.turns(1e4, rotary, np.arange(self.n_pos)) if rotary else None
        self.qw, self.kw = ((1 + 0.3 * rng.standard_normal(ge.d)).astype(np.float16) for _ in range(2)) if norm else (None, None)
        self.off = np.cumsum([0] + counts).astype(np.int32)
        self.upload()

    def upload(self):
        none = lambda a: None if a is None else dev(a)  # noqa: E731
        self.d = dict(qkv=dev(self.qkv), table=dev(self.table), pool=dev(self.pool.bytes), turns=none(self.turns),
                      qw=none(self.qw), kw=none(self.kw), off=dev(self.off), lens=dev(np.array(self.lens, np.int32)))
        self.out = empty((self.t, self.hq + 1, self.ge.d), np.float16)  # rows of one head more
        self.out.fill_(np.float16(123.0).view(np.int16).item())

    def run(self, queries=True, inplace=False, stream=None):
        g, a = self.ge, lambda n: None if self.d[n] is None else self.d[n].data_ptr()  # noqa: E731
        at = a("qkv")
        cb.check(cb.lib().cactus_cuda_kv4_rope_append(
            at if queries else None, self.width, at if inplace else self.out.data_ptr(),
            self.width if inplace else (self.hq + 1) * g.d, at + 2 * self.hq * g.d, at + 2 * (self.hq + g.hkv) * g.d,
            self.width, a("turns"), self.n_pos, self.rotary, a("qw"), a("kw"), self.eps, a("off"), a("lens"), a("table"),
            self.table.shape[1], a("pool"), self.pool.pages, self.pool.stride, len(self.counts), self.t, self.hq, *g.args(),
            stream), "rope_append")

    def rows(self):
        """(token, sequence, position) of each token that has a place."""
        for b, (n, l) in enumerate(zip(self.counts, self.lens)):
            for i in range(n):
                yield self.off[b] + i, b, l - n + i

    def expected(self, x, weight):
        pos = np.zeros(self.t, np.int64)
        for t, _, p in self.rows():
            pos[t] = max(p, 0)
        turn = self.turns[np.minimum(pos, self.n_pos - 1)] if self.rotary else None
        v, e = B.rotate(x, weight, self.eps, turn, self.rotary)
        return v, e, (B.rotate32(x, turn, self.rotary) if weight is None else None)

    def check(self, queries=True, inplace=False, err=0):
        g = self.ge
        placed = {t: (b, p) for t, b, p in self.rows()}
        live = [t for t, (b, p) in placed.items() if 0 <= p and (not self.rotary or p < self.n_pos)]
        if queries:
            got = host(self.d["qkv"], np.float16)[:, :self.hq * g.d].reshape(self.t, self.hq, g.d) if inplace else \
                host(self.out, np.float16)
            v, e, exact = self.expected(self.q, self.qw)
            if exact is None:
                B.within(got[live, :self.hq], v[live], e[live] + B.fp16_step(v[live]))
            else:
                assert np.array_equal(got[live, :self.hq].view(np.uint16), exact[live].view(np.uint16))
            zero = [t for t in placed if t not in set(live)]
            assert (got[zero, :self.hq] == 0).all()
            rest = [t for t in range(self.t) if t not in placed]
            same = self.q[rest] if inplace else np.full((len(rest), self.hq, g.d), 123.0, np.float16)
            assert np.array_equal(got[rest, :self.hq].view(np.uint16), same.view(np.uint16))
            if not inplace:
                assert (got[:, self.hq:] == np.float16(123.0)).all()
        # the pool: exact keys and all values byte for byte, normalised keys within half a step
        v, e, exact = self.expected(self.k, self.kw)
        now = U.Pool(g, self.pool.pages, np.random.default_rng(0), self.pool.stride)
        now.bytes = host(self.d["pool"], np.uint8).reshape(self.pool.bytes.shape)
        wanted = self.pool.bytes.copy()
        want = U.Pool(g, self.pool.pages, np.random.default_rng(0), self.pool.stride)
        want.bytes = wanted
        for t in live:
            b, p = placed[t]
            page = int(self.table[b, p // g.page])
            if page < 0:
                continue
            want.write(1, page, p % g.page, self.v[t])
            if exact is not None:
                want.write(0, page, p % g.page, exact[t])
                continue
            codes, par = now._parts(0)
            code, pair = codes[page, :, p % g.page], np.ascontiguousarray(par[page, :, p % g.page]).view(np.float16)
            full = np.empty((g.hkv, g.d), np.uint8)
            full[:, 0::2], full[:, 1::2] = code & 15, code >> 4
            pair = pair.reshape(g.hkv, g.ng, 2)
            stands = U.values(full, pair[..., 0], pair[..., 1], g.g).astype(np.float64)
            x = v[t].reshape(g.hkv, g.ng, g.g)
            one = e[t] + B.fp16_step(v[t])  # of the key in fp16
            step = (x.max(-1) - x.min(-1)) / 15 + one.reshape(x.shape).max(-1) / 7
            tol = np.repeat(step, g.g, -1) * (0.5 + 15 * 2.0 ** -10) + one + B.fp16_step(stands)
            assert (np.abs(stands - v[t]) <= tol).all()
            want._parts(0)[0][page, :, p % g.page], want._parts(0)[1][page, :, p % g.page] = code, par[page, :, p % g.page]
        assert np.array_equal(now.bytes, want.bytes)
        assert _err() == err


GEOMS = [(16, 2, 64, 32), (64, 1, 128, 32), (32, 3, 128, 128), (16, 2, 256, 64), (256, 1, 64, 64), (128, 5, 256, 32)]


@pytest.mark.parametrize("geom", GEOMS)
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("part", [4, 3, 2, 1, 0])
def test_heads_rotary_and_norm(geom, norm, part):
    ge = U.Geom(*geom)
    rng = np.random.default_rng(ge.d + part)
    call = Call(ge, [1, 40, 3], [70, 40, 1000], 2 * ge.hkv, ge.d * part // 4, rng, norm, extra=4, pad=8)
    call.run()
    call.check()


@pytest.mark.parametrize("counts,lens", [([1], [1]), ([0, 1, 0], [5, 1, 0]), ([33], [33]), ([1] * 70, list(range(1, 71))),
                                         ([5, 31, 32, 64], [5, 100, 32, 65]), ([300], [4000])])
def test_counts(counts, lens):
    ge = U.Geom(16, 2, 128, 64)
    rng = np.random.default_rng(len(counts))
    call = Call(ge, counts, lens, 4, 128, rng, True, extra=2)
    call.run()
    call.check()


@pytest.mark.parametrize("norm", [False, True])
def test_in_place_and_without_queries(norm):
    ge = U.Geom(32, 2, 64, 32)
    rng = np.random.default_rng(3)
    call = Call(ge, [40, 2], [50, 9], 6, 48, rng, norm, extra=3)
    call.run(inplace=True)
    call.check(inplace=True)
    call = Call(ge, [40, 2], [50, 9], 6, 48, rng, norm)
    call.run(queries=False)
    call.check(queries=False)


def test_values_that_are_no_numbers_and_constant_groups():
    ge = U.Geom(16, 2, 128, 32)
    rng = np.random.default_rng(4)
    call = Call(ge, [40], [40], 4, 0, rng)
    call.v[3, 0, 5], call.v[4, 1, 127], call.v[5, 0, :32], call.v[6] = np.nan, np.inf, 0.5, 0
    call.k[3, 0, 5], call.k[4, 1, 127], call.k[5, 0, :32], call.k[6] = -np.inf, np.nan, -7, 65504
    call.upload()
    call.run()
    codes = {n: host(call.d[n], np.uint8) for n in ("pool",)}["pool"].reshape(call.pool.bytes.shape)
    now = U.Pool(ge, call.pool.pages, rng, call.pool.stride)
    now.bytes = codes
    for which, x in ((0, call.k), (1, call.v)):
        got = now.rows(which, call.table[0].tolist(), 40)
        q, step, low = U.quantise(x, ge.g)
        want = U.values(q, step, low, ge.g)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)])
    assert np.array_equal(host(call.out, np.float16)[:, :4].view(np.uint16), call.q.view(np.uint16)) and _err() == 0


def test_norm_of_zeros_and_large_rows():
    ge = U.Geom(16, 1, 64, 32)
    rng = np.random.default_rng(5)
    call = Call(ge, [20], [20], 2, 64, rng, True, eps=1e-5)
    call.q[0], call.k[1], call.q[2], call.k[3], call.q[4] = 0, 0, 60000, -60000, 6e-8
    call.upload()
    call.run()
    call.check()


def test_positions_below_zero_and_past_the_table():
    ge = U.Geom(16, 2, 64, 64)
    rng = np.random.default_rng(6)
    call = Call(ge, [6, 3, 40], [4, 0, 40], 4, 64, rng)  # two tokens, three, before position 0
    call.run()
    call.check()
    call = Call(ge, [6, 3], [60, 3], 4, 32, rng, True, positions=57)  # three past the table's end
    call.run()
    call.check(err=3)
    call = Call(ge, [6, 3], [60, 3], 4, 0, rng, positions=0)  # no rotation: no table is needed
    call.run()
    call.check()


def test_bad_pages_are_skipped():
    ge = U.Geom(16, 2, 128, 32)
    rng = np.random.default_rng(7)
    call = Call(ge, [40, 5], [40, 90], 4, 128, rng)
    call.table[0, 1], call.table[1, 5] = -1, call.pool.pages
    call.upload()
    call.run()
    keep = call.table[1, 5]
    call.table[1, 5] = -1
    call.check(err=3)
    assert keep == call.pool.pages
    call = Call(ge, [3], [16 * 5 + 2], 4, 128, rng)  # positions past a table that is cut short
    call.table = np.ascontiguousarray(call.table[:, :5])
    call.upload()
    call.run()
    call.table = np.concatenate([call.table, [[-1]]], 1).astype(np.int32)
    call.check(err=3)


def test_replayed_as_the_sequences_grow():
    t = torch()
    ge = U.Geom(16, 2, 128, 32)
    rng = np.random.default_rng(8)
    call = Call(ge, [1, 1, 1], [60, 33, 100], 4, 128, rng, positions=200)
    call.lens = [40, 32, 99]
    call.upload()
    call.run()
    call.check()
    call.pool.bytes = host(call.d["pool"], np.uint8).reshape(call.pool.bytes.shape).copy()
    graph = t.cuda.CUDAGraph()
    t.cuda.synchronize()
    with t.cuda.graph(graph):
        call.run(stream=t.cuda.current_stream().cuda_stream)
    for step in range(3):
        call.lens = [n + 1 for n in call.lens] if step else call.lens
        call.lens = [min(n, m) for n, m in zip(call.lens, [60, 33, 100])]
        call.d["lens"].copy_(t.tensor(call.lens, dtype=t.int32))
        graph.replay()
        call.check()
        call.pool.bytes = host(call.d["pool"], np.uint8).reshape(call.pool.bytes.shape).copy()


@pytest.mark.parametrize("theta,rotary,positions", [(1e4, 64, 100), (1e6, 128, 5000), (500000.0, 48, 131072), (1e4, 256, 1),
                                                    (2.5, 2, 1000)])
def test_table(theta, rotary, positions):
    t = empty((positions, rotary // 2, 2), np.float32)
    kv4.rope_table(theta, rotary, positions, t)
    # rounding of numbers up to 1, and 8 units of 64 bits of the angle
    angle = np.arange(positions)[:, None] * float(np.float32(theta)) ** (-np.arange(rotary // 2) * 2.0 / rotary)
    tol = (2.0 ** -25 + 8 * 2.0 ** -53 * angle)[..., None]
    assert (np.abs(host(t, np.float32) - np.stack([np.cos(angle), np.sin(angle)], -1)) <= tol).all()


def test_handle_appends_what_the_entry_points_do():
    """KVCache4.rope_append against rotated keys through KVCache4.append: the same rows back, bit for bit."""
    ge, hq, rng = U.Geom(16, 2, 64, 32), 4, np.random.default_rng(9)
    caches = [kv4.KVCache4(2, hq, ge.hkv, ge.d, 64, 4, 400, 128, ge.g, ge.page) for _ in range(2)]
    table = empty((400, ge.d // 2, 2), np.float32)
    kv4.rope_table(1e4, ge.d, 400, table)
    turns, done = host(table, np.float32), [0, 0, 0]
    for counts in ([50, 1, 20], [1, 1, 1], [30, 0, 2]):
        t = sum(counts)
        q, k, v = (rng.standard_normal((t, h, ge.d)).astype(np.float16) for h in (hq, ge.hkv, ge.hkv))
        pos = np.concatenate([np.arange(d, d + n) for d, n in zip(done, counts)])
        turned = B.rotate32(k, turns[pos], ge.d)
        dq, dk, dv, dt, out = dev(q), dev(k), dev(v), dev(turned), empty((t, hq, ge.d), np.float16)
        for c in caches:
            c.begin([0, 1, 2], counts)
        for layer in range(2):
            caches[0].rope_append(layer, dk, dv, table, 400, ge.d, dq, out)
            caches[1].append(layer, dt, dv)
        assert np.array_equal(host(out, np.float16), B.rotate32(q, turns[pos], ge.d))
        done = [d + n for d, n in zip(done, counts)]
        for s, n in enumerate(done):
            got = []
            for c in caches:
                kk, vv = empty((n, ge.hkv, ge.d), np.float16), empty((n, ge.hkv, ge.d), np.float16)
                c.read(1, s, 0, n, kk, vv)
                got.append((host(kk, np.uint16), host(vv, np.uint16)))
            assert np.array_equal(got[0][0], got[1][0]) and np.array_equal(got[0][1], got[1][1])
    with pytest.raises(cb.CactusError, match="rope_append"):
        caches[0].rope_append(2, dk, dv, table, 400, ge.d)
    for c in caches:
        c.close()
    assert _err() == 0
