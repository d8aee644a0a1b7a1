"""The 4-bit paged KV cache's kernels (include/cactus_b200_kv4.h) against a plain 64-bit statement.

Quantisation, page copies and compaction are compared bit for bit over the whole pool; attention
within bounds derived from the number formats (tests/kv4_util.py:attention)."""
import math

import numpy as np
import pytest

import cactus_b200 as cb
from tests import kv4_util as U
from tests.gpu_util import dev, empty, host, ptr, torch

pytestmark = pytest.mark.gpu


def _err():
    return cb.lib().cactus_cuda_device_error(None)


def _offsets(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


# ------------------------------------------------------------------------------------ append, read
APPEND = [
    # counts of new rows, rows before them, (page, hkv, d, g), extra row stride, extra page stride
    ([1], [0], (16, 1, 64, 32), 0, 0),
    ([1, 1, 1], [0, 15, 40], (16, 8, 128, 32), 0, 0),
    ([5, 0, 33, 1], [11, 3, 0, 16], (32, 2, 128, 64), 64, 16),
    ([70, 0, 0, 129], [1, 0, 9, 63], (64, 3, 64, 64), 8, 0),
    ([31, 32, 33], [0, 0, 0], (128, 1, 256, 128), 256, 48),
    ([300, 2], [7, 250], (256, 5, 256, 32), 0, 0),
    ([17, 100], [0, 5], (16, 2, 128, 128), 8, 0),
]


def _rows(rng, n, width, g):
    x = rng.standard_normal((n, width)).astype(np.float32)
    x = (x * np.exp(rng.standard_normal((n, 1)))).astype(np.float16)
    flat = x.reshape(n, -1, g)
    for i in range(n):  # groups at the edges of the format
        j = i % flat.shape[1]
        kind = i % 9
        if kind == 0:
            flat[i, j] = 0.25
        elif kind == 1:
            flat[i, j] = np.where(np.arange(g) % 2, np.float16(65504), np.float16(-65504))
        elif kind == 2:
            flat[i, j] = (np.arange(g) % 29) * np.float16(2.0 ** -24)
        elif kind == 3:
            flat[i, j] = np.float16(1000) + (np.arange(g) % 3 == 0)
        elif kind == 4:
            flat[i, j] = (np.arange(g) % 31) * np.float16(0.5)  # quotients at exact halves
        elif kind == 5:
            flat[i, j] = np.where(np.arange(g) == 3, np.float16(0), np.float16(-0.0))
    return x


@pytest.mark.parametrize("counts,before,geom,row_extra,page_extra", APPEND)
def test_append_then_read(counts, before, geom, row_extra, page_extra):
    L, ge = cb.lib(), U.Geom(*geom)
    rng = np.random.default_rng(sum(counts) + ge.d)
    lens = [a + b for a, b in zip(counts, before)]
    table, pages, _ = U.tables(lens, ge.page, rng)
    pool = U.Pool(ge, pages, rng, ge.block * ge.hkv + page_extra)
    n, width = sum(counts), ge.hkv * ge.d
    pad = 3  # rows past the last offset are ignored
    k = np.zeros((n + pad, width + row_extra), np.float16)
    v = np.zeros_like(k)
    k[:, :width], v[:, :width] = _rows(rng, n + pad, width, ge.g), _rows(rng, n + pad, width, ge.g)
    dpool, off = dev(pool.bytes), _offsets(counts)
    d = [dev(a) for a in (k, v, off, np.array(lens, np.int32), table)]
    cb.check(L.cactus_cuda_kv4_append(ptr(d[0]), ptr(d[1]), width + row_extra, ptr(d[2]), ptr(d[3]), ptr(d[4]),
                                      table.shape[1], ptr(dpool), pages, pool.stride, len(counts), n + pad, *ge.args(),
                                      None), "append")
    for b, (c, f) in enumerate(zip(counts, before)):
        for i in range(c):
            page, row = table[b, (f + i) // ge.page], (f + i) % ge.page
            for which, x in ((0, k), (1, v)):
                pool.write(which, page, row, x[off[b] + i, :width].reshape(ge.hkv, ge.d))
    assert np.array_equal(host(dpool, np.uint8), pool.bytes)
    # the new rows and up to five before them
    first = np.array([max(0, f - 5) for f in before], np.int32)
    want = [a - f for a, f in zip(lens, first)]
    total = sum(want)
    got = [empty((total, ge.hkv, ge.d), np.float16) for _ in range(2)]
    dro, dfirst = dev(_offsets(want)), dev(first)
    cb.check(L.cactus_cuda_kv4_read(ptr(dpool), pages, pool.stride, ptr(d[4]), table.shape[1], ptr(dro), ptr(dfirst),
                                    ptr(got[0]), ptr(got[1]), len(counts), total, *ge.args(), None), "read")
    for which in (0, 1):
        ref = [pool.rows(which, table[b], lens[b])[first[b]:] for b in range(len(lens))]
        assert np.array_equal(host(got[which], np.float16), np.concatenate(ref), equal_nan=True)
    only = empty((total, ge.hkv, ge.d), np.float16)
    cb.check(L.cactus_cuda_kv4_read(ptr(dpool), pages, pool.stride, ptr(d[4]), table.shape[1], ptr(dro), ptr(dfirst),
                                    None, ptr(only), len(counts), total, *ge.args(), None), "read values")
    assert np.array_equal(host(only, np.uint16), host(got[1], np.uint16))
    assert _err() == 0


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_append_of_a_non_finite_value_reads_as_nan_in_its_group_alone(bad):
    L, ge = cb.lib(), U.Geom(16, 2, 128, 32)
    x = np.random.default_rng(3).standard_normal((4, ge.hkv * ge.d)).astype(np.float16)
    x[1, 40] = bad
    dpool, dx = dev(np.zeros((1, ge.block * ge.hkv), np.uint8)), dev(x)
    meta = [dev(np.array(a, np.int32)) for a in ([0, 4], [4], [[0]])]
    cb.check(L.cactus_cuda_kv4_append(ptr(dx), ptr(dx), ge.hkv * ge.d, ptr(meta[0]), ptr(meta[1]), ptr(meta[2]), 1,
                                      ptr(dpool), 1, ge.block * ge.hkv, 1, 4, *ge.args(), None))
    got = [empty((4, ge.hkv, ge.d), np.float16) for _ in range(2)]
    cb.check(L.cactus_cuda_kv4_read(ptr(dpool), 1, ge.block * ge.hkv, ptr(meta[2]), 1, ptr(meta[0]), None,
                                    ptr(got[0]), ptr(got[1]), 1, 4, *ge.args(), None))
    for g in got:
        nan = np.isnan(host(g, np.float16).reshape(4, -1))
        assert nan[1, 32:64].all() and nan.sum() == 32
    assert _err() == 0


def test_append_of_negative_positions_writes_nothing():
    L, ge = cb.lib(), U.Geom(16, 1, 64, 32)
    rng = np.random.default_rng(5)
    pool = U.Pool(ge, 2, rng)
    x = rng.standard_normal((5, 64)).astype(np.float16)
    dpool, dx = dev(pool.bytes), dev(x)
    meta = [dev(np.array(a, np.int32)) for a in ([0, 5], [2], [[1]])]
    cb.check(L.cactus_cuda_kv4_append(ptr(dx), ptr(dx), 64, ptr(meta[0]), ptr(meta[1]), ptr(meta[2]), 1, ptr(dpool), 2,
                                      pool.stride, 1, 5, *ge.args(), None))
    for i in (3, 4):
        for which in (0, 1):
            pool.write(which, 1, i - 3, x[i].reshape(1, 64))
    assert np.array_equal(host(dpool, np.uint8), pool.bytes)
    assert _err() == 0


# ------------------------------------------------------------------------------------ attention
def _filled(ge, lens, rng, stride_extra=0, loud=True):
    """A pool with realistic rows in the sequences' pages, NaN parameters in the rows past their ends."""
    table, pages, rest = U.tables(lens, ge.page, rng)
    pool = U.Pool(ge, pages, rng, ge.block * ge.hkv + stride_extra)
    for which in (0, 1):
        x = rng.standard_normal((pages, ge.hkv, ge.page, ge.d))
        if loud and which == 0:
            x *= np.where(rng.random(ge.d) < 0.05, 4.0, 1.0)
        q, step, low = U.quantise(x.astype(np.float16), ge.g)
        codes, par = pool._parts(which)
        codes[:] = q[..., 0::2] | (q[..., 1::2] << 4)
        par[:] = np.ascontiguousarray(np.stack([step, low], -1)).view(np.uint8).reshape(par.shape)
    for p in rest:
        pool.spoil(p, 0)
    for b, n in enumerate(lens):
        if n % ge.page:
            pool.spoil(table[b, n // ge.page], n % ge.page)
    return pool, table


def _attend(pool, table, q, counts, lens, hq, causal=True, window=0, scale=None, q_extra=0, lse=True, max_q=None,
            stream=None, ws=None):
    L, ge = cb.lib(), pool.ge
    t = q.shape[0]
    qs = np.full((t, hq * ge.d + q_extra), np.nan, np.float16)
    qs[:, :hq * ge.d] = q.reshape(t, -1)
    d = [dev(a) for a in (qs, _offsets(counts), np.array(lens, np.int32), table, pool.bytes)]
    out, dl = empty((t, hq, ge.d), np.float16), empty((t, hq), np.float32)
    if ws is None:
        size = L.cactus_cuda_kv4_attention_workspace(len(lens), t, hq, ge.hkv, ge.d)
        assert size > 0
        ws = empty((size,), np.uint8)
    torch().cuda.synchronize()
    cb.check(L.cactus_cuda_kv4_attention(
        ptr(d[0]), qs.shape[1], ptr(d[1]), ptr(d[2]), ptr(d[3]), table.shape[1], ptr(d[4]), pool.pages, pool.stride,
        ptr(out), ptr(dl) if lse else None, len(lens), t, max_q or max(max(counts), 1), hq, *ge.args(),
        1.0 / math.sqrt(ge.d) if scale is None else scale, window, int(causal), ptr(ws), ws.numel(), stream),
        "attention")
    torch().cuda.synchronize()
    return host(out, np.float16), host(dl, np.float32), ws


def _check(pool, table, q, counts, lens, hq, causal, window, got, lse, scale=None):
    at = 0
    for b, (c, n) in enumerate(zip(counts, lens)):
        if c == 0:
            continue
        k, v = (pool.rows(w, table[b], n) if n else np.zeros((0, pool.ge.hkv, pool.ge.d), np.float16) for w in (0, 1))
        out, rl, tol, ltol = U.attention(q[at:at + c], k, v, 1.0 / math.sqrt(pool.ge.d) if scale is None else scale,
                                         causal, window)
        o, l = got[at:at + c].astype(np.float64), lse[at:at + c].astype(np.float64)
        none = np.isinf(rl)
        assert np.array_equal(none, np.isneginf(l)), b
        assert np.all(o[none] == 0)
        assert np.all(np.abs(o - out) <= tol), (b, np.max(np.abs(o - out) / tol))
        assert np.all(np.abs(np.where(none, 0, l) - np.where(none, 0, rl)) <= ltol + none), b
        at += c


ATTENTION = [
    # counts, lens, (page, hkv, d, g), hq, causal, window, page stride extra
    ([1], [1], (16, 1, 64, 32), 1, True, 0, 0),
    ([1], [512], (64, 8, 128, 32), 16, True, 0, 0),
    ([1, 1, 1], [17, 1, 2500], (16, 2, 128, 64), 2, True, 0, 16),
    ([1] * 9, [1, 2, 15, 16, 17, 63, 64, 65, 1000], (16, 2, 64, 64), 8, True, 0, 0),
    ([1, 1], [777, 5000], (256, 1, 256, 128), 4, True, 0, 32),
    ([1, 1, 1], [300, 129, 4100], (32, 3, 256, 32), 21, True, 0, 0),
    ([1, 1], [4097, 130], (64, 2, 128, 128), 16, True, 100, 0),
    ([1, 0, 1], [40, 0, 3], (16, 1, 128, 32), 7, True, 0, 0),
    ([2, 1, 5], [900, 1, 33], (32, 2, 128, 32), 4, True, 0, 0),
    ([3, 8], [3, 700], (16, 4, 64, 32), 8, True, 20, 0),
    ([4, 4], [1000, 70], (64, 1, 256, 64), 8, False, 0, 0),
    ([9, 2], [1200, 400], (64, 8, 128, 64), 16, True, 0, 0),
    ([33], [33], (16, 1, 64, 32), 4, True, 0, 0),
    ([64, 1, 130, 0, 7], [64, 900, 300, 12, 7], (32, 2, 128, 32), 4, True, 0, 0),
    ([200], [1111], (64, 2, 128, 128), 6, True, 0, 0),
    ([257, 3], [700, 700], (128, 1, 256, 64), 4, True, 0, 0),
    ([100, 260], [400, 260], (16, 2, 256, 32), 2, True, 65, 0),
    ([300], [300], (64, 1, 64, 64), 8, False, 0, 0),
    ([150, 40], [500, 640], (32, 2, 64, 32), 2, False, 37, 16),
    ([513], [1500], (64, 1, 128, 64), 3, True, 0, 0),
    ([140], [140], (64, 1, 128, 32), 1, True, 1, 0),
    # more queries than rows: the first ones stand before the sequence's start and see nothing
    ([6, 40], [4, 30], (16, 2, 128, 32), 4, True, 0, 0),
    ([300], [100], (64, 1, 64, 32), 2, True, 0, 0),
    ([5, 1], [0, 0], (16, 1, 64, 32), 2, True, 0, 0),
    ([150], [0], (16, 1, 256, 32), 2, False, 0, 0),
]


@pytest.mark.parametrize("counts,lens,geom,hq,causal,window,extra", ATTENTION)
def test_attention(counts, lens, geom, hq, causal, window, extra):
    ge = U.Geom(*geom)
    rng = np.random.default_rng(sum(counts) * 31 + sum(lens) + hq)
    pool, table = _filled(ge, lens, rng, extra)
    t = sum(counts)
    q = rng.standard_normal((t, hq, ge.d)).astype(np.float16)
    out, lse, ws = _attend(pool, table, q, counts, lens, hq, causal, window, q_extra=8 * (t % 3))
    _check(pool, table, q, counts, lens, hq, causal, window, out, lse)
    # again on the same workspace, without the log-sum-exp: the same bits
    again, _, _ = _attend(pool, table, q, counts, lens, hq, causal, window, lse=False, ws=ws)
    assert np.array_equal(again.view(np.uint16), out.view(np.uint16))
    assert _err() == 0


MIXED = [
    # counts, (page, hkv, d, g), hq, window: a prompt's chunk among sequences of a token, and one or two of some
    ([1] * 20 + [130] + [1] * 9, (32, 2, 128, 32), 4, 0),
    ([1] * 30 + [16, 100] + [1] * 30 + [12], (16, 1, 128, 64), 2, 0),
    ([1] * 40 + [90, 24], (16, 2, 64, 32), 4, 33),
    ([1] * 24 + [48] + [1] * 8 + [7, 0], (16, 2, 256, 64), 4, 0),
    ([17, 16, 15, 40, 16], (32, 1, 128, 32), 2, 0),
]


@pytest.mark.parametrize("counts,geom,hq,window", MIXED)
def test_attention_of_a_chunk_among_single_tokens(counts, geom, hq, window):
    ge = U.Geom(*geom)
    rng = np.random.default_rng(sum(counts) + hq)
    lens = [int(c + rng.integers(0, 400)) for c in counts]
    pool, table = _filled(ge, lens, rng)
    q = rng.standard_normal((sum(counts), hq, ge.d)).astype(np.float16)
    out, lse, ws = _attend(pool, table, q, counts, lens, hq, True, window)
    _check(pool, table, q, counts, lens, hq, True, window, out, lse)
    again, _, _ = _attend(pool, table, q, counts, lens, hq, True, window, ws=ws)
    assert np.array_equal(again.view(np.uint16), out.view(np.uint16))
    assert _err() == 0


@pytest.mark.parametrize("count", [1, 4, 90])
def test_attention_with_scores_far_apart(count):
    """Scores of hundreds: one key's weight is 1 and the others vanish; the maximum comes late, early or between."""
    ge = U.Geom(32, 1, 128, 32)
    rng = np.random.default_rng(count)
    lens = [700]
    pool, table = _filled(ge, lens, rng)
    big = rng.standard_normal(128)
    for row, f in ((5, 30.0), (350, -30.0), (690, 40.0)):
        pool.write(0, table[0, row // 32], row % 32, (big * f).astype(np.float16).reshape(1, 128))
    q = np.stack([big * s for s in rng.uniform(-4, 4, count * 2)]).reshape(count, 2, 128).astype(np.float16)
    out, lse, _ = _attend(pool, table, q, [count], lens, 2)
    _check(pool, table, q, [count], lens, 2, True, 0, out, lse)
    assert _err() == 0


@pytest.mark.parametrize("count,window", [(1, 0), (1, 50), (3, 0), (80, 0), (80, 50)])
def test_attention_shows_a_nan_to_those_that_see_it_alone(count, window):
    """A row poisoned by a non-finite key or value: NaN in the outputs of its kv head's queries that see it."""
    ge = U.Geom(16, 2, 64, 32)
    lens, hq, bad = [200], 4, 130
    rng = np.random.default_rng(count)
    pool, table = _filled(ge, lens, rng)
    x = rng.standard_normal((2, 64)).astype(np.float16)
    x[1, 3] = np.inf
    pool.write(1, table[0, bad // 16], bad % 16, x)
    q = rng.standard_normal((count, hq, 64)).astype(np.float16)
    out, lse, _ = _attend(pool, table, q, [count], lens, hq, window=window)
    pos = np.arange(lens[0] - count, lens[0])
    sees = (bad <= pos) & ((bad > pos - window) if window else True)
    nan = np.isnan(out)
    assert not nan[:, :2].any() and not nan[~sees].any()
    assert nan[sees][:, 2:, :32].all() and not nan[:, :, 32:].any()
    assert not np.isnan(lse).any()
    pool.write(0, table[0, bad // 16], bad % 16, x)  # the key too: every output of the head
    out, lse, _ = _attend(pool, table, q, [count], lens, hq, window=window)
    assert not np.isnan(out[:, :2]).any() and not np.isnan(out[~sees]).any()
    assert np.isnan(out[sees][:, 2:]).all() and np.isnan(lse[sees][:, 2:]).all()
    assert _err() == 0


def test_attention_workspace_is_ready_for_other_shapes():
    L = cb.lib()
    size = max(L.cactus_cuda_kv4_attention_workspace(4, 400, 16, 8, 128),
               L.cactus_cuda_kv4_attention_workspace(9, 9, 8, 1, 256))
    ws = empty((size,), np.uint8)
    for counts, lens, geom, hq in (([1, 1], [3000, 70], (64, 8, 128, 32), 16), ([200, 1], [400, 2000], (32, 2, 64, 32), 8),
                                   ([1] * 9, [1500] * 9, (16, 1, 256, 64), 8), ([1], [9], (16, 1, 64, 32), 1),
                                   ([1, 1], [3000, 70], (64, 8, 128, 32), 16)):
        ge = U.Geom(*geom)
        rng = np.random.default_rng(len(counts))
        pool, table = _filled(ge, lens, rng)
        q = rng.standard_normal((sum(counts), hq, ge.d)).astype(np.float16)
        out, lse, _ = _attend(pool, table, q, counts, lens, hq, ws=ws)
        _check(pool, table, q, counts, lens, hq, True, 0, out, lse)
    assert _err() == 0


def test_attention_does_not_touch_pages_out_of_the_window():
    """Entries of pages before every window are -1 (freed), those of a stranger's rows NaN."""
    ge = U.Geom(16, 2, 128, 32)
    rng = np.random.default_rng(8)
    for count in (1, 5, 100):
        lens, hq, window = [900], 4, 60
        pool, table = _filled(ge, lens, rng)
        q = rng.standard_normal((count, hq, 128)).astype(np.float16)
        first = lens[0] - count - window + 1
        cut = table.copy()
        cut[0, :first // 16] = -1
        out, lse, _ = _attend(pool, cut, q, [count], lens, hq, window=window)
        _check(pool, table, q, [count], lens, hq, True, window, out, lse)
        assert _err() == 0


@pytest.mark.parametrize("count", [1, 6, 70])
def test_attention_skips_pages_that_the_table_lacks_and_reports_them(count):
    ge = U.Geom(16, 1, 64, 32)
    rng = np.random.default_rng(9)
    lens = [100, 200]
    pool, table = _filled(ge, lens, rng)
    q = rng.standard_normal((2 * count, 2, 64)).astype(np.float16)
    for wrong in (-1, pool.pages, 1 << 30):
        cut = table.copy()
        cut[1, 1] = wrong
        out, lse, _ = _attend(pool, cut, q, [count, count], lens, 2)
        assert _err() == 3
        _check(pool, table, q[:count], [count], lens[:1], 2, True, 0, out[:count], lse[:count])
        # the second sequence: as if those 16 rows were not there
        k, v = (np.delete(pool.rows(w, table[1], lens[1]), np.s_[16:32], axis=0) for w in (0, 1))
        ref, rl, tol, ltol = U.attention(q[count:], k, v, 0.125, True, 0)
        assert np.all(np.abs(out[count:].astype(np.float64) - ref) <= tol)
        assert np.all(np.abs(lse[count:] - rl) <= ltol)
    # a length past the table's end
    out, lse, _ = _attend(pool, table, q, [count, count], [100, 16 * table.shape[1] + 5], 2)
    assert _err() == 3
    assert not np.isnan(out[:count].astype(np.float64)).any()


def test_attention_cuts_a_sequence_longer_than_max_query_len_and_reports_it():
    ge = U.Geom(16, 1, 64, 32)
    rng = np.random.default_rng(10)
    pool, table = _filled(ge, [100, 50], rng)
    q = rng.standard_normal((12, 2, 64)).astype(np.float16)
    out, lse, _ = _attend(pool, table, q, [9, 3], [100, 50], 2, max_q=3)
    assert _err() == 3
    _check(pool, table[1:], q[9:], [3], [50], 2, True, 0, out[9:], lse[9:])


def test_attention_far_into_a_large_pool():
    """Page offsets past 2^32 bytes."""
    t = torch()
    L, ge = cb.lib(), U.Geom(64, 8, 128, 32)
    rng = np.random.default_rng(12)
    lens = [200]
    small, table = _filled(ge, lens, rng)
    stride = ge.block * ge.hkv
    pages = (5 << 30) // stride
    big = t.empty((pages, stride), dtype=t.uint8, device="cuda")
    big[-small.pages:] = dev(small.bytes)
    far = (table + pages - small.pages).astype(np.int32)
    for count in (1, 100):
        q = rng.standard_normal((count, 16, 128)).astype(np.float16)
        d = [dev(a) for a in (q, _offsets([count]), np.array(lens, np.int32), far)]
        out, lse = empty((count, 16, 128), np.float16), empty((count, 16), np.float32)
        ws = empty((L.cactus_cuda_kv4_attention_workspace(1, count, 16, 8, 128),), np.uint8)
        cb.check(L.cactus_cuda_kv4_attention(ptr(d[0]), 2048, ptr(d[1]), ptr(d[2]), ptr(d[3]), far.shape[1],
                                             big.data_ptr(), pages, stride, ptr(out), ptr(lse), 1, count, count, 16,
                                             *ge.args(), 1 / math.sqrt(128), 0, 1, ptr(ws), ws.numel(), None))
        _check(small, table, q, [count], lens, 16, True, 0, host(out, np.float16), host(lse, np.float32))
    assert _err() == 0


def test_attention_on_a_stream_and_in_a_graph():
    t = torch()
    L, ge = cb.lib(), U.Geom(32, 2, 128, 32)
    rng = np.random.default_rng(14)
    for count in (1, 50):
        lens, hq = [600, 90], 8
        counts = [count, count]
        pool, table = _filled(ge, lens, rng)
        q = rng.standard_normal((2 * count, hq, 128)).astype(np.float16)
        ref, rlse, _ = _attend(pool, table, q, counts, lens, hq)
        d = [dev(a) for a in (q, _offsets(counts), np.array(lens, np.int32), table, pool.bytes)]
        out, lse = empty((2 * count, hq, 128), np.float16), empty((2 * count, hq), np.float32)
        ws = empty((L.cactus_cuda_kv4_attention_workspace(2, 2 * count, hq, 2, 128),), np.uint8)

        def call(stream):
            cb.check(L.cactus_cuda_kv4_attention(ptr(d[0]), hq * 128, ptr(d[1]), ptr(d[2]), ptr(d[3]), table.shape[1],
                                                 ptr(d[4]), pool.pages, pool.stride, ptr(out), ptr(lse), 2, 2 * count,
                                                 count, hq, *ge.args(), 1 / math.sqrt(128), 0, 1, ptr(ws), ws.numel(),
                                                 stream))
        t.cuda.synchronize()
        side = t.cuda.Stream()
        call(side.cuda_stream)
        side.synchronize()
        assert np.array_equal(host(out, np.uint16), ref.view(np.uint16))
        graph = t.cuda.CUDAGraph()
        with t.cuda.graph(graph):
            call(t.cuda.current_stream().cuda_stream)
        # the captured call follows the lengths on the device
        for now in ([600, 90], [517, 64], [600, 90]):
            d[2].copy_(dev(np.array(now, np.int32)))
            graph.replay()
            t.cuda.synchronize()
            _check(pool, table, q, counts, now, hq, True, 0, host(out, np.float16), host(lse, np.float32))
        assert np.array_equal(host(out, np.uint16), ref.view(np.uint16))
    assert _err() == 0


# ------------------------------------------------------------------------------------ pages
@pytest.mark.parametrize("planes,pages,page_bytes,gap,n,page_first", [
    (1, 3, 16, 0, 1, False), (3, 40, 1296, 16, 9, False), (2, 600, 16400, 0, 290, True), (28, 12, 5120, 0, 5, True),
    (5, 9, 81920, 48, 4, False)])
def test_copy_pages(planes, pages, page_bytes, gap, n, page_first):
    L = cb.lib()
    rng = np.random.default_rng(pages)
    step = page_bytes + gap
    # [plane][page] or, page_first, every page with all its planes
    page_stride, plane_stride = (step * planes, step) if page_first else (step, step * pages)
    img = rng.integers(0, 256, planes * pages * step, dtype=np.uint8)
    order = rng.permutation(pages)
    dst, src = order[:n].astype(np.int32), rng.choice(order[n:], n).astype(np.int32)
    d, ds, dd = dev(img), dev(src), dev(dst)
    cb.check(L.cactus_cuda_kv_copy_pages(ptr(d), pages, page_bytes, page_stride, planes, plane_stride, ptr(ds), ptr(dd),
                                         n, None))
    ref = img.copy()
    for pl in range(planes):
        for s, t in zip(src.astype(np.int64), dst.astype(np.int64)):
            a, b = pl * plane_stride + s * page_stride, pl * plane_stride + t * page_stride
            ref[b:b + page_bytes] = img[a:a + page_bytes]
    assert np.array_equal(host(d, np.uint8), ref)
    assert _err() == 0


def test_copy_pages_skips_ids_out_of_the_pool_and_reports_them():
    L = cb.lib()
    img = np.random.default_rng(1).integers(0, 256, (4, 64), dtype=np.uint8)
    d, ds, dd = dev(img), dev(np.array([0, -1, 4, 1], np.int32)), dev(np.array([2, 3, 3, 7], np.int32))
    cb.check(L.cactus_cuda_kv_copy_pages(ptr(d), 4, 64, 64, 1, 0, ptr(ds), ptr(dd), 4, None))
    img[2] = img[0]
    assert np.array_equal(host(d, np.uint8), img)
    assert _err() == 3


COMPACT = [
    # lens, kept rows of each (a list, or a number of random ones), geometry, planes
    ([5], [[0, 4]], (16, 1, 64, 32), 1),
    ([100, 40], [37, 1], (16, 2, 128, 32), 3),
    ([300, 7, 64], [299, 0, 64], (64, 3, 64, 64), 2),
    ([1000], [[0, 1, 2, 3] + list(range(700, 1000))], (32, 1, 256, 32), 4),
    ([513, 90], [200, 90], (256, 2, 256, 128), 1),
    ([70], [[69, 3, 3, 0]], (16, 5, 128, 128), 2),
]


@pytest.mark.parametrize("lens,kept,geom,planes", COMPACT)
def test_compact(lens, kept, geom, planes):
    L, ge = cb.lib(), U.Geom(*geom)
    rng = np.random.default_rng(sum(lens))
    rows = [np.sort(rng.choice(n, k, replace=False)) if isinstance(k, int) else np.array(k) for n, k in zip(lens, kept)]
    counts = [len(r) for r in rows]
    need = sum(-(-c // ge.page) for c in counts)
    src, pages, rest = U.tables(lens, ge.page, rng, extra=need + 1)
    dst = np.full_like(src, -1)
    at = 0
    for b, c in enumerate(counts):
        k = -(-c // ge.page)
        dst[b, :k] = rest[at:at + k]
        at += k
    stride = ge.block * ge.hkv + 16
    pools = [U.Pool(ge, pages, rng, stride) for _ in range(planes)]
    img = np.stack([p.bytes for p in pools])
    d = [dev(a) for a in (img, src, dst, np.concatenate(rows).astype(np.int32), _offsets(counts))]
    cb.check(L.cactus_cuda_kv4_compact(ptr(d[0]), pages, stride, planes, stride * pages, ptr(d[1]), ptr(d[2]),
                                       src.shape[1], ptr(d[3]), ptr(d[4]), len(lens), sum(counts), *ge.args(), None))
    for p in pools:
        for which in (0, 1):
            for part in p._parts(which):
                old = part.copy()
                for b, r in enumerate(rows):
                    for j, k in enumerate(r):
                        part[dst[b, j // ge.page], :, j % ge.page] = old[src[b, k // ge.page], :, k % ge.page]
    assert np.array_equal(host(d[0], np.uint8), np.stack([p.bytes for p in pools]))
    assert _err() == 0


def test_compact_skips_rows_that_the_tables_lack_and_reports_them():
    L, ge = cb.lib(), U.Geom(16, 1, 64, 32)
    rng = np.random.default_rng(2)
    pool = U.Pool(ge, 4, rng)
    d = [dev(pool.bytes)] + [dev(np.array(a, np.int32)) for a in ([[0, 9]], [[2, -1]], [3, 20, -1, 32, 5], [0, 5])]
    cb.check(L.cactus_cuda_kv4_compact(ptr(d[0]), 4, pool.stride, 1, 0, ptr(d[1]), ptr(d[2]), 2, ptr(d[3]), ptr(d[4]), 1,
                                       5, *ge.args(), None))
    for which in (0, 1):
        for part in pool._parts(which):
            part[2, :, 0], part[2, :, 4] = part[0, :, 3].copy(), part[0, :, 5].copy()
    assert np.array_equal(host(d[0], np.uint8), pool.bytes)
    assert _err() == 3


# ------------------------------------------------------------------------------------ the handle
def _rows_of(cache, ge, layer, seq):
    n = cache.length(seq)
    got = [empty((n, ge.hkv, ge.d), np.float16) for _ in range(2)]
    cache.read(layer, seq, 0, n, *(ptr(g) for g in got))
    return [host(g, np.float16) for g in got]


def _quantised(x, g):
    return U.values(*U.quantise(x, g), g)


@pytest.mark.parametrize("geom", [(16, 2, 64, 32), (32, 1, 128, 64)])
def test_cache_keeps_what_sequences_hold(geom):
    """Random growth, forks, cuts and compactions of a cache of three layers against lists of rows."""
    from cactus_b200.kv4 import KVCache4
    ge, layers, seqs, hq = U.Geom(*geom), 3, 5, 4
    rng = np.random.default_rng(ge.d)
    cache = KVCache4(layers, hq, ge.hkv, ge.d, num_pages=60, max_seqs=seqs, max_context=300, max_tokens=200,
                     group_size=ge.g, page_size=ge.page)
    width = ge.hkv * ge.d
    rows = [[[np.zeros((0, ge.hkv, ge.d), np.float16)] * 2 for _ in range(layers)] for _ in range(seqs)]
    for step in range(40):
        kind = rng.integers(6)
        if kind <= 2:
            ids = rng.permutation(seqs)[:rng.integers(1, seqs + 1)].tolist()
            counts = [int(rng.integers(0, 4)) if rng.random() < 0.7 else int(rng.integers(0, 40)) for _ in ids]
            if sum(counts) == 0 or any(rows[s][0][0].shape[0] + c > 300 for s, c in zip(ids, counts)):
                continue
            free = cache.info()["free_pages"]
            try:
                cache.begin(ids, counts)
            except cb.CactusError as e:
                assert "out of pages" in str(e) and cache.info()["free_pages"] == free
                cache.free(range(seqs))
                rows = [[[np.zeros((0, ge.hkv, ge.d), np.float16)] * 2 for _ in range(layers)] for _ in range(seqs)]
                continue
            t, off = sum(counts), _offsets(counts)
            for l in range(layers):
                kv = rng.standard_normal((2, t, width)).astype(np.float16)
                q = rng.standard_normal((t, hq, ge.d)).astype(np.float16)
                d = [dev(kv[0]), dev(kv[1]), dev(q)]
                out, lse = empty((t, hq, ge.d), np.float16), empty((t, hq), np.float32)
                cache.append(l, ptr(d[0]), ptr(d[1]))
                cache.attention(l, ptr(d[2]), ptr(out), 0.1, lse=ptr(lse))
                out = host(out, np.float16).astype(np.float64)
                for i, s in enumerate(ids):
                    at = slice(off[i], off[i + 1])
                    rows[s][l] = [np.concatenate([rows[s][l][w], _quantised(kv[w, at].reshape(-1, ge.hkv, ge.d), ge.g)])
                                  for w in (0, 1)]
                    if counts[i]:
                        ref, _, tol, _ = U.attention(q[at], *rows[s][l], 0.1, True, 0)
                        assert np.all(np.abs(out[at] - ref) <= tol)
        elif kind == 3:
            src = [int(s) for s in rng.integers(0, seqs, seqs)]
            cache.fork(src, list(range(seqs)))
            rows = [[list(rows[s][l]) for l in range(layers)] for s in src]
        elif kind == 4:
            s = int(rng.integers(seqs))
            n = int(rng.integers(0, rows[s][0][0].shape[0] + 1))
            cache.truncate(s, n)
            rows[s] = [[x[:n] for x in kv] for kv in rows[s]]
        else:
            ids = rng.permutation(seqs)[:2].tolist()
            kept = [np.flatnonzero(rng.random(rows[s][0][0].shape[0]) < 0.7) for s in ids]
            try:
                cache.compact(ids, kept)
            except cb.CactusError as e:
                assert "out of pages" in str(e)
                continue
            for s, k in zip(ids, kept):
                rows[s] = [[x[k] for x in kv] for kv in rows[s]]
        for s in range(seqs):
            assert cache.length(s) == rows[s][0][0].shape[0]
            for l in range(layers):
                if cache.length(s):
                    got = _rows_of(cache, ge, l, s)
                    assert all(np.array_equal(g, r) for g, r in zip(got, rows[s][l])), (step, s, l)
    cache.free(range(seqs))
    assert cache.info()["free_pages"] == 60
    cache.close()
    assert _err() == 0


def test_cache_slide_and_refusals():
    from cactus_b200.kv4 import KVCache4
    ge = U.Geom(16, 1, 64, 32)
    cache = KVCache4(1, 2, 1, 64, num_pages=12, max_seqs=2, max_context=128, max_tokens=128, page_size=16)
    x = np.random.default_rng(1).standard_normal((100, 64)).astype(np.float16)
    d = dev(x)
    with pytest.raises(cb.CactusError, match="no batch"):
        cache.append(0, ptr(d), ptr(d))
    cache.begin([1], [100])
    cache.append(0, ptr(d), ptr(d))
    cache.slide([1], sink=4, window=20)
    kept = list(range(4)) + list(range(84, 100))
    assert np.array_equal(_rows_of(cache, ge, 0, 1)[0].reshape(-1, 64), _quantised(x, 32)[kept])
    assert cache.info()["free_pages"] == 10
    for call, why in ((lambda: cache.begin([0], [129]), "max_tokens"), (lambda: cache.begin([1], [120]), "longest context"),
                      (lambda: cache.begin([2], [1]), "no sequence"), (lambda: cache.begin([0, 0], [1, 1]), "twice"),
                      (lambda: cache.append(0, ptr(d), ptr(d)), "no batch"), (lambda: cache.truncate(1, 21), "length"),
                      (lambda: cache.compact([1], [[20]]), "kept row"), (lambda: cache.compact([1], [[-1]]), "kept row"),
                      (lambda: cache.read(0, 1, 15, 6, ptr(d), ptr(d)), "rows"), (lambda: cache.fork([0], [5]), "no sequence"),
                      (lambda: cache.read(1, 1, 0, 1, ptr(d), ptr(d)), "layer"), (lambda: cache.free([0, 7]), "no sequence")):
        with pytest.raises(cb.CactusError, match=why):
            call()
    assert cache.length(1) == 20 and cache.length(0) == 0
    cache.close()
    assert _err() == 0


def test_example_runs(capsys):
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "kv4_sampling.py")
    spec = importlib.util.spec_from_file_location("kv4_sampling", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    # 4 bits a value: a step is a fifteenth of a group's range (about 4 deviations of 32 normal values), so
    # its rounding is 0.27 / sqrt(12) = 8 % of a deviation, in the values and, through the scores, again
    assert example.main(["--prompt", "300", "--samples", "4", "--steps", "20"]) < 0.25
    assert "samples" in capsys.readouterr().out
    assert _err() == 0


@pytest.mark.parametrize("count", [2, 80])
@pytest.mark.parametrize("wrong", ["past", "falling", "negative", "again"])
def test_attention_leaves_out_token_rows_that_are_not_there(count, wrong):
    """Offsets past num_tokens, falling, negative, or naming rows twice: reported, and nothing else is written."""
    t = torch()
    L, ge = cb.lib(), U.Geom(16, 1, 64, 32)
    rng = np.random.default_rng(21)
    lens = [100, 100, 100]
    pool, table = _filled(ge, lens, rng)
    n = 3 * count
    q = rng.standard_normal((n, 2, 64)).astype(np.float16)
    off = {"past": [0, count, 2 * count, n + 1], "falling": [0, count, 0, n], "negative": [-1, count, 2 * count, n],
           "again": [0, n, 0, n]}[wrong]
    d = [dev(a) for a in (q, np.array(off, np.int32), np.array(lens, np.int32), table, pool.bytes)]
    out = t.full((n + 64, 2, 64), 7.0, dtype=t.float16, device="cuda")
    ws = empty((L.cactus_cuda_kv4_attention_workspace(3, n, 2, 1, 64),), np.uint8)
    for _ in range(2):
        cb.check(L.cactus_cuda_kv4_attention(ptr(d[0]), 128, ptr(d[1]), ptr(d[2]), ptr(d[3]), table.shape[1], ptr(d[4]),
                                             pool.pages, pool.stride, out.data_ptr(), None, 3, n, n, 2, *ge.args(), 0.125,
                                             0, 1, ptr(ws), ws.numel(), None))
        assert _err() == 3
    assert bool((out[n:] == 7.0).all())
    got = out.cpu().numpy()
    if wrong in ("past", "negative"):  # the sequences whose rows are there
        b = 0 if wrong == "past" else 1
        at = slice(b * count, (b + 1) * count)
        k, v = (pool.rows(w, table[b], 100) for w in (0, 1))
        ref, _, tol, _ = U.attention(q[at], k, v, 0.125, True, 0)
        assert np.all(np.abs(got[at].astype(np.float64) - ref) <= tol)
