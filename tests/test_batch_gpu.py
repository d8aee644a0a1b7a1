"""A ragged batch's operators (include/cactus_b200_batch.h) against the 64-bit statements of tests/batch_util.py."""
import numpy as np
import pytest

import cactus_b200 as cb
from cactus_b200 import batch
from tests import batch_util as U
from tests.gpu_util import dev, empty, host, torch

pytestmark = pytest.mark.gpu


def _err():
    return cb.lib().cactus_cuda_device_error(None)


def _padded(a, stride, rng, offset=0):
    """Rows of `a` on the device, `stride` elements apart behind `offset` elements of something else."""
    flat = (rng.integers(0, 1 << 16, offset + a.shape[0] * stride + 64, dtype=np.uint64).astype(np.uint16)).view(a.dtype)
    rows = flat[offset:offset + a.shape[0] * stride].reshape(a.shape[0], stride)
    rows[:, :a.shape[1]] = a
    t = dev(flat)
    return t, t.data_ptr() + offset * a.itemsize


# ---------------------------------------------------------------------------------------- residual, RMSNorm, 8 bits
def _check_norm(x, r, w, eps, got_sum, codes, scales, normed):
    s = U.add16(x, r) if r is not None else x
    if got_sum is not None:
        assert np.array_equal(got_sum.view(np.uint16)[~np.isnan(s)], s.view(np.uint16)[~np.isnan(s)])
        assert np.isnan(got_sum[np.isnan(s)]).all()
    y, tol = U.norm(s, w, eps)
    if normed is not None:
        U.within(normed, np.where(np.abs(y) > 65519, np.copysign(np.inf, y), y), tol + U.fp16_step(y))
    if codes is not None:
        with np.errstate(invalid="ignore"):
            top = np.abs(y).max(-1)
            bad = ~(top < 3.4e38)
        assert np.isnan(scales[bad]).all() and (codes[bad] == 0).all()
        unit = np.maximum(top / 127, float(np.float32(1e-10)))[~bad]
        assert (np.abs(scales[~bad] - unit) <= 5 * U.U32 * unit).all()
        # a code is off its quotient by a half, and by what the quotient's steps leave: 8 of 2^-24 of 127
        q = y[~bad] / unit[:, None]
        assert (np.abs(codes[~bad] - q) <= 0.5 + 127 * 8 * U.U32).all()


def _norm(x, w, r=None, xs=None, rs=None, eps=1e-6, want="sqn", inplace=None, rng=None, offset=0):
    rows, dims = x.shape
    rng = rng or np.random.default_rng(0)
    tx, px = _padded(x, xs or dims, rng, offset)
    tr, pr = _padded(r, rs or dims, rng, offset) if r is not None else (None, None)
    tw = dev(w)
    total = empty((rows, dims), np.float16) if "s" in want else None
    codes, scales = (empty((rows, dims), np.int8), empty((rows,), np.float32)) if "q" in want else (None, None)
    normed = empty((rows, dims), np.float16) if "n" in want else None
    before = host(tx, np.uint16).copy()
    ps, ss = (None, None) if total is None else (total.data_ptr(), dims)
    if inplace:
        ps, ss = (px, xs or dims) if inplace == "x" else (pr, rs or dims)
    batch.add_rms_norm_q8(px, tw, rows, dims, codes, scales, normed, pr, ps, eps, xs or dims, rs or dims, ss)
    if inplace:
        flat = host(tx if inplace == "x" else tr, np.float16)
        got = flat[offset:offset + rows * ss].reshape(rows, ss)[:, :dims].copy()
    else:
        got = None if total is None else host(total, np.float16)
        assert np.array_equal(host(tx, np.uint16), before)
    got = got, None if codes is None else host(codes, np.int8), None if codes is None else host(scales, np.float32), \
        None if normed is None else host(normed, np.float16)
    _check_norm(x, r, w, eps, *got)
    assert _err() == 0
    return got


def _rows(rng, rows, dims, scale=1.0):
    return (rng.standard_normal((rows, dims)) * scale).astype(np.float16)


@pytest.mark.parametrize("dims", [1, 2, 7, 8, 31, 64, 100, 256, 1000, 1024, 1032, 2048, 2056, 4096, 5000, 8192, 8200, 12288, 16384,
                                  20001, 32760, 32768])
@pytest.mark.parametrize("rows", [1, 5])
def test_norm_dims(rows, dims):
    rng = np.random.default_rng(dims)
    _norm(_rows(rng, rows, dims, 2.0), _rows(rng, 1, dims)[0], _rows(rng, rows, dims))


@pytest.mark.parametrize("want", ["s", "q", "n", "sq", "qn", "sqn", "sn"])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_outputs(want, residual):
    if "q" not in want and "n" not in want:
        want += "n"
    rng = np.random.default_rng(3)
    for dims in (264, 1030):
        _norm(_rows(rng, 6, dims), _rows(rng, 1, dims)[0], _rows(rng, 6, dims) if residual else None, want=want)


@pytest.mark.parametrize("dims,xs,rs,offset", [(512, 1024, 520, 0), (512, 515, 600, 0), (512, 512, 512, 1), (512, 520, 512, 8),
                                               (77, 80, 77, 3), (4096, 12288, 4096, 0), (16384, 16385, 16400, 5)])
@pytest.mark.parametrize("inplace", [None, "x", "r"])
def test_norm_strides_alignment_and_in_place(dims, xs, rs, offset, inplace):
    rng = np.random.default_rng(dims + offset)
    _norm(_rows(rng, 7, dims), _rows(rng, 1, dims)[0], _rows(rng, 7, dims), xs, rs, inplace=inplace, rng=rng, offset=offset)


def test_norm_many_rows_and_extreme_values():
    rng = np.random.default_rng(9)
    x, r = _rows(rng, 1500, 192), _rows(rng, 1500, 192)
    x[0], r[0] = 0, 0                       # eps alone
    x[1] *= np.float16(2.0 ** -10)          # near fp16's smallest
    x[2], r[2] = 6e-8, 0
    x[3], r[3] = 60000, 0
    x[4, 5], r[4, 5] = 60000, 60000         # the sum is infinite: a row that shows it
    x[5, 0] = np.nan
    x[6, 191], r[6, 191] = np.inf, -np.inf
    x[7], r[7, :] = 0, 0
    x[7, 3] = 1.0                           # one element has all of the norm
    w = _rows(rng, 1, 192)[0]
    w[10], w[11] = 0, -w[11]
    for eps in (1e-6, 1e-5, 0.1):
        _norm(x, w, r, eps=eps)
    _norm(x[1:], w, r[1:], eps=0.0)
    w[20] = np.inf
    _norm(x[8:12], w, r[8:12])


def test_norm_codes_feed_the_projection():
    """matmul_int8 of the codes: the product of what they stand for, to its own two roundings."""
    rng = np.random.default_rng(12)
    rows, k, n, g = 20, 256, 96, 32
    x, w = _rows(rng, rows, k), _rows(rng, 1, k)[0]
    q, s = empty((rows, k), np.int8), empty((rows,), np.float32)
    tx, tw = dev(x), dev(w)
    batch.add_rms_norm_q8(tx, tw, rows, k, q, s)
    b = rng.integers(-127, 128, (n, k)).astype(np.int8)
    bs = (rng.random((n, k // g)) * 0.01 + 0.001).astype(np.float16)
    tb, tbs, c = dev(b), dev(bs), empty((rows, n), np.float16)
    cb.check(cb.lib().cactus_cuda_matmul_int8(q.data_ptr(), s.data_ptr(), tb.data_ptr(), tbs.data_ptr(), c.data_ptr(), rows, k,
                                              n, g, None))
    a = host(q, np.int8).astype(np.float64) * host(s, np.float32).astype(np.float64)[:, None]
    full = b.astype(np.float64) * np.repeat(bs.astype(np.float64), g, 1)
    ref, size = a @ full.T, np.abs(a) @ np.abs(full).T
    U.within(host(c, np.float16), ref, U.fp16_step(ref) + (k // g + 4) * U.U32 * size)


# ---------------------------------------------------------------------------------------- adapters
class Lora:
    """Arguments of a lora call on the device; rows and columns past an adapter's rank hold NaN."""

    def __init__(self, counts, ids, ranks, k, n, rng, top=None, pad=0, extra=0, tokens=None, integers=False, scales=True,
                 spread=1.0):
        self.ids, self.ranks, self.k, self.n, self.ad = list(ids), list(ranks), k, n, len(ranks)
        self.top = top or max(8, -(-max(list(ranks) + [1]) // 8) * 8)
        ends = np.cumsum(counts).tolist()
        self.seqs = list(zip([0] + ends[:-1], ends))
        self.t = tokens or ends[-1] + extra
        make = (lambda *s: rng.integers(-3, 4, s).astype(np.float16)) if integers else \
            (lambda *s: rng.standard_normal(s).astype(np.float16))
        self.x, self.base = make(self.t, k), make(self.t, n)
        ad = max(self.ad, 1)
        self.a, self.b = make(ad, self.top, k), make(ad, n, self.top)
        if not integers:
            self.a = (self.a * (max(k, 1) ** -0.5 * spread)).astype(np.float16)
        for i, r in enumerate(self.ranks):
            self.a[i, r:], self.b[i, :, r:] = np.nan, np.nan
        self.scales = (rng.random(ad) + 0.5).astype(np.float32) if scales else np.ones(ad, np.float32)
        self.dx, self.px = _padded(self.x, k + pad, rng)
        self.dbase, self.pbase = _padded(self.base, n + pad, rng)
        self.pad = pad
        self.da, self.db = dev(self.a), dev(self.b)
        self.dr, self.ds = dev(np.array(self.ranks + [0], np.int32)), dev(self.scales) if scales else None
        self.off = dev(np.array([0] + ends, np.int32))
        self.did = dev(np.array(self.ids, np.int32))
        s = len(self.ids)
        self.pb = batch.lora_plan_bytes(s, self.t, self.ad)
        self.wb = batch.lora_workspace(self.t, self.top)
        self.dplan, self.ws = dev(rng.integers(0, 256, self.pb).astype(np.uint8)), dev(np.full(self.wb, 0xFF, np.uint8))
        self.out = empty((self.t, n + pad), np.float16)
        self.out.fill_(np.float16(123.0).view(np.int16).item())

    def plan(self, stream=0):
        batch.lora_plan(self.off, self.did, len(self.ids), self.t, self.ad, self.dplan, self.pb, stream)

    def run(self, base=True, out=None, ranks=True, stream=0):
        batch.lora(self.px, self.da, self.db, self.out if out is None else out, self.dplan, self.pb, len(self.ids), self.t,
                   self.ad, self.top, self.k, self.n, self.ws, self.wb, self.pbase if base else None,
                   self.dr if ranks else None, self.ds, self.k + self.pad, self.n + self.pad, self.n + self.pad, stream)

    def got(self, flat=None):
        return (host(self.out, np.float16) if flat is None else flat)[:, :self.n]

    def check(self, base=True, got=None):
        got = self.got() if got is None else got
        ref, tol = U.lora(self.x, self.a, self.b, self.ranks, self.scales, self.base if base else np.zeros_like(self.base),
                          self.seqs, self.ids)
        end = self.seqs[-1][1]
        U.within(got[:end], ref[:end], tol[:end])
        assert (got[end:] == np.float16(123.0)).all()  # rows of no sequence
        if self.pad:
            assert (host(self.out, np.float16)[:, self.n:] == np.float16(123.0)).all()
        assert _err() == 0

    def both(self, **kw):
        self.plan()
        self.run(**kw)
        self.check(kw.get("base", True))


@pytest.mark.parametrize("counts", [[1], [1] * 9, [1, 0, 3], [2, 5, 1, 8], [63], [64], [65], [200, 1, 0, 130], [7] * 40])
@pytest.mark.parametrize("rank", [1, 8, 13, 16, 40, 64])
def test_lora_counts_and_ranks(counts, rank):
    rng = np.random.default_rng(rank * 100 + len(counts))
    ids = [i % 3 for i in range(len(counts))]
    Lora(counts, ids, [rank, max(1, rank // 2), rank], 128, 136, rng, extra=5, pad=8).both()


@pytest.mark.parametrize("k", [8, 16, 24, 40, 64, 72, 200, 1024, 2056])
@pytest.mark.parametrize("n", [8, 24, 64, 264, 1000])
@pytest.mark.parametrize("counts", [[1, 1, 3], [90, 20]])
def test_lora_features(k, n, counts):
    rng = np.random.default_rng(k + n)
    Lora(counts, [0, 1, 0][:len(counts)], [16, 5], k, n, rng).both()


@pytest.mark.parametrize("rank,top", [(128, 128), (256, 256), (200, 256), (72, 72), (3, 256), (250, 256), (104, 104)])
@pytest.mark.parametrize("counts", [[4], [150]])
def test_lora_large_ranks(rank, top, counts):
    rng = np.random.default_rng(rank)
    Lora(counts, [0], [rank], 264, 200, rng, top=top).both()


def test_lora_many_adapters_bare_sequences_and_none_at_all():
    rng = np.random.default_rng(4)
    ids = rng.integers(-1, 50, 300).tolist()
    Lora(rng.integers(0, 4, 300).tolist(), ids, rng.integers(0, 20, 50).tolist(), 72, 96, rng, extra=3).both()
    Lora([3, 4], [-1, -1], [8], 64, 64, rng, extra=2).both()
    Lora([5, 80], [0, -1], [0], 64, 64, rng).both()        # an adapter of rank 0
    call = Lora([5, 80], [-1, -1], [], 64, 64, rng)        # no adapters
    call.both()
    Lora([0, 0, 0], [0, 1, 0], [8, 8], 64, 64, rng, tokens=4).both()  # no rows
    Lora([2] * 1500, (np.arange(1500) % 1200).tolist(), [8] * 1200, 64, 32, rng).both()
    Lora([3, 70], [0, 1], [4, 8], 64, 64, rng, scales=False).both(base=False)


def test_lora_in_place_and_without_ranks():
    rng = np.random.default_rng(5)
    for counts in ([1, 2, 1], [100, 3, 64]):
        call = Lora(counts, [1, -1, 0], [16, 16], 96, 104, rng)
        call.plan()
        call.run(out=call.pbase, ranks=False)
        call.check(got=host(call.dbase, np.float16)[:call.t * call.n].reshape(call.t, call.n))


@pytest.mark.parametrize("counts", [[3], [120]])
def test_lora_middle_product_keeps_its_bits(counts):
    """Whole numbers whose middle product has 15 bits and more: every step is exact but the last rounding."""
    rng = np.random.default_rng(6)
    call = Lora(counts, [0], [24], 512, 80, rng, integers=True, scales=False)
    call.x[:, ::2], call.a[0, :24, ::2] = 29, 31   # 256 * 899 = 230144 of 18 bits
    call.b[0, :, 0] = 1 + call.b[0, :, 1]          # large parts that cancel
    call.b[0, :, 2:24] = 0
    call.b[0, :, 1] = -call.b[0, :, 0]
    call.dx, call.px = _padded(call.x, 512, rng)
    call.da, call.db = dev(call.a), dev(call.b)
    call.plan()
    call.run()
    x, a, b = call.x.astype(np.float64), call.a[0, :24].astype(np.float64), call.b[0, :, :24].astype(np.float64)
    want = (call.base.astype(np.float64) + (x @ a.T) @ b.T).astype(np.float16)
    assert np.array_equal(call.got(), want)


def test_lora_infinities_and_nan_stay_in_their_rows():
    rng = np.random.default_rng(7)
    for counts, ids in (([6, 6], [0, 1]), ([100, 90], [0, 1])):
        call = Lora(counts, ids, [16, 8], 128, 72, rng)
        x = call.x.copy()
        x[2, 5], x[4, 100], x[counts[0] + 1] = np.nan, np.inf, 60000
        call.x = x
        call.dx, call.px = _padded(x, 128, rng)
        call.plan()
        call.run()
        got = call.got()
        rows = np.ones(call.t, bool)
        rows[[2, 4]] = False
        ref, tol = U.lora(call.x, call.a, call.b, call.ranks, call.scales, call.base, call.seqs, call.ids)
        with np.errstate(over="ignore"):
            over = np.abs(ref) + tol > 65504  # may be infinite
        ok = np.abs(got[rows].astype(np.float64) - ref[rows]) <= tol[rows]
        assert (ok | (over[rows] & (np.sign(got[rows]) == np.sign(ref[rows])))).all()
        assert np.isnan(got[2]).all() and not np.isfinite(got[4]).any()


@pytest.mark.parametrize("rank", [1, 3, 8, 21])
@pytest.mark.parametrize("counts,ids,n", [([6], [0], 72), ([40], [0], 72), ([100], [0], 72), (None, [0, 0], 1608), ([300], [0], 2800)])
def test_lora_an_infinity_keeps_its_sign(counts, ids, n, rank):
    """Factors of one sign: the row's results are infinities, whatever the rank is padded with."""
    rng = np.random.default_rng(rank)
    top = 40 if n == 2800 else 24 if counts else 64  # 40, 64: both products by the kernels of much work
    call = Lora(counts or _wide(n, top, [70, 60]), ids, [rank], 128, n, rng, top=top)
    call.a, call.b, call.x = np.abs(call.a), np.abs(call.b) + np.float16(0.01), np.abs(call.x) + np.float16(0.01)
    call.a[0, :rank] += np.float16(0.01)
    call.x[2, 5], call.x[4, 127] = np.inf, -np.inf
    call.da, call.db = dev(call.a), dev(call.b)
    call.dx, call.px = _padded(call.x, 128, rng)
    call.plan()
    call.run()
    got, rows = call.got(), np.ones(call.t, bool)
    rows[[2, 4]] = False
    ref, tol = U.lora(call.x, call.a, call.b, call.ranks, call.scales, call.base, call.seqs, call.ids)
    U.within(got[rows], ref[rows], tol[rows])
    assert (got[2] == np.inf).all() and (got[4] == -np.inf).all()


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("rank", [2, 7, 21])
@pytest.mark.parametrize("counts,n,top", [
    ([6, 2], 72, 24),        # one kernel, a cluster of blocks a tile
    ([40, 20], 72, 24), ([40, 20], 72, 256), ([130], 264, 24), ([5, 90], 264, 200),  # both products by lora.cu's two kernels
    ([520, 3], 8192, 32),    # the second product by tcgen05
    ([300, 20], 2800, 40), ([300, 20], 2800, 104),  # both of them
])
def test_lora_an_infinity_of_an_adapter_beside_large_sums(counts, n, top, rank, sign):
    """One infinity in a's first row, sums past fp16's end in its others: their products are finite, of either sign, so that
    the results are the infinity's, rows of the other adapter what they are without it."""
    rng = np.random.default_rng(1000 * rank + top)
    call = Lora(counts, range(len(counts)), [rank, 8][:len(counts)], 128, n, rng, top=top)
    call.x[:counts[0]] = rng.uniform(50, 100, (counts[0], 128))
    call.x[:counts[0], 77] *= np.where(np.arange(counts[0]) % 3 == 1, -1, 1).astype(np.float16)
    call.a[0, 1:rank] = rng.uniform(20, 40, (rank - 1, 128))  # sums from 126 * 50 * 20 on: above 65504
    call.a[0, 0, 77] = np.inf
    call.b[0, :, :rank] = np.abs(call.b[0, :, :rank]) + np.float16(0.01)
    call.b[0, :, 1:rank] *= np.float16(sign)
    call.da, call.db = dev(call.a), dev(call.b)
    call.dx, call.px = _padded(call.x, 128, rng)
    call.plan()
    call.run()
    got = call.got()
    want = np.where(call.x[:counts[0], 77] > 0, np.inf, -np.inf)[:, None]
    assert (got[:counts[0]] == want).all()
    call.ids[0] = -1  # the others' rows
    ref, tol = U.lora(call.x, call.a, call.b, call.ranks, call.scales, call.base, call.seqs, call.ids)
    U.within(got[counts[0]:], ref[counts[0]:], tol[counts[0]:])
    assert _err() == 0


def test_lora_refuses_lists_on_the_device():
    """Offsets that fall or pass the tokens: no row; ids and ranks that are none: rows as without an adapter."""
    rng = np.random.default_rng(8)
    for off in ([0, 5, 3, 9], [0, 4, 8, 500], [-1, 3, 5, 9]):
        call = Lora([3, 3, 3], [0, 1, 0], [8, 8], 64, 64, rng)
        call.off = dev(np.array(off, np.int32))
        call.plan()
        call.run()
        assert (call.got() == np.float16(123.0)).all() and _err() == 4
    call = Lora([3, 3, 3], [0, 1, 2], [8, 8], 64, 64, rng)
    call.ids = [0, 2, -2]
    call.did = dev(np.array(call.ids, np.int32))
    call.plan()
    call.run()
    assert _err() == 4
    call.ids = [0, -1, -1]
    call.check()
    for rank in (9, -1):
        call = Lora([3, 70], [0, 1], [8, 8], 64, 64, rng)
        call.dr = dev(np.array([8, rank], np.int32))
        call.plan()
        call.run()
        assert _err() == 4
        call.ids = [0, -1]
        call.check()
    call = Lora([3, 3], [0, 1], [8, 8], 64, 64, rng)  # a plan of other numbers
    call.plan()
    call.did = dev(np.array([0, 1, 0], np.int32))
    call.ids = [0, 1, 0]
    call.pb = batch.lora_plan_bytes(3, call.t, 2)
    call.dplan = torch().cat([call.dplan, call.dplan])
    call.run()
    assert (call.got() == np.float16(123.0)).all() and _err() == 4


def test_lora_is_the_same_every_time_and_when_replayed():
    """Bits of repeated calls, a captured plan and call whose adapters, offsets and inputs change, two streams."""
    t = torch()
    rng = np.random.default_rng(10)
    for counts in ([1] * 20, [150, 1, 90, 3]):
        ids = rng.integers(-1, 3, len(counts)).tolist()
        call = Lora(counts, ids, [16, 8, 24], 512, 264, rng)
        call.both()
        first = call.got().view(np.uint16).copy()
        for _ in range(10):
            call.ws.fill_(255)
            call.plan()
            call.run()
            assert np.array_equal(call.got().view(np.uint16), first)
        t.cuda.synchronize()
        graph = t.cuda.CUDAGraph()
        with t.cuda.graph(graph):
            stream = t.cuda.current_stream().cuda_stream
            call.plan(stream)
            call.run(stream=stream)
        graph.replay()
        call.check()
        call.ids = [2 - max(i, 0) for i in call.ids]
        call.did.copy_(t.tensor(call.ids, dtype=t.int32))
        ends = np.cumsum(counts[::-1])
        call.seqs = list(zip([0] + ends[:-1].tolist(), ends.tolist()))
        call.off.copy_(t.tensor([0] + ends.tolist(), dtype=t.int32))
        graph.replay()
        call.check()
    one, two = (Lora([40, 1, 9], [0, 1, 0], [16, 8], 256, 128, rng) for _ in range(2))
    streams = t.cuda.Stream(), t.cuda.Stream()
    t.cuda.synchronize()
    for _ in range(20):
        for call, stream in zip((one, two), streams):
            call.plan(stream.cuda_stream)
            call.run(stream=stream.cuda_stream)
    t.cuda.synchronize()
    one.check()
    two.check()


def test_lora_split_product_over_a_long_row():
    rng = np.random.default_rng(11)
    Lora([1], [0], [16], 16384, 64, rng).both()
    Lora([1, 1], [0, 1], [64, 64], 8200, 64, rng).both()
    Lora([130], [0], [64], 8200, 72, rng).both()


# Few tokens for as many adapters as there may be: both products by a cluster of blocks a tile, of 8 or of 4.
@pytest.mark.parametrize("seqs", [1, 6, 30, 60])
@pytest.mark.parametrize("k,n", [(8, 8), (40, 24), (264, 1000), (2048, 72), (1000, 2056)])
@pytest.mark.parametrize("rank", [3, 16, 29, 64])
def test_lora_tokens_by_clusters(seqs, k, n, rank):
    rng = np.random.default_rng(seqs + k + rank)
    ids = rng.integers(-1, seqs, seqs).tolist()
    ranks = rng.integers(0, rank + 1, seqs).tolist()
    ranks[0] = rank
    Lora(rng.integers(0, 4, seqs).tolist() if seqs > 1 else [8], ids, ranks, k, n, rng, extra=3, pad=8).both()


def test_lora_tokens_by_clusters_skewed_in_place_and_replayed():
    t = torch()
    rng = np.random.default_rng(31)
    # all rows of one adapter: tiles of 64 rows, 8 at a time; none of any; one of each
    for ids in ([3] * 50, [-1] * 50, list(range(50)), [7] * 49 + [-1]):
        call = Lora([8] * 50, ids, [16] * 50, 136, 264, rng)
        call.both()
        call.both(base=False)
        call = Lora([8] * 50, ids, [16] * 50, 136, 264, rng)
        call.plan()
        call.run(out=call.pbase)
        call.check(got=host(call.dbase, np.float16)[:call.t * call.n].reshape(call.t, call.n))
    call = Lora([1] * 64, rng.integers(-1, 64, 64).tolist(), [24] * 64, 512, 392, rng)
    call.both()
    first = call.got().view(np.uint16).copy()
    for _ in range(20):
        call.ws.fill_(255)
        call.out.fill_(0)
        call.run()
        assert np.array_equal(call.got().view(np.uint16), first)
    t.cuda.synchronize()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        stream = t.cuda.current_stream().cuda_stream
        call.plan(stream)
        call.run(stream=stream)
    for ids in ([5] * 64, [-1] * 63 + [0], rng.integers(-1, 64, 64).tolist()):
        call.ids = ids
        call.did.copy_(t.tensor(ids, dtype=t.int32))
        call.out.fill_(np.float16(123.0).view(np.int16).item())
        for _ in range(3):
            graph.replay()
        call.check()
    x = call.x.copy()
    x[2, 5], x[40, 100] = np.nan, np.inf
    call.x = x
    call.ids = list(range(64))
    call.did.copy_(t.arange(64, dtype=t.int32))
    call.dx, call.px = _padded(x, 512, rng)
    call.plan()
    call.run()
    got, rows = call.got(), np.ones(64, bool)
    rows[[2, 40]] = False
    ref, tol = U.lora(call.x, call.a, call.b, call.ranks, call.scales, call.base, call.seqs, call.ids)
    U.within(got[rows], ref[rows], tol[rows])
    assert np.isnan(got[2]).all() and not np.isfinite(got[40]).any()


# Batches of so much work (tokens * outputs * rank) that the second product has tiles of 128 rows and goes over items
# ahead of one another.
WIDE = 1 << 27


def _wide(n, top, pattern):
    """Token counts in the pattern's proportions that make enough work."""
    t = WIDE // (n * top) + 1
    counts = [max(p > 0, p * t // sum(pattern)) for p in pattern]
    counts[0] += max(0, t - sum(counts))
    return counts


@pytest.mark.parametrize("pattern", [[1], [511, 1], [1] * 4, [129, 0, 127, 300], [70] * 12, [37] * 40, [1] * 900])
@pytest.mark.parametrize("rank", [1, 16, 40, 64, 100, 128])
def test_lora_many_rows(pattern, rank):
    rng = np.random.default_rng(rank * 100 + len(pattern))
    n = 1544
    counts = _wide(n, -(-rank // 8) * 8, pattern)
    ids = [(i * 5) % 4 - 1 for i in range(len(counts))] if len(counts) > 1 else [1]
    Lora(counts, ids, [rank, max(1, rank // 2), rank], 72, n, rng, extra=5, pad=8).both()


@pytest.mark.parametrize("n", [8, 64, 120, 128, 136, 264, 2000])
@pytest.mark.parametrize("k", [8, 200])
@pytest.mark.parametrize("top", [64, 128])
def test_lora_many_rows_features(n, k, top):
    if n * k == 1600:
        k = 40
    rng = np.random.default_rng(n + k + top)
    counts = _wide(n, top, [300, 40, 260, 5])
    for base in (True, False):
        Lora(counts, [0, 1, -1, 0], [top - 11, 5], k, n, rng, top=top).both(base=base)


def test_lora_many_rows_of_many_adapters_and_of_few():
    rng = np.random.default_rng(14)
    ids = rng.integers(-1, 60, 400).tolist()
    for top in (64, 128):
        counts = rng.integers(0, 9, 400) * (WIDE // (1032 * top * 1600) + 1)
        Lora(counts.tolist(), ids, rng.integers(0, top + 1, 60).tolist(), 72, 1032, rng, extra=WIDE // (1032 * top), top=top).both()
        counts = _wide(776, top, [300, 400])
        Lora(counts, [-1, -1], [8], 64, 776, rng, extra=2, top=top).both()
        Lora(counts, [0, -1], [0], 64, 776, rng, top=top).both()
        call = Lora(_wide(776, top, [100, 350, 164, 30]), [1, -1, 0, 1], [top, 16], 96, 776, rng, top=top)
        call.plan()
        call.run(out=call.pbase)  # in place
        call.check(got=host(call.dbase, np.float16)[:call.t * call.n].reshape(call.t, call.n))
    Lora([1300, 3], [0, 1], [4, 200], 64, 1320, rng).both()  # a rank past that kernel's


def test_lora_many_rows_keep_their_bits():
    """As test_lora_middle_product_keeps_its_bits; and calls repeated, and replayed with other lists."""
    rng = np.random.default_rng(15)
    call = Lora(_wide(1040, 24, [1]), [0], [24], 512, 1040, rng, integers=True, scales=False)
    call.x[:, ::2], call.a[0, :24, ::2] = 29, 31
    call.b[0, :, 0] = 1 + call.b[0, :, 1]
    call.b[0, :, 2:24] = 0
    call.b[0, :, 1] = -call.b[0, :, 0]
    call.dx, call.px = _padded(call.x, 512, rng)
    call.da, call.db = dev(call.a), dev(call.b)
    call.plan()
    call.run()
    x, a, b = call.x.astype(np.float64), call.a[0, :24].astype(np.float64), call.b[0, :, :24].astype(np.float64)
    assert np.array_equal(call.got(), (call.base.astype(np.float64) + (x @ a.T) @ b.T).astype(np.float16))
    t = torch()
    counts = _wide(1608, 64, [150, 1, 290, 3, 300, 65])
    call = Lora(counts, [2, 1, 0, -1, 2, 0], [64, 8, 24], 512, 1608, rng)
    call.both()
    first = call.got().view(np.uint16).copy()
    for _ in range(20):
        call.ws.fill_(255)
        call.out.fill_(0)
        call.run()
        assert np.array_equal(call.got().view(np.uint16), first)
    t.cuda.synchronize()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        stream = t.cuda.current_stream().cuda_stream
        call.plan(stream)
        call.run(stream=stream)
    for ids, order in (([0, 0, 1, 2, -1, 1], counts[::-1]), ([-1] * 6, counts), ([1] * 6, [0, call.t - 9, 0, 0, 9, 0])):
        call.ids = ids
        call.did.copy_(t.tensor(ids, dtype=t.int32))
        ends = np.cumsum(order)
        call.seqs = list(zip([0] + ends[:-1].tolist(), ends.tolist()))
        call.off.copy_(t.tensor([0] + ends.tolist(), dtype=t.int32))
        call.out.fill_(np.float16(123.0).view(np.int16).item())
        for _ in range(3):
            graph.replay()
        call.check()


# Ranks above 32 and 2^25 of work: the first product on the same tensor cores, its tiles of 64 or 128 rows, whole or in
# parts of K.
@pytest.mark.parametrize("k", [0, 8, 72, 136, 264, 1000, 2056])
@pytest.mark.parametrize("ranks", [[33], [64, 3, 17], [100, 0, 128]])
def test_lora_first_product_of_many_rows(k, ranks):
    rng = np.random.default_rng(k + len(ranks))
    counts = [150, 64, 0, 65, 1, 130]
    ids = [0, 1, 2, 2, -1, 0] if len(ranks) > 1 else [0, 0, 0, 0, -1, 0]
    top = max(40, -(-max(ranks) // 8) * 8)
    n = -(-2 ** 25 // (sum(counts) * top) // 8) * 8 + 8
    Lora(counts, ids, ranks, k, n, rng, top=top, extra=7, pad=8).both()


@pytest.mark.parametrize("t,k,ranks", [(64, 4096, [48]), (300, 14344, [40, 33]), (9600, 136, [64]), (30000, 136, [64, 20]),
                                       (20000, 136, [40]), (16400, 2056, [16]), (8200, 4104, [8, 32])])
def test_lora_first_product_by_tiles_and_parts(t, k, ranks):
    """Few tiles in many parts; more tiles than there are blocks, of either height; ranks up to 32 of much work."""
    rng = np.random.default_rng(t)
    top = -(-max(ranks) // 8) * 8
    work = 2 ** 25 if top > 32 else 2 ** 27
    n = max(24, -(-work // (t * top) // 8) * 8 + 8)
    counts = [t // 2 + 3, t - t // 2 - 3]
    Lora(counts, [0, len(ranks) - 1], ranks, k, n, rng, top=top, extra=3).both()


def test_lora_first_product_of_many_rows_replayed():
    """Other tokens, adapters and rows by the same graph, its second kernel launched while the first one ends."""
    t = torch()
    rng = np.random.default_rng(91)
    call = Lora([200, 100, 90], [0, 1, 1], [64, 40], 1032, 2048, rng)
    stream = t.cuda.Stream()
    stream.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(stream):
        call.plan(stream.cuda_stream)
        call.run(stream=stream.cuda_stream)
    stream.synchronize()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph, stream=stream):
        call.plan(t.cuda.current_stream().cuda_stream)
        call.run(stream=t.cuda.current_stream().cuda_stream)
    for ids in ([1, 0, 0], [-1, -1, 0], [0, 0, 0]):
        call.ids = ids
        call.did.copy_(t.tensor(ids, dtype=t.int32))
        call.out.fill_(np.float16(123.0).view(np.int16).item())
        for _ in range(3):
            graph.replay()
        call.check()


def test_lora_first_product_of_many_rows_refuses_lists_on_the_device():
    """As test_lora_refuses_lists_on_the_device."""
    rng = np.random.default_rng(92)
    for rank in (65, -1):
        call = Lora([200, 100], [0, 1], [64, 40], 136, 2048, rng)
        call.dr = dev(np.array([64, rank], np.int32))
        call.plan()
        call.run()
        assert _err() == 4
        call.ids = [0, -1]
        call.check()
    call = Lora([200, 100], [0, 1], [64, 40], 136, 2048, rng)  # a plan of other numbers
    call.plan()
    call.did = dev(np.array([0, 1, 0], np.int32))
    call.ids = [0, 1, 0]
    call.pb = batch.lora_plan_bytes(3, call.t, 2)
    call.dplan = torch().cat([call.dplan, call.dplan])
    call.run()
    assert (call.got() == np.float16(123.0)).all() and _err() == 4
    call = Lora([200, 100], [0, 1], [64, 40], 136, 2048, rng)  # lists that fall: a plan without rows
    call.off = dev(np.array([0, 200, 100], np.int32))
    call.plan()
    call.run()
    assert (call.got() == np.float16(123.0)).all() and _err() == 4


def test_lora_many_rows_infinities_and_nan_stay_in_their_rows():
    rng = np.random.default_rng(16)
    call = Lora(_wide(1608, 64, [300, 290]), [0, 1], [64, 40], 128, 1608, rng)
    odd = call.seqs[0][1]
    call.x[2, 5], call.x[odd - 10, 100], call.x[odd + 1] = np.nan, np.inf, 60000
    call.dx, call.px = _padded(call.x, 128, rng)
    call.plan()
    call.run()
    got = call.got()
    rows = np.ones(call.t, bool)
    rows[[2, odd - 10]] = False
    ref, tol = U.lora(call.x, call.a, call.b, call.ranks, call.scales, call.base, call.seqs, call.ids)
    with np.errstate(over="ignore"):
        over = np.abs(ref) + tol > 65504  # may be infinite
    ok = np.abs(got[rows].astype(np.float64) - ref[rows]) <= tol[rows]
    assert (ok | (over[rows] & (np.sign(got[rows]) == np.sign(ref[rows])))).all()
    assert np.isnan(got[2]).all() and not np.isfinite(got[odd - 10]).any()


def test_lora_many_rows_on_two_streams():
    t = torch()
    rng = np.random.default_rng(17)
    one, two = (Lora(_wide(1544, top, [40, 1, 9]), [0, 1, 0], [top, 8], 256, 1544, rng) for top in (64, 128))
    streams = t.cuda.Stream(), t.cuda.Stream()
    t.cuda.synchronize()
    for _ in range(10):
        for call, stream in zip((one, two), streams):
            call.plan(stream.cuda_stream)
            call.run(stream=stream.cuda_stream)
    t.cuda.synchronize()
    one.check()
    two.check()


# ---------------------------------------------------------------------------------------- logits
class Logits:
    def __init__(self, rows, vocab, rng, history=None, biases=None, masks=None, penalties=None, prompts=None, pad=0, opad=None,
                 offset=0, mask_pad=0, x=None):
        self.rows, self.v, self.pad, self.opad = rows, vocab, pad, pad if opad is None else opad
        self.x = (rng.standard_normal((rows, vocab)) * 4).astype(np.float16) if x is None else x
        self.histories = history
        self.prompts = prompts if prompts is not None else ([0] * rows if history is not None else None)
        self.penalties = penalties if penalties is not None else np.tile(np.float32([1.3, 0.25, 0.5]), (rows, 1))
        if history is None:
            self.penalties = None
        self.biases, self.masks = biases, masks
        self.dx, self.px = _padded(self.x, vocab + pad, rng, offset)
        self.offset = offset
        flat = np.full(offset + rows * (vocab + self.opad), 123.0, np.float16)
        self.dout = dev(flat)
        self.pout = self.dout.data_ptr() + 2 * offset
        self.kw = {}
        if history is not None:
            flat = np.concatenate([np.asarray(h, np.uint32) for h in history] + [np.zeros(1, np.uint32)])
            self.kw.update(penalties=dev(self.penalties), history=dev(flat),
                           history_offsets=dev(np.cumsum([0] + [len(h) for h in history]).astype(np.int32)),
                           num_history=flat.size - 1, prompt_lens=None if prompts is None else dev(np.array(prompts, np.int32)))
        if biases is not None:
            ids = np.array([i for b in biases for i, _ in b] + [0], np.uint32)
            vals = np.array([v for b in biases for _, v in b] + [0], np.float32)
            self.kw.update(bias_ids=dev(ids), bias_values=dev(vals), num_biases=ids.size - 1,
                           bias_offsets=dev(np.cumsum([0] + [len(b) for b in biases]).astype(np.int32)))
        if masks is not None:
            words = -(-vocab // 32) + mask_pad
            have = [m for m in masks if m is not None]
            self.kw.update(masks=dev(np.stack([U.pack_bits(m, words) for m in have] + [np.zeros(words, np.uint32)])),
                           mask_stride=words, num_masks=len(have))
            at = iter(range(len(have)))
            self.kw.update(mask_ids=dev(np.array([-1 if m is None else next(at) for m in masks], np.int32)))

    def run(self, inplace=False, stream=0):
        batch.logits_process(self.px, self.px if inplace else self.pout, self.rows, self.v, logits_stride=self.v + self.pad,
                             output_stride=self.v + (self.pad if inplace else self.opad), stream=stream, **self.kw)
        flat, pad = (self.dx, self.pad) if inplace else (self.dout, self.opad)
        flat = host(flat, np.float16)[self.offset:self.offset + self.rows * (self.v + pad)].reshape(self.rows, -1)
        if not inplace:
            assert (flat[:, self.v:] == np.float16(123.0)).all()
        return flat[:, :self.v]

    def check(self, inplace=False, err=0):
        got = self.run(inplace)
        ref, tol = U.logits(self.x, self.penalties, self.histories, self.prompts, self.biases, self.masks)
        U.within(got, ref, tol)
        assert _err() == err
        return got


def _histories(rng, rows, vocab, lengths):
    return [(rng.random(lengths[b % len(lengths)]) ** 3 * vocab).astype(np.int64) for b in range(rows)]


def _biases(rng, rows, vocab, n):
    return [[(int(i), float(v)) for i, v in zip(rng.integers(0, vocab, n), rng.standard_normal(n) * 3)] for _ in range(rows)]


def _masks(rng, rows, vocab, free=0.3):
    return [None if b % 3 == 1 else rng.random(vocab) < free for b in range(rows)]


@pytest.mark.parametrize("vocab", [1, 7, 8, 31, 32, 33, 100, 1000, 4096, 4099, 20011, 32768, 65537, 151936])
@pytest.mark.parametrize("rows", [1, 5])
def test_logits_all_together(vocab, rows):
    rng = np.random.default_rng(vocab + rows)
    call = Logits(rows, vocab, rng, _histories(rng, rows, vocab, [0, 300, 1, 77]), _biases(rng, rows, vocab, 9),
                  _masks(rng, rows, vocab), prompts=[0, 100, 1, 20, 5][:rows])
    call.check()


@pytest.mark.parametrize("parts", ["h", "b", "m", "hb", "bm", "hm", ""])
@pytest.mark.parametrize("inplace", [False, True])
def test_logits_parts(parts, inplace):
    rng = np.random.default_rng(len(parts))
    for vocab in (1001, 5000):
        call = Logits(4, vocab, rng, _histories(rng, 4, vocab, [50, 200]) if "h" in parts else None,
                      _biases(rng, 4, vocab, 20) if "b" in parts else None, _masks(rng, 4, vocab) if "m" in parts else None)
        call.check(inplace)


@pytest.mark.parametrize("pad,opad,offset", [(0, 0, 1), (8, 8, 0), (3, 3, 0), (8, 16, 0), (1, 0, 0), (0, 5, 2), (24, 24, 8)])
def test_logits_strides_and_alignment(pad, opad, offset):
    rng = np.random.default_rng(pad * 10 + offset)
    for vocab in (2000, 9001):
        def make():
            return Logits(5, vocab, rng, _histories(rng, 5, vocab, [100, 30]), _biases(rng, 5, vocab, 7), _masks(rng, 5, vocab),
                          pad=pad, opad=opad, offset=offset, mask_pad=3)
        make().check()
        make().check(inplace=True)


def test_logits_penalties_of_all_kinds():
    """Counts of one and of many, the prompt alone, negative penalties, logits of either sign, 0 and infinite."""
    rng = np.random.default_rng(20)
    vocab = 3000
    x = (rng.standard_normal((7, vocab)) * 4).astype(np.float16)
    x[:, 5], x[:, 6], x[:, 7], x[:, 8], x[:, 9] = 0, np.inf, -np.inf, np.nan, 60000
    hist = [np.r_[np.arange(20), np.full(70000, 11), [vocab - 1]]] * 7
    pen = np.float32([[1.5, 0.1, 0.2], [0.5, -0.5, -1], [1, 0, 0], [2, 0, 0], [1, 0.5, 0], [1, 0, 3], [1e-3, 100, 1000]])
    call = Logits(7, vocab, rng, hist, penalties=pen, prompts=[0, 10, 70021, 70021, 15, 3, 21], x=x)
    got = call.check()
    assert np.isnan(got[:, 8]).all() and got[6, 9] == 65504 and got[6, 11] == -65504


def test_logits_biases_of_one_token_and_of_extreme_values():
    rng = np.random.default_rng(21)
    b = [[(3, 1.0), (3, 2.0), (4, -np.inf), (5, np.inf), (6, 1e6), (7, -1e6), (999, 0.5), (3, -7.0)], [], [(0, 0.0)]]
    got = Logits(3, 1000, rng, biases=b).check()
    assert got[0, 4] == -np.inf and got[0, 5] == np.inf and got[0, 6] == 65504 and got[0, 7] == -65504


def test_logits_masks_that_leave_nothing_or_everything_over_any_value():
    rng = np.random.default_rng(22)
    vocab = 5003
    x = (rng.standard_normal((4, vocab)) * 4).astype(np.float16)
    x[:, ::7], x[:, 1::7], x[:, 2::7] = np.nan, np.inf, -np.inf
    one = np.zeros(vocab, bool)
    one[vocab - 1] = True
    masks = [np.zeros(vocab, bool), np.ones(vocab, bool), one, None]
    got = Logits(4, vocab, rng, masks=masks, x=x).check()
    assert (got[0] == -np.inf).all() and np.array_equal(got[1].view(np.uint16), x[1].view(np.uint16))
    # without ids row i has mask i
    call = Logits(3, vocab, rng, masks=masks[:3], x=x[:3].copy())
    call.kw["mask_ids"] = None
    call.check()
    # the greedy choice of a masked row
    call = Logits(1, vocab, rng, masks=[one])
    call.run()
    token = empty((1,), np.uint32)
    cb.check(cb.lib().cactus_cuda_argmax_f16(call.pout, 1, vocab, token.data_ptr(), None))
    assert host(token, np.uint32)[0] == vocab - 1


@pytest.mark.parametrize("vocab", [5003, 40000])
def test_logits_then_a_sample_is_what_the_mask_leaves(vocab):
    """Penalties, bans and masks, then a token of each row by temperature, top-k and top-p: one that is left."""
    rng = np.random.default_rng(28)
    left = [1, 2, 40, 3000]
    masks = [np.zeros(vocab, bool) for _ in left]
    for mask, n in zip(masks, left):
        mask[rng.permutation(vocab)[:n]] = True
    ban = [int(np.flatnonzero(m)[-1]) for m in masks]
    bias = [[(ban[b], -np.inf)] if left[b] > 1 else [] for b in range(4)]
    call = Logits(4, vocab, rng, _histories(rng, 4, vocab, [50]), bias, masks)
    got = call.check(inplace=True)
    token, work = empty((1,), np.uint32), empty((vocab,), np.float16)
    for b in range(4):
        if left[b] > 1:
            masks[b][ban[b]] = False
        assert np.array_equal(np.isfinite(got[b]), masks[b])
        for top_k, top_p in ((0, 0.9), (0, 1.0), (20, 0.9), (5, 1.0)):
            for uniform in (1e-7, 0.5, 1 - 2.0 ** -24):
                cb.check(cb.lib().cactus_cuda_sample_f16(call.px + 2 * b * vocab, 1, vocab, 0.8, top_p, top_k, uniform, None, 0,
                                                         work.data_ptr(), token.data_ptr(), None))
                assert masks[b][host(token, np.uint32)[0]]


@pytest.mark.parametrize("rows,vocab", [(1, 6000), (2, 40000), (300, 20000)])
def test_logits_of_many_named_tokens(rows, vocab):
    """More tokens of one slice in the lists than are counted at a time; every token, named by history or biases."""
    rng = np.random.default_rng(25)
    every = rng.permutation(vocab)
    hist = [np.r_[every[:vocab * 4 // 5], every[:50]] if b % 3 == 0 else every[:b + 1] for b in range(rows)]
    bias = [[(int(i), float(i % 7) - 3.0) for i in (every[::2] if b % 3 == 0 else every[:5])] for b in range(rows)]
    call = Logits(rows, vocab, rng, hist, bias, _masks(rng, rows, vocab, 0.7), prompts=[(b * 37) % 4000 for b in range(rows)])
    call.check()
    call.check(inplace=True)


def test_logits_refuses_lists_on_the_device():
    """Ids past the vocabulary, offsets and mask ids that are none, penalties that are no factors: skipped, and said so."""
    rng = np.random.default_rng(23)
    call = Logits(2, 500, rng, [[1, 2, 500, 2 ** 32 - 1, 3], [4]], [[(7, 1.0), (500, 2.0)], [(2 ** 31, 1.0)]])
    call.check(err=4)
    for name, bad in (("history_offsets", [0, 9, 4]), ("history_offsets", [0, 2, 99]), ("history_offsets", [-3, -1, 0])):
        call = Logits(2, 500, rng, [[1, 2], [3, 4, 5]])
        call.kw[name] = dev(np.array(bad, np.int32))
        call.run()
        assert _err() == 4
    call = Logits(2, 500, rng, biases=[[(1, 1.0)], [(2, 2.0)]])
    call.kw["bias_offsets"] = dev(np.array([0, 1, 7], np.int32))
    call.biases = [[(1, 1.0)], []]
    call.check(err=4)
    call = Logits(3, 500, rng, masks=_masks(rng, 3, 500))
    call.kw["mask_ids"] = dev(np.array([0, 7, -2], np.int32))
    call.masks = [call.masks[0], None, None]
    call.check(err=4)
    pen = np.float32([[0, 0.5, 0.5], [-1, 0, 0], [np.nan, 0, 1], [np.inf, 1, 0]])
    Logits(4, 500, rng, [[1, 2, 3]] * 4, penalties=pen).check(err=4)


@pytest.mark.parametrize("vocab,rows", [(500, 3), (40000, 3), (40000, 300)])
def test_logits_refuses_lengths_and_penalties_of_every_row(vocab, rows):
    """A prompt of less than no tokens counts as none, a repetition penalty that is no factor as 1, and both are said of
    rows without a history too; a prompt of more than the history is all of it."""
    rng = np.random.default_rng(26)
    hist = [[1, 2, 1], [], [vocab - 1]] * (rows // 3)
    for at, value in ((0, -1), (1, -7), (rows - 1, -2 ** 31), (rows - 2, -1)):
        prompts = [b % 3 for b in range(rows)]
        prompts[at] = value
        call = Logits(rows, vocab, rng, hist, prompts=prompts)
        call.prompts = [max(p, 0) for p in prompts]
        call.check(err=4)
    for at, value in ((1, 0.0), (rows - 2, np.nan), (2, -1.0), (0, np.inf)):
        pen = np.tile(np.float32([1.3, 0.25, 0.5]), (rows, 1))
        pen[at, 0] = value
        Logits(rows, vocab, rng, hist, penalties=pen).check(err=4)
    Logits(rows, vocab, rng, hist, prompts=[2 ** 31 - 1] * rows).check()


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("offsets,rest", [([0, 9, 4], [[], []]), ([0, 2, 99], [[1, 2], []]), ([-3, -1, 0], [[], []]),
                                          ([5, 3, 5], [[], [4, 5]]), ([-1, 2, 5], [[], [3, 4, 5]])])
def test_logits_rows_with_refused_lists_stay_as_they_are(offsets, rest, inplace):
    rng = np.random.default_rng(27)
    for vocab in (500, 40000):
        call = Logits(2, vocab, rng, [[1, 2], [3, 4, 5]])
        call.kw["history_offsets"] = dev(np.array(offsets, np.int32))
        call.histories = rest
        got = call.check(inplace, err=4)
        for row in range(2):
            if not rest[row]:
                assert np.array_equal(got[row].view(np.uint16), call.x[row].view(np.uint16))


def test_logits_replayed_with_other_lists():
    t = torch()
    rng = np.random.default_rng(24)
    call = Logits(3, 10000, rng, _histories(rng, 3, 10000, [300]), masks=_masks(rng, 3, 10000))
    call.check()
    t.cuda.synchronize()
    graph = t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        batch.logits_process(call.px, call.pout, 3, 10000, stream=t.cuda.current_stream().cuda_stream, **call.kw)
    call.histories = _histories(rng, 3, 10000, [100, 5, 200])
    flat = np.concatenate(call.histories).astype(np.int32)
    call.kw["history"][:flat.size].copy_(t.from_numpy(flat))
    call.kw["history_offsets"].copy_(t.tensor([0, 100, 105, 305], dtype=t.int32))
    call.dout.fill_(0)
    graph.replay()
    got = host(call.dout, np.float16).reshape(3, -1)
    U.within(got, *U.logits(call.x, call.penalties, call.histories, call.prompts, call.biases, call.masks))
    assert _err() == 0
