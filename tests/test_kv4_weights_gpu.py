"""How exactly the 4-bit KV cache's attention holds its softmax weights: as well as 32-bit ones would.

tests/test_kv4_gpu.py allows for weights of one fp16 number, as large an error as the rounding of the
result. Here the values cancel, so that the result and its rounding are small beside the weights."""
import math

import numpy as np
import pytest

from tests import kv4_util as U
from tests.test_kv4_gpu import _attend, _err

pytestmark = pytest.mark.gpu

# tokens (2 heads share a kv head), head_dim: tiles of 4, 8 and 16 rows, and the kernel for many queries with
# one row tile and two
FORMS = [(1, 64), (2, 128), (1, 256), (4, 64), (4, 128), (4, 256), (7, 64), (8, 128), (13, 128), (24, 64), (16, 256),
         (40, 64), (40, 128), (40, 256), (150, 64), (150, 128), (150, 256)]


def _pool(ge, k, v, rng):
    """One sequence with the rows k, v [n, hkv, D]."""
    table, pages, _ = U.tables([k.shape[0]], ge.page, rng)
    pool = U.Pool(ge, pages, rng)
    for row in range(k.shape[0]):
        for which, x in ((0, k), (1, v)):
            pool.write(which, table[0, row // ge.page], row % ge.page, x[row].astype(np.float16))
    return pool, table


def _exact(q, keys, vals, scale, unit=0.0):
    """Causal attention in 64 bits, and what fp32 weights and one fp16 rounding of the result may be off by.

    With mag = sum_k w_k |v_k| >= |out| and a = the largest scale * sum |q||k|: 2^-11 |out| (2^-25 at
    least) for the result's rounding; of mag, 2^-18 a for the fp32 scores (as in kv4_util.attention),
    2^-19 for the exponential (2^-22), for its argument, of up to 8 beside a (2^-21), and for weights of
    22 bits (2^-22), and 2^-24 a term for each of the two sums. A quarter is added. `unit`: what a weight may
    be off by however small it is, relative to the largest."""
    s, hq, _ = q.shape
    n, hkv = keys.shape[:2]
    q, keys, vals = q.astype(np.float64), keys.astype(np.float64), vals.astype(np.float64)
    see = np.arange(n)[None, :] <= np.arange(n - s, n)[:, None]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(hq):
        kh, vh = keys[:, h * hkv // hq], vals[:, h * hkv // hq]
        sc = np.where(see, q[:, h] @ kh.T * scale, -np.inf)
        w = np.exp(sc - sc.max(-1, keepdims=True))
        w /= w.sum(-1, keepdims=True)
        a = np.where(see, np.abs(q[:, h]) @ np.abs(kh).T * scale, 0.0).max(-1, keepdims=True)
        out[:, h] = w @ vh
        tol[:, h] = 1.25 * (np.maximum(2.0 ** -11 * np.abs(out[:, h]), 2.0 ** -25) +
                            (w @ np.abs(vh)) * (2.0 ** -18 * a + 2.0 ** -19 + 2 * n * 2.0 ** -24) +
                            unit * w.max(-1, keepdims=True) * (see @ np.abs(vh)))
    return out, tol


@pytest.mark.parametrize("count,d", FORMS)
def test_weights_are_not_rounded_to_fp16(count, d):
    """Scores of about 0.1 and values of +-1 that nearly cancel: what is left of the weights' rounding shows."""
    ge, hq = U.Geom(16, 2, d, 32), 4
    rng = np.random.default_rng(count + d)
    n = count + 39
    k = 0.1 * rng.standard_normal((n, ge.hkv, d))
    v = rng.permuted(np.broadcast_to(np.where(np.arange(n) % 2, 1.0, -1.0)[:, None, None], (n, ge.hkv, d)), axis=0)
    pool, table = _pool(ge, k, v, rng)
    q = rng.standard_normal((count, hq, d)).astype(np.float16)
    got, _, _ = _attend(pool, table, q, [count], [n], hq)
    out, tol = _exact(q, pool.rows(0, table[0], n), pool.rows(1, table[0], n), 1 / math.sqrt(d))
    assert np.all(np.abs(got.astype(np.float64) - out) <= tol), np.max(np.abs(got - out) / tol)
    assert _err() == 0


@pytest.mark.parametrize("every", [0, 16])
@pytest.mark.parametrize("count,d", FORMS)
def test_a_tail_of_small_weights_keeps_its_bits(count, d, every):
    """One row, or one in 16, has nearly all the weight and values of zero; the result comes from the others' weights,
    each 2^-18 to 2^-24.5 of theirs."""
    ge, hq, n = U.Geom(64, 2, d, 32), 4, 600 if every else 2900
    rng = np.random.default_rng(count * d + every)
    k, v = np.zeros((n, ge.hkv, d)), np.full((n, ge.hkv, d), 512.0 if every else 1.0)
    heavy = np.s_[3::every] if every else np.s_[3:4]
    k[heavy], v[heavy] = 1.0, 0.0
    pool, table = _pool(ge, k, v, rng)
    # the heavy rows' score is d times an element of the query, the others' is 0
    score = rng.uniform(18.0, 24.5, (count, hq, 1)) * math.log(2)
    q = np.broadcast_to((score / math.sqrt(d)).astype(np.float16), (count, hq, d))
    got, _, _ = _attend(pool, table, q, [count], [n], hq)
    # two fp16 numbers a weight, the largest 2^7 or more: their last bit is 2^-24 at most, half of it the error
    out, tol = _exact(q, pool.rows(0, table[0], n), pool.rows(1, table[0], n), 1 / math.sqrt(d), unit=2.0 ** -32)
    assert np.all(np.abs(got.astype(np.float64) - out) <= tol), np.max(np.abs(got - out) / tol)
    assert np.all(out > 1e-4)
    assert _err() == 0
