"""Plain 64-bit statement of the 4-bit paged KV cache for its tests (numpy, no code of the library)."""
import numpy as np


class Geom:
    def __init__(self, page, hkv, d, g):
        self.page, self.hkv, self.d, self.g, self.ng = page, hkv, d, g, d // g
        self.half = page * d // 2            # code bytes of keys (or values) in a block
        self.par = page * 4 * self.ng        # parameter bytes
        self.block = 2 * (self.half + self.par)

    def args(self):
        return self.page, self.hkv, self.d, self.g


def quantise(x, g):
    """fp16 [..., D] -> codes uint8 [..., D], step and low fp16 [..., D/g]."""
    x = np.asarray(x, np.float16).astype(np.float64)
    x = x.reshape(*x.shape[:-1], x.shape[-1] // g, g)
    with np.errstate(invalid="ignore", over="ignore"):
        bad = ~np.isfinite(x).all(-1)
        y = np.where(bad[..., None], 0.0, x)
        lo, hi = y.min(-1), y.max(-1)
        wide = (hi - lo) / 15.0
        step = wide.astype(np.float16)
        over = step.astype(np.float64) > wide
        step = np.where(over, np.nextafter(step, np.float16(0)), step).astype(np.float16)
        s = step.astype(np.float64)
        q = np.where(s[..., None] > 0, (y - lo[..., None]) / np.where(s > 0, s, 1.0)[..., None], 0.0)
    codes = np.clip(np.rint(q), 0, 15).astype(np.uint8)
    step = np.where(bad, np.float16(np.nan), step).astype(np.float16)
    low = np.where(bad, np.float16(np.nan), lo.astype(np.float16)).astype(np.float16)
    return codes.reshape(*x.shape[:-2], x.shape[-2] * g), step, low


def values(codes, step, low, g):
    """fp16 values the codes stand for: one rounding of the exact c * step + low."""
    s, b = (np.repeat(t.astype(np.float64), g, axis=-1) for t in (step, low))
    with np.errstate(invalid="ignore"):
        return (codes.astype(np.float64) * s + b).astype(np.float16)


class Pool:
    """Host image of a pool: bytes [pages][stride]."""

    def __init__(self, ge, pages, rng, stride=None):
        self.ge, self.pages = ge, pages
        self.stride = stride or ge.block * ge.hkv
        self.bytes = rng.integers(0, 256, (pages, self.stride), dtype=np.uint8)

    def _parts(self, which):
        ge = self.ge
        blocks = self.bytes[:, :ge.block * ge.hkv].reshape(self.pages, ge.hkv, ge.block)
        at = which * (ge.half + ge.par)
        codes = blocks[:, :, at:at + ge.half].reshape(self.pages, ge.hkv, ge.page, ge.d // 2)
        par = blocks[:, :, at + ge.half:at + ge.half + ge.par].reshape(self.pages, ge.hkv, ge.page, ge.ng * 4)
        return codes, par  # views

    def write(self, which, page, row, x):
        """x fp16 [hkv, D] into one row."""
        q, step, low = quantise(x, self.ge.g)
        codes, par = self._parts(which)
        codes[page, :, row] = q[..., 0::2] | (q[..., 1::2] << 4)
        par[page, :, row] = np.ascontiguousarray(np.stack([step, low], -1)).view(np.uint8).reshape(self.ge.hkv, -1)

    def rows(self, which, pages, n):
        """fp16 values [n, hkv, D] of the first n rows of a page list."""
        ge = self.ge
        codes, par = self._parts(which)
        pages = np.asarray(pages[:-(-n // ge.page)], np.int64)
        c = codes[pages].transpose(0, 2, 1, 3).reshape(-1, ge.hkv, ge.d // 2)[:n]
        p = np.ascontiguousarray(par[pages].transpose(0, 2, 1, 3).reshape(-1, ge.hkv, ge.ng * 4)[:n])
        p = p.view(np.float16).reshape(n, ge.hkv, ge.ng, 2)
        q = np.empty((n, ge.hkv, ge.d), np.uint8)
        q[..., 0::2], q[..., 1::2] = c & 15, c >> 4
        return values(q, p[..., 0], p[..., 1], ge.g)

    def spoil(self, page, first):
        """NaN parameters in the rows from `first` on."""
        for which in (0, 1):
            self._parts(which)[1][page, :, first:] = 0x7F


def tables(lens, page, rng, extra=2, width=None):
    """Block tables over shuffled pages; entries past a sequence's end are -1."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + extra
    order = rng.permutation(total).astype(np.int32)
    t = np.full((len(lens), width or max(max(need), 1)), -1, np.int32)
    at = 0
    for b, k in enumerate(need):
        t[b, :k] = order[at:at + k]
        at += k
    return t, total, order[at:]


def attention(q, keys, vals, scale, causal, window):
    """One sequence: q [S, hq, D], keys and vals fp16 [n, hkv, D] -> out, lse, bound, lse bound (64 bits).

    The bounds are what an implementation with fp32 scores, fp16 weights (or better) and one fp16
    rounding of the result may be off by: with m = sum_k w_k |v_k| >= |out| and a = the largest
    scale * sum |q||k|, the rounding of the weights and of the result give 2^-11 m each, weights below
    fp16's normal range another 2^-25 sum |v| over the weights' sum (>= 1 at the running maximum), and
    an fp32 dot product in any order is off by at most 2^-19 a (D <= 256 terms of 2^-24, and as much
    again for the scaling and the exponent), which moves each weight by twice that. A quarter is added.
    """
    s, hq, d = q.shape
    n, hkv = keys.shape[:2]
    q, keys, vals = q.astype(np.float64), keys.astype(np.float64), vals.astype(np.float64)
    pos, k = np.arange(n - s, n)[:, None], np.arange(n)[None, :]
    see = np.ones((s, n), bool)
    if causal:
        see &= k <= pos
    if window:
        see &= k > pos - window
    out, lse = np.zeros((s, hq, d)), np.full((s, hq), -np.inf)
    tol, ltol = np.full((s, hq, d), 2.0 ** -25), np.zeros((s, hq))
    for h in range(hq):
        kh, vh = keys[:, h // (hq // hkv)], vals[:, h // (hq // hkv)]
        if n == 0:
            continue
        sc = np.where(see, q[:, h] @ kh.T * scale, -np.inf)
        a = np.where(see, np.abs(q[:, h]) @ np.abs(kh).T * scale, 0.0).max(-1)
        m = sc.max(-1)
        ok = np.isfinite(m)
        w = np.where(see, np.exp(sc - np.where(ok, m, 0.0)[:, None]), 0.0)
        l = w.sum(-1)
        safe = np.where(ok, l, 1.0)
        out[:, h] = w @ vh / safe[:, None]
        lse[:, h] = np.where(ok, m + np.log(safe), -np.inf)
        mag = w @ np.abs(vh) / safe[:, None]
        small = see.astype(np.float64) @ np.abs(vh) / safe[:, None] * 2.0 ** -25
        tol[:, h] += 1.25 * (mag * (2.0 ** -10 + 2 * 2.0 ** -19 * a[:, None]) + small)
        ltol[:, h] = 1.25 * (2.0 ** -19 * a + 2.0 ** -21 * (1 + np.abs(np.where(ok, lse[:, h], 0.0))))
    return out, lse, tol, ltol
