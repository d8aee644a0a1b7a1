"""Plain 64-bit statements of a ragged batch's operators for their tests (numpy, no code of the library).

Each returns results with what an implementation may be off by: fp32 steps are off by 2^-24 of their result
each (sums of n terms, in any order and cut instead of rounded, by n 2^-23 of the sum of magnitudes), a rounding
to fp16 by 2^-11 of the result, 2^-25 at the least."""
import numpy as np

U32, CUT = 2.0 ** -24, 2.0 ** -23


def fp16_step(v):
    with np.errstate(invalid="ignore"):
        return np.maximum(2.0 ** -11 * np.abs(v), 2.0 ** -25)


def within(got, ref, tol):
    """got (fp16 or fp32) against ref and tol (64 bits): the same infinities and NaN, the rest within tol. An
    fp16 result may also be infinite where ref is within tol of fp16's end."""
    got = got.astype(np.float64)
    with np.errstate(invalid="ignore"):
        ok = (np.isnan(got) & np.isnan(ref)) | (got == ref) | (np.abs(got - ref) <= tol)
    assert ok.all(), f"{(~ok).sum()} of {ok.size} off: {got[~ok][:4]} for {ref[~ok][:4]}, allowed {np.broadcast_to(tol, ref.shape)[~ok][:4]}"


def add16(x, r):
    with np.errstate(over="ignore", invalid="ignore"):
        return (x.astype(np.float64) + r.astype(np.float64)).astype(np.float16)


def norm(s, w, eps):
    """y and its tolerance before any rounding to fp16 or 8 bits: the factor, then two products."""
    s, w = s.astype(np.float64), w.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        y = s / np.sqrt((s * s).mean(-1, keepdims=True) + float(np.float32(eps))) * w
    return y, 3.01 * U32 * np.abs(y)


def lora(x, a, b, ranks, scales, base, seqs, ids):
    """seqs: (first, end) rows of each sequence; returns out and tolerance, base where there is no adapter."""
    out = base.astype(np.float64).copy()
    tol = np.zeros(out.shape)
    for (t0, t1), i in zip(seqs, ids):
        if i < 0 or t1 <= t0:
            continue
        r, c = int(ranks[i]), float(np.float32(scales[i]))
        xs, aa, bb = x[t0:t1].astype(np.float64), a[i, :r].astype(np.float64), b[i, :, :r].astype(np.float64)
        with np.errstate(invalid="ignore", over="ignore"):
            h = xs @ aa.T
            eh = (x.shape[1] + 64) * CUT * (np.abs(xs) @ np.abs(aa).T)
            out[t0:t1] += c * (h @ bb.T)
            mag = np.abs(h) @ np.abs(bb).T
            # the low-rank sums, their parts of 22 bits of the row's largest, the second sum, scale and addition
            top = np.abs(h).max(-1, keepdims=True) if r else np.zeros((t1 - t0, 1))
            e = eh @ np.abs(bb).T + 2.0 ** -21 * top * np.abs(bb).sum(-1)[None] + ((2 * r + 8) * CUT) * mag
            tol[t0:t1] = abs(c) * e + 2 * U32 * (np.abs(out[t0:t1]) + abs(c) * mag)
            tol[t0:t1] += fp16_step(out[t0:t1])
    return out, tol


def logits(x, penalties, histories, prompts, biases, masks):
    """x fp16 [rows, vocab]; histories, biases ((id, value) lists) and masks (bool [vocab]) of each row or None."""
    out = x.astype(np.float64)
    size = np.abs(out)  # magnitudes of all that was added up
    rows, vocab = x.shape
    hidden = np.zeros(x.shape, bool)
    for b in range(rows):
        if penalties is not None and histories is not None:
            rep, freq, pres = (float(v) for v in penalties[b])
            if not (0 < rep < np.inf):
                rep = 1.0
            h = np.asarray(histories[b], np.int64)
            h, made = h[h < vocab], np.asarray(histories[b], np.int64)[prompts[b]:]
            seen = np.bincount(h, minlength=vocab) > 0
            n = np.bincount(made[made < vocab], minlength=vocab)
            with np.errstate(invalid="ignore"):
                l = out[b]
                out[b] = np.where(seen, np.where(l > 0, l / rep, l * rep), l) - freq * n - np.where(n > 0, pres, 0.0)
                size[b] = np.where(seen, size[b] * max(rep, 1 / rep), size[b]) + np.abs(freq) * n + np.abs(pres) * (n > 0)
        if biases is not None:
            last = {int(i): np.float32(v) for i, v in biases[b] if i < vocab}
            for i, v in last.items():
                out[b, i] += float(v)
                size[b, i] += abs(float(v))
        if masks is not None and masks[b] is not None:
            hidden[b] = ~masks[b]
    with np.errstate(invalid="ignore"):
        tol = np.where(np.isfinite(size), 5 * U32 * size, 0.0) + fp16_step(np.where(np.isfinite(out), out, 0.0))
        untouched = (out == x.astype(np.float64)) & (size == np.abs(x.astype(np.float64)))
        tol = np.where(untouched, 0.0, tol)
        out = np.where(np.isfinite(out), np.clip(out, -65504.0, 65504.0), out)
    out[hidden] = -np.inf
    return out, tol


def pack_bits(mask, words=None):
    """bool [vocab] -> uint32 words, bit t % 32 of word t / 32."""
    n = words or -(-mask.size // 32)
    bits = np.zeros(n * 32, np.uint64)
    bits[:mask.size] = mask
    return (bits.reshape(n, 32) << np.arange(32, dtype=np.uint64)).sum(1).astype(np.uint32)


def turns(theta, rotary, positions):
    """(cos, sin) fp32 [positions, rotary / 2, 2] rounded from 64 bits."""
    a = np.asarray(positions, np.float64)[:, None] * float(np.float32(theta)) ** (-np.arange(rotary // 2) * 2.0 / rotary)
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


def rotate(x, weight, eps, turn, rotary):
    """x fp16 [T, H, D], turn fp32 [T, rotary / 2, 2] -> values before the rounding to fp16, and tolerance."""
    v = x.astype(np.float64)
    d = x.shape[-1]
    e = np.zeros(v.shape)
    if weight is not None:
        with np.errstate(invalid="ignore"):
            v = v / np.sqrt((v * v).mean(-1, keepdims=True) + float(np.float32(eps))) * weight.astype(np.float64)
        # the sum's terms, the mean, eps, root, quotient (the root halves what precedes it), two products
        e = (d / 2 + 6) * U32 * np.abs(v)
    half = rotary // 2
    if rotary:
        c, s = (turn[:, None, :, i].astype(np.float64) for i in (0, 1))
        a, b, ea, eb = v[..., :half], v[..., half:rotary], e[..., :half], e[..., half:rotary]
        lo, hi = a * c - b * s, b * c + a * s
        tl = np.abs(c) * ea + np.abs(s) * eb + 2.01 * U32 * (np.abs(a * c) + np.abs(b * s))
        th = np.abs(c) * eb + np.abs(s) * ea + 2.01 * U32 * (np.abs(b * c) + np.abs(a * s))
        v = np.concatenate([lo, hi, v[..., rotary:]], -1)
        e = np.concatenate([tl, th, e[..., rotary:]], -1)
    return v, e


def rotate32(x, turn, rotary):
    """The same without a norm in fp32, step by step: bits that have to be met."""
    v, half = x.astype(np.float32), rotary // 2
    if not rotary:
        return x
    c, s = turn[:, None, :, 0], turn[:, None, :, 1]
    a, b = v[..., :half], v[..., half:rotary]
    with np.errstate(over="ignore", invalid="ignore"):
        return np.concatenate([a * c - b * s, b * c + a * s, v[..., rotary:]], -1).astype(np.float16)
