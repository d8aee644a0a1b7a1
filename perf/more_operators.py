"""Cases and plain forms of the operators around a ragged batch's projections and its 4-bit cache: the
residual's addition with RMSNorm and 8-bit rows, low-rank adapters of many requests beside a shared
projection, the append that normalises and rotates keys (and queries) on the way into the cache, and the
penalties, biases and grammar masks on a batch's logits.

norm     s = fp16(x + residual); y = s / sqrt(mean(s^2) + eps) * weight; scale = max(max|y| / 127, 1e-10) of the
         row; code = round_half_even(y / scale). `normed` is y in fp16.
lora     row t of a sequence with adapter a: base + scale[a] * (x A[a]^T) B[a]^T, where only the first rank[a] rows
         of A[a] [max_rank][in] and columns of B[a] [out][max_rank] exist (the rest holds anything). A sequence
         without an adapter (-1) keeps its base rows.
rope     the token at position p of its sequence: queries and keys of each head normalised (y = x / sqrt(mean(x^2) +
         eps) * weight, where there are weights), then element i and i + R/2 of the first R turned by the angle of
         row p of the table, rounded to fp16; keys and values go into the pages of the 4-bit cache
         (include/cactus_b200_kv4.h has its format) and are read back as what their codes stand for.
logits   l of a token that the row's history holds: l / repetition where l > 0, else l * repetition; minus
         frequency * count and minus presence where the count, of what was generated (the history after its first
         prompt_len tokens), is not 0; plus the row's bias for the token; -inf where the row's mask has a 0 bit. A
         finite result past fp16's range is its largest number.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"


# ---------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one conversation's next token: nothing but latency
        dict(op="norm", name="norm_token_1x1024", rows=1, dims=1024, normed=False, residual=True, slice=1),
        # the tokens of a full server, the adapters' fp16 rows written too
        dict(op="norm", name="norm_tokens_256x2048", rows=256, dims=2048, normed=True, residual=True, slice=1),
        # a chunk of prompts in a wide model; x is half of a wider projection's output
        dict(op="norm", name="norm_prompts_16384x4096", rows=16384, dims=4096, normed=False, residual=True, slice=2),
        # one request with an adapter of rank 16
        dict(op="lora", name="lora_token_1x1024", seqs=1, q_len=1, ragged=0.0, k=1024, n=2048, rank=16, mixed=False,
             adapters=4, bare=0.0),
        # a full server whose requests bring 40 adapters of different ranks, some requests none
        dict(op="lora", name="lora_tokens_128_of_40", seqs=128, q_len=1, ragged=0.0, k=2048, n=2048, rank=32,
             mixed=True, adapters=40, bare=0.1),
        # prompts of very different lengths, a few adapters, into a wide projection
        dict(op="lora", name="lora_prompts_9000", seqs=14, q_len=1031, ragged=0.8, k=2048, n=8192, rank=64,
             mixed=True, adapters=5, bare=0.1),
        # the new token of every running sequence, heads normalised before they turn (16 / 8 heads of 128)
        dict(op="rope", name="rope_tokens_64", seqs=64, q_len=1, context=1913, ragged=0.8, hq=16, hkv=8, d=128,
             rotary=128, g=32, page=16, norm=True),
        # a batch of whole prompts (24 / 8 heads of 64)
        dict(op="rope", name="rope_prompts_24x4096", seqs=24, q_len=4096, context=4096, ragged=0.7, hq=24, hkv=8, d=64,
             rotary=64, g=64, page=64, norm=False),
        # chunks behind long contexts, one key head of 256 of which half turns
        dict(op="rope", name="rope_chunks_16x256", seqs=16, q_len=256, context=30011, ragged=0.5, hq=4, hkv=1, d=256,
             rotary=128, g=32, page=64, norm=True),
        # one request with penalties and a few biased words
        dict(op="logits", name="logits_1x151936", rows=1, vocab=151936, history=700, biases=20, masks=0, free=0.5,
             penalties=True, inplace=False),
        # a full server: penalties everywhere, a grammar on every third row
        dict(op="logits", name="logits_256x128256", rows=256, vocab=128256, history=1500, biases=50, masks=8, free=0.03,
             penalties=True, inplace=False),
        # grammars alone, written over the logits where they stand
        dict(op="logits", name="logits_masks_48x262144", rows=48, vocab=262144, history=0, biases=0, masks=48, free=0.01,
             penalties=False, inplace=True),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


#: The most that a drawn case moves and computes: below each operator's largest listed one.
_MOST = {"norm": (4.5e8, 2e9), "lora": (3.4e8, 1.0e10), "rope": (7.4e8, 2e10), "logits": (1.2e8, 1e9)}


def draw(rng):
    while True:
        c = _drawn(rng)
        w = work(c)
        if w["bytes"] <= _MOST[c["op"]][0] and w["flops"] <= _MOST[c["op"]][1]:
            return c


def _drawn(rng):
    op = rng.choice(("norm", "lora", "lora", "rope", "logits"))
    if op == "norm":
        dims = _spread(rng, 64, 8192)
        return {"op": op, "rows": _spread(rng, 1, 16384), "dims": dims if rng.random() < 0.2 else max(64, dims // 8 * 8),
                "normed": rng.random() < 0.5, "residual": rng.random() < 0.8, "slice": rng.choice((1, 1, 2, 3))}
    if op == "lora":
        tokens = rng.random() < 0.5
        return {"op": op, "seqs": _spread(rng, 1, 300 if tokens else 24),
                "q_len": rng.choice((1, 1, 2, 5)) if tokens else _spread(rng, 6, 3000), "ragged": rng.choice((0.0, 0.5, 0.95)),
                "k": 8 * _spread(rng, 8, 1024), "n": 8 * _spread(rng, 8, 1024), "rank": _spread(rng, 1, 128),
                "mixed": rng.random() < 0.6, "adapters": _spread(rng, 1, 48), "bare": rng.choice((0.0, 0.1, 0.6))}
    if op == "rope":
        d = rng.choice((64, 128, 256))
        hkv = rng.choice((1, 2, 3, 4, 5, 8))
        prompt = rng.random() < 0.6
        q_len = _spread(rng, 2, 4000) if prompt else 1
        return {"op": op, "seqs": _spread(rng, 1, 32 if prompt else 256), "q_len": q_len,
                "context": q_len + (0 if rng.random() < 0.4 else _spread(rng, 1, 30000)), "ragged": rng.choice((0.0, 0.5, 0.9)),
                "hq": hkv * rng.choice((1, 2, 3, 4, 7, 8)), "hkv": hkv, "d": d,
                "rotary": rng.choice((d, d, d, d // 2, d // 4 * 3)),
                "g": rng.choice([g for g in (32, 64, 128) if d % g == 0]), "page": rng.choice((16, 32, 64, 128)),
                "norm": rng.random() < 0.5}
    kind = rng.choice(("all", "all", "penalties", "masks", "biases"))
    rows = _spread(rng, 1, 256)
    return {"op": op, "rows": rows, "vocab": _spread(rng, 1000, 262144),
            "history": _spread(rng, 1, 4000) if kind in ("all", "penalties") else 0,
            "biases": _spread(rng, 1, 300) if kind in ("all", "biases") else 0,
            "masks": (rows if rng.random() < 0.5 else min(rows, 8)) if kind in ("all", "masks") else 0,
            "free": rng.choice((0.0005, 0.02, 0.5, 0.98)), "penalties": kind in ("all", "penalties"),
            "inplace": kind == "masks" and rng.random() < 0.7}


def _lengths(c):
    """(new rows, context) of each sequence: the longest first, the others down to (1 - ragged) of it."""
    got = []
    for b in range(c["seqs"]):
        f = 1.0 - c["ragged"] * ((b * 0.6180339887498949) % 1.0)
        s = max(1, int(round(c["q_len"] * f))) if c["q_len"] > 16 else c["q_len"]
        got.append((s, max(s, int(round(c.get("context", s) * f)))))
    return got


def _adapters(c):
    """Each sequence's adapter (-1: none) and each adapter's rank."""
    rng = random.Random(c["seqs"] * 7919 + c["adapters"])
    ids = [-1 if rng.random() < c["bare"] else rng.randrange(c["adapters"]) for _ in range(c["seqs"])]
    ranks = [max(1, c["rank"] // rng.choice((1, 1, 2, 4))) if c["mixed"] else c["rank"] for _ in range(c["adapters"])]
    return ids, ranks


def _row_bytes(c):
    """Bytes of one row of one key head in the cache: keys and values, codes and parameters."""
    return 2 * (c["d"] // 2 + 4 * (c["d"] // c["g"]))


def _masked(c):
    """Which mask each row uses: all rows where they alone are wanted, else every third."""
    if not c["masks"]:
        return None
    return [b % c["masks"] if c["inplace"] or c["masks"] == c["rows"] or b % 3 == 0 else -1 for b in range(c["rows"])]


def work(c):
    if c["op"] == "norm":
        n = c["rows"] * c["dims"]
        per = 2 + 1 + (4 if c["residual"] else 0) + (2 if c["normed"] else 0)
        return {"bytes": float(n * per + 2 * c["dims"] + 4 * c["rows"]), "flops": 10.0 * n}
    if c["op"] == "lora":
        ids, ranks = _adapters(c)
        tokens = sum(s for s, _ in _lengths(c))
        size = 4.0 * tokens * c["n"]
        flops = 0.0
        for (s, _), a in zip(_lengths(c), ids):
            if a >= 0:
                size += 2.0 * s * c["k"]
                flops += 2.0 * s * ranks[a] * (c["k"] + c["n"])
        return {"bytes": size + sum(2.0 * ranks[a] * (c["k"] + c["n"]) for a in set(ids) - {-1}), "flops": flops}
    if c["op"] == "rope":
        tokens = sum(s for s, _ in _lengths(c))
        positions = len({p for s, n in _lengths(c) for p in (range(n - s, n) if s < 100 else (n,))}) if c["q_len"] < 100 else \
            max(n for _, n in _lengths(c)) - min(n - s for s, n in _lengths(c))
        # queries read and written, keys and values read, written as codes and read back
        per = 4 * c["hq"] * c["d"] + c["hkv"] * (4 * c["d"] + 2 * _row_bytes(c) + 4 * c["d"])
        return {"bytes": float(tokens * per + min(positions, tokens) * 4 * c["rotary"]),
                "flops": float(tokens * c["d"] * (8 * c["hq"] + 20 * c["hkv"]))}
    n = c["rows"] * c["vocab"]
    lists = c["rows"] * (4.0 * c["history"] + 8.0 * c["biases"])
    if c["inplace"]:  # what a mask leaves out is written, the rest stays
        return {"bytes": 2.0 * n * (1.0 - c["free"]) + n / 8, "flops": float(n)}
    return {"bytes": 4.0 * n + lists + c["masks"] * c["vocab"] / 8.0, "flops": 4.0 * n}


# ---------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    return {"norm": _prepare_norm, "lora": _prepare_lora, "rope": _prepare_rope, "logits": _prepare_logits}[c["op"]](c, gen)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEVICE)


def _normal(shape, gen):
    return torch.randn(shape, generator=gen, device=DEVICE)


def _prepare_norm(c, gen):
    rows, dims = c["rows"], c["dims"]
    loud = 1.0 + 20.0 * (torch.rand(dims, generator=gen, device=DEVICE) < 0.003)  # the few large channels of a decoder
    width = dims * c["slice"]
    x = _normal((rows, width), gen).half()
    residual = (_normal((rows, dims), gen) * 2.0 * loud).half() if c["residual"] else None
    return {"case": c, "x": x, "width": width, "residual": residual, "eps": 1e-6,
            "weight": (1.0 + 0.2 * _normal((dims,), gen)).half()}


def _prepare_lora(c, gen):
    ids, ranks = _adapters(c)
    lengths = [s for s, _ in _lengths(c)]
    starts = [0]
    for s in lengths:
        starts.append(starts[-1] + s)
    top = -(-c["rank"] // 8) * 8
    # a projection's weights and an adapter's: the products are of the size of the base rows' own rounding and up
    a = _normal((c["adapters"], top, c["k"]), gen).mul_(c["k"] ** -0.5).half()
    b = _normal((c["adapters"], c["n"], top), gen).mul_(0.05).half()
    for i, r in enumerate(ranks):  # rows and columns that an adapter does not have
        a[i, r:] = math.nan
        b[i, :, r:] = math.nan
    rows_of = {}
    for i, s, n in zip(ids, starts, lengths):
        rows_of.setdefault(i, []).append(torch.arange(s, s + n, device=DEVICE))
    return {"case": c, "x": _normal((starts[-1], c["k"]), gen).half(), "a": a, "b": b, "top": top,
            "base": _normal((starts[-1], c["n"]), gen).half(), "offsets": _ints(starts), "ids": _ints(ids),
            "ranks": _ints(ranks), "scales": torch.rand(c["adapters"], generator=gen, device=DEVICE) + 0.5,
            "tokens": starts[-1], "host_ranks": ranks, "rows_of": {i: torch.cat(v) for i, v in rows_of.items()}}


def _prepare_rope(c, gen):
    sizes = _lengths(c)
    need = [-(-n // c["page"]) for _, n in sizes]
    # pages of the rows before the new ones are shared or long written: the table names them, nothing reads them
    first = [(n - s) // c["page"] for s, n in sizes]
    pages = sum(n - f for n, f in zip(need, first)) + 2
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((len(sizes), max(need)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, (n, f) in enumerate(zip(need, first)):
        table[b, f:n] = order[at:at + n - f]
        at += n - f
    pool = torch.randint(0, 256, (pages, c["hkv"], _row_bytes(c) * c["page"]), generator=gen, device=DEVICE, dtype=torch.uint8)
    starts = [0]
    for s, _ in sizes:
        starts.append(starts[-1] + s)
    tokens, d = starts[-1], c["d"]
    qkv = _normal((tokens, (c["hq"] + 2 * c["hkv"]) * d), gen).half()  # a fused projection's output
    qkv[:, c["hq"] * d:c["hq"] * d + c["g"]] *= 3.0
    counts = torch.tensor([s for s, _ in sizes], device=DEVICE)
    seq = torch.repeat_interleave(torch.arange(len(sizes), device=DEVICE), counts)
    offsets, context = _ints(starts), _ints([n for _, n in sizes])
    position = torch.arange(tokens, device=DEVICE) - offsets[1:].long()[seq] + context.long()[seq]
    half, most = c["rotary"] // 2, max(n for _, n in sizes)
    turn = torch.arange(most, device=DEVICE, dtype=torch.float64)[:, None] * \
        torch.pow(1e6, -torch.arange(half, device=DEVICE, dtype=torch.float64) * (2.0 / c["rotary"]))
    state = {"case": c, "pool": pool, "table": table, "qkv": qkv, "offsets": offsets, "context": context, "tokens": tokens,
             "turns": torch.stack([turn.cos(), turn.sin()], -1).float(), "first": context - _ints([s for s, _ in sizes]),
             "seq": seq, "position": position, "eps": 1e-6, "q_weight": None, "k_weight": None}
    if c["norm"]:
        state["q_weight"], state["k_weight"] = ((1.0 + 0.2 * _normal((d,), gen)).half() for _ in range(2))
    return state


def _prepare_logits(c, gen):
    rows, vocab = c["rows"], c["vocab"]
    state = {"case": c, "logits": (_normal((rows, vocab), gen) * 2.5 - 1.0).half(), "history": None, "biases": None,
             "masks": None}
    if c["penalties"]:
        # words come again: ids by a steep law, the lengths of the rows from a half to all of `history`
        lengths = [max(1, int(c["history"] * (1.0 - 0.5 * ((b * 0.618) % 1.0)))) for b in range(rows)]
        starts = [0]
        for n in lengths:
            starts.append(starts[-1] + n)
        ids = (torch.rand(starts[-1], generator=gen, device=DEVICE).pow(4) * vocab).long().clamp(max=vocab - 1)
        ids = (ids * 7919 + 13) % vocab
        per = torch.stack([1.0 + 0.3 * torch.rand(rows, generator=gen, device=DEVICE),
                           0.5 * torch.rand(rows, generator=gen, device=DEVICE),
                           torch.rand(rows, generator=gen, device=DEVICE) - 0.2], 1).contiguous()
        state.update(history=ids.to(torch.int32), history_offsets=_ints(starts), penalties=per,
                     prompt_lens=_ints([n // 3 for n in lengths]),
                     history_row=torch.repeat_interleave(torch.arange(rows, device=DEVICE), torch.tensor(lengths, device=DEVICE)))
    if c["biases"]:
        k = min(c["biases"], vocab)
        start = torch.randint(0, vocab, (rows, 1), generator=gen, device=DEVICE)
        ids = (start + torch.arange(k, device=DEVICE) * max(1, vocab // k)) % vocab  # a row's ids are all different
        values = _normal((rows, k), gen) * 4.0
        values[:, ::7] = -math.inf  # banned words
        state.update(biases=ids.to(torch.int32).reshape(-1).contiguous(), bias_values=values.reshape(-1).contiguous(),
                     bias_offsets=_ints([b * k for b in range(rows + 1)]), bias_rows=k)
    if c["masks"]:
        words = -(-vocab // 32)
        bits = torch.rand((c["masks"], words, 32), generator=gen, device=DEVICE) < c["free"]
        state["masks"] = (bits.long() << torch.arange(32, device=DEVICE)).sum(-1).to(torch.int32).contiguous()
        state["mask_ids"] = _ints(_masked(c))
    return state


# ---------------------------------------------------------------------------------------- plain forms
def _plain_norm(s):
    c = s["case"]
    x = s["x"][:, :c["dims"]]
    out = {}
    if s["residual"] is not None:
        x = (x.float() + s["residual"].float()).half()
        out["sum"] = x
    v = x.float()
    mean = v.double().square().mean(-1, keepdim=True)  # a long sum
    y = v * (1.0 / torch.sqrt(mean + s["eps"])).float() * s["weight"].float()
    if c["normed"]:
        out["normed"] = y.half()
    scale = (y.abs().amax(-1, keepdim=True) / torch.full((), 127.0, device=DEVICE)).clamp(min=1e-10)
    code = torch.round(y * (torch.ones((), device=DEVICE) / scale)).clamp(-127, 127)
    out["values"], out["scales"] = (code * scale).half(), scale[:, 0]
    return out


def _plain_lora(s):
    out = s["base"].clone()
    for a, rows in s["rows_of"].items():
        if a >= 0:
            r = s["host_ranks"][a]
            low = s["x"][rows].float() @ s["a"][a, :r].float().T
            out[rows] = (s["base"][rows].float() + s["scales"][a] * (low @ s["b"][a, :, :r].float().T)).half()
    return {"output": out}


def _quantise(x, c):
    """Codes [..., D] and (step, low) pairs [..., D/G, 2] of fp16 rows [..., D], as the cache's format has them."""
    g = x.float().reshape(*x.shape[:-1], x.shape[-1] // c["g"], c["g"])
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    wide = (hi - lo) / 15.0
    step = wide.half()
    step = torch.where(step.float() > wide, (step.view(torch.int16) - 1).view(torch.float16), step)
    some = step.float() > 0
    q = torch.round((g - lo) / torch.where(some, step.float(), 1.0)).clamp(0, 15)
    return torch.where(some, q, 0.0).to(torch.uint8).reshape(x.shape), torch.cat([step, lo.half()], -1)


def _turned(x, weight, s):
    """Heads [T, H, D] fp16, normalised and turned."""
    v, half = x.float(), s["case"]["rotary"] // 2
    if weight is not None:
        v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + s["eps"]) * weight.float()
    turn = s["turns"][s["position"]]
    cos, sin = turn[:, None, :, 0], turn[:, None, :, 1]
    a, b = v[..., :half], v[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, v[..., 2 * half:]], -1).half()


def _plain_rope(s):
    c = s["case"]
    p, hq, hkv, d, ng = c["page"], c["hq"], c["hkv"], c["d"], c["d"] // c["g"]
    heads = s["qkv"].reshape(-1, hq + 2 * hkv, d)
    queries = _turned(heads[:, :hq], s["q_weight"], s)
    page, row = s["table"][s["seq"], s["position"] // p].long(), s["position"] % p
    half, par = p * d // 2, 4 * ng
    out = {"queries": queries}
    for which, name in ((0, "keys"), (1, "values")):
        x = _turned(heads[:, hq:hq + hkv], s["k_weight"], s) if which == 0 else heads[:, hq + hkv:]
        q, params = _quantise(x, c)
        at = which * (half + p * par)
        codes = s["pool"][..., at:at + half].unflatten(-1, (p, d // 2))
        codes[page, :, row] = q[..., 0::2] | (q[..., 1::2] << 4)
        pairs = s["pool"][..., at + half:at + half + p * par].unflatten(-1, (p, par))
        pairs[page, :, row] = params.contiguous().view(torch.uint8).flatten(-2)
        # read back from the pages
        code, pair = codes[page, :, row], pairs[page, :, row].contiguous().view(torch.float16).reshape(-1, hkv, ng, 1, 2).float()
        code = torch.stack([code & 15, code >> 4], -1).reshape(-1, hkv, ng, c["g"]).float()
        out[name] = (code * pair[..., 0] + pair[..., 1]).half().flatten(-2)
    return out


def _plain_logits(s):
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    v = s["logits"].float()
    if s["history"] is not None:
        ids = s["history"].long()
        at = torch.arange(ids.numel(), device=DEVICE) - s["history_offsets"].long()[s["history_row"]]
        made = (at >= s["prompt_lens"].long()[s["history_row"]]).int()
        seen = torch.zeros((rows, vocab), dtype=torch.bool, device=DEVICE)
        seen[s["history_row"], ids] = True
        count = torch.zeros((rows, vocab), dtype=torch.int32, device=DEVICE)
        count.index_put_((s["history_row"], ids), made, accumulate=True)
        rep, freq, pres = (s["penalties"][:, i:i + 1] for i in range(3))
        v = torch.where(seen, torch.where(v > 0, v / rep, v * rep), v)
        v = v - freq * count.float()
        v = v - torch.where(count > 0, pres, 0.0)
    if s["biases"] is not None:
        v = v.scatter_add(1, s["biases"].long().reshape(rows, -1), s["bias_values"].reshape(rows, -1))
    v = torch.where(torch.isfinite(v), v.clamp(-65504.0, 65504.0), v).half()
    if s["masks"] is not None:
        bits = (s["masks"][:, :, None] >> torch.arange(32, device=DEVICE, dtype=torch.int32)) & 1
        allowed = bits.flatten(1)[:, :vocab].bool()[s["mask_ids"].long().clamp(min=0)] | (s["mask_ids"] < 0)[:, None]
        v = torch.where(allowed, v, -math.inf)
    if c["inplace"]:
        s["logits"].copy_(v)
        v = s["logits"]
    return {"logits": v}


# ---------------------------------------------------------------------------------------- the framework's
def _stream():
    return torch.cuda.current_stream().cuda_stream


def _at(t):
    return None if t is None else t.data_ptr()


def _empty(shape, dtype=torch.float16):
    return torch.empty(shape, dtype=dtype, device=DEVICE)


def _own_norm(s, cb):
    c = s["case"]
    rows, dims = c["rows"], c["dims"]
    out = {}
    if c["residual"]:
        out["sum"] = _empty((rows, dims))
    if c["normed"]:
        out["normed"] = _empty((rows, dims))
    codes, scales = _empty((rows, dims), torch.int8), _empty((rows,), torch.float32)
    cb.check(cb.lib().cactus_cuda_add_rms_norm_q8(
        s["x"].data_ptr(), s["width"], _at(s["residual"]), dims, s["weight"].data_ptr(), _at(out.get("sum")), dims,
        codes.data_ptr(), scales.data_ptr(), _at(out.get("normed")), rows, dims, s["eps"], _stream()), "add_rms_norm_q8")
    out["values"] = torch.mul(codes, scales[:, None], out=_empty((rows, dims)))  # what the codes stand for
    out["scales"] = scales
    return out


def _own_lora(s, cb):
    c, lib, seqs, tokens = s["case"], cb.lib(), s["ids"].numel(), s["tokens"]
    if "plan" not in s:  # a step's plan serves the projections of all its layers; the workspace any call
        size = lib.cactus_cuda_lora_plan_bytes(seqs, tokens, c["adapters"])
        s["plan"] = _empty((size,), torch.uint8)
        cb.check(lib.cactus_cuda_lora_plan(s["offsets"].data_ptr(), s["ids"].data_ptr(), seqs, tokens, c["adapters"],
                                           s["plan"].data_ptr(), size, _stream()), "lora_plan")
        s["workspace"] = _empty((lib.cactus_cuda_lora_workspace(tokens, s["top"]),), torch.uint8)
    out = _empty((tokens, c["n"]))
    cb.check(lib.cactus_cuda_lora_f16(
        s["x"].data_ptr(), c["k"], s["a"].data_ptr(), s["b"].data_ptr(), s["ranks"].data_ptr(), s["scales"].data_ptr(),
        s["base"].data_ptr(), c["n"], out.data_ptr(), c["n"], s["plan"].data_ptr(), s["plan"].numel(), seqs, tokens,
        c["adapters"], s["top"], c["k"], c["n"], s["workspace"].data_ptr(), s["workspace"].numel(), _stream()), "lora_f16")
    return {"output": out}


def _own_rope(s, cb):
    c, lib, stream = s["case"], cb.lib(), _stream()
    hq, hkv, d, width, tokens = c["hq"], c["hkv"], c["d"], s["qkv"].shape[1], s["tokens"]
    queries, keys, values = _empty((tokens, hq, d)), _empty((tokens, hkv, d)), _empty((tokens, hkv, d))
    at, geometry = s["qkv"].data_ptr(), (c["page"], hkv, d, c["g"])
    table = (s["table"].data_ptr(), s["table"].shape[1])
    pool = (s["pool"].data_ptr(), s["pool"].shape[0], s["pool"].stride(0))
    cb.check(lib.cactus_cuda_kv4_rope_append(
        at, width, queries.data_ptr(), hq * d, at + 2 * hq * d, at + 2 * (hq + hkv) * d, width, s["turns"].data_ptr(),
        s["turns"].shape[0], c["rotary"], _at(s["q_weight"]), _at(s["k_weight"]), s["eps"], s["offsets"].data_ptr(),
        s["context"].data_ptr(), *table, *pool, c["seqs"], tokens, hq, *geometry, stream), "kv4_rope_append")
    cb.check(lib.cactus_cuda_kv4_read(*pool, *table, s["offsets"].data_ptr(), s["first"].data_ptr(), keys.data_ptr(),
                                      values.data_ptr(), c["seqs"], tokens, *geometry, stream), "kv4_read")
    return {"queries": queries, "keys": keys, "values": values}


def _own_logits(s, cb):
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    out = s["logits"] if c["inplace"] else _empty((rows, vocab))
    history, biases, masks = s["history"], s["biases"], s["masks"]
    cb.check(cb.lib().cactus_cuda_logits_process_f16(
        s["logits"].data_ptr(), vocab, out.data_ptr(), vocab, rows, vocab, _at(s.get("penalties")), _at(history),
        _at(s.get("history_offsets")), _at(s.get("prompt_lens")), 0 if history is None else history.numel(), _at(biases),
        _at(s.get("bias_values")), _at(s.get("bias_offsets")), 0 if biases is None else biases.numel(), _at(masks),
        0 if masks is None else masks.shape[1], c["masks"], _at(s.get("mask_ids")), _stream()), "logits_process_f16")
    return {"logits": out}


_PLAIN = {"norm": _plain_norm, "lora": _plain_lora, "rope": _plain_rope, "logits": _plain_logits}
_OWN = {"norm": _own_norm, "lora": _own_lora, "rope": _own_rope, "logits": _own_logits}


def run(state):
    op = state["case"]["op"]
    if own:
        import cactus_b200
        return _OWN[op](state, cactus_b200)
    return _PLAIN[op](state)


# ---------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "lora": _exact_lora, "rope": _exact_rope, "logits": _exact_logits}[s["case"]["op"]](s)


def _exact_norm(s):
    c = s["case"]
    x = s["x"][:, :c["dims"]].double()
    out = {}
    if s["residual"] is not None:
        x = (x + s["residual"].double()).half().double()
        out["sum"] = x
    y = x / ((x * x).sum(1, keepdim=True) / c["dims"] + s["eps"]).sqrt() * s["weight"].double()[None]
    if c["normed"]:
        out["normed"] = y
    unit = torch.maximum(y.abs().max(1, keepdim=True).values / 127, torch.full((), 1e-10, device=DEVICE, dtype=torch.float64))
    out["values"], out["scales"] = (y / unit).round() * unit, unit[:, 0]
    return out


def _exact_lora(s):
    c, starts, ids = s["case"], s["offsets"].tolist(), s["ids"].tolist()
    out = s["base"].double()
    for i, (t0, t1) in enumerate(zip(starts, starts[1:])):
        a = ids[i]
        if a < 0:
            continue
        r = s["host_ranks"][a]
        low = torch.einsum("tk,rk->tr", s["x"][t0:t1].double(), s["a"][a, :r].double())
        out[t0:t1] += torch.einsum("tr,nr->tn", low, s["b"][a, :, :r].double()) * s["scales"][a].double()
    return {"output": out}


def _exact_rope(s):
    c = s["case"]
    hq, hkv, d, g, half = c["hq"], c["hkv"], c["d"], c["g"], c["rotary"] // 2
    rows = s["qkv"].double().reshape(-1, hq + 2 * hkv, d)
    speed = 1e6 ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) * 2.0 / c["rotary"])
    angle = s["position"].double()[:, None, None] * speed

    def turned(x, weight):
        if weight is not None:
            x = x / ((x * x).sum(-1, keepdim=True) / d + s["eps"]).sqrt() * weight.double()
        z = torch.polar(torch.ones_like(angle), angle) * torch.complex(x[..., :half], x[..., half:2 * half])
        return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)

    def stored(x):
        x = x.half().double().unflatten(-1, (d // g, g))
        low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
        # fifteenths of the range, cut to the 11 bits of fp16 (2^-24 at the least)
        wide = (high - low) / 15
        unit = torch.exp2(torch.floor(torch.log2(wide.clamp(min=2.0 ** -14))) - 10)
        step = torch.floor(wide / unit) * unit
        code = torch.where(step > 0, ((x - low) / torch.where(step > 0, step, 1.0)).round().clamp(0, 15), 0.0)
        return (code * step + low).half().double().flatten(-2)

    return {"queries": turned(rows[:, :hq], s["q_weight"]), "keys": stored(turned(rows[:, hq:hq + hkv], s["k_weight"])),
            "values": stored(rows[:, hq + hkv:])}


def _exact_logits(s):
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    out = s["logits"].double()
    if s["history"] is not None:
        starts, prompt = s["history_offsets"].tolist(), s["prompt_lens"].tolist()
        per = s["penalties"].double()
        for b in range(rows):
            ids = s["history"][starts[b]:starts[b + 1]].long()
            every = torch.bincount(ids, minlength=vocab)
            made = torch.bincount(ids[prompt[b]:], minlength=vocab)
            line = out[b]
            line = torch.where(every > 0, torch.where(line > 0, line / per[b, 0], line * per[b, 0]), line)
            out[b] = line - made * per[b, 1] - (made > 0) * per[b, 2]
    if s["biases"] is not None:
        k = s["bias_rows"]
        for b in range(rows):
            out[b, s["biases"][b * k:(b + 1) * k].long()] += s["bias_values"][b * k:(b + 1) * k].double()
    out = torch.where(out.isfinite(), out.clamp(-65504.0, 65504.0), out)
    if s["masks"] is not None:
        for b, m in enumerate(_masked(c)):
            if m >= 0:
                token = torch.arange(vocab, device=DEVICE)
                bit = s["masks"][m].long()[token // 32].bitwise_right_shift(token % 32) & 1
                out[b] = out[b].masked_fill(bit == 0, -math.inf)
    return {"logits": out}
