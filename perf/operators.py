"""Cases and plain forms of the 4-bit paged KV cache: the append that quantises keys and values into
pages, the attention that reads them, the copy of pages when a sequence is forked, and the compaction
that moves the rows a sequence keeps into new pages.

A cache is a pool of pages, bytes [num_pages][kv heads][block]. One block holds, for its page_size rows,

    key codes [rows][D/2] | key parameters [rows][D/G] | value codes [rows][D/2] | value parameters [rows][D/G]

with two 4-bit codes in a byte (the even element in the low half) and one pair of fp16 numbers (step, low)
for each group of G elements. A code c stands for fp16(c * step + low), rounded once. For a group with the
smallest element lo and the largest hi, low = lo, step = (hi - lo) / 15 rounded towards zero to fp16, and
c = round_half_even((x - low) / step) held within 0..15; a constant group has step 0 and codes 0, and a
group with an infinity or a NaN reads as NaN. Row r of sequence b is row r % page_size of page
table[b][r / page_size]; the rows of a page that no sequence has reached hold anything, NaN among it.

The queries of a sequence are its last ones: query i of S, at context length n (which counts them), has
position n - S + i. It sees the cached rows at positions 0..n-1 that are not after it (where causal) and,
with a window W, less than W before it. A query that sees nothing gives zeros, and -inf as its log-sum-exp.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"


# ---------------------------------------------------------------------------------------- cases
def listed():
    attn = {"op": "attention", "causal": True, "window": 0, "ragged": 0.0}
    return [
        # one interactive request early in a conversation (16 / 8 heads): nothing but latency
        dict(attn, name="attn_one_token_512", seqs=1, q_len=1, context=512, hq=16, hkv=8, d=128, g=32, page=64),
        # a full server at long contexts: the cache is all of the traffic
        dict(attn, name="attn_tokens_64x32768", seqs=64, q_len=1, context=32768, hq=16, hkv=8, d=128, g=32, page=64,
             ragged=0.5),
        # many short conversations in small pages (32 / 8 heads of 64)
        dict(attn, name="attn_tokens_256x1061", seqs=256, q_len=1, context=1061, hq=32, hkv=8, d=64, g=64, page=16,
             ragged=0.9),
        # a few drafted tokens checked in one pass over a long cache, one group for a whole head
        dict(attn, name="attn_verify_5x7919", seqs=12, q_len=5, context=7919, hq=16, hkv=8, d=128, g=128, page=32,
             ragged=0.3),
        # a prompt's chunk with a sliding window, one key head of 256 for four query heads
        dict(attn, name="attn_chunk_256_window", seqs=16, q_len=256, context=4349, hq=4, hkv=1, d=256, g=32, page=64,
             window=512),
        # long prompts in large chunks: the one that the tensor cores bound
        dict(attn, name="attn_prompt_2048x8192", seqs=4, q_len=2048, context=8192, hq=16, hkv=8, d=128, g=64, page=64,
             ragged=0.1),
        # the new token of every running sequence, appended and read back with what stood before it
        dict(op="append", name="append_one_token_64", seqs=64, q_len=1, context=33, hkv=8, d=128, g=32, page=16,
             ragged=0.8),
        # a batch of whole prompts of very different lengths, appended and read back
        dict(op="append", name="append_prompts_32x4096", seqs=32, q_len=4096, context=4096, hkv=8, d=128, g=64,
             page=64, ragged=0.97),
        # four samples forked from one prompt: their last pages in every one of 28 layers
        dict(op="copy", name="copy_fork_4x28", copies=4, layers=28, pages=64, hkv=8, d=128, g=32, page=16),
        # a batch moved as a whole: pages of 16 layers
        dict(op="copy", name="copy_batch_640x16", copies=640, layers=16, pages=1600, hkv=8, d=64, g=32, page=64),
        # one sequence slides: 4 rows at its start and its latest ones stay
        dict(op="compact", name="compact_slide_1x28", seqs=1, context=512, kept=260, scattered=False, layers=28, hkv=8,
             d=128, g=32, page=16),
        # scattered rows of a batch stay, as an eviction by score leaves them
        dict(op="compact", name="compact_evict_16x4096", seqs=16, context=4096, kept=2045, scattered=True, layers=16,
             hkv=8, d=128, g=64, page=64),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


#: The most that a drawn case reads, writes and computes: below the largest listed ones.
_MOST_BYTES, _MOST_FLOPS, _MOST_PADDED = 1.4e9, 3.5e11, 1.2e9


def draw(rng):
    while True:
        c = _drawn(rng)
        w = work(c)
        padded = c["seqs"] * c["context"] * c["hkv"] * c["d"] * 2 if c["op"] in ("attention", "append") else 0
        if c["op"] == "attention":
            padded = max(padded, c["seqs"] * c["q_len"] * c["hq"] * c["context"])
        if w["bytes"] <= _MOST_BYTES and w["flops"] <= _MOST_FLOPS and padded <= _MOST_PADDED:
            return c


def _drawn(rng):
    op = rng.choice(("attention", "attention", "attention", "append", "copy", "compact"))
    d = rng.choice((64, 128, 256))
    c = {"op": op, "hkv": rng.choice((1, 2, 3, 4, 5, 8)), "d": d,
         "g": rng.choice([g for g in (32, 64, 128) if d % g == 0]), "page": rng.choice((16, 32, 64, 128))}
    if op == "attention":
        c["hq"] = c["hkv"] * rng.choice((1, 2, 3, 4, 7, 8))
        form = rng.choice(("token", "verify", "chunk", "prompt"))
        c["seqs"] = _spread(rng, 1, {"token": 256, "verify": 48, "chunk": 16, "prompt": 6}[form])
        c["q_len"] = {"token": lambda: 1, "verify": lambda: rng.randint(2, 9), "chunk": lambda: _spread(rng, 10, 300),
                      "prompt": lambda: _spread(rng, 300, 2500)}[form]()
        c["context"] = c["q_len"] + _spread(rng, 1, {"token": 30000, "verify": 16000}.get(form, 8000)) - 1
        c["causal"] = rng.random() < 0.85
        c["window"] = _spread(rng, 16, 2048) if rng.random() < 0.25 else 0
        c["ragged"] = rng.choice((0.0, 0.3, 0.9))
    elif op == "append":
        prompt = rng.random() < 0.6
        c["seqs"] = _spread(rng, 1, 48 if prompt else 256)
        c["q_len"] = _spread(rng, 2, 4000) if prompt else 1
        c["context"] = c["q_len"] + (0 if prompt else rng.randint(0, 60))
        c["ragged"] = rng.choice((0.0, 0.5, 0.97))
    elif op == "copy":
        c["layers"] = rng.randint(1, 28)
        c["copies"] = _spread(rng, 1, 400)
        c["pages"] = 2 * c["copies"] + rng.randint(0, 50)
    else:
        c["layers"] = rng.randint(1, 28)
        c["seqs"] = _spread(rng, 1, 16)
        c["context"] = _spread(rng, 2, 4000)
        c["kept"] = max(1, int(c["context"] * rng.uniform(0.1, 0.9)))
        c["scattered"] = rng.random() < 0.5
    return c


def _lengths(c):
    """(queries, context) of each sequence: the longest first, the others down to (1 - ragged) of it."""
    r = c.get("ragged", 0.0)
    got = []
    for b in range(c["seqs"]):
        f = 1.0 - r * ((b * 0.6180339887498949) % 1.0)
        s = max(1, int(round(c["q_len"] * f))) if c["q_len"] > 16 else c["q_len"]
        got.append((s, max(s, int(round(c["context"] * f)))))
    return got


def _row_bytes(c):
    """Bytes of one row of one key head: keys and values, codes and parameters."""
    return 2 * (c["d"] // 2 + 4 * (c["d"] // c["g"]))


def work(c):
    row = _row_bytes(c) * c["hkv"]
    if c["op"] == "attention":
        rows = pairs = tokens = 0
        for s, n in _lengths(c):
            w = c["window"]
            tokens += s
            first = max(0, n - s - w + 1) if w else 0
            rows += n - first
            for_all = s * n
            if c["causal"] or w:
                # query i sees positions max(0, p - w + 1) .. p (or .. n - 1), p = n - s + i
                for_all = 0
                lo, hi = n - s, n - 1
                ends = (lo + hi) * s // 2 + s if c["causal"] else s * n
                if w:
                    k = max(0, hi - max(lo, w) + 1)  # queries with p >= w: the first p - w + 1 positions are out
                    ends -= sum((max(lo, w) - w + 1, hi - w + 1)) * k // 2 if k else 0
                for_all = ends
            pairs += for_all
        return {"bytes": rows * row + tokens * c["hq"] * (4 * c["d"] + 4), "flops": 4.0 * pairs * c["hq"] * c["d"]}
    if c["op"] == "append":
        new, live = (sum(v) for v in zip(*_lengths(c)))
        values = 4 * c["hkv"] * c["d"]  # fp16 keys and values of a row
        return {"bytes": new * (values + row) + live * (row + values), "flops": 6.0 * (new + live) * c["hkv"] * c["d"]}
    if c["op"] == "copy":
        return {"bytes": 2.0 * c["copies"] * c["layers"] * c["page"] * row, "flops": 0.0}
    return {"bytes": 2.0 * c["seqs"] * c["kept"] * c["layers"] * row, "flops": 0.0}


# ---------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c = dict(case)
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    return {"attention": _prepare_attention, "append": _prepare_append, "copy": _prepare_copy,
            "compact": _prepare_compact}[c["op"]](c, gen)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEVICE)


def _table(lengths, page, extra, gen):
    """Block tables over shuffled pages, and the number of pages; entries past a sequence's end are -1."""
    need = [-(-n // page) for n in lengths]
    total = sum(need) + extra
    order = torch.randperm(total, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total, order[at:]


def _fill(pool, c, gen):
    """Quantised keys (some channels much larger, as rotated keys have them) and values in every page."""
    n, hkv, p, d = pool.shape[0], c["hkv"], c["page"], c["d"]
    loud = 1.0 + 3.0 * (torch.rand(d, generator=gen, device=DEVICE) < 0.05)
    step = max(1, (1 << 27) // (hkv * p * d))
    for at in range(0, n, step):
        m = min(step, n - at)
        k = torch.randn((m, hkv, p, d), generator=gen, device=DEVICE) * loud
        v = torch.randn((m, hkv, p, d), generator=gen, device=DEVICE) + 0.25
        pool[at:at + m] = _block(k.half(), v.half(), c)


def _spoil(pool, table, lengths, c):
    """NaN parameters in the rows of the last pages that no sequence has reached."""
    p, half, par = c["page"], c["page"] * c["d"] // 2, 4 * (c["d"] // c["g"])
    for b, n in enumerate(lengths):
        if n % p:
            for at in (half, 2 * half + p * par):
                pool[int(table[b, n // p]), :, at + (n % p) * par:at + p * par] = 0x7F


def _prepare_attention(c, gen):
    sizes = _lengths(c)
    s, n = [x[0] for x in sizes], [x[1] for x in sizes]
    table, pages, _ = _table(n, c["page"], 3, gen)
    pool = torch.empty((pages, c["hkv"], _row_bytes(c) * c["page"]), dtype=torch.uint8, device=DEVICE)
    _fill(pool, c, gen)
    _spoil(pool, table, n, c)
    # queries are a slice of a fused projection's output, as a layer has them
    tokens, width = sum(s), (c["hq"] + 2 * c["hkv"]) * c["d"]
    qkv = torch.randn((tokens, width), generator=gen, device=DEVICE).half()
    starts = [0]
    for x in s:
        starts.append(starts[-1] + x)
    seq = torch.repeat_interleave(torch.arange(len(s), device=DEVICE), torch.tensor(s, device=DEVICE))
    return {"case": c, "pool": pool, "table": table, "qkv": qkv, "offsets": _ints(starts), "context": _ints(n),
            "tokens": tokens, "longest": max(s), "seq": seq,
            "at": torch.arange(tokens, device=DEVICE) - _ints(starts)[seq].long()}


def _prepare_append(c, gen):
    sizes = _lengths(c)
    s, n = [x[0] for x in sizes], [x[1] for x in sizes]
    table, pages, _ = _table(n, c["page"], 2, gen)
    pool = torch.empty((pages, c["hkv"], _row_bytes(c) * c["page"]), dtype=torch.uint8, device=DEVICE)
    _fill(pool, c, gen)
    tokens, width = sum(s), c["hkv"] * c["d"]
    loud = 1.0 + 3.0 * (torch.rand(c["d"], generator=gen, device=DEVICE) < 0.05)
    kv = torch.randn((tokens, 2, c["hkv"], c["d"]), generator=gen, device=DEVICE) * loud
    kv[:, 1, 0, :c["g"]] = 0.5  # a constant group
    kv = kv.half().reshape(tokens, 2 * width)
    starts, rows = [0], [0]
    for x, y in sizes:
        starts.append(starts[-1] + x)
        rows.append(rows[-1] + y)
    seq = torch.repeat_interleave(torch.arange(len(s), device=DEVICE), torch.tensor(s, device=DEVICE))
    row_seq = torch.repeat_interleave(torch.arange(len(n), device=DEVICE), torch.tensor(n, device=DEVICE))
    offsets, context, row_offsets = _ints(starts), _ints(n), _ints(rows)
    ends = torch.arange(tokens, device=DEVICE) - offsets[1:].long()[seq]
    return {"case": c, "pool": pool, "table": table, "kv": kv, "offsets": offsets, "context": context,
            "row_offsets": row_offsets, "tokens": tokens, "rows": rows[-1], "seq": seq, "row_seq": row_seq,
            "position": context[seq].long() + ends,
            "row": torch.arange(rows[-1], device=DEVICE) - row_offsets[row_seq].long()}


def _prepare_copy(c, gen):
    block = _row_bytes(c) * c["page"] * c["hkv"]
    pool = torch.randint(-2**31, 2**31, (c["layers"], c["pages"], block // 4), generator=gen, device=DEVICE,
                         dtype=torch.int32)
    order = torch.randperm(c["pages"], generator=gen, device=DEVICE).to(torch.int32)
    k = c["copies"]
    # forks of one parent share its last page as their source: a quarter of the copies here
    src = torch.where(torch.rand(k, generator=gen, device=DEVICE) < 0.25, order[:1].expand(k), order[:k])
    return {"case": c, "pool": pool, "src": src.contiguous(), "dst": order[k:2 * k].contiguous(), "page_bytes": block}


def _prepare_compact(c, gen):
    n, kept, b, p = c["context"], c["kept"], c["seqs"], c["page"]
    src, total, rest = _table([n] * b, p, b * (-(-kept // p)), gen)
    dst = torch.full_like(src, -1)
    dst[:, :-(-kept // p)] = rest.reshape(b, -1)
    if c["scattered"]:
        rows = torch.rand((b, n), generator=gen, device=DEVICE).argsort(1)[:, :kept].sort(1).values
    else:
        first = min(4, kept)
        one = torch.cat([torch.arange(first, device=DEVICE), torch.arange(n - (kept - first), n, device=DEVICE)])
        rows = one.expand(b, kept)
    words = _row_bytes(c) * p // 4
    pool = torch.randint(-2**31, 2**31, (c["layers"], total, c["hkv"], words), generator=gen, device=DEVICE,
                         dtype=torch.int32)
    return {"case": c, "pool": pool, "src": src, "dst": dst, "kept": rows.reshape(-1).to(torch.int32).contiguous(),
            "offsets": _ints([i * kept for i in range(b + 1)])}


# ---------------------------------------------------------------------------------------- plain forms
def _quantise(x, c):
    """Codes [..., D] and (step, low) pairs [..., D/G, 2] of fp16 rows [..., D]."""
    g = x.float().reshape(*x.shape[:-1], x.shape[-1] // c["g"], c["g"])
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    wide = (hi - lo) / 15.0
    step = wide.half()
    step = torch.where(step.float() > wide, (step.view(torch.int16) - 1).view(torch.float16), step)
    bad = ~torch.isfinite(wide)
    step, low = (t.masked_fill(bad, math.nan) for t in (step, lo.half()))
    some = step.float() > 0
    q = torch.round((g - lo) / torch.where(some, step.float(), 1.0)).clamp(0, 15)
    q = torch.where(some, q, 0.0).to(torch.uint8).reshape(x.shape)
    return q, torch.cat([step, low], -1)


def _block(k, v, c):
    """The bytes [..., block] of rows [..., page, D] of keys and values."""
    parts = []
    for x in (k, v):
        q, par = _quantise(x, c)
        parts.append((q[..., 0::2] | (q[..., 1::2] << 4)).flatten(-2))
        parts.append(par.contiguous().view(torch.uint8).flatten(-3))
    return torch.cat(parts, -1)


def _rows(block, which, c):
    """fp32 values [..., page, D] of keys (0) or values (1) of blocks [..., block]."""
    p, d, ng = c["page"], c["d"], c["d"] // c["g"]
    size = p * (d // 2 + 4 * ng)
    part = block[..., which * size:(which + 1) * size]
    code = part[..., :p * d // 2].reshape(*block.shape[:-1], p, ng, c["g"] // 2)
    par = part[..., p * d // 2:].contiguous().view(torch.float16).reshape(*block.shape[:-1], p, ng, 1, 2).float()
    code = torch.stack([code & 15, code >> 4], -1).flatten(-2).float()
    return (code * par[..., 0] + par[..., 1]).half().float().flatten(-2)


def _plain_attention(s):
    c = s["case"]
    b, longest, d, hkv, share = c["seqs"], s["longest"], c["d"], c["hkv"], c["hq"] // c["hkv"]
    blocks = s["pool"][s["table"].clamp(min=0).long()]  # [B, pages, kv heads, block]
    n = blocks.shape[1] * c["page"]
    context, count = s["context"].long(), (s["offsets"][1:] - s["offsets"][:-1]).long()
    q = torch.zeros((b, longest, hkv, share, d), dtype=torch.float32, device=DEVICE)
    q[s["seq"], s["at"]] = s["qkv"][:, :c["hq"] * d].float().reshape(-1, hkv, share, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(b, hkv, share * longest, d)
    key = torch.arange(n, device=DEVICE)
    pos = (context - count)[:, None] + torch.arange(longest, device=DEVICE)  # [B, S]
    live = (key < context[:, None])[:, None, :]
    if c["causal"]:
        live = live & (key <= pos[..., None])
    if c["window"]:
        live = live & (key > pos[..., None] - c["window"])
    live = live[:, None, None]  # [B, 1, 1, S, N]
    rows = _rows(blocks, 0, c).transpose(1, 2).reshape(b, hkv, n, d)
    rows = torch.where((key < context[:, None])[:, None, :, None], rows, 0.0)
    score = (q @ rows.transpose(-1, -2)).reshape(b, hkv, share, longest, n) * (1.0 / math.sqrt(d))
    score = torch.where(live, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    score = torch.exp(score - torch.where(torch.isfinite(top), top, 0.0))
    total = score.sum(-1, keepdim=True)
    rows = _rows(blocks, 1, c).transpose(1, 2).reshape(b, hkv, n, d)
    rows = torch.where((key < context[:, None])[:, None, :, None], rows, 0.0)
    out = (score.reshape(b, hkv, share * longest, n) @ rows).reshape(b, hkv, share, longest, d)
    out = out / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total)).squeeze(-1)
    out, lse = out.permute(0, 3, 1, 2, 4)[s["seq"], s["at"]], lse.permute(0, 3, 1, 2)[s["seq"], s["at"]]
    return {"output": out.reshape(-1, c["hq"], d).half(), "lse": lse.reshape(-1, c["hq"])}


def _plain_append(s):
    c = s["case"]
    p, hkv, d, ng = c["page"], c["hkv"], c["d"], c["d"] // c["g"]
    kv = s["kv"].reshape(-1, 2, hkv, d)
    page = s["table"][s["seq"], s["position"] // p].long()
    row, pool, half, par = s["position"] % p, s["pool"], p * d // 2, 4 * ng
    for which, at in ((0, 0), (1, half + p * par)):
        q, params = _quantise(kv[:, which], c)
        codes = pool[..., at:at + half].unflatten(-1, (p, d // 2))
        codes[page, :, row] = q[..., 0::2] | (q[..., 1::2] << 4)
        pairs = pool[..., at + half:at + half + p * par].unflatten(-1, (p, par))
        pairs[page, :, row] = params.contiguous().view(torch.uint8).flatten(-2)
    blocks = pool[s["table"].clamp(min=0).long()]
    out = [_rows(blocks, which, c).transpose(2, 3).flatten(1, 2)[s["row_seq"], s["row"]].half() for which in (0, 1)]
    return {"keys": out[0], "values": out[1]}


def _plain_copy(s):
    s["pool"][:, s["dst"].long()] = s["pool"][:, s["src"].long()]
    return {"pool": s["pool"]}


def _plain_compact(s):
    c, pool = s["case"], s["pool"]
    b, kept, p, ng = c["seqs"], c["kept"], c["page"], c["d"] // c["g"]
    to = torch.arange(kept, device=DEVICE)
    rows = s["kept"].reshape(b, kept).long()
    from_page = s["src"].gather(1, rows // p).long()
    to_page = s["dst"][:, to // p].long()
    at = 0
    for words in (c["d"] // 8, ng, c["d"] // 8, ng):  # a row's part of each region, in 32-bit words
        region = pool[..., at:at + p * words].unflatten(-1, (p, words))
        region[:, to_page, :, (to % p).expand(b, kept)] = region[:, from_page, :, rows % p]
        at += p * words
    return {"pool": pool}


# ---------------------------------------------------------------------------------------- the framework's
def _geometry(c):
    return c["page"], c["hkv"], c["d"], c["g"]


def _own_attention(s, cb):
    c, lib = s["case"], cb.lib()
    if "workspace" not in s:  # kept between calls; the kernels leave it as they find it: zero
        size = lib.cactus_cuda_kv4_attention_workspace(c["seqs"], s["tokens"], c["hq"], c["hkv"], c["d"])
        s["workspace"] = torch.zeros(size, dtype=torch.uint8, device=DEVICE)
    out = torch.empty((s["tokens"], c["hq"], c["d"]), dtype=torch.float16, device=DEVICE)
    lse = torch.empty((s["tokens"], c["hq"]), dtype=torch.float32, device=DEVICE)
    rc = lib.cactus_cuda_kv4_attention(
        s["qkv"].data_ptr(), s["qkv"].shape[1], s["offsets"].data_ptr(), s["context"].data_ptr(),
        s["table"].data_ptr(), s["table"].shape[1], s["pool"].data_ptr(), s["pool"].shape[0], s["pool"].stride(0),
        out.data_ptr(), lse.data_ptr(), c["seqs"], s["tokens"], s["longest"], c["hq"], *_geometry(c),
        1.0 / math.sqrt(c["d"]), c["window"], int(c["causal"]), s["workspace"].data_ptr(), s["workspace"].numel(),
        torch.cuda.current_stream().cuda_stream)
    cb.check(rc, "kv4_attention")
    return {"output": out, "lse": lse}


def _own_append(s, cb):
    c, lib, stream = s["case"], cb.lib(), torch.cuda.current_stream().cuda_stream
    width = c["hkv"] * c["d"]
    out = [torch.empty((s["rows"], c["hkv"], c["d"]), dtype=torch.float16, device=DEVICE) for _ in range(2)]
    rc = lib.cactus_cuda_kv4_append(
        s["kv"].data_ptr(), s["kv"].data_ptr() + 2 * width, 2 * width, s["offsets"].data_ptr(),
        s["context"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1], s["pool"].data_ptr(),
        s["pool"].shape[0], s["pool"].stride(0), c["seqs"], s["tokens"], *_geometry(c), stream)
    cb.check(rc, "kv4_append")
    rc = lib.cactus_cuda_kv4_read(
        s["pool"].data_ptr(), s["pool"].shape[0], s["pool"].stride(0), s["table"].data_ptr(), s["table"].shape[1],
        s["row_offsets"].data_ptr(), None, out[0].data_ptr(), out[1].data_ptr(), c["seqs"], s["rows"], *_geometry(c),
        stream)
    cb.check(rc, "kv4_read")
    return {"keys": out[0], "values": out[1]}


def _own_copy(s, cb):
    c, pool = s["case"], s["pool"]
    rc = cb.lib().cactus_cuda_kv_copy_pages(
        pool.data_ptr(), c["pages"], s["page_bytes"], 4 * pool.stride(1), c["layers"], 4 * pool.stride(0),
        s["src"].data_ptr(), s["dst"].data_ptr(), c["copies"], torch.cuda.current_stream().cuda_stream)
    cb.check(rc, "kv_copy_pages")
    return {"pool": pool}


def _own_compact(s, cb):
    c, pool = s["case"], s["pool"]
    rc = cb.lib().cactus_cuda_kv4_compact(
        pool.data_ptr(), pool.shape[1], 4 * pool.stride(1), c["layers"], 4 * pool.stride(0), s["src"].data_ptr(),
        s["dst"].data_ptr(), s["src"].shape[1], s["kept"].data_ptr(), s["offsets"].data_ptr(), c["seqs"],
        s["kept"].numel(), *_geometry(c), torch.cuda.current_stream().cuda_stream)
    cb.check(rc, "kv4_compact")
    return {"pool": pool}


_PLAIN = {"attention": _plain_attention, "append": _plain_append, "copy": _plain_copy, "compact": _plain_compact}
_OWN = {"attention": _own_attention, "append": _own_append, "copy": _own_copy, "compact": _own_compact}


def run(state):
    op = state["case"]["op"]
    if own:
        import cactus_b200
        return _OWN[op](state, cactus_b200)
    return _PLAIN[op](state)


# ---------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    c = dict(case)
    if c["op"] == "attention":
        return _exact_attention(prepare(c, seed))
    if c["op"] == "append":
        return _exact_append(prepare(c, seed))
    return None  # bytes that move: no computed numbers


def _exact_values(raw, pairs, g):
    """Values [rows, heads, D] from code bytes [rows, heads, D/2] and fp16 pairs [rows, heads, D/G, 2]."""
    codes = torch.empty((*raw.shape[:-1], 2 * raw.shape[-1]), dtype=torch.float64, device=DEVICE)
    codes[..., 0::2] = raw.remainder(16).double()
    codes[..., 1::2] = raw.div(16, rounding_mode="floor").double()
    step, low = (pairs[..., i].double().repeat_interleave(g, dim=-1) for i in (0, 1))
    return torch.addcmul(low, codes, step).half().double()


def _exact_attention(s):
    c = s["case"]
    p, d, ng, hkv = c["page"], c["d"], c["d"] // c["g"], c["hkv"]
    share, half = c["hq"] // hkv, p * d // 2
    outs, lses = [], []
    for b, (count, n) in enumerate(_lengths(c)):
        blocks = s["pool"][s["table"][b, :-(-n // p)].long()].transpose(0, 1)  # [heads, pages, block]
        got = []
        for at in (0, half + 4 * ng * p):
            raw = blocks[..., at:at + half].reshape(hkv, -1, d // 2)[:, :n]
            par = blocks[..., at + half:at + half + 4 * ng * p].contiguous().view(torch.float16)
            got.append(_exact_values(raw, par.reshape(hkv, -1, ng, 2)[:, :n], c["g"]))
        t0 = int(s["offsets"][b])
        q = s["qkv"][t0:t0 + count, :c["hq"] * d].double().reshape(count, hkv, share, d)
        place = torch.arange(n - count, n, device=DEVICE)[:, None]
        key = torch.arange(n, device=DEVICE)[None, :]
        hidden = torch.zeros((count, n), dtype=torch.bool, device=DEVICE)
        if c["causal"]:
            hidden |= key > place
        if c["window"]:
            hidden |= key <= place - c["window"]
        out = torch.empty((count, c["hq"], d), dtype=torch.float64, device=DEVICE)
        lse = torch.empty((count, c["hq"]), dtype=torch.float64, device=DEVICE)
        for h in range(c["hq"]):
            score = (q[:, h // share, h % share] @ got[0][h // share].T / d ** 0.5).masked_fill(hidden, -math.inf)
            lse[:, h] = torch.logsumexp(score, -1)
            weight = torch.exp(score - lse[:, h:h + 1]).nan_to_num(0.0)
            out[:, h] = weight @ got[1][h // share]
        outs.append(out)
        lses.append(lse)
    return {"output": torch.cat(outs), "lse": torch.cat(lses)}


def _exact_append(s):
    c = s["case"]
    p, d, g, hkv = c["page"], c["d"], c["g"], c["hkv"]
    ng, half = d // g, p * d // 2
    kv = s["kv"].reshape(-1, 2, hkv, d).double()
    got = []
    for which in (0, 1):
        x = kv[:, which].unflatten(-1, (ng, g))
        low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
        # fifteenths of the range, cut to the 11 bits of fp16 (2^-24 at the least)
        wide = (high - low) / 15
        unit = torch.exp2(torch.floor(torch.log2(wide.clamp(min=2.0 ** -14))) - 10)
        step = torch.floor(wide / unit) * unit
        code = torch.where(step > 0, ((x - low) / torch.where(step > 0, step, 1.0)).round().clamp(0, 15), 0.0)
        new = (code * step + low).half().double().flatten(-2)
        at = which * (half + 4 * ng * p)
        rows = []
        for b, (count, n) in enumerate(_lengths(c)):
            blocks = s["pool"][s["table"][b, :-(-n // p)].long()].transpose(0, 1)
            raw = blocks[..., at:at + half].reshape(hkv, -1, d // 2)[:, :n]
            par = blocks[..., at + half:at + half + 4 * ng * p].contiguous().view(torch.float16)
            old = _exact_values(raw, par.reshape(hkv, -1, ng, 2)[:, :n], g).transpose(0, 1).clone()
            t0 = int(s["offsets"][b])
            old[n - count:] = new[t0:t0 + count]
            rows.append(old)
        got.append(torch.cat(rows))
    return {"keys": got[0], "values": got[1]}
