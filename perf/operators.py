"""Operators around a paged cache held in 4 bits, as cases that can be timed and checked.

``store``    a step's q|k|v rows: q and k rotated with the step's table of cosines and sines, k and v quantised into their page
             slots, and the written rows read back (what a move of cached rows to another cache reads).  Outputs: the rotated q
             rows and the values that the cache now stands for.
``decode``   attention of one new row a request over its 4-bit pages.  Output: the rows.
``prefill``  attention of portions of several rows a request over its 4-bit pages, the portion's own keys among them.
``tables``   a step's integer arrays from the requests' lengths: page tables with new pages taken from a stack of free ones,
             slots, positions, rows' requests, tiles of portions.  Outputs: all of them.

The cache: a page of a KV head is ``page`` rows of dim/2 bytes of codes, then ``page`` pairs (scale, zero) in bfloat16, the whole
rounded up to 16 bytes.  A row of x stands for zero + scale * code with zero = min(x), scale = (max(x) - min(x)) / 15 (both
rounded to bfloat16) and code = round((x - zero) / scale) within 0..15.  The little-endian 32-bit word m of a row of codes holds
element 8m + 2i at bits 4i and element 8m + 2i + 1 at bits 16 + 4i.

Sizes: the heads of the tools' presets (32/4 of 64, 32/32 and 32/8 of 128) and of ``bench.py --compare`` (16/4 of 128 with a
window, capped scores and sinks), pages of 16, contexts up to 8,192 positions.
"""
import math
import random
import types

import torch

own = False

DEVICE = "cuda:0"
CACHE_SEED = 0x51ED


# ------------------------------------------------------------------------------------------------ cases

def _store(rows, heads, kv_heads, dim, page=16, rotary=None, interleaved=False, skip=0):
    return dict(op="store", rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, page=page, rotary=dim if rotary is None else rotary,
                interleaved=interleaved, skip=skip)


def _decode(batch, median, sigma, cap, heads, kv_heads, dim, page=16, window=0, softcap=0.0, sink=False, pad=0, mix=1):
    """``batch`` requests of lognormal contexts (median, sigma; at most cap), ``pad`` padded entries without keys behind them."""
    return dict(op="decode", batch=batch, median=median, sigma=sigma, cap=cap, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                window=window, softcap=softcap, sink=sink, pad=pad, mix=mix)


def _prefill(batch, median, sigma, cap, past, heads, kv_heads, dim, page=16, window=0, softcap=0.0, sink=False, mix=1):
    """``batch`` portions of lognormal lengths (median, sigma; at most cap), each behind up to ``past`` cached positions."""
    return dict(op="prefill", batch=batch, median=median, sigma=sigma, cap=cap, past=past, heads=heads, kv_heads=kv_heads, dim=dim,
                page=page, window=window, softcap=softcap, sink=sink, mix=mix)


def _tables(batch, portion, sigma, past, page=16, limit=8192, pad=0, mix=1):
    """``batch`` requests that bring ``portion`` rows each (lognormal where sigma > 0), behind up to ``past`` cached positions."""
    return dict(op="tables", batch=batch, portion=portion, sigma=sigma, past=past, page=page, limit=limit, pad=pad, mix=mix)


def listed():
    return [
        # a layer of a decode step of 8 requests: latency
        dict(_store(8, 32, 4, 64), name="store_decode8"),
        # a layer of a step of 8,192 prompt rows
        dict(_store(8192, 32, 8, 128, skip=5), name="store_rows8192"),
        # one user in a chat
        dict(_decode(1, 148, 0.0, 148, 32, 4, 64), name="decode_chat"),
        # the headline batch: 8 requests around 1,536 positions
        dict(_decode(8, 1536, 0.1, 2048, 32, 4, 64), name="decode_batch8"),
        # a sliding window, capped scores and a sink, ragged requests, a padded batch
        dict(_decode(27, 900, 1.0, 4096, 16, 4, 128, window=1024, softcap=50.0, sink=True, pad=5), name="decode_window32"),
        # a loaded server: 64 ragged requests
        dict(_decode(64, 1024, 0.9, 8192, 32, 8, 128), name="decode_ragged64"),
        # a full one: 64 long requests
        dict(_decode(64, 8192, 0.0, 8192, 32, 8, 128), name="decode_long64"),
        # the first portion of a chat
        dict(_prefill(1, 148, 0.0, 148, 0, 32, 4, 64), name="prefill_chat"),
        # a whole prompt of 2,048 tokens
        dict(_prefill(1, 2048, 0.0, 2048, 0, 32, 8, 128), name="prefill_2048"),
        # ragged portions behind long cached prefixes
        dict(_prefill(4, 1500, 0.4, 2048, 6000, 32, 8, 128), name="prefill_behind"),
        # a decode step of a full batch, padded to its bucket
        dict(_tables(250, 1, 0.0, 8000, pad=6), name="tables_decode250"),
        # 64 ragged portions
        dict(_tables(64, 120, 1.0, 4000), name="tables_portions64"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


SHAPES = [(32, 4, 64), (32, 8, 128), (32, 32, 128), (16, 4, 128), (8, 1, 64), (12, 12, 64), (24, 2, 128), (10, 5, 96), (4, 2, 256)]


def draw(rng):
    op = rng.choice(["store", "decode", "decode", "prefill", "prefill", "tables"])
    heads, kv, dim = rng.choice(SHAPES)
    page = rng.choice([8, 16, 16, 32, 64])
    masks = rng.choice([{}, {}, dict(window=_log_int(rng, 40, 2000)), dict(softcap=30.0, sink=True)])
    mix = rng.randrange(1 << 20)
    if op == "store":
        rows = _log_int(rng, 1, 8192 * 48 * 128 // ((heads + 2 * kv) * dim))
        rotary = rng.choice([dim, dim, dim // 2])
        return _store(min(rows, 16384), heads, kv, dim, page, rotary, rng.random() < 0.3, rng.randrange(0, 4))
    if op == "decode":
        batch = _log_int(rng, 1, 64)
        most = min(8192, 64 * 8192 * 8 * 128 // (batch * kv * dim))
        cap = _log_int(rng, 1, most)
        return _decode(batch, max(1, cap // 2), rng.uniform(0.0, 1.2), cap, heads, kv, dim, page, pad=rng.randrange(0, 4), mix=mix, **masks)
    if op == "prefill":
        batch = _log_int(rng, 1, 8)
        cap = _log_int(rng, 2, min(2048, 4 * 2048 // batch))
        past = rng.choice([0, _log_int(rng, 1, min(6000, 4 * 6000 // batch))])
        heads, kv, dim = rng.choice([s for s in SHAPES if s[0] * s[2] <= 32 * 128])
        return _prefill(batch, max(2, cap // 2), rng.uniform(0.0, 1.0), cap, past, heads, kv, dim, page, mix=mix, **masks)
    batch = _log_int(rng, 1, 512)
    portion = rng.choice([1, 1, _log_int(rng, 2, max(2, 8192 // batch))])
    return _tables(batch, portion, 0.0 if portion == 1 else rng.uniform(0.0, 0.8), _log_int(rng, 1, 6000), page, pad=rng.randrange(0, 8), mix=mix)


def _lognormal(rng, median, sigma, low, high):
    return max(low, min(high, int(round(median * math.exp(sigma * rng.gauss(0.0, 1.0))))))


def _lengths(case):
    """Per request (cached positions before the step, rows of the step)."""
    rng = random.Random(case["mix"])
    if case["op"] == "decode":
        ends = [_lognormal(rng, case["median"], case["sigma"], 1, case["cap"]) for _ in range(case["batch"])]
        return [(e - 1, 1) for e in ends]
    if case["op"] == "prefill":
        out = []
        for _ in range(case["batch"]):
            n = _lognormal(rng, case["median"], case["sigma"], 2, case["cap"])
            out.append((rng.randrange(case["past"] // 2, case["past"] + 1), n))
        return out
    out = []
    for _ in range(case["batch"]):
        n = 1 if case["portion"] == 1 else _lognormal(rng, case["portion"], case["sigma"], 1, case["limit"] // 4)
        out.append((rng.randrange(0, min(case["past"], case["limit"] - n) + 1), n))
    return out


def work(case):
    h, kv, d = case.get("heads"), case.get("kv_heads"), case.get("dim")
    if case["op"] == "store":
        T = case["rows"]
        cached = T * 2 * kv * (d // 2 + 4)
        moved = T * ((h + 2 * kv) * d * 2 + h * d * 2 + case["rotary"] * 4 + 4)
        return {"bytes": moved + 2 * cached + T * 2 * kv * d * 2, "flops": T * (3 * (h + kv) * d + 8 * 2 * kv * d)}
    if case["op"] == "tables":
        spans = _lengths(case)
        rows, page = sum(n for _, n in spans), case["page"]
        new = sum(-(-(s + n) // page) - -(-s // page) for s, n in spans)
        return {"bytes": 4 * (2 * len(spans) + 3 * rows + 2 * new + 2 * len(spans)), "flops": 4 * rows}
    keys = pairs = rows = 0
    w = case["window"]
    for start, n in _lengths(case):
        end = start + n
        first = max(0, start + 1 - w) if w else 0
        keys += end - first
        rows += n
        full = n * start + n * (n + 1) // 2
        pairs += full if not w else sum(min(start + i + 1, w) for i in range(n))
    return {"bytes": keys * kv * (d // 2 + 4) * 2 + rows * h * d * 4, "flops": 4 * h * d * pairs}


# ------------------------------------------------------------------------------------------------ the cache in plain operations

def _page_bytes(page, dim):
    return (page * (dim // 2 + 4) + 15) // 16 * 16


def _parts(cache, page, dim):
    """The code bytes [.., page, dim/2] and the (scale, zero) pairs [.., page, 2] of pages [.., bytes]."""
    n = page * (dim // 2)
    codes = cache[..., :n].unflatten(-1, (page, dim // 2))
    pairs = cache[..., n:n + 4 * page].contiguous().view(torch.bfloat16).unflatten(-1, (page, 2))
    return codes, pairs


def _unpacked(codes, dim):
    """uint8 [.., dim/2] -> integers [.., dim]: byte 0 of a word holds elements 0, 2, byte 1 4, 6, byte 2 1, 3, byte 3 5, 7."""
    b = codes.unflatten(-1, (dim // 8, 4))
    both = torch.stack((b & 15, b >> 4), dim=-1)                              # [.., words, byte, half]
    both = both.unflatten(-2, (2, 2))                                         # [.., words, odd, pair of bytes, half]
    return both.movedim(-3, -1).flatten(-4)                                   # [.., words, (byte pair, half, odd)]


def _packed(codes, dim):
    """Integers [.., dim] -> uint8 [.., dim/2]."""
    c = codes.to(torch.uint8).unflatten(-1, (dim // 8, 2, 2, 2)).movedim(-1, -3)    # [.., words, odd, byte pair, half]
    return (c[..., 0] | (c[..., 1] << 4)).flatten(-3)


def _quantised(x):
    """float32 [.., dim] -> codes (float32 whole numbers), scale and zero (bfloat16)."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    zero = low.to(torch.bfloat16)
    scale = ((high - low) / 15.0).to(torch.bfloat16)
    s = scale.float()
    code = torch.where(s > 0, ((x - zero.float()) / s), torch.zeros_like(x)).round().clamp(0, 15)
    return code, scale, zero


def _filled(pages, kv, page, dim, gen, base):
    """Pages of keys or values that were quantised: normal rows around an offset of each channel (``base``)."""
    out = torch.zeros((pages, kv, _page_bytes(page, dim)), dtype=torch.uint8, device=DEVICE)
    step = max(1, (1 << 27) // (kv * page * dim))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        x = torch.randn((n, kv, page, dim), generator=gen, device=DEVICE) + base
        code, scale, zero = _quantised(x)
        k = page * (dim // 2)
        out[at:at + n, :, :k] = _packed(code, dim).flatten(-2)
        out[at:at + n, :, k:k + 4 * page] = torch.cat((scale, zero), dim=-1).flatten(-2).view(torch.uint8)
    return out


# ------------------------------------------------------------------------------------------------ inputs

def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _context(spans, pad):
    """A step's integer arrays, as the batch builder makes them (portions in tiles of 64 rows)."""
    starts, tiles, at = [], [], 0
    for i, (s, n) in enumerate(spans):
        starts.append(at)
        if n > 1:
            tiles += [(i, q) for q in range(0, n, 64)]
        at += n
    single = all(n == 1 for _, n in spans)
    ends = [s + n for s, n in spans]
    rows = at + pad
    return types.SimpleNamespace(
        rows=rows, seqs=len(spans) + pad, decode_seqs=rows if single else 0, prefill_rows=0 if single else rows,
        prefill_tiles=len(tiles), tile_rows=64, max_ctx=max(ends), max_decode_ctx=max(ends) if single else 0,
        max_q_len=max(n for _, n in spans),
        positions=_ints([s + i for s, n in spans for i in range(n)] + [-1] * pad),
        row_seq=_ints([i for i, (_, n) in enumerate(spans) for _ in range(n)] + list(range(len(spans), len(spans) + pad))),
        seq_q_start=_ints(starts + [at + i for i in range(pad)]), seq_q_len=_ints([n for _, n in spans] + [1] * pad),
        seq_ctx_len=_ints(ends + [0] * pad),
        decode_order=_ints(sorted(range(len(spans) + pad), key=lambda i: -(ends + [0] * pad)[i])),
        tile_seq=_ints([t for t, _ in tiles]), tile_q0=_ints([q for _, q in tiles]), options={})


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    s = types.SimpleNamespace(case=case)
    if case["op"] == "tables":
        spans = _lengths(case)
        page, pad = case["page"], case["pad"]
        held = [-(-a // page) for a, _ in spans]
        need = sum(-(-(a + n) // page) for a, n in spans)
        width = -(-case["limit"] // page)
        total = need + 37
        ids = torch.randperm(total, generator=gen, device=DEVICE).to(torch.int32)
        table = torch.full((len(spans), width), -1, dtype=torch.int32)
        host, at = ids.cpu(), 0
        for i, n in enumerate(held):
            table[i, :n] = host[at:at + n]
            at += n
        s.table = table.to(DEVICE)
        s.free = ids[at:].contiguous()
        s.count = _ints([total - at])
        s.start, s.n = _ints([a for a, _ in spans]), _ints([n for _, n in spans])
        s.rows = sum(n for _, n in spans) + pad
        s.tiles = sum(-(-n // 64) for _, n in spans if n > 1) + (0 if case["portion"] == 1 else 3)
        # where a program keeps the arrays of its steps
        def room(n):
            return torch.empty(n, dtype=torch.int32, device=DEVICE)
        s.step = {"seq_q_start": room(len(spans)), "seq_ctx_len": room(len(spans)), "positions": room(s.rows), "row_seq": room(s.rows),
                  "slot_mapping": room(s.rows), "tile_seq": room(s.tiles), "tile_q0": room(s.tiles), "free_left": room(1)}
        s.status = room(4)
        return s
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if case["op"] == "store":
        T, rot = case["rows"], case["rotary"]
        s.qkv = torch.randn((T, (h + 2 * kv) * d), generator=gen, device=DEVICE).to(torch.bfloat16)
        where = torch.randint(0, 8192, (T,), generator=gen, device=DEVICE).double()
        angle = where[:, None] * (10000.0 ** (-torch.arange(0, rot, 2, device=DEVICE).double() / rot))
        s.table = torch.cat((angle.cos(), angle.sin()), dim=1).float()
        pages = -(-T // page) + 3
        s.slots = torch.randperm((pages - 1) * page, generator=gen, device=DEVICE)[:T].to(torch.int32)     # the last page is nobody's
        s.slots[:case["skip"]] = -1
        s.k = torch.zeros((pages, kv, _page_bytes(page, d)), dtype=torch.uint8, device=DEVICE)
        s.v = torch.zeros_like(s.k)
        return s
    spans = _lengths(case)
    pad = case.get("pad", 0)
    blocks = [-(-(a + n) // page) for a, n in spans]
    s.ctx = _context(spans, pad)
    pages = sum(blocks) + 2
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32).cpu()
    width = max(blocks)
    table = torch.full((len(spans) + pad, width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(blocks):
        table[i, :n] = order[at:at + n]
        at += n
    s.tables = table.to(DEVICE)
    outliers = 2.0 * torch.randn((kv, 1, d), generator=gen, device=DEVICE) * (torch.rand((kv, 1, d), generator=gen, device=DEVICE) < 0.1)
    s.k = _filled(pages, kv, page, d, gen, outliers)
    s.v = _filled(pages, kv, page, d, gen, 0.0)
    s.q = (1.5 * torch.randn((s.ctx.rows, h * d), generator=gen, device=DEVICE)).to(torch.bfloat16)
    s.sink = torch.randn((h,), generator=gen, device=DEVICE) if case["sink"] else None
    return s


# ------------------------------------------------------------------------------------------------ one pass

def _turned(x, table, rotary, interleaved):
    """x float32 [T, heads, dim] rotated over its first ``rotary`` elements; table [T, cosines | sines]."""
    cos, sin = table[:, None, :rotary // 2], table[:, None, rotary // 2:]
    head, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = head[..., :rotary // 2], head[..., rotary // 2:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1)


def _store_plain(s):
    c = s.case
    h, kv, d, page, T = c["heads"], c["kv_heads"], c["dim"], c["page"], c["rows"]
    x = s.qkv.float().view(T, h + 2 * kv, d)
    qk = _turned(x[:, :h + kv], s.table, c["rotary"], c["interleaved"])
    used = (s.slots >= 0)
    slot = torch.where(used, s.slots.long(), torch.full_like(s.slots, s.k.shape[0] * page - 1, dtype=torch.long))
    at, off = slot // page, slot % page
    kept = {"q": qk[:, :h].reshape(T, h * d).to(torch.bfloat16)}
    n = page * (d // 2)
    for name, rows, cache in (("k", qk[:, h:], s.k), ("v", x[:, h + kv:], s.v)):
        code, scale, zero = _quantised(rows)
        codes = cache[..., :n].unflatten(-1, (page, d // 2))
        pairs = cache[..., n:n + 4 * page].unflatten(-1, (page, 4))
        old = codes[at, :, off]
        codes[at, :, off] = torch.where(used[:, None, None], _packed(code, d), old)
        both = torch.cat((scale, zero), dim=-1).view(torch.uint8)
        pairs[at, :, off] = torch.where(used[:, None, None], both, pairs[at, :, off])
        got = _unpacked(codes[at, :, off], d).float()
        two = pairs[at, :, off].contiguous().view(torch.bfloat16).float()
        values = (two[..., 1:] + two[..., :1] * got).to(torch.bfloat16)
        kept[name] = torch.where(used[:, None, None], values, torch.zeros_like(values)).view(T, kv * d)
    return kept


def _gathered(cache, tables, page, dim):
    """float32 [requests, kv heads, positions, dim] of the requests' pages."""
    codes, pairs = _parts(cache[tables.clamp(min=0).long()], page, dim)        # [S, blocks, kv, page, ..]
    two = pairs.float()
    x = two[..., 1:] + two[..., :1] * _unpacked(codes, dim).float()
    return x.movedim(2, 1).flatten(2, 3)


def _softmax_rows(scores, seen, sink, softcap):
    """Probabilities of float32 scores [.., rows, keys]; rows that see nothing are zero."""
    if softcap:
        scores = softcap * torch.tanh(scores / softcap)
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    if sink is not None:
        total = total + torch.where(total > 0, torch.exp(sink - top), torch.zeros_like(total))
    return e / torch.where(total > 0, total, torch.ones_like(total))


def _attention_plain(s):
    c = s.case
    h, kv, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    x, S = s.ctx, s.tables.shape[0]
    n, G = x.max_q_len, h // kv
    k, v = _gathered(s.k, s.tables, page, d), _gathered(s.v, s.tables, page, d)
    L = k.shape[2]
    # rows of the requests side by side, [S, n]; those behind a request's own read row 0 and are not returned
    i = torch.arange(n, device=DEVICE)
    row = (x.seq_q_start[:, None] + i).long()
    real = i < x.seq_q_len[:, None]
    q = s.q[torch.where(real, row, torch.zeros_like(row))].float().view(S, n, kv, G, d).permute(0, 2, 3, 1, 4)
    at = (x.seq_ctx_len - x.seq_q_len)[:, None] + i
    key = torch.arange(L, device=DEVICE)
    seen = key <= at[..., None]
    if c["window"]:
        seen &= key > at[..., None] - c["window"]
    scores = torch.matmul(q.reshape(S, kv, G * n, d), k.transpose(-1, -2)).view(S, kv, G, n, L) * (d ** -0.5)
    sink = s.sink.view(1, kv, G, 1, 1) if s.sink is not None else None
    p = _softmax_rows(scores, seen[:, None, None], sink, c["softcap"])
    o = torch.matmul(p.view(S, kv, G * n, L), v).view(S, kv, G, n, d).permute(0, 3, 1, 2, 4).reshape(S, n, h * d)
    out = torch.empty((x.rows, h * d), dtype=torch.bfloat16, device=DEVICE)
    out[row[real]] = o[real].to(torch.bfloat16)
    return out


def _tables_plain(s):
    c = s.case
    page, width = c["page"], s.table.shape[1]
    start, n = s.start.long(), s.n.long()
    ends = start + n
    held, need = (start + page - 1) // page, (ends + page - 1) // page
    new = need - held
    first = torch.cumsum(new, 0) - new                                     # new pages of the requests before
    q_start = torch.cumsum(n, 0) - n
    j = torch.arange(width, device=DEVICE)
    fresh = (j >= held[:, None]) & (j < need[:, None])
    pick = s.count.long() - 1 - (first[:, None] + j - held[:, None])
    table = torch.where(fresh, s.free[torch.where(fresh, pick, torch.zeros_like(pick))], s.table)
    r = torch.arange(s.rows, device=DEVICE)
    total = n.sum()
    seq = (torch.searchsorted(q_start, r, right=True) - 1)
    real = r < total
    at = torch.where(real, start[seq] + r - q_start[seq], torch.full_like(r, -1))
    slot = table[seq, at.clamp(min=0) // page] * page + at.clamp(min=0) % page
    t = torch.where(n > 1, (n + 63) // 64, torch.zeros_like(n))
    t_start = torch.cumsum(t, 0) - t
    k = torch.arange(s.tiles, device=DEVICE)
    t_seq = torch.searchsorted(t_start + t, k, right=True).clamp(max=len(n) - 1)
    t_real = k < t.sum()
    none = torch.full_like(k, -1)
    out = {"block_tables": table, "free_left": s.count - new.sum(), "seq_q_start": q_start, "seq_ctx_len": ends, "positions": at,
           "row_seq": torch.where(real, seq, torch.zeros_like(seq)), "slot_mapping": torch.where(real, slot, torch.full_like(r, -1)),
           "tile_seq": torch.where(t_real, t_seq, none), "tile_q0": torch.where(t_real, (k - t_start[t_seq]) * 64, none)}
    return {name: v.to(torch.int32) for name, v in out.items()}


def run(state):
    s = state
    c = s.case
    if not own:
        return {"store": _store_plain, "decode": _attention_plain, "prefill": _attention_plain, "tables": _tables_plain}[c["op"]](s)
    from kvcm.kernels import library as K
    if c["op"] == "tables":
        K.step_tables(s.start, s.n, s.table, s.free, s.count, c["page"], **s.step, status=s.status, tile_rows=64)
        return {"block_tables": s.table, **s.step}
    h, kv, d, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    if c["op"] == "store":
        q = torch.empty((c["rows"], h * d), dtype=torch.bfloat16, device=DEVICE)
        k = torch.zeros((c["rows"], kv * d), dtype=torch.bfloat16, device=DEVICE)
        v = torch.zeros_like(k)
        K.rope_cache_q4(s.qkv, s.table, c["interleaved"], s.slots, s.k, s.v, q, h, kv, d, page)
        K.read_cache_q4(s.k, s.v, s.slots, k, v, kv, d, page)
        return {"q": q, "k": k, "v": v}
    out = torch.empty_like(s.q)
    K.paged_attention_q4(s.q, out, s.k, s.v, s.tables, s.ctx, h, kv, d, page, d ** -0.5, c["window"], c["softcap"], s.sink)
    return out


# ------------------------------------------------------------------------------------------------ in 64 bits

def _words(cache, page, dim):
    """Values float64 [.., page, dim] of pages [.., bytes], element by element from the 32-bit words of the codes."""
    n = page * (dim // 2)
    words = cache[..., :n].contiguous().view(torch.int32).to(torch.int64).unflatten(-1, (page, dim // 8))
    shift = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=cache.device)
    code = ((words[..., None] >> shift) & 15).flatten(-2).double()
    pair = cache[..., n:n + 4 * page].contiguous().view(torch.int16).to(torch.int32).unflatten(-1, (page, 2))
    pair = (pair << 16).view(torch.float32).double()
    return pair[..., 1].unsqueeze(-1) + pair[..., 0].unsqueeze(-1) * code


def _exact_store(s):
    c = s.case
    h, kv, d, T, rot = c["heads"], c["kv_heads"], c["dim"], c["rows"], c["rotary"]
    x = s.qkv.double().view(T, h + 2 * kv, d).clone()
    z = torch.complex(s.table[:, :rot // 2].double(), s.table[:, rot // 2:].double())[:, None]
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if c["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
    w = torch.complex(x[:, :h + kv, first], x[:, :h + kv, second]) * z
    x[:, :h + kv, first], x[:, :h + kv, second] = w.real, w.imag
    out = {"q": x[:, :h].reshape(T, h * d)}
    for name, rows in (("k", x[:, h:h + kv]), ("v", x[:, h + kv:])):
        low, high = rows.min(-1, keepdim=True).values, rows.max(-1, keepdim=True).values
        scale, zero = ((high - low) / 15).to(torch.bfloat16).double(), low.to(torch.bfloat16).double()
        code = torch.round((rows - zero) / torch.where(scale > 0, scale, torch.ones_like(scale))).clamp(0, 15)
        out[name] = torch.where((s.slots >= 0)[:, None, None], zero + scale * code, torch.zeros_like(rows)).reshape(T, kv * d)
    return out


def _exact_attention(s):
    c = s.case
    h, kv, d, page, w = c["heads"], c["kv_heads"], c["dim"], c["page"], c["window"]
    out = torch.zeros((s.ctx.rows, h * d), dtype=torch.float64, device=DEVICE)
    row = 0
    for i, (start, n) in enumerate(_lengths(c)):
        end = start + n
        ids = s.tables[i, :-(-end // page)].long()
        k, v = (_words(x[ids], page, d).transpose(0, 1).flatten(1, 2)[:, :end] for x in (s.k, s.v))
        at = torch.arange(start, end, device=DEVICE)[:, None]
        j = torch.arange(end, device=DEVICE)
        hidden = (j > at) if not w else (j > at) | (j <= at - w)
        for head in range(h):
            g = head // (h // kv)
            q = s.q[row:row + n, head * d:(head + 1) * d].double()
            score = (q @ k[g].T) / math.sqrt(d)
            if c["softcap"]:
                score = c["softcap"] * torch.tanh(score / c["softcap"])
            score[hidden] = -math.inf
            if s.sink is not None:
                score = torch.cat((score, s.sink[head].double().expand(n, 1)), dim=1)
            p = torch.softmax(score, dim=1)[:, :end]
            out[row:row + n, head * d:(head + 1) * d] = p @ v[g]
        row += n
    return out


def exact(case, seed):
    if case["op"] == "tables":
        return None                                                        # whole numbers only
    s = prepare(case, seed)
    return _exact_store(s) if case["op"] == "store" else _exact_attention(s)
