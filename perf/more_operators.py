"""Operators around a paged cache held in 8 bits, as cases that can be timed and checked.

``store``    a step's q|k|v rows: q and k rotated, k and v quantised into their page slots with one scale for each page and KV head
             (a page that grows beyond its scale is brought to the new one), and every row of the touched pages read back.
             Outputs: the rotated q rows and the values that the touched pages now stand for.
``attend``   attention of a step's rows over their pages in 8 bits: one new row a request, or portions of several rows.  Output: the rows.
``prompt``   attention of whole prompts, packed one behind another, over their own rows (nothing cached).  Output: the rows; those
             behind the last prompt stay as they were.
``fork``     requests that begin as copies of others: whole pages shared, the last one, which both would write to, copied in the
             pools of all layers.  Outputs: lengths, page tables, holders of pages, free pages left, the pools.
``compact``  requests that end give their pages back, and the pages in use move to the front of the pools.  Outputs: lengths, page
             tables, holders, the stack of free pages, where every page went, the pools.

The cache: codes in 8 bits (e4m3: a sign, four bits of exponent, three of fraction) [pages, KV heads, page, dim], a float32 scale
[pages, KV heads] which is a power of two, the least 2^e (e >= -60) with 448 * 2^e not below the page's largest element; a row
stands for scale * code.  A page whose first row is written begins anew; else its scale never shrinks, and where it grows the rows
that are there are rounded to the new one.

Sizes: the heads of the tools' presets (32/4 of 64, 32/32 and 32/8 of 128) and of ``bench.py --compare`` (16/4 of 128 with a window,
capped scores and sinks), pages of 16, contexts and prompts up to 8,192 positions.
"""
import math
import random
import types

import torch

own = False

DEVICE = "cuda:0"
FP8 = torch.float8_e4m3fn
LEAST = -60                        # exponent of the smallest scale


# ------------------------------------------------------------------------------------------------ cases

def _store(batch, rows, sigma, heads, kv_heads, dim, page=16, past=0, rotary=None, interleaved=False, dtype="bfloat16", skip=0, mix=1):
    """``batch`` requests that bring about ``rows`` rows each behind up to ``past`` cached ones; ``skip`` rows without a slot."""
    return dict(op="store", batch=batch, rows=rows, sigma=sigma, heads=heads, kv_heads=kv_heads, dim=dim, page=page, past=past,
                rotary=dim if rotary is None else rotary, interleaved=interleaved, dtype=dtype, skip=skip, mix=mix)


def _attend(batch, rows, median, sigma, cap, heads, kv_heads, dim, page=16, window=0, softcap=0.0, sink=False, pad=0, mix=1):
    """``batch`` requests of lognormal contexts (median, sigma; at most cap), of which the last ``rows`` (or fewer) are the step's;
    ``pad`` padded entries without keys behind single rows."""
    return dict(op="attend", batch=batch, rows=rows, median=median, sigma=sigma, cap=cap, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                window=window, softcap=softcap, sink=sink, pad=pad, mix=mix)


def _prompt(batch, median, sigma, cap, heads, kv_heads, dim, window=0, softcap=0.0, sink=False, pad=0, mix=1):
    """``batch`` prompts of lognormal lengths, ``pad`` rows behind the last."""
    return dict(op="prompt", batch=batch, median=median, sigma=sigma, cap=cap, heads=heads, kv_heads=kv_heads, dim=dim, window=window,
                softcap=softcap, sink=sink, pad=pad, mix=mix)


def _fork(batch, children, median, sigma, cap, layers, kv_heads, dim, page=16, pad=0, mix=1):
    """``batch`` requests, each forked into ``children`` more; ``pad`` entries of the call name nobody."""
    return dict(op="fork", batch=batch, children=children, median=median, sigma=sigma, cap=cap, layers=layers, kv_heads=kv_heads, dim=dim,
                page=page, pad=pad, mix=mix)


def _compact(batch, gone, median, sigma, cap, layers, kv_heads, dim, page=16, pad=0, mix=1):
    """``batch`` requests, of which ``gone`` end, in a pool with an eighth of its pages free before."""
    return dict(op="compact", batch=batch, gone=gone, median=median, sigma=sigma, cap=cap, layers=layers, kv_heads=kv_heads, dim=dim,
                page=page, pad=pad, mix=mix)


def listed():
    return [
        # a layer of a decode step of 64 requests: latency
        dict(_store(64, 1, 0.0, 32, 8, 128, past=2000), name="store_decode64"),
        # a layer of a step of about 8,192 prompt rows, some behind cached ones, five of them cached already
        dict(_store(6, 1400, 0.3, 32, 8, 128, past=100, skip=5), name="store_rows8192"),
        # the headline batch: 8 requests around 1,536 positions
        dict(_attend(8, 1, 1536, 0.1, 2048, 32, 4, 64), name="attend_batch8"),
        # a full server: 64 long requests
        dict(_attend(64, 1, 8192, 0.0, 8192, 32, 8, 128), name="attend_long64"),
        # ragged portions behind long cached prefixes
        dict(_attend(4, 1500, 6500, 0.2, 8192, 32, 8, 128), name="attend_behind"),
        # a few chat prompts of a small model
        dict(_prompt(5, 110, 0.5, 300, 32, 4, 64, pad=3), name="prompt_chat"),
        # a packed batch of ragged prompts, a sliding window, capped scores and sinks
        dict(_prompt(16, 600, 0.9, 2048, 16, 4, 128, window=1024, softcap=50.0, sink=True), name="prompt_packed16"),
        # one long prompt
        dict(_prompt(1, 8192, 0.0, 8192, 32, 8, 128), name="prompt_8192"),
        # four samples of one chat
        dict(_fork(1, 3, 300, 0.0, 300, 4, 4, 64), name="fork_chat"),
        # four samples each of 48 ragged requests
        dict(_fork(48, 3, 700, 0.8, 4096, 8, 8, 128, pad=16), name="fork_samples48"),
        # one of eight chats ends
        dict(_compact(8, 1, 300, 0.5, 1000, 4, 4, 64), name="compact_chat8"),
        # 100 of 250 requests end, and the pool is given back
        dict(_compact(250, 100, 150, 1.0, 2048, 8, 8, 128, pad=28), name="compact_250"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


SHAPES = [(32, 4, 64), (32, 8, 128), (32, 32, 128), (16, 4, 128), (8, 1, 64), (12, 12, 64), (24, 2, 128), (10, 5, 96), (4, 2, 256)]


def draw(rng):
    op = rng.choice(["store", "attend", "attend", "attend", "prompt", "prompt", "fork", "compact"])
    heads, kv, dim = rng.choice(SHAPES)
    page = rng.choice([8, 16, 16, 32, 64])
    masks = rng.choice([{}, {}, dict(window=_log_int(rng, 40, 2000)), dict(softcap=30.0, sink=True)])
    mix = rng.randrange(1 << 20)
    if op == "store":
        total = _log_int(rng, 1, min(8192, 8192 * 48 * 128 // ((heads + 2 * kv) * dim)))
        batch = rng.choice([total, max(1, total // 300), 1]) if total <= 512 else max(1, total // _log_int(rng, 100, 2000))
        rotary = rng.choice([dim, dim, dim // 2])
        return _store(batch, max(1, total // batch), 0.0 if total == batch else rng.uniform(0.0, 0.4), heads, kv, dim, page, rng.choice([0, 100, 1000]),
                      rotary, rng.random() < 0.3, rng.choice(["bfloat16", "bfloat16", "float32"]), rng.randrange(0, 4), mix)
    if op == "attend":
        if rng.random() < 0.5:
            batch = _log_int(rng, 1, 64)
            most = min(8192, 64 * 8192 * 8 * 128 // (batch * kv * dim))
            cap = _log_int(rng, 1, most)
            return _attend(batch, 1, max(1, cap // 2), rng.uniform(0.0, 1.2), cap, heads, kv, dim, page, pad=rng.randrange(0, 4), mix=mix, **masks)
        batch = _log_int(rng, 1, 8)
        rows = _log_int(rng, 2, min(2048, 4 * 1500 // batch))
        cap = max(rows, _log_int(rng, 2, min(8192, 4 * 8192 // batch)))
        heads, kv, dim = rng.choice([s for s in SHAPES if s[0] * s[2] <= 32 * 128])
        return _attend(batch, rows, max(2, cap // 2), rng.uniform(0.0, 0.8), cap, heads, kv, dim, page, mix=mix, **masks)
    if op == "prompt":
        heads, kv, dim = rng.choice([s for s in SHAPES if s[2] <= 128 and s[0] * s[2] <= 32 * 128])
        cap = _log_int(rng, 1, 8192)
        batch = _log_int(rng, 1, max(1, min(64, (8192 // cap) ** 2, 16384 // cap)))
        return _prompt(batch, max(1, cap // 2), rng.uniform(0.0, 1.0), cap, heads, kv, dim, pad=rng.randrange(0, 4), mix=mix, **masks)
    layers = rng.choice([1, 2, 4, 8])
    kv, dim = rng.choice([(4, 64), (8, 128), (1, 64), (5, 96), (2, 256)])
    batch = _log_int(rng, 1, 250)
    cap = _log_int(rng, 8, min(4096, 8 * 8 * 128 * 250 * 300 // (layers * kv * dim * batch)))
    if op == "fork":
        return _fork(batch, rng.choice([1, 1, 3, 7]), max(1, cap // 2), rng.uniform(0.0, 0.9), cap, layers, kv, dim, page, rng.randrange(0, 9), mix)
    return _compact(batch, rng.randrange(0, batch + 1), max(1, cap // 2), rng.uniform(0.0, 0.9), cap, layers, kv, dim, page, rng.randrange(0, 9), mix)


def _lognormal(rng, median, sigma, low, high):
    return max(low, min(high, int(round(median * math.exp(sigma * rng.gauss(0.0, 1.0))))))


def _spans(case):
    """Per request (cached positions before the step, rows of the step); for forks and ends (0, positions)."""
    rng = random.Random(case["mix"])
    out = []
    for _ in range(case["batch"]):
        if case["op"] == "store":
            n = _lognormal(rng, case["rows"], case["sigma"], 1, 2 * case["rows"])
            out.append((rng.randrange(0, case["past"] + 1), n))
        elif case["op"] == "attend":
            end = _lognormal(rng, case["median"], case["sigma"], 1 if case["rows"] == 1 else 2, case["cap"])
            n = 1 if case["rows"] == 1 else max(2, min(end, _lognormal(rng, case["rows"], 0.2, 2, case["rows"])))
            out.append((end - n, n))
        else:
            out.append((0, _lognormal(rng, case["median"], case["sigma"], 1, case["cap"])))
    return out


def _tails(case):
    """Pages that a fork has to copy."""
    return case["children"] * sum(n % case["page"] > 0 for _, n in _spans(case))


def _pool(case):
    """Pages in all, pages held, pages free before."""
    held = sum(-(-n // case["page"]) for _, n in _spans(case))
    if case["op"] == "fork":
        free = _tails(case) + 9
    else:
        free = held // 8 + 3
    return held + free, held, free


def _gone(case):
    """The requests that end."""
    return random.Random(case["mix"] + 1).sample(range(case["batch"]), case["gone"])


def work(case):
    h, kv, d, page = case.get("heads"), case["kv_heads"], case["dim"], case.get("page")
    spans = _spans(case)
    rows = sum(n for _, n in spans)
    if case["op"] == "store":
        size = 2 if case["dtype"] == "bfloat16" else 4
        touched = sum(-(-(s + n) // page) * page - s // page * page for s, n in spans)
        moved = rows * ((h + 2 * kv) * d * size + h * d * size + case["rotary"] * 4 + 4)
        return {"bytes": moved + rows * 2 * kv * d + touched * 2 * kv * d * 3, "flops": rows * (3 * (h + kv) * d + 4 * 2 * kv * d)}
    if case["op"] in ("fork", "compact"):
        page_bytes = 2 * case["layers"] * kv * (page * d + 4)
        if case["op"] == "fork":
            pages = _tails(case)
            ints = 2 * case["children"] * sum(-(-n // page) for _, n in spans) + 2 * len(spans) * (1 + case["children"])
        else:
            total, held, free = _pool(case)
            gone = sum(-(-spans[i][1] // page) for i in _gone(case))
            # (pages lie anywhere: those in use beyond the first `left` move)
            left = held - gone
            pages = left * (total - left) // total
            ints = 2 * held + 2 * total
        return {"bytes": 2 * pages * page_bytes + 4 * ints, "flops": ints}
    w = case["window"]
    keys = pairs = 0
    for start, n in spans:
        first = max(0, start + 1 - w) if w else 0
        keys += start + n - first
        pairs += n * start + n * (n + 1) // 2 if not w else sum(min(start + i + 1, w) for i in range(n))
    each = 1 if case["op"] == "attend" else 2
    return {"bytes": keys * kv * d * each * 2 + rows * h * d * 4, "flops": 4 * h * d * pairs}


# ------------------------------------------------------------------------------------------------ the cache in plain operations

def _needed(largest):
    """The scale for a largest element: the least 2^e with 448 * 2^e >= largest, e >= LEAST (float32, exact)."""
    fraction, e = torch.frexp(largest)                                        # largest = fraction * 2^e, fraction in [0.5, 1)
    e = torch.where(fraction > 0.875, e - 8, e - 9)                           # 448 = 0.875 * 2^9
    e = torch.where(largest > 0, e, torch.full_like(e, LEAST)).clamp(min=LEAST)
    return torch.ldexp(torch.ones_like(largest), e)


def _values(codes, scale):
    """float32 [.., page, dim] of codes [.., page, dim] and scales [..]."""
    return codes.float() * scale[..., None, None]


def _filled(pages, kv, page, dim, gen, base, size):
    """Codes and scales of pages of normal rows around an offset of each channel (``base``), ``size`` [pages, kv] times as large."""
    codes = torch.empty((pages, kv, page, dim), dtype=FP8, device=DEVICE)
    scale = torch.empty((pages, kv), dtype=torch.float32, device=DEVICE)
    step = max(1, (1 << 27) // (kv * page * dim))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        x = (torch.randn((n, kv, page, dim), generator=gen, device=DEVICE) + base) * size[at:at + n, :, None, None]
        scale[at:at + n] = _needed(x.abs().amax((-1, -2)))
        codes[at:at + n] = (x / scale[at:at + n, :, None, None]).to(FP8)
    return codes, scale


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


def _page_rows(counts, ids, width):
    """Page tables [requests, width] that take ``counts`` of the page ids in turn, the rest of a row -1."""
    table, at = torch.full((len(counts), width), -1, dtype=torch.int32), 0
    for i, n in enumerate(counts):
        table[i, :n] = ids[at:at + n]
        at += n
    return table


def _prepare_store(s, gen):
    c = s.case
    h, kv, d, page, rot = c["heads"], c["kv_heads"], c["dim"], c["page"], c["rotary"]
    spans = _spans(c)
    blocks = [-(-(a + n) // page) for a, n in spans]
    # the pages that the rows go to (of those before, a program has many more), in any order
    firsts = [a // page for a, _ in spans]
    touched = sum(b - f for b, f in zip(blocks, firsts))
    pages = touched + 3
    order = torch.randperm(pages - 1, generator=gen, device=DEVICE).cpu().tolist()      # (the last page is nobody's)
    slots, look, at = [], [], 0
    for (a, n), f, b in zip(spans, firsts, blocks):
        mine = order[at:at + b - f]
        at += b - f
        slots += [mine[(a + i) // page - f] * page + (a + i) % page for i in range(n)]
        look += [mine[j // page - f] * page + j % page for j in range(f * page, a + n)]      # and the rows before in the first page
    T = len(slots)
    s.rows = T
    s.qkv = torch.randn((T, (h + 2 * kv) * d), generator=gen, device=DEVICE).to(getattr(torch, c["dtype"]))
    where = torch.tensor([a + i for a, n in spans for i in range(n)], device=DEVICE).double()
    angle = where[:, None] * (10000.0 ** (-torch.arange(0, rot, 2, device=DEVICE).double() / rot))
    s.table = torch.cat((angle.cos(), angle.sin()), dim=1).float()
    # (the first rows of a step that a prefix cache had already)
    skip = min(c["skip"], T)
    s.slots = _ints([-1] * skip + slots[skip:])
    s.look = _ints(look)
    sizes = 2.0 ** torch.randint(-2, 2, (2, pages, kv), generator=gen, device=DEVICE).float()
    s.k, s.k_scale = _filled(pages, kv, page, d, gen, 0.0, sizes[0])
    s.v, s.v_scale = _filled(pages, kv, page, d, gen, 0.0, sizes[1])


def _prepare_attend(s, gen):
    c = s.case
    h, kv, d, page, pad = c["heads"], c["kv_heads"], c["dim"], c["page"], c["pad"]
    spans = _spans(c)
    blocks = [-(-(a + n) // page) for a, n in spans]
    s.ctx = _context(spans, pad)
    pages = sum(blocks) + 2
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32).cpu()
    s.tables = _page_rows(blocks + [0] * pad, order, max(blocks)).to(DEVICE)
    outliers = 2.0 * torch.randn((kv, 1, d), generator=gen, device=DEVICE) * (torch.rand((kv, 1, d), generator=gen, device=DEVICE) < 0.1)
    s.k, s.k_scale = _filled(pages, kv, page, d, gen, outliers, torch.ones((pages, kv), device=DEVICE))
    s.v, s.v_scale = _filled(pages, kv, page, d, gen, 0.0, 2.0 ** torch.randint(-1, 2, (pages, kv), generator=gen, device=DEVICE).float())
    s.q = (1.5 * torch.randn((s.ctx.rows, h * d), generator=gen, device=DEVICE)).to(torch.bfloat16)
    s.sink = torch.randn((h,), generator=gen, device=DEVICE) if c["sink"] else None


def _prepare_prompt(s, gen):
    c = s.case
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    spans = _spans(c)
    # prompts of one row come first, as the batch builder puts them
    spans.sort(key=lambda span: span[1] > 1)
    s.ctx = _context(spans, 0)
    s.ctx.decode_seqs = sum(n == 1 for _, n in spans)
    s.ctx.rows += c["pad"]
    # q, k and v as a fused projection leaves them; the rows behind the last prompt hold anything
    s.qkv = torch.randn((s.ctx.rows, (h + 2 * kv) * d), generator=gen, device=DEVICE)
    s.qkv[:, :h * d] *= 1.5
    s.qkv = s.qkv.to(torch.bfloat16)
    s.sink = torch.randn((h,), generator=gen, device=DEVICE) if c["sink"] else None
    s.out = torch.zeros((s.ctx.rows, h * d), dtype=torch.bfloat16, device=DEVICE)


def _prepare_pages(s, gen):
    c = s.case
    kv, d, page = c["kv_heads"], c["dim"], c["page"]
    lengths = [n for _, n in _spans(c)]
    pages, held, free = _pool(c)
    blocks = [-(-n // page) for n in lengths]
    width = -(-c["cap"] // page)
    ids = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    more = c["children"] * c["batch"] if c["op"] == "fork" else 0
    s.tables = _page_rows(blocks + [0] * more, ids.cpu(), width).to(DEVICE)
    s.length = _ints(lengths + [0] * more)
    s.stack = torch.full((pages,), -1, dtype=torch.int32, device=DEVICE)
    s.stack[:free] = ids[held:]
    s.count = _ints([free])
    s.shared = torch.zeros((pages,), dtype=torch.int32, device=DEVICE)
    if c["op"] == "fork":
        s.parents = _ints([i for i in range(c["batch"]) for _ in range(c["children"])] + [-1] * c["pad"])
        s.children = _ints([c["batch"] + i for i in range(more)] + [-1] * c["pad"])
    else:
        s.gone = _ints(_gone(c) + [-1] * c["pad"])
        s.new_tables = torch.empty_like(s.tables)
        s.new_stack = torch.full_like(s.stack, -1)
        s.map = torch.empty_like(s.shared)
        s.new_shared = torch.empty_like(s.shared)
    # where a program keeps what comes of it
    s.new_length, s.holders, s.left = torch.empty_like(s.length), torch.empty_like(s.shared), torch.empty_like(s.count)
    s.status = torch.empty(4, dtype=torch.int32, device=DEVICE)
    # the pools of all layers' keys and values, bytes and scales
    n = 2 * c["layers"]
    s.codes = torch.randint(0, 256, (n, pages, kv, page, d), generator=gen, device=DEVICE, dtype=torch.uint8)
    s.scales = 2.0 ** torch.randint(-9, 3, (n, pages, kv), generator=gen, device=DEVICE).float()


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    s = types.SimpleNamespace(case=case)
    {"store": _prepare_store, "attend": _prepare_attend, "prompt": _prepare_prompt, "fork": _prepare_pages, "compact": _prepare_pages}[case["op"]](s, gen)
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


def _written(codes, scale, rows, slots, page):
    """Rows float32 [T, kv, dim] into the pages of their slots (below zero: nowhere)."""
    pages, used = codes.shape[0], slots >= 0
    # (rows without a slot count for one more page, and leave the last one, which is nobody's, as it was)
    at = torch.where(used, slots.long() // page, torch.full_like(slots, pages, dtype=torch.long))
    off = slots.long().clamp(min=0) % page
    largest = torch.zeros((pages + 1, rows.shape[1]), device=DEVICE)
    largest.scatter_reduce_(0, at[:, None].expand(-1, rows.shape[1]), rows.abs().amax(-1), "amax")
    anew = torch.zeros(pages + 1, device=DEVICE).scatter_reduce_(0, at, (off == 0).float(), "amax") > 0
    mine = at.clamp(max=pages - 1)
    old = scale[mine]
    kept = torch.where(anew[mine][:, None], torch.zeros_like(old), old)
    new = torch.maximum(_needed(largest[mine]), kept)
    # what the touched pages held, at their new scales (a page of several rows is formed for each of them, alike)
    bytes_of = codes.view(torch.uint8)
    before = bytes_of[mine]
    after = torch.where((kept < new)[..., None, None], (_values(before.view(FP8), old) / new[..., None, None]).clamp(-448.0, 448.0).to(FP8).view(torch.uint8), before)
    bytes_of[mine] = torch.where(used[:, None, None, None], after, bytes_of[mine])
    scale[mine] = torch.where(used[:, None], new, scale[mine])
    code = (rows / new[..., None]).to(FP8).view(torch.uint8)
    bytes_of[mine, :, off] = torch.where(used[:, None, None], code, bytes_of[mine, :, off])


def _store_plain(s):
    c = s.case
    h, kv, d, page, T = c["heads"], c["kv_heads"], c["dim"], c["page"], s.rows
    x = s.qkv.float().view(T, h + 2 * kv, d)
    qk = _turned(x[:, :h + kv], s.table, c["rotary"], c["interleaved"])
    out = {"q": qk[:, :h].reshape(T, h * d).to(s.qkv.dtype)}
    look, off = s.look.long() // page, s.look.long() % page
    for name, rows, codes, scale in (("k", qk[:, h:], s.k, s.k_scale), ("v", x[:, h + kv:], s.v, s.v_scale)):
        _written(codes, scale, rows, s.slots, page)
        got = codes.view(torch.uint8)[look, :, off].view(FP8).float() * scale[look][..., None]
        out[name] = got.to(s.qkv.dtype).reshape(-1, kv * d)
    return out


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


def _attention_plain(q, k, v, x, c, at, sink, out):
    """q rows of a step, k and v float32 [requests, kv, keys, dim], ``at`` the position of each request's first row."""
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    S, n, G, L = k.shape[0], x.max_q_len, h // kv, k.shape[2]
    # rows of the requests side by side, [S, n]; those behind a request's own read row 0 and are not returned
    i = torch.arange(n, device=DEVICE)
    row = (x.seq_q_start[:, None] + i).long()
    real = i < x.seq_q_len[:, None]
    q = q[torch.where(real, row, torch.zeros_like(row))].float().view(S, n, kv, G, d).permute(0, 2, 3, 1, 4)
    at = at[:, None] + i
    key = torch.arange(L, device=DEVICE)
    seen = key <= at[..., None]
    if c["window"]:
        seen &= key > at[..., None] - c["window"]
    scores = torch.matmul(q.reshape(S, kv, G * n, d), k.transpose(-1, -2)).view(S, kv, G, n, L) * (d ** -0.5)
    sink = sink.view(1, kv, G, 1, 1) if sink is not None else None
    p = _softmax_rows(scores, seen[:, None, None], sink, c["softcap"])
    o = torch.matmul(p.view(S, kv, G * n, L), v).view(S, kv, G, n, d).permute(0, 3, 1, 2, 4).reshape(S, n, h * d)
    out[row[real]] = o[real].to(torch.bfloat16)
    return out


def _attend_plain(s):
    c, x = s.case, s.ctx
    ids = s.tables.clamp(min=0).long()
    k, v = (_values(codes.view(torch.uint8)[ids].view(FP8), scale[ids]).movedim(2, 1).flatten(2, 3) for codes, scale in ((s.k, s.k_scale), (s.v, s.v_scale)))
    return _attention_plain(s.q, k, v, x, c, x.seq_ctx_len - x.seq_q_len, s.sink, torch.empty_like(s.q))


def _prompt_plain(s):
    c, x = s.case, s.ctx
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    i = torch.arange(x.max_q_len, device=DEVICE)
    row = (x.seq_q_start[:, None] + torch.minimum(i, x.seq_q_len[:, None] - 1)).long()
    k, v = (s.qkv[:, at * d:(at + kv) * d][row].float().view(row.shape[0], row.shape[1], kv, d).transpose(1, 2) for at in (h, h + kv))
    return _attention_plain(s.qkv[:, :h * d], k, v, x, c, torch.zeros_like(x.seq_q_len), s.sink, s.out)


def _fork_plain(s):
    page, width = s.case["page"], s.tables.shape[1]
    real = s.parents >= 0
    p, child = s.parents.clamp(min=0).long(), torch.where(real, s.children, s.children[0]).long()
    p = torch.where(real, p, p[0])                                            # (entries of nobody repeat the first)
    n = s.length[p].long()
    full, tail = n // page, real & (n % page > 0)
    rank = torch.cumsum(tail, 0) - 1
    new = s.stack[(s.count.long() - 1 - rank).clamp(min=0)]
    j = torch.arange(width, device=DEVICE)
    rows = s.tables[p]
    last = rows.gather(1, full.clamp(max=width - 1)[:, None])[:, 0]
    first_new = torch.where(real, new, new[0])
    first_tail = torch.where(real, tail, tail[0])
    s.tables[child] = torch.where(j < full[:, None], rows, torch.where((j == full[:, None]) & first_tail[:, None], first_new[:, None], s.tables[child]))
    s.new_length.copy_(s.length)
    s.new_length[child] = n.to(torch.int32)
    s.holders.copy_(s.shared)
    held = (j < full[:, None]) & real[:, None]
    s.holders.index_put_((torch.where(held, rows, torch.zeros_like(rows)).long().flatten(),), held.flatten().to(torch.int32), accumulate=True)
    s.left.copy_(s.count - tail.sum())
    # (entries without a page to copy write a page over itself)
    src = torch.where(tail, last, s.stack[0]).long()
    dst = torch.where(tail, new, s.stack[0]).long()
    for pool in (s.codes, s.scales):
        pool[:, dst] = pool[:, src]
    return {"length": s.new_length, "tables": s.tables, "shared": s.holders, "left": s.left, "codes": s.codes, "scales": s.scales}


def _compact_plain(s):
    page, pages = s.case["page"], s.shared.numel()
    real = s.gone >= 0
    ends = torch.zeros(s.length.numel() + 1, dtype=torch.bool, device=DEVICE)
    ends[torch.where(real, s.gone, s.length.numel()).long()] = True
    ends = ends[:-1]
    blocks = (s.length.long() + page - 1) // page
    held = torch.arange(s.tables.shape[1], device=DEVICE) < blocks[:, None]
    given = held & ends[:, None]
    s.holders.copy_(s.shared)
    s.holders.index_put_((torch.where(given, s.tables, torch.zeros_like(s.tables)).long().flatten(),), -given.flatten().to(torch.int32), accumulate=True)
    freed = s.holders < 0
    s.holders.clamp_(min=0)
    # freed pages onto the stack, the lowest on top
    count = int(s.count)
    ids = torch.nonzero(freed)[:, 0].flip(0).to(torch.int32)
    s.stack[count:count + ids.numel()] = ids
    s.new_length.copy_(torch.where(ends, torch.zeros_like(s.length), s.length))
    s.left.copy_(s.count + ids.numel())
    # pages in use behind the first `used` move into the free ones before, in their order
    free = count + ids.numel()
    used = pages - free
    is_free = torch.zeros(pages, dtype=torch.bool, device=DEVICE)
    is_free[s.stack[:free].long()] = True
    holes = torch.nonzero(is_free[:used])[:, 0]
    movers = torch.nonzero(~is_free[used:])[:, 0] + used
    s.map.copy_(torch.where(is_free, -1, torch.arange(pages, device=DEVICE)))
    s.map[movers] = holes.to(torch.int32)
    live = held & ~ends[:, None]
    s.new_tables.copy_(torch.where(live, s.map[torch.where(live, s.tables, torch.zeros_like(s.tables)).long()], s.tables))
    s.new_shared.zero_()
    s.new_shared[:used] = s.holders[:used]
    s.new_shared[holes] = s.holders[movers]
    s.new_stack[:free] = torch.arange(pages - 1, used - 1, -1, device=DEVICE)
    for pool in (s.codes, s.scales):
        pool[:, holes] = pool[:, movers]
    return _compacted(s)


def _compacted(s):
    return {"length": s.new_length, "tables": s.new_tables, "shared": s.new_shared, "stack": s.new_stack, "left": s.left, "map": s.map,
            "codes": s.codes, "scales": s.scales}


def run(state):
    s = state
    c = s.case
    if not own:
        return {"store": _store_plain, "attend": _attend_plain, "prompt": _prompt_plain, "fork": _fork_plain, "compact": _compact_plain}[c["op"]](s)
    from kvcm.kernels import library as K
    if c["op"] == "fork":
        K.fork_requests(s.parents, s.children, s.length, s.tables, s.shared, s.stack, s.count, c["page"], [s.codes, s.scales],
                        seq_len_out=s.new_length, shared_out=s.holders, free_left=s.left, status=s.status)
        return {"length": s.new_length, "tables": s.tables, "shared": s.holders, "left": s.left, "codes": s.codes, "scales": s.scales}
    if c["op"] == "compact":
        K.release_requests(s.gone, s.length, s.tables, s.shared, s.stack, s.count, c["page"],
                           seq_len_out=s.new_length, shared_out=s.holders, free_left=s.left, status=s.status)
        K.compact_pages(s.new_length, s.tables, s.holders, s.stack, s.left, c["page"], [s.codes, s.scales],
                        tables_out=s.new_tables, shared_out=s.new_shared, free_out=s.new_stack, page_map=s.map, status=s.status)
        return _compacted(s)
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    if c["op"] == "store":
        q = torch.empty((s.rows, h * d), dtype=s.qkv.dtype, device=DEVICE)
        k = torch.empty((s.look.numel(), kv * d), dtype=s.qkv.dtype, device=DEVICE)
        v = torch.empty_like(k)
        K.rope_cache_q8(s.qkv, s.table, c["interleaved"], s.slots, s.k, s.v, s.k_scale, s.v_scale, q, h, kv, d)
        K.read_cache_q8(s.k, s.v, s.k_scale, s.v_scale, s.look, k, v)
        return {"q": q, "k": k, "v": v}
    if c["op"] == "attend":
        out = torch.empty_like(s.q)
        K.paged_attention_q8(s.q, out, s.k, s.v, s.k_scale, s.v_scale, s.tables, s.ctx, h, kv, d, d ** -0.5, c["window"], c["softcap"], s.sink)
        return out
    q, k, v = s.qkv[:, :h * d], s.qkv[:, h * d:(h + kv) * d], s.qkv[:, (h + kv) * d:]
    K.prompt_attention(q, k, v, s.out, s.ctx, h, kv, d, d ** -0.5, c["window"], c["softcap"], s.sink)
    return s.out


# ------------------------------------------------------------------------------------------------ in 64 bits

def _code_value(y):
    """The e4m3 value next to y (float64, |y| <= 448): three bits of fraction, exponents from -6 on, ties to even."""
    e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20))).clamp(min=-6.0)
    step = torch.exp2(e - 3.0)
    return torch.round(y / step) * step


def _exact_store(s):
    c = s.case
    h, kv, d, page, T, rot = c["heads"], c["kv_heads"], c["dim"], c["page"], s.rows, c["rotary"]
    x = s.qkv.double().view(T, h + 2 * kv, d).clone()
    z = torch.complex(s.table[:, :rot // 2].double(), s.table[:, rot // 2:].double())[:, None]
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if c["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
    w = torch.complex(x[:, :h + kv, first], x[:, :h + kv, second]) * z
    x[:, :h + kv, first], x[:, :h + kv, second] = w.real, w.imag
    out = {"q": x[:, :h].reshape(T, h * d)}
    slots = s.slots.long()
    slots, x = slots[slots >= 0], x[slots >= 0]
    look = s.look.long()
    for name, rows, codes, scale in (("k", x[:, h:h + kv], s.k, s.k_scale), ("v", x[:, h + kv:], s.v, s.v_scale)):
        value = codes.float().double() * scale.double()[..., None, None]
        old = scale.double()
        old[torch.unique(slots[slots % page == 0] // page)] = 0.0
        where, back = torch.unique(slots // page, return_inverse=True)
        top = torch.zeros((where.numel(), kv), dtype=torch.float64, device=DEVICE).index_reduce_(0, back, rows.abs().amax(-1), "amax")
        need = torch.exp2(torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0)).clamp(min=LEAST))
        new = torch.maximum(need, old[where])[..., None, None]
        value[where] = _code_value((value[where] / new).clamp(-448.0, 448.0)) * new
        value[slots // page, :, slots % page] = _code_value(rows / new[back][..., 0]) * new[back][..., 0]
        out[name] = value[look // page, :, look % page].reshape(-1, kv * d)
    return out


def _exact_rows(q, k, v, at, c, sink, out):
    """Rows of one request: q [n, heads * dim], k and v [kv, keys, dim] in float64, positions ``at`` [n]."""
    h, kv, d, w = c["heads"], c["kv_heads"], c["dim"], c["window"]
    j = torch.arange(k.shape[1], device=DEVICE)
    hidden = (j > at[:, None]) if not w else (j > at[:, None]) | (j <= at[:, None] - w)
    for head in range(h):
        g = head // (h // kv)
        score = (q[:, head * d:(head + 1) * d].double() @ k[g].T) / math.sqrt(d)
        if c["softcap"]:
            score = c["softcap"] * torch.tanh(score / c["softcap"])
        score[hidden] = -math.inf
        if sink is not None:
            score = torch.cat((score, sink[head].double().expand(score.shape[0], 1)), dim=1)
        out[:, head * d:(head + 1) * d] = torch.softmax(score, dim=1)[:, :k.shape[1]] @ v[g]


def _exact_attend(s):
    c = s.case
    out = torch.zeros((s.ctx.rows, c["heads"] * c["dim"]), dtype=torch.float64, device=DEVICE)
    row = 0
    for i, (start, n) in enumerate(_spans(c)):
        ids = s.tables[i, :-(-(start + n) // c["page"])].long()
        k, v = ((codes.view(torch.uint8)[ids].view(FP8).float().double() * scale[ids].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :start + n]
                for codes, scale in ((s.k, s.k_scale), (s.v, s.v_scale)))
        _exact_rows(s.q[row:row + n], k, v, torch.arange(start, start + n, device=DEVICE), c, s.sink, out[row:row + n])
        row += n
    return out


def _exact_prompt(s):
    c = s.case
    h, kv, d = c["heads"], c["kv_heads"], c["dim"]
    out = torch.zeros((s.ctx.rows, h * d), dtype=torch.float64, device=DEVICE)
    starts, counts = s.ctx.seq_q_start.tolist(), s.ctx.seq_q_len.tolist()
    for a, n in zip(starts, counts):
        k, v = (s.qkv[a:a + n, at * d:(at + kv) * d].double().view(n, kv, d).transpose(0, 1) for at in (h, h + kv))
        _exact_rows(s.qkv[a:a + n, :h * d], k, v, torch.arange(n, device=DEVICE), c, s.sink, out[a:a + n])
    return out


def exact(case, seed):
    if case["op"] in ("fork", "compact"):
        return None                                                        # whole numbers and bytes only
    s = prepare(case, seed)
    return {"store": _exact_store, "attend": _exact_attend, "prompt": _exact_prompt}[case["op"]](s)
