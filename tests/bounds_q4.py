"""How far attention over the cache in 4 bits may be off, row by row and element by element, from the roundings that its kernels do.

With x_j = zero_j + scale_j code_j and probabilities p_j (sum 1), in units in the last place of the types, half a step each:
 * bfloat16 results: 2^-8 |o|; float32 results 2^-24 |o|.
 * weights: the kernels on tensor cores round p_j scale_j once where it enters a product with code_j - 8 (float16 2^-11 in single rows,
   bfloat16 2^-8 in portions, there up to three times more where a maximum is renewed inside a tile): ``weight`` * sum p scale |code - 8|.
   float16 weights below 2^-14 of the unit, which is at most twice the largest, are off by up to 2^-25 of it:
   2^-24 max(p scale) * sum |code - 8|, ``small`` times.
 * float32 sums: 2^-24 of the sum of the terms' sizes, sum p (15 scale + |zero|), for each addition that a term goes through: at most
   one a key and hd; in single rows a fourth of the keys (four warps), one a piece of 128 where pieces are joined, and 16.
 * scores that are off by e_j change the result by at most sum p_j e_j |x_j - o|, whatever all of them are off by together.  A
   score's terms are q_d code_d scale and zero q_d: e is (hd + 8) * 2^-24 of their sizes (portions: of q_d (code_d - 8) scale
   and (zero + 8 scale) q_d), single rows' q in addition max|q| / 65024 * sum |scale code - mean over the keys| (q in 16 bits);
   exponentials and products around them 8 * 2^-24 (1 + |score|).
 * pages laid out in bfloat16: keys, values and probabilities are rounded there, 2^-8 of each.
"""
import torch

import plain_q4 as P


def parts(cache, hd, B):
    """Codes, scale, zero (float64) of all rows of a cache: [pages, nkv, B, hd], [pages, nkv, B, 1] twice."""
    pages, nkv, _ = cache.shape
    n = B * hd // 2
    pair = cache[..., n:n + 4 * B].contiguous().view(torch.bfloat16).double().view(pages, nkv, B, 2)
    scale, zero = pair[..., :1], pair[..., 1:]
    x = P.read(cache, hd, B)
    code = torch.where(scale > 0, (x - zero) / torch.where(scale > 0, scale, torch.ones_like(scale)), torch.zeros_like(x)).round()
    return code, scale, zero


KINDS = {"single": dict(weight=2.0 ** -11, small=1, result=2.0 ** -8, q16=True, centred=False),
         "portion": dict(weight=2.0 ** -8, small=0, result=2.0 ** -8, q16=False, centred=True),
         "climbing portion": dict(weight=4 * 2.0 ** -8, small=0, result=2.0 ** -8, q16=False, centred=True),
         "laid out": dict(weight=0.0, small=0, result=2.0 ** -8, q16=False, centred=False, again=2.0 ** -8),
         "plain bfloat16": dict(weight=0.0, small=0, result=2.0 ** -8, q16=False, centred=False),
         "plain float32": dict(weight=0.0, small=0, result=2.0 ** -24, q16=False, centred=False)}


def attention(kind, q, kc, vc, tables, spans, nh, nkv, hd, B, scale, window=0, lost=None):
    """float64 rows [rows, nh, hd] and the room around each; ``lost``: (first, last) keys left out of the sums (a planted mistake)."""
    c = KINDS[kind]
    eps = 2.0 ** -24
    k_of, v_of = parts(kc, hd, B), parts(vc, hd, B)
    want, room = torch.zeros_like(q), torch.zeros_like(q)
    row = 0
    for i, (start, n) in enumerate(spans):
        end = start + n
        ids = tables[i, :(end + B - 1) // B].long()
        kcode, ks, kz, vcode, vs, vz = (x[ids].transpose(0, 1).flatten(1, 2)[:, :end] for x in (*k_of, *v_of))
        at = torch.arange(start, end)[:, None]
        key = torch.arange(end)
        seen = (key <= at) & (key > at - window if window else torch.ones_like(key, dtype=torch.bool))
        if lost is not None:
            seen = seen & ~((key >= lost[0]) & (key < lost[1]))
        depth = end / 4 + end / 128 + 16 if c["q16"] else end + hd
        for h in range(nh):
            g = h // (nh // nkv)
            x, s1, z1 = vz[g] + vs[g] * vcode[g], vs[g], vz[g]
            rows = q[row:row + n, h]
            s = (rows @ (kz[g] + ks[g] * kcode[g]).T) * scale
            s = s.masked_fill(~seen, -torch.inf)
            p = torch.nan_to_num(torch.softmax(s, -1))
            o = p @ x
            middle = 8 if c["centred"] else 0
            size = (rows.abs() @ (ks[g] * (kcode[g] - middle).abs() + (kz[g] + middle * ks[g]).abs()).T) * scale     # of a score's terms
            e = (hd + 8) * eps * size + 8 * eps * (1 + s.abs())
            if c["q16"]:
                coded = ks[g] * kcode[g]
                e = e + rows.abs().amax(-1, keepdim=True) / 65024 * (coded - coded.mean(0)).abs().sum(-1) * scale
            again = c.get("again", 0.0)
            e = e + again * (rows.abs() @ (kz[g] + ks[g] * kcode[g]).abs().T) * scale
            e = torch.where(seen, e, torch.zeros_like(e))
            moved = torch.stack([((p[r] * e[r])[:, None] * (x - o[r]).abs()).sum(0) for r in range(n)])
            centred = (vcode[g] - 8).abs()
            top = (p * s1[:, 0]).amax(-1, keepdim=True)
            want[row:row + n, h] = o
            room[row:row + n, h] = (c["result"] * o.abs() + c["weight"] * ((p * s1[:, 0]) @ centred) + c["small"] * eps * top * (seen.double() @ centred)
                                    + depth * eps * (p @ (15 * s1 + z1.abs())) + moved
                                    + 2 * again * (p @ x.abs()))
        row += n
    return want, room * 1.05                                         # products of the roundings with one another


def check(got, want, room):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    over = ((got - want).abs() / room.clamp(min=1e-300)).nan_to_num(0.0)
    assert over.max() <= 1, (over.max().item(), int(over.argmax()))


def cache_of(x):
    """The pages of rows x [pages, nkv, B, hd]."""
    return pages_of(*P.quantised(x))


def pages_of(code, scale, zero):
    """The pages of rows of codes [pages, nkv, B, hd] (whole numbers), scales and zeros [pages, nkv, B, 1] (bfloat16)."""
    pages, nkv, B, hd = code.shape
    w = sum(code[..., e::8] << P.SHIFTS[e] for e in range(8))
    cache = torch.zeros((pages, nkv, P.page_bytes(B, hd)), dtype=torch.uint8)
    n = B * hd // 2
    cache[..., :n] = torch.stack([(w >> (8 * b)) & 255 for b in range(4)], dim=-1).flatten(2).to(torch.uint8)
    cache[..., n:n + 4 * B] = torch.cat((scale, zero), dim=-1).flatten(2).contiguous().view(torch.uint8)
    return cache


def inputs(spans, nh, nkv, hd, B, dtype, seed=0):
    """Queries, pages and tables of requests (start, rows).  Every 128 keys of a request have values around a point of their own, so that
    each such piece moves the result by more than all roundings together."""
    g = torch.Generator().manual_seed(seed)
    blocks = [-(-(s + n) // B) for s, n in spans]
    pages = sum(blocks) + 2
    ids = torch.randperm(pages, generator=g).int()
    tables = torch.full((len(spans), max(blocks)), -1, dtype=torch.int32)
    k, v = torch.randn((pages, nkv, B, hd), generator=g) + 0.5, torch.randn((pages, nkv, B, hd), generator=g)
    at = 0
    for i, n in enumerate(blocks):
        tables[i, :n] = ids[at:at + n]
        at += n
        points = 3 * torch.randn((-(-n * B // 128), nkv, hd), generator=g)
        of_key = torch.arange(n * B) // 128
        v[tables[i, :n].long()] += points[of_key].view(n, B, nkv, hd).transpose(1, 2)
    q = torch.randn((sum(n for _, n in spans), nh * hd), generator=g).to(dtype)
    return q, cache_of(k), cache_of(v), tables


# (kind, requests, query heads, KV heads, head size, page, options of the step)
CASES = [("single", [(5000, 1), (0, 1), (3, 1), (700, 1)], 12, 4, 128, 16, {"attn_parts": -1}),
         ("single", [(20000, 1)], 4, 1, 64, 16, {"attn_parts": -1}),              # more than 128 pieces of one head
         ("single", [(28000, 1), (17000, 1), (9, 1)], 8, 1, 128, 16, {"attn_parts": -1}),
         ("single", [(1500, 1), (1000, 1), (129, 1)], 8, 2, 64, 16, {"attn_parts": 3}),
         ("single", [(1500, 1), (1000, 1), (129, 1)], 5, 1, 96, 7, {"attn_parts": 12}),
         ("single", [(1100, 1), (255, 1)], 2, 2, 256, 32, {}),
         ("portion", [(700, 300), (0, 130), (131, 5)], 2, 1, 64, 16, {}),
         ("portion", [(900, 140), (0, 513)], 2, 1, 128, 16, {}),
         ("laid out", [(500, 70), (0, 200)], 2, 1, 96, 16, {}),
         ("plain bfloat16", [(511, 1), (512, 1), (1300, 1)], 2, 1, 40, 16, {"attention": "plain"}),
         ("plain float32", [(511, 1), (512, 1), (1300, 1)], 2, 1, 32, 16, {}),
         ("plain float32", [(2000, 3), (40, 70)], 3, 1, 24, 7, {})]
