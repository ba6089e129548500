"""Portions over the cache in 4 bits where the order of things inside the kernel counts (bounds: bounds_q4.py)."""
import pytest
import torch

import bounds_q4 as bounds
import plain_q4 as P
from test_gpu_q4 import DEV, K, make_step

pytestmark = pytest.mark.gpu


def climbing(step, nh, nkv, hd, B, spans, seed):
    """A request whose scores climb by about ``step`` (in log2) from 32 keys to the next, values falling by as much: every piece of 32 keys has
    its share of the result, and a row renews its maximum up to four times a tile."""
    tables, pages, ctx = make_step(spans, B, seed)
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((2, pages, B, nkv, hd), generator=g)
    per_key = step / (hd ** 0.5 * 1.4426950408889634)                      # q is about one: q.k hd^-0.5 log2(e) = step
    for i, (start, n) in enumerate(spans):
        for t in range(start + n):
            page, piece = int(tables[i, t // B]), t // 32
            x[0, page, t % B] = piece * per_key + 0.05 * x[0, page, t % B]
            x[1, page, t % B] *= 2.0 ** (-step * piece)
    kc, vc = (torch.zeros((pages, nkv, P.page_bytes(B, hd)), dtype=torch.uint8) for _ in range(2))
    for p in range(pages):
        for o in range(B):
            P.write(kc, B, p, o, x[0, p, o])
            P.write(vc, B, p, o, x[1, p, o])
    q = (1 + 0.25 * torch.randn((ctx.rows, nh * hd), generator=g)).to(torch.bfloat16)
    return tables, ctx, kc, vc, q


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("step", [5, 9, 13])
def test_maxima_renewed_inside_a_tile(hd, step):
    nh, nkv, B, spans = 2, 1, 16, [(0, 200), (40, 140)]
    tables, ctx, kc, vc, q = climbing(step, nh, nkv, hd, B, spans, step)
    out = torch.full_like(q, 9.0, device=DEV)
    K().attention_prefill_q4(q.to(DEV), out, kc.to(DEV), vc.to(DEV), tables.to(DEV), ctx, nh, nkv, hd, B, hd ** -0.5)
    torch.cuda.synchronize()
    K().check_errors()
    want, room = bounds.attention("climbing portion", q.double().view(-1, nh, hd), kc, vc, tables, spans, nh, nkv, hd, B, hd ** -0.5)
    bounds.check(out.view(-1, nh, hd), want, room)


@pytest.mark.parametrize("hd", [64, 128, 96])
@pytest.mark.parametrize("n,keys", [(300, 32), (300, 160), (140, 16), (600, 16), (129, 64)])
def test_rows_before_the_first_key_of_a_short_table(hd, n, keys):
    """A portion longer than its page table: the context ends with the table, and the rows in front of its keys see nothing and are zero."""
    from test_gpu_q4 import make_cache
    nh, nkv, B = 2, 1, 16
    tables, pages, ctx = make_step([(0, keys), (5, 200)], B, 2)
    kc, vc = make_cache(pages, nkv, B, hd, 3), make_cache(pages, nkv, B, hd, 4)
    tables = tables[:, :keys // B].contiguous()                     # the second request too is longer than its table
    rows = n + 200
    q = torch.randn((rows, nh * hd), generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    tiles = [(0, t) for t in range(0, n, 64)] + [(1, t) for t in range(0, 200, 64)]
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    ctx.rows, ctx.prefill_tiles, ctx.max_ctx = rows, len(tiles), max(n, 205)
    ctx.seq_q_start, ctx.seq_q_len, ctx.seq_ctx_len = i([0, n]), i([n, 200]), i([n, 205])
    ctx.tile_seq, ctx.tile_q0 = i([t for t, _ in tiles]), i([t for _, t in tiles])
    for _ in range(3):
        out = torch.full_like(q, 9.0, device=DEV)
        K().attention_prefill_q4(q.to(DEV), out, kc.to(DEV), vc.to(DEV), tables.to(DEV), ctx, nh, nkv, hd, B, hd ** -0.5)
        torch.cuda.synchronize()
        K().check_errors()
        for request, first, count in ((0, 0, n), (1, n, 200)):
            blind = max(0, count - keys)
            assert not out[first:first + blind].any()
            got = out[first + blind:first + count].cpu()
            want, room = bounds.attention("portion" if hd != 96 else "laid out", q.double()[first + blind:first + count].view(-1, nh, hd), kc, vc, tables[request:request + 1],
                                          [(keys - (count - blind), count - blind)], nh, nkv, hd, B, hd ** -0.5)
            bounds.check(got.view(-1, nh, hd), want, room)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size", [1.0, 100.0])
def test_large_queries_and_keys_that_all_score_the_same(hd, size):
    """Queries of very different elements, up to ``size``; keys of two scales, every one of which scores zero because its codes lie around 8 in
    pairs that cancel.  Values are 1 under one scale and -1 under the other: a score's error that grows with its scale shows at once."""
    nh, nkv, B, n = 2, 1, 16, 320
    tables, pages, ctx = make_step([(40, n - 40)], B, 1)
    g = torch.Generator().manual_seed(hd)
    half = torch.randint(1, 8, (pages, nkv, B, hd // 2), generator=g)
    code = torch.stack((8 + half, 8 - half), -1).flatten(-2)
    large = torch.rand((pages, nkv, B, 1), generator=g) < 0.5
    scale = torch.where(large, 1.0, 1.0 / 64).to(torch.bfloat16)
    kc = bounds.pages_of(code, scale, (-8 * scale.float()).to(torch.bfloat16))
    vc = bounds.pages_of(torch.zeros_like(code), torch.zeros_like(scale), torch.where(large, 1.0, -1.0).to(torch.bfloat16))
    q = size * torch.exp2(-14 * torch.rand((ctx.rows, nh * hd // 2), generator=g))
    q = q.repeat_interleave(2, dim=-1).to(torch.bfloat16)
    out = torch.full_like(q, 9.0, device=DEV)
    K().attention_prefill_q4(q.to(DEV), out, kc.to(DEV), vc.to(DEV), tables.to(DEV), ctx, nh, nkv, hd, B, hd ** -0.5)
    torch.cuda.synchronize()
    K().check_errors()
    want, room = bounds.attention("portion", q.double().view(-1, nh, hd), kc, vc, tables, [(40, n - 40)], nh, nkv, hd, B, hd ** -0.5)
    bounds.check(out.view(-1, nh, hd), want, room)
