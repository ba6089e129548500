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
