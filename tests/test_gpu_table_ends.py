"""Contexts that are longer than their page table (a step that was refused may leave such lengths): rows keep their positions, their keys end
with the table.  On the GPU, within the bounds of plain_q8.py."""
import pytest
import torch

import plain_q8 as P
from test_gpu_q4 import make_step
from test_gpu_q8 import DEV, K, gpu_pool

pytestmark = pytest.mark.gpu


def check_q8(kind, spans, columns, nh, nkv, hd, B, seed, window=0, softcap=0.0, sink=False, options=None):
    """Requests (start, rows) whose tables end after ``columns`` pages."""
    g = torch.Generator().manual_seed(seed)
    tables, pages, ctx = make_step(spans, B, seed)
    tables = tables[:, :columns].contiguous()
    ctx.options = options or {}
    (kc, ks), (vc, vs) = P.pool(pages, nkv, B, hd, seed + 1, spread=2), P.pool(pages, nkv, B, hd, seed + 2, spread=2)
    k, k_scale = gpu_pool(kc, ks)
    v, v_scale = gpu_pool(vc, vs)
    q = (1.5 * torch.randn((ctx.rows, nh * hd), generator=g)).bfloat16()
    s = torch.randn((nh,), generator=g) if sink else None
    out = torch.full((ctx.rows, nh * hd), 7.0, dtype=torch.bfloat16, device=DEV)
    K().paged_attention_q8(q.to(DEV), out, k, v, k_scale, v_scale, tables.to(DEV), ctx, nh, nkv, hd, hd ** -0.5, window, softcap,
                           s.to(DEV) if sink else None)
    K().check_errors()
    got = out.cpu().double().view(ctx.rows, nh, hd)
    row = 0
    for i, (start, n) in enumerate(spans):
        keys = min(start + n, columns * B)
        want, room = P.attend(kind, q[row:row + n].double().view(n, nh, hd), P.gathered(kc, ks, tables[i], keys), P.gathered(vc, vs, tables[i], keys),
                              torch.arange(start, start + n), hd ** -0.5, window, softcap, s)
        far = (got[row:row + n] - want).abs()
        assert bool((far <= room).all()), (i, float((far - room).max()))
        row += n


# rows on both sides of a table's end, in both groups of a block; whole blocks behind it; tables of one page
PORTIONS = [([(0, 200)], 8), ([(0, 200)], 12), ([(100, 300), (0, 40)], 10), ([(0, 700)], 3), ([(0, 700)], 1), ([(900, 300), (3, 70)], 5), ([(0, 513)], 32)]
MASKS = [dict(), dict(window=100), dict(window=3), dict(window=60, softcap=9.0, sink=True)]


@pytest.mark.parametrize("masks", MASKS)
@pytest.mark.parametrize("spans,columns", PORTIONS)
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 128), (4, 1, 64)])
def test_portions_q8(spans, columns, nh, nkv, hd, masks):
    check_q8("portion", spans, columns, nh, nkv, hd, 16, 41, **masks)


@pytest.mark.parametrize("masks", MASKS)
def test_plain_rows_q8(masks):
    check_q8("plain bfloat16", [(5, 1), (900, 1), (40, 200)], 6, 4, 2, 64, 16, 42, options=dict(attention="plain"), **masks)


@pytest.mark.parametrize("masks", MASKS)
@pytest.mark.parametrize("spans,columns", PORTIONS + [([(400, 1), (100, 300)], 12)])
@pytest.mark.parametrize("nh,nkv,hd,options", [(4, 2, 96, {}), (2, 1, 256, {}), (4, 2, 128, dict(attn_prefill="unpack"))])
def test_portions_q8_through_laid_out_pages(spans, columns, nh, nkv, hd, options, masks):
    check_q8("laid out", spans, columns, nh, nkv, hd, 16, 43, options=options, **masks)


@pytest.mark.parametrize("masks", MASKS + [dict(window=900)])
@pytest.mark.parametrize("options", [{}, dict(attn_parts=1), dict(attn_parts=4), dict(attn_parts=11), dict(attn_parts=4, attn_merge="kernel"), dict(attn_parts=-1)])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 128), (12, 1, 64), (4, 4, 96)])
def test_single_rows_q8(nh, nkv, hd, options, masks):
    """Windows inside the table, across its end and behind it; contexts that fit between them."""
    check_q8("single", [(2500, 1), (100, 1), (1000, 1), (959, 1), (960, 1), (1023, 1), (1300, 1), (0, 1), (1059, 1)], 60, nh, nkv, hd, 16, 44, options=options, **masks)
