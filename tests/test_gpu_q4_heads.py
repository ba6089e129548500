"""Single rows over the cache in 4 bits: what a head gives does not depend on the heads beside it (bounds: bounds_q4.py)."""
import types

import pytest
import torch

import bounds_q4 as bounds
import plain_q4 as P
from test_gpu_q4 import DEV, K, make_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nh,nkv,hd", [(4, 1, 128), (3, 1, 64), (8, 1, 96), (6, 1, 128), (16, 2, 64), (17, 1, 256), (8, 2, 32)])
@pytest.mark.parametrize("bits", [8, 13, 24, 100])
@pytest.mark.parametrize("force", [1, 3, -1])
def test_a_large_value_with_weight_in_one_head_only(nh, nkv, hd, bits, force):
    """A value 2^bits times the others: all the weight of one head of each KV head, none (below 2^-200) of the others."""
    B, n, at = 16, 400, 37
    tables, pages, ctx = make_step([(n - 1, 1), (n - 1, 1)], B, 21)
    g = torch.Generator().manual_seed(22)
    x = torch.randn((2, pages, B, nkv, hd), generator=g)
    q = torch.randn((2, nh, hd), generator=g).abs().add(0.5)
    q[:, torch.arange(nh) % (nh // nkv) != 1] *= -1.0
    for i in range(2):
        page = int(tables[i, at // B])
        x[0, page, at % B] = 6.0 + 0.1 * x[0, page, at % B]
        x[1, page, at % B] *= 2.0 ** bits
    q = q.flatten(1).to(torch.bfloat16)
    kc, vc = (torch.zeros((pages, nkv, P.page_bytes(B, hd)), dtype=torch.uint8) for _ in range(2))
    for p in range(pages):
        for o in range(B):
            P.write(kc, B, p, o, x[0, p, o])
            P.write(vc, B, p, o, x[1, p, o])
    out = torch.empty((2, nh * hd), dtype=torch.bfloat16, device=DEV)
    ctx.options = {"attn_parts": force}
    scale = 4.0 * hd ** -0.5
    K().attention_decode_q4(q.to(DEV), out, kc.to(DEV), vc.to(DEV), tables.to(DEV), ctx, nh, nkv, hd, B, scale)
    want, room = bounds.attention("single", q.double().view(2, nh, hd), kc, vc, tables, [(n - 1, 1), (n - 1, 1)], nh, nkv, hd, B, scale)
    bounds.check(out.view(2, nh, hd), want, room)


@pytest.mark.parametrize("nh,nkv,hd", [(4, 1, 128), (8, 1, 64), (2, 2, 96), (6, 1, 256)])
@pytest.mark.parametrize("climb", [0.3, 0.9, 1.1, 3.0])
@pytest.mark.parametrize("force", [1, 3, -1])
def test_a_large_value_that_scores_climb_away_from(nh, nkv, hd, climb, force):
    """Scores that climb by ``climb`` (in log2) from 128 keys to the next, and a value 2^20 times the others among the first 32: at the end
    it has little or no weight, however slowly it was left behind."""
    B, n = 16, 4000
    tables, pages, _ = make_step([(n - 1, 1)], B, 5)
    g = torch.Generator().manual_seed(6)
    k, v = 0.02 * torch.randn((pages, nkv, B, hd), generator=g), torch.randn((pages, nkv, B, hd), generator=g)
    per_key = climb / (hd ** 0.5 * 1.4426950408889634)                     # q is about one: q.k hd^-0.5 log2(e) = climb
    blocks = -(-n // B)
    steps = torch.arange(blocks * B).view(blocks, 1, B, 1) // 128
    k[tables[0, :blocks].long()] += steps * per_key
    v[int(tables[0, 0]), :, 7] *= 2.0 ** 20
    kc, vc = bounds.cache_of(k), bounds.cache_of(v)
    q = (1 + 0.1 * torch.randn((1, nh * hd), generator=g)).to(torch.bfloat16)
    out = torch.empty_like(q, device=DEV)
    ctx = types.SimpleNamespace(seq_ctx_len=torch.tensor([n], dtype=torch.int32, device=DEV), max_decode_ctx=n, options={"attn_parts": force})
    K().attention_decode_q4(q.to(DEV), out, kc.to(DEV), vc.to(DEV), tables.to(DEV), ctx, nh, nkv, hd, B, hd ** -0.5)
    want, room = bounds.attention("single", q.double().view(1, nh, hd), kc, vc, tables, [(n - 1, 1)], nh, nkv, hd, B, hd ** -0.5)
    bounds.check(out.view(1, nh, hd), want, room)
