"""Attention over the cache in 4 bits within the bounds of its roundings, row by row, where a piece of keys that got lost would show
(test_q4_bounds.py); contexts of more pieces than the joining kernel weighs at once."""
import types

import pytest
import torch

import bounds_q4 as bounds
from test_gpu_q4 import DEV, K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,spans,nh,nkv,hd,B,options", bounds.CASES, ids=str)
def test_within_the_bounds(kind, spans, nh, nkv, hd, B, options):
    q, kc, vc, tables = bounds.inputs(spans, nh, nkv, hd, B, torch.float32 if kind == "plain float32" else torch.bfloat16)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    single = kind == "single" or all(n == 1 for _, n in spans)
    tiles = [(i, t) for i, (_, n) in enumerate(spans) if not single for t in range(0, n, 64)]
    ends = [s + n for s, n in spans]
    starts = [sum(n for _, n in spans[:i]) for i in range(len(spans))]
    ctx = types.SimpleNamespace(
        rows=q.shape[0], seqs=len(spans), decode_seqs=len(spans) if single else 0, prefill_tiles=len(tiles), tile_rows=64, max_ctx=max(ends),
        max_decode_ctx=max(ends), max_q_len=max(n for _, n in spans), positions=i32([s + r for s, n in spans for r in range(n)]),
        row_seq=i32([i for i, (_, n) in enumerate(spans) for _ in range(n)]), seq_q_start=i32(starts), seq_q_len=i32([n for _, n in spans]),
        seq_ctx_len=i32(ends), tile_seq=i32([t for t, _ in tiles]), tile_q0=i32([t for _, t in tiles]), options=options)
    out = torch.full_like(q, 9.0, device=DEV)
    K().paged_attention_q4(q.to(DEV), out, kc.to(DEV), vc.to(DEV), tables.to(DEV), ctx, nh, nkv, hd, B, hd ** -0.5)
    torch.cuda.synchronize()
    K().check_errors()
    want, room = bounds.attention(kind, q.double().view(-1, nh, hd), kc, vc, tables, spans, nh, nkv, hd, B, hd ** -0.5)
    bounds.check(out.view(-1, nh, hd), want, room)
