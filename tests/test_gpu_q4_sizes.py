"""Attention over the cache in 4 bits with keys and queries whose sizes are far apart while their products are ordinary (bounds: bounds_q4.py)."""
import types

import pytest
import torch

import bounds_q4 as bounds
from test_gpu_q4 import DEV, K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [-110, -60, 60, 110])
@pytest.mark.parametrize("kind,hd", [("single", 64), ("single", 128), ("single", 96), ("portion", 64), ("portion", 128), ("plain bfloat16", 64),
                                     ("plain float32", 40)])
def test_large_keys_and_small_queries(kind, hd, bits):
    """Keys times 2^bits, queries times 2^-bits: the results of ordinary ones."""
    nh, nkv, B = 4, 1, 16
    spans = [(200, 1), (33, 1)] if kind == "single" else [(0, 90), (130, 40)]
    dtype = torch.float32 if kind == "plain float32" else torch.bfloat16
    q, _, vc, tables = bounds.inputs(spans, nh, nkv, hd, B, dtype, 3)
    g = torch.Generator().manual_seed(4)
    kc = bounds.cache_of((torch.randn((vc.shape[0], nkv, B, hd), generator=g) + 0.5) * 2.0 ** bits)
    q = q * 2.0 ** -bits
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    single = kind == "single"
    tiles = [(i, t) for i, (_, n) in enumerate(spans) if not single for t in range(0, n, 64)]
    ends = [s + n for s, n in spans]
    ctx = types.SimpleNamespace(
        rows=q.shape[0], seqs=2, decode_seqs=2 if single else 0, prefill_tiles=len(tiles), tile_rows=64, max_ctx=max(ends), max_decode_ctx=max(ends),
        max_q_len=max(n for _, n in spans), positions=i32([s + r for s, n in spans for r in range(n)]),
        row_seq=i32([i for i, (_, n) in enumerate(spans) for _ in range(n)]), seq_q_start=i32([0, spans[0][1]]), seq_q_len=i32([n for _, n in spans]),
        seq_ctx_len=i32(ends), tile_seq=i32([t for t, _ in tiles]), tile_q0=i32([t for _, t in tiles]),
        options={"attention": "plain"} if kind == "plain bfloat16" else {})
    out = torch.full_like(q, 9.0, device=DEV)
    K().paged_attention_q4(q.to(DEV), out, kc.to(DEV), vc.to(DEV), tables.to(DEV), ctx, nh, nkv, hd, B, hd ** -0.5)
    torch.cuda.synchronize()
    K().check_errors()
    want, room = bounds.attention(kind, q.double().view(-1, nh, hd), kc, vc, tables, spans, nh, nkv, hd, B, hd ** -0.5)
    assert want.abs().max() > 0.5
    bounds.check(out.view(-1, nh, hd), want, room)
