"""Portions over the cache in 4 bits through pages laid out in bfloat16: what the scratch held before does not matter."""
import pytest
import torch

from test_gpu_q4 import DEV, K, make_cache, make_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,B", [(64, 16), (128, 16), (64, 64), (128, 8), (96, 16), (256, 16), (64, 7)])
@pytest.mark.parametrize("window", [0, 20, 100])
def test_scratch_that_held_no_numbers(hd, B, window):
    nh, nkv, spans = 4, 2, [(33, 1), (300, 90), (131, 70), (0, 200), (777, 3)]
    tables, pages, ctx = make_step(spans, B, 5)
    ctx.options = {"attn_prefill": "unpack"}
    kc, vc = make_cache(pages, nkv, B, hd, 6).to(DEV), make_cache(pages, nkv, B, hd, 7).to(DEV)
    q = torch.randn((ctx.rows, nh * hd), generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).to(DEV)
    tables = tables.to(DEV)
    blocks = min(tables.shape[1], -(-ctx.max_ctx // B))
    outs = []
    for held in (0.0, float("nan"), float("inf")):
        out = torch.full_like(q, 9.0)
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        scratch = torch.full((2, (len(spans) - 1) * blocks, nkv, B, hd), held, dtype=torch.bfloat16, device=DEV)
        at = scratch.data_ptr()
        del scratch
        again = torch.empty((2, (len(spans) - 1) * blocks, nkv, B, hd), dtype=torch.bfloat16, device=DEV)
        assert again.data_ptr() == at                               # the call's scratch will be this memory
        del again
        K().attention_prefill_q4(q, out, kc, vc, tables, ctx, nh, nkv, hd, B, hd ** -0.5, window)
        torch.cuda.synchronize()
        outs.append(out)
    assert outs[0][1:].isfinite().all() and (outs[0][0] == 9).all()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    K().check_errors()
