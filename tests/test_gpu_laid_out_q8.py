"""Portions over pages in 8 bits that are laid out in bfloat16 first (heads that the kernel on tensor cores does not take, and on demand), on the
GPU: behind windows that skip whole pages, capped, with sinks, behind single rows.  The memory that the pages are laid out in holds
not-a-number before, so that what is read without having been written shows."""
import pytest
import torch

from test_gpu_q8 import DEV, check

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def stale_memory():
    """What the allocator hands out next holds not-a-number."""
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    sizes = [1 << 28] + [1 << n for n in range(16, 24)] * 2
    blocks = [torch.full((n // 2,), float("nan"), dtype=torch.bfloat16, device=DEV) for n in sizes]
    torch.cuda.synchronize()
    del blocks
    yield
    torch.cuda.empty_cache()


SPANS = [[(700, 200), (0, 130)], [(300, 1), (0, 1), (520, 90), (3, 64)], [(1000, 2)], [(40, 1), (129, 65)]]
MASKS = [dict(), dict(window=100), dict(window=1), dict(window=40, softcap=9.0, sink=True), dict(softcap=20.0), dict(sink=True)]


@pytest.mark.parametrize("masks", MASKS)
@pytest.mark.parametrize("spans", SPANS)
@pytest.mark.parametrize("nh,nkv,hd,B,options", [(4, 2, 96, 16, {}), (2, 1, 256, 7, {}), (4, 2, 32, 8, {}), (4, 2, 128, 20, {}),
                                                 (4, 2, 128, 16, dict(attn_prefill="unpack")), (4, 1, 64, 64, dict(attn_prefill="unpack"))])
def test_portions_through_laid_out_pages(nh, nkv, hd, B, options, spans, masks):
    check("laid out", spans, nh, nkv, hd, B, 51, options=options, **masks)
