"""Portions over pages in 4 bits that are laid out in bfloat16 first, where a context says more keys than its table has pages for and a window
starts inside it: the pages of the window that is attended are the ones that are laid out.  The memory that they are laid out in holds
not-a-number before, so that what is read without having been written shows."""
import pytest
import torch

from test_gpu_laid_out_q8 import stale_memory                       # noqa: F401 (a fixture of every test here)
from test_gpu_q4 import DEV, K, make_cache, make_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,options", [(96, {}), (128, dict(attn_prefill="unpack"))])
@pytest.mark.parametrize("window", [0, 20, 100])
@pytest.mark.parametrize("more", [1, 40, 2000])
def test_a_window_in_a_context_that_ends_with_its_table(more, window, hd, options):
    nh, nkv, B = 4, 2, 16
    tables, pages, ctx = make_step([(330, 70), (0, 400)], B, 1, width_extra=0)
    ctx.options, ctx.max_ctx = options, 3000
    kc, vc = make_cache(pages, nkv, B, hd, 2).to(DEV), make_cache(pages, nkv, B, hd, 3).to(DEV)
    q = torch.randn((ctx.rows, nh * hd), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(DEV)

    def run():
        out = torch.full_like(q, 9.0)
        K().paged_attention_q4(q, out, kc, vc, tables.to(DEV), ctx, nh, nkv, hd, B, hd ** -0.5, window)
        K().check_errors()
        return out
    want = run()
    assert not bool(torch.isnan(want).any())
    ctx.seq_ctx_len = ctx.seq_ctx_len + more
    assert torch.equal(run(), want)
