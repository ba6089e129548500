"""Portions and prompts on the GPU within narrower bounds than plain_q8.py's: a tile's weights are always formed from its products, also where a row's
maximum is renewed inside the tile, so each is rounded once, and not up to four times.

 * portions: 2^-11 of a weight (float16), which its row's sum does not see: 2^-11 sum p |v|.
 * prompts: 2^-8 (bfloat16), which the sum sees in masked tiles alone: |sum d_j p_j (v_j - o)| <= 2^-8 (sum p |v| + |o|) <= 2 * 2^-8 sum p |v|."""
import pytest
import torch

import plain_q8 as P
from test_gpu_prompt_attention import check as check_prompts
from test_gpu_q8 import check as check_pages

ONCE = {"portion once": dict(P.KINDS["portion"], weight=2.0 ** -11), "prompt once": dict(P.KINDS["prompt"], weight=2 * 2.0 ** -8)}


@pytest.fixture(autouse=True)
def kinds(monkeypatch):
    for name, kind in ONCE.items():
        monkeypatch.setitem(P.KINDS, name, kind)


@pytest.mark.gpu
@pytest.mark.parametrize("masks", [dict(), dict(window=100), dict(softcap=20.0), dict(window=77, softcap=5.0, sink=True)])
@pytest.mark.parametrize("nh,nkv,hd,B", [(4, 1, 64, 16), (4, 2, 128, 16)])
def test_portions(nh, nkv, hd, B, masks):
    check_pages("portion once", [(700, 200), (0, 300), (3, 40)], nh, nkv, hd, B, 61, **masks)


@pytest.mark.gpu
@pytest.mark.parametrize("spread,q_size,k_size", [(30, 1.5, 1.0), (0, 100.0, 1.0), (0, 1e-3, 1.0), (12, 1.5, 30.0)])
def test_portions_of_other_sizes(spread, q_size, k_size):
    check_pages("portion once", [(500, 200)], 4, 2, 128, 16, 62, spread=spread, q_size=q_size, k_size=k_size)


@pytest.mark.gpu
@pytest.mark.parametrize("masks", [dict(), dict(window=100), dict(window=1), dict(softcap=20.0), dict(window=77, softcap=5.0, sink=True)])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 1, 64), (4, 2, 128), (2, 1, 96)])
def test_prompts(nh, nkv, hd, masks):
    check_prompts([1, 700, 130, 3], nh, nkv, hd, kind="prompt once", **masks)


@pytest.mark.gpu
@pytest.mark.parametrize("q_size", [1e-3, 60.0])
def test_prompts_of_other_sizes(q_size):
    check_prompts([400], 4, 2, 128, kind="prompt once", q_size=q_size)


@pytest.mark.parametrize("kind,rows", [("portion once", 600), ("prompt once", 420), ("prompt once", 700)])
def test_no_key_lost(kind, rows):
    """Eight keys that get lost leave these bounds."""
    nh, nkv, hd = 4, 1, 128
    g = torch.Generator().manual_seed(9)
    q = torch.randn((1, nh, hd), generator=g).double()
    k, v = torch.randn((2, nkv, rows, hd), generator=g).double()
    want, room = P.attend(kind, q, k, v, torch.tensor([rows - 1]), hd ** -0.5)
    off, _ = P.attend(kind, q, k, v, torch.tensor([rows - 1]), hd ** -0.5, lost=(128, 136))
    assert bool(((off - want).abs() > room).any())
