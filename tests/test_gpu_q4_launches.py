"""The calls around the cache in 4 bits between kernels that start before the one in front of them has ended: what each reads has been
written, what each writes is there for the next."""
import types

import pytest
import torch

import plain_q4 as P
from test_gpu_q4 import DEV, K

pytestmark = pytest.mark.gpu
I32 = dict(dtype=torch.int32, device=DEV)


def random_cache(pages, nkv, B, hd, seed):
    """Pages of random codes, scales of 0.1 to 0.4 and zeros of -3 to -1."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    cache = torch.randint(0, 256, (pages, nkv, P.page_bytes(B, hd)), generator=g, device=DEV).to(torch.uint8)
    r = torch.rand((pages, nkv, B, 2), generator=g, device=DEV)
    pair = torch.stack((0.1 + 0.3 * r[..., 0], -1 - 2 * r[..., 1]), -1).to(torch.bfloat16).flatten(-2).contiguous().view(torch.uint8)
    n = B * hd // 2
    cache[..., n:n + 4 * B] = pair
    return cache


class Step:
    """``S`` requests of one row each over pages of 16 keys, an entry behind them that brings nothing, and the arrays of the step."""
    def __init__(self, S, ends, nh, nkv, hd, tiles, seed=0):
        self.S, self.nh, self.nkv, self.hd, self.B = S, nh, nkv, hd, 16
        width = -(-max(ends) // 16) + 1
        g = torch.Generator().manual_seed(seed)
        self.tables = torch.randperm((S + 1) * width, generator=g).int().view(S + 1, width).to(DEV)
        self.k, self.v = (random_cache((S + 1) * width, nkv, 16, hd, seed + i) for i in (1, 2))
        self.q = torch.randn((S + 3, nh * hd), generator=g).to(torch.bfloat16).to(DEV)
        i = lambda n, v: torch.full((n,), v, **I32)
        self.ctx = types.SimpleNamespace(
            rows=S + 3, seqs=S + 1, decode_seqs=S, prefill_tiles=tiles, tile_rows=64, max_ctx=width * 16, max_decode_ctx=width * 16, max_q_len=1,
            positions=torch.tensor([e - 1 for e in ends] + [-1] * 3, **I32), row_seq=torch.tensor(list(range(S)) + [0] * 3, **I32),
            seq_q_start=torch.tensor(list(range(S + 1)), **I32), seq_q_len=torch.tensor([1] * S + [0], **I32),
            seq_ctx_len=torch.tensor(list(ends) + [5], **I32), tile_seq=i(tiles, -1), tile_q0=i(tiles, -1), options={})

    def attend(self, out, **kw):
        K().paged_attention_q4(self.q, out, self.k, self.v, self.tables, self.ctx, self.nh, self.nkv, self.hd, 16, self.hd ** -0.5, **kw)


def captured(f):
    f()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        f()
    return g


@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("parts", [0, 3, -1])
def test_tiles_of_no_request_between_single_rows_and_their_reader(hd, parts):
    """Long single rows, a launch of nothing but empty tiles, and at once a kernel that reads the single rows' results (here: writes them
    into another cache, the first heads' rows as they are)."""
    S = 12
    s = Step(S, [6000 + 37 * i for i in range(S)], 4, 1, hd, 6)
    s.ctx.options = {"attn_parts": parts}
    want = torch.full_like(s.q, 9.0)
    s.attend(want)
    torch.cuda.synchronize()
    assert (want[S:] == 9).all() and not (want[:S] == 9).any()
    out, first = torch.empty_like(want), torch.empty((S + 3, 2 * hd), dtype=torch.bfloat16, device=DEV)
    k2, v2 = torch.zeros((1, 1, P.page_bytes(16, hd)), dtype=torch.uint8, device=DEV), torch.zeros((1, 1, P.page_bytes(16, hd)), dtype=torch.uint8, device=DEV)
    slots = torch.arange(S + 3, **I32)

    def step():
        out.fill_(9.0)
        s.attend(out)
        K().rope_cache_q4(out, None, False, slots, k2, v2, first, 2, 1, hd, 16)
    g = captured(step)
    caches = (k2.clone(), v2.clone())
    for _ in range(100):
        first.zero_(), k2.zero_(), v2.zero_()
        g.replay()
        assert torch.equal(first, want[:, :2 * hd]) and torch.equal(k2, caches[0]) and torch.equal(v2, caches[1])
    K().check_errors()
