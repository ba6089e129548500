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


@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("parts", [0, 3, -1])
def test_lengths_from_the_kernel_right_before(hd, parts):
    """The contexts' ends are formed on the device by the launch in front of the call, others every time."""
    S = 12
    s = Step(S, [3000] * S, 4, 1, hd, 0)
    s.ctx.options, s.ctx.rows, s.q = {"attn_parts": parts}, S, s.q[:S].contiguous()
    source, lengths = torch.zeros(S + 1, **I32), s.ctx.seq_ctx_len
    out = torch.empty_like(s.q)

    def step():
        torch.add(source, 1, out=lengths)
        s.attend(out)
    g = captured(step)
    for i in range(40):
        ends = torch.tensor([(97 * i + 211 * j) % 2990 for j in range(S)] + [0], dtype=torch.int32)
        source.copy_(ends)
        g.replay()
        got = out.clone()
        lengths.copy_(ends + 1)
        torch.cuda.synchronize()
        s.attend(out)
        torch.cuda.synchronize()
        assert torch.equal(got, out), i
    K().check_errors()


@pytest.mark.parametrize("hd", [64, 96, 128])
def test_tiles_from_the_kernel_right_before(hd):
    """Portions whose tiles, starts and lengths are formed by the launches in front of the call: another division of 300 rows every time."""
    nh, nkv, B, T, tiles = 4, 1, 16, 300, 9
    k, v = random_cache(60, nkv, B, hd, 1), random_cache(60, nkv, B, hd, 2)
    tables = torch.randperm(60, generator=torch.Generator().manual_seed(3)).int().view(2, 30).to(DEV)
    q = torch.randn((T, nh * hd), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(DEV)
    i = lambda n: torch.full((n,), -1, **I32)
    ctx = types.SimpleNamespace(rows=T, seqs=2, decode_seqs=0, prefill_tiles=tiles, tile_rows=64, max_ctx=480, max_decode_ctx=0, max_q_len=T, options={},
                                positions=i(T), row_seq=i(T), seq_q_start=i(2).zero_(), seq_q_len=i(2).zero_(), seq_ctx_len=i(2).zero_(), tile_seq=i(tiles),
                                tile_q0=i(tiles))
    names = ("seq_q_start", "seq_q_len", "seq_ctx_len", "tile_seq", "tile_q0")
    source = {n: getattr(ctx, n) - 1 for n in names}
    out = torch.empty_like(q)

    def attend():
        K().paged_attention_q4(q, out, k, v, tables, ctx, nh, nkv, hd, B, hd ** -0.5)

    def step():
        for n in names:
            torch.add(source[n], 1, out=getattr(ctx, n))
        attend()
    g = captured(step)
    for r in range(30):
        a = 2 + (37 * r) % (T - 4)
        of = [(s, q0) for s, n in enumerate((a, T - a)) for q0 in range(0, n, 64)]
        of += [(-1, -1)] * (tiles - len(of))
        values = dict(seq_q_start=[0, a], seq_q_len=[a, T - a], seq_ctx_len=[a + r, T - a + 3 * r], tile_seq=[t for t, _ in of], tile_q0=[t for _, t in of])
        for n in names:
            source[n].copy_(torch.tensor(values[n], dtype=torch.int32) - 1)
        g.replay()
        got = out.clone()
        for n in names:
            getattr(ctx, n).copy_(torch.tensor(values[n], dtype=torch.int32))
        torch.cuda.synchronize()
        attend()
        torch.cuda.synchronize()
        assert torch.equal(got, out), r
    K().check_errors()


@pytest.mark.parametrize("hd", [64, 96, 128])
def test_steps_of_many_rows_made_in_place_and_attended(hd):
    """Steps of more rows than one block of ``step_tables`` takes (a cluster makes them), lengths and the free pages' count advanced in
    place, from a graph: rows written, attention over them."""
    from test_gpu_q4_steps import Loop
    loop = Loop([0, 37, 64], 2, 1, hd, 16, 170, 400, 2750, 50, seed=hd)
    portions = [[1100, 900, 702], [2, 1400, 1040], [0, 30, 600]]
    loop.fill(portions[0])
    loop.launch()
    loop.check(portions[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loop.launch()
    for ns in portions[1:]:
        loop.fill(ns)
        g.replay()
        loop.check(ns)


def test_single_rows_in_bfloat16_behind_the_tables_of_their_step():
    """Kernels that read a step's integers ahead of their wait, right behind the launch that makes them: the bfloat16 attention, lengths
    advanced in place, from a graph."""
    S, nh, nkv, hd, B, width = 300, 4, 1, 64, 16, 24
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn((S * width, nkv, B, hd), generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    q = torch.randn((S, nh * hd), generator=g).to(torch.bfloat16).to(DEV)
    i = lambda n, x=0: torch.full((n,), x, **I32)
    tables, free, count, status = i(S * width, -1).view(S, width), torch.randperm(S * width, generator=g).int().to(DEV), i(1, S * width), i(4)
    ctx = types.SimpleNamespace(rows=S, seqs=S, decode_seqs=S, prefill_tiles=0, tile_rows=64, max_ctx=width * B, max_decode_ctx=width * B, max_q_len=1,
                                positions=i(S), row_seq=i(S), slot_mapping=i(S), seq_q_start=i(S), seq_q_len=i(S, 1), seq_ctx_len=i(S), options={})
    out = torch.empty_like(q)

    def attend(o):
        K().paged_attention(q, o, k, v, tables, ctx, nh, nkv, hd, hd ** -0.5)

    def step():
        K().step_tables(ctx.seq_ctx_len, ctx.seq_q_len, tables, free, count, B, seq_q_start=ctx.seq_q_start, seq_ctx_len=ctx.seq_ctx_len,
                        positions=ctx.positions, row_seq=ctx.row_seq, slot_mapping=ctx.slot_mapping, free_left=count, status=status)
        attend(out)
    graph = captured(step)
    for n in range(2, 60):
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert ctx.seq_ctx_len.tolist() == [n] * S and status.tolist() == [0, 0, S, 0]
        attend(out)
        assert torch.equal(got, out), n


@pytest.mark.parametrize("parts", [0, 1, 3, 8, 12])
@pytest.mark.parametrize("window", [0, 900])
def test_contexts_longer_than_was_said(parts, window):
    """The longest context only says how the keys are divided: one that grew beyond it is attended whole."""
    S, ends = 5, [10, 300, 700, 1500, 64]
    s = Step(S, ends, 4, 1, 64, 0)
    s.ctx.rows, s.q = S, s.q[:S].contiguous()
    want, got = torch.empty_like(s.q), torch.empty_like(s.q)
    s.ctx.options = {"attention": "plain"}
    s.attend(want, window=window)
    s.ctx.options = {"attn_parts": parts}
    for longest in (1500, 1000, 300, 1):
        s.ctx.max_decode_ctx = longest
        s.attend(got, window=window)
        # two roundings to bfloat16 and the weights' (2^-11 of at most the largest value)
        room = 2.0 ** -7 * want.float().abs() + 2.0 ** -10 * 4.0
        assert ((got.float() - want.float()).abs() <= room).all(), longest
    K().check_errors()
