"""The cache in 4 bits as it is used: steps whose arrays are made on the device, rows written, attention read, in order on one stream
and from CUDA graphs; calls side by side on two streams; tables, tiles and rows that are not there or not numbers.  Tolerances as
in test_gpu_q4.py; where two calls do the same work their results are equal."""
import types

import pytest
import torch

import plain_q4 as P
from test_gpu_q4 import DEV, K, check_attention, make_cache, make_step

pytestmark = pytest.mark.gpu
I32 = dict(dtype=torch.int32, device=DEV)
NAN = torch.tensor([0xc0, 0x7f, 0xc0, 0x7f], dtype=torch.uint8)


class Loop:
    """Requests over one layer's cache; the CPU keeps a copy of the cache, written by the plain form."""
    def __init__(self, starts, nh, nkv, hd, B, width, pages, rows, tiles, seed=0):
        self.S, self.nh, self.nkv, self.hd, self.B, self.rows = len(starts), nh, nkv, hd, B, rows
        g = torch.Generator().manual_seed(seed)
        self.g, self.at, self.width = g, list(starts), width
        free = torch.randperm(pages, generator=g).int()
        self.tables, count = torch.full((self.S, width), -1, dtype=torch.int32), pages
        for i, s in enumerate(starts):
            for b in range(-(-s // B)):
                count -= 1
                self.tables[i, b] = free[count]
        self.kc, self.vc = make_cache(pages, nkv, B, hd, seed + 1), make_cache(pages, nkv, B, hd, seed + 2)
        i = lambda n, v=0: torch.full((n,), v, **I32)
        self.dk, self.dv, self.dt = self.kc.to(DEV), self.vc.to(DEV), self.tables.to(DEV)
        self.free, self.count, self.status = free.to(DEV), i(1, count), i(4)
        self.qkv = torch.zeros((rows, (nh + 2 * nkv) * hd), dtype=torch.bfloat16, device=DEV)
        self.angles = torch.empty((rows, hd), device=DEV)
        self.q, self.out = (torch.zeros((rows, nh * hd), dtype=torch.bfloat16, device=DEV) for _ in range(2))
        self.inv_freq = (10000.0 ** (-torch.arange(0, hd, 2).double() / hd)).float().to(DEV)
        self.n = i(self.S)
        length = torch.tensor(starts, **I32)
        self.ctx = types.SimpleNamespace(
            rows=rows, seqs=self.S, decode_seqs=0, prefill_tiles=tiles, tile_rows=64, max_ctx=width * B, max_decode_ctx=width * B, max_q_len=rows,
            positions=i(rows), row_seq=i(rows), slot_mapping=i(rows), seq_q_start=i(self.S), seq_q_len=self.n, seq_ctx_len=length, tile_seq=i(tiles),
            tile_q0=i(tiles), options={})

    def launch(self):
        c = self.ctx
        K().step_tables(c.seq_ctx_len, self.n, self.dt, self.free, self.count, self.B, seq_q_start=c.seq_q_start, seq_ctx_len=c.seq_ctx_len,
                        positions=c.positions, row_seq=c.row_seq, slot_mapping=c.slot_mapping, free_left=self.count, status=self.status,
                        tile_seq=c.tile_seq, tile_q0=c.tile_q0)
        K().rope_table(c.positions, self.inv_freq, self.angles)
        K().rope_cache_q4(self.qkv, self.angles, False, c.slot_mapping, self.dk, self.dv, self.q, self.nh, self.nkv, self.hd, self.B)
        K().paged_attention_q4(self.q, self.out, self.dk, self.dv, self.dt, c, self.nh, self.nkv, self.hd, self.B, self.hd ** -0.5)

    def fill(self, ns):
        """New rows of the next step."""
        self.n.copy_(torch.tensor(ns, dtype=torch.int32))
        self.x = torch.randn((self.rows, (self.nh + 2 * self.nkv) * self.hd), generator=self.g).to(torch.bfloat16)
        self.qkv.copy_(self.x)
        self.out.fill_(9.0)

    def check(self, ns):
        """What the step of ``ns`` rows has left, against the plain forms."""
        K().check_errors()
        status = self.status.tolist()
        K().raise_on_step_tables(status)
        T, B = sum(ns), self.B
        assert status[2] == T
        spans = [(a, n) for a, n in zip(self.at, ns)]
        rows = [(i, a + r) for i, (a, n) in enumerate(spans) for r in range(n)]
        self.at = [a + n for a, n in spans]
        assert self.ctx.seq_ctx_len.tolist() == self.at
        tables = self.dt.cpu()
        held = [int(p) for i, a in enumerate(self.at) for p in tables[i, :-(-a // B)]]
        assert len(set(held)) == len(held) and min(held) >= 0               # no page twice
        slots = [int(tables[i, p // B]) * B + p % B for i, p in rows]
        assert self.ctx.slot_mapping[:T].tolist() == slots and self.ctx.positions[:T].tolist() == [p for _, p in rows]
        table = self.angles.cpu()
        x = self.x.float().view(self.rows, -1, self.hd)
        half = self.hd // 2
        turned = P.rotated(x[:, :self.nh + self.nkv], table[:, :half], table[:, half:], False)
        for t, s in enumerate(slots):
            P.write(self.kc, B, s // B, s % B, turned[t, self.nh:])
            P.write(self.vc, B, s // B, s % B, x[t, self.nh + self.nkv:])
        assert torch.equal(self.dk.cpu(), self.kc) and torch.equal(self.dv.cpu(), self.vc)
        q = self.q[:T].cpu()
        assert torch.equal(q, turned[:T, :self.nh].reshape(T, -1).to(torch.bfloat16))
        k, v = P.read(self.kc, self.hd, B), P.read(self.vc, self.hd, B)
        want = P.attention(q.double().view(T, self.nh, self.hd), k, v, tables, spans, self.nh, self.nkv, B, self.hd ** -0.5)
        check_attention(self.out[:T].view(T, self.nh, self.hd), want, v.abs().max().item(), "bfloat16", max(self.at) + self.hd)


@pytest.mark.parametrize("nh,nkv,hd,B", [(4, 2, 64, 16), (6, 1, 128, 16), (4, 4, 96, 7), (2, 1, 256, 8)])
@pytest.mark.parametrize("parts", [0, -1])
def test_prompts_then_single_rows_from_a_graph(nh, nkv, hd, B, parts):
    """Two steps of portions with tiles to spare, then single rows replayed over the ends of pages, then a step that has no page."""
    starts, steps = [0, 5, 2 * B, 70, 0], 2 * B + 3
    portions = [[2, 130, 65, 3, 200], [64, 2, 0, 70, 5]]
    width = (max(starts) + 264 + steps) // B + 2
    ends = [s + sum(p[i] for p in portions) + steps for i, s in enumerate(starts)]
    loop = Loop(starts, nh, nkv, hd, B, width, sum(-(-e // B) for e in ends), 402, 14, seed=hd)
    for ns in portions:
        loop.fill(ns)
        loop.launch()
        loop.check(ns)
    c = loop.ctx
    one = lambda *names: {n: getattr(c, n)[:loop.S].contiguous() for n in names}
    loop.ctx = types.SimpleNamespace(**{**vars(c), **one("positions", "row_seq", "slot_mapping"), "rows": loop.S, "decode_seqs": loop.S,
                                        "prefill_tiles": 0, "tile_seq": None, "tile_q0": None, "options": {"attn_parts": parts}})
    loop.rows = loop.S
    loop.qkv, loop.angles, loop.q, loop.out = (t[:loop.S].contiguous() for t in (loop.qkv, loop.angles, loop.q, loop.out))
    ns = [1] * loop.S
    loop.fill(ns)
    loop.launch()
    loop.check(ns)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loop.launch()
    for _ in range(steps - 1):
        loop.fill(ns)
        g.replay()
        loop.check(ns)
    while True:                                                              # to the end of the pages that are left
        loop.fill(ns)
        before = [t.clone() for t in (loop.dk, loop.dv, loop.dt, loop.count, loop.ctx.seq_ctx_len)]
        g.replay()
        if int(loop.status[0]):
            break
        loop.check(ns)
    with pytest.raises(K().KernelError, match="missing"):
        K().raise_on_step_tables(loop.status.tolist())
    K().check_errors()
    for was, t in zip(before, (loop.dk, loop.dv, loop.dt, loop.count, loop.ctx.seq_ctx_len)):
        assert torch.equal(was, t)


def test_requests_without_rows_behind_the_others():
    """A padded batch: entries that bring nothing, with and without a context, stand behind those that do; their rows stay apart."""
    loop = Loop([9, 40, 30, 0], 4, 2, 64, 16, 6, 16, 4, 0)
    loop.ctx.decode_seqs, loop.ctx.tile_seq, loop.ctx.tile_q0 = 4, None, None
    for _ in range(3):
        loop.fill([1, 1, 0, 0])
        loop.launch()
        loop.check([1, 1, 0, 0])
        assert not loop.out[3].any()                                         # nothing to see


# ------------------------------------------------------------------------------------------- side by side, again and again

def attend(kind, B=16, seed=0):
    """(inputs' owner, a call that writes a new result) of one kind."""
    nh, nkv, hd = 8, 2, 128 if kind != "unpack" else 96
    spans = [(700 * (i % 5) + 3, 1) for i in range(20)] if kind in ("shares", "kernel", "cluster", "plain") else [(300, 90), (0, 200), (5, 70)]
    tables, pages, ctx = make_step(spans, B, seed)
    ctx.options = {"shares": {"attn_parts": -1}, "kernel": {"attn_parts": 9}, "cluster": {"attn_parts": 4}, "plain": {"attention": "plain"}}.get(kind, {})
    kc, vc = make_cache(pages, nkv, B, hd, seed + 1).to(DEV), make_cache(pages, nkv, B, hd, seed + 2).to(DEV)
    q = torch.randn((ctx.rows, nh * hd), generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(DEV)
    tables = tables.to(DEV)

    def call(out):
        K().paged_attention_q4(q, out, kc, vc, tables, ctx, nh, nkv, hd, B, hd ** -0.5)
        return out
    return q, call


KINDS = ["shares", "kernel", "cluster", "plain", "portions", "unpack"]


@pytest.mark.parametrize("kind", KINDS)
def test_two_streams_at_once(kind):
    cases = [attend(kind, seed=s) for s in (0, 10)]
    want = [call(torch.empty_like(q)) for q, call in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = [[torch.full_like(q, 9.0) for _ in range(20)] for q, _ in cases]
    torch.cuda.synchronize()
    for i in range(20):
        for (q, call), s, o in zip(cases, streams, outs):
            with torch.cuda.stream(s):
                call(o[i])
    torch.cuda.synchronize()
    K().check_errors()
    for w, o in zip(want, outs):
        assert all(torch.equal(w, x) for x in o)


@pytest.mark.parametrize("kind", KINDS)
def test_two_graphs_by_turns(kind):
    cases = [attend(kind, seed=s) for s in (0, 10)]
    want = [call(torch.empty_like(q)) for q, call in cases]
    outs, graphs = [torch.empty_like(q) for q, _ in cases], []
    for (q, call), o in zip(cases, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(o)
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.fill_(9.0)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(w, o) for w, o in zip(want, outs))
    K().check_errors()


# ------------------------------------------------------------------------------------------- what is not there

@pytest.mark.parametrize("kind", KINDS)
def test_a_context_ends_with_its_table(kind):
    """A request that says more keys than its table has pages for sees those of its table: no other request's, nothing behind it."""
    nh, nkv, hd, B = 4, 2, 128 if kind != "unpack" else 96, 16
    single = kind not in ("portions", "unpack")
    spans = [(47, 1), (47, 1), (47, 1)] if single else [(0, 48), (0, 48), (0, 48)]
    tables, pages, ctx = make_step(spans, B, 1, width_extra=0)
    ctx.options = {"shares": {"attn_parts": -1}, "kernel": {"attn_parts": 9}, "cluster": {"attn_parts": 4}, "plain": {"attention": "plain"}}.get(kind, {})
    ctx.max_ctx = ctx.max_decode_ctx = 3000
    kc, vc = make_cache(pages, nkv, B, hd, 2).to(DEV), make_cache(pages, nkv, B, hd, 3).to(DEV)
    q = torch.randn((ctx.rows, nh * hd), generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(DEV)

    def run():
        out = torch.full_like(q, 9.0)
        K().paged_attention_q4(q, out, kc, vc, tables.to(DEV), ctx, nh, nkv, hd, B, hd ** -0.5)
        torch.cuda.synchronize()
        K().check_errors()
        return out
    want = run()
    longer = torch.tensor([48, 2900, 1000], **I32)
    if kind == "plain":
        ctx.positions = longer - 1
    else:
        ctx.seq_ctx_len = longer
    assert torch.equal(run(), want)


@pytest.mark.parametrize("hd,how", [(64, "unpack"), (128, "unpack"), (96, "auto"), (256, "auto"), (32, "auto"), (128, "auto")])
@pytest.mark.parametrize("window", [0, 20])
def test_tiles_of_no_request(hd, how, window):
    """Tiles behind the last one, and a step of nothing else: the rows' results are those without them, other rows stay."""
    nh, nkv, B = 4, 2, 16
    spans = [(33, 1), (300, 90), (0, 200)]
    tables, pages, ctx = make_step(spans, B, 5)
    ctx.options = {"attn_prefill": how}
    kc, vc = make_cache(pages, nkv, B, hd, 6).to(DEV), make_cache(pages, nkv, B, hd, 7).to(DEV)
    q = torch.randn((ctx.rows, nh * hd), generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).to(DEV)

    def run():
        out = torch.full_like(q, 9.0)
        K().attention_prefill_q4(q, out, kc, vc, tables.to(DEV), ctx, nh, nkv, hd, B, hd ** -0.5, window)
        torch.cuda.synchronize()
        K().check_errors()
        return out
    want = run()
    assert (want[0] == 9).all() and not (want[1:] == 9).any()
    none = torch.full((5,), -1, **I32)
    real = ctx.tile_seq, ctx.tile_q0, ctx.prefill_tiles
    ctx.tile_seq, ctx.tile_q0, ctx.prefill_tiles = torch.cat((real[0], none)), torch.cat((real[1], none)), real[2] + 5
    assert torch.equal(run(), want)
    ctx.tile_seq, ctx.tile_q0, ctx.prefill_tiles = none, none, 5
    assert (run() == 9).all()


@pytest.mark.parametrize("hd,how", [(64, "auto"), (128, "auto")])
def test_portions_do_not_see_masked_rows_that_are_no_numbers(hd, how):
    """A key or value that is not a number: rows before it and rows whose window has passed it are as they were, the others are none."""
    nh, nkv, B = 2, 1, 16
    tables, pages, ctx = make_step([(30, 300)], B, 9)
    kc, vc = make_cache(pages, nkv, B, hd, 6), make_cache(pages, nkv, B, hd, 7)
    q = torch.randn((ctx.rows, nh * hd), generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).to(DEV)

    def run(k, v, window):
        out = torch.full_like(q, 9.0)
        K().attention_prefill_q4(q, out, k.to(DEV), v.to(DEV), tables.to(DEV), ctx, nh, nkv, hd, B, hd ** -0.5, window)
        torch.cuda.synchronize()
        return out
    for window in (0, 40):
        clean = run(kc, vc, window)
        assert clean.isfinite().all()
        for key in (3, 100, 128, 290):
            for which in (0, 1):
                bad = [kc.clone(), vc.clone()]
                off = B * hd // 2 + 4 * (key % B)
                bad[which][int(tables[0, key // B]), 0, off:off + 4] = NAN
                got = run(*bad, window)
                pos = torch.arange(30, 330, device=DEV)
                sees = (pos >= key) & ((pos < key + window) if window else True)
                assert got[sees].isnan().all() and torch.equal(got[~sees], clean[~sees]), (window, key, which)
    K().check_errors()


# ------------------------------------------------------------------------------------------- values of very different size

@pytest.mark.parametrize("nh,nkv,hd", [(4, 1, 128), (1, 1, 64), (8, 1, 96), (6, 2, 128)])
@pytest.mark.parametrize("force", [1, 3, -1])
def test_a_large_value_without_weight_does_not_cost_the_others_their_bits(nh, nkv, hd, force):
    """Values 2^24 times the others, whose keys have scores far below the rest (p < 2^-200): one in the midst of a request, and the first
    32 of another, which are all there is until the rest comes.  The result is the others', to a rounding of it and of their
    weights (2^-12 each, below the 2^-8 of max |v|)."""
    B, n, at = 16, 400, [[37], range(32)]
    tables, pages, ctx = make_step([(n - 1, 1), (n - 1, 1)], B, 21)
    g = torch.Generator().manual_seed(22)
    x = torch.randn((2, pages, B, nkv, hd), generator=g)
    q = torch.randn((2, nh * hd), generator=g).abs().add(0.5).to(torch.bfloat16)
    for i, t in ((i, t) for i in range(2) for t in at[i]):
        page = int(tables[i, t // B])
        x[0, page, t % B] = -6.0 + 0.1 * x[0, page, t % B]                 # q > 0: its scores are low in every head
        x[1, page, t % B] *= 2.0 ** 24
    kc, vc = (torch.zeros((pages, nkv, P.page_bytes(B, hd)), dtype=torch.uint8) for _ in range(2))
    for p in range(pages):
        for o in range(B):
            P.write(kc, B, p, o, x[0, p, o])
            P.write(vc, B, p, o, x[1, p, o])
    out = torch.empty((2, nh * hd), dtype=torch.bfloat16, device=DEV)
    ctx.options = {"attn_parts": force}
    scale = 4.0 * hd ** -0.5
    K().attention_decode_q4(q.to(DEV), out, kc.to(DEV), vc.to(DEV), tables.to(DEV), ctx, nh, nkv, hd, B, scale)
    k, v = P.read(kc, hd, B), P.read(vc, hd, B)
    want = P.attention(q.double().view(2, nh, hd), k, v, tables, [(n - 1, 1), (n - 1, 1)], nh, nkv, B, scale)
    check_attention(out.view(2, nh, hd), want, 6.0, "bfloat16", n + hd)
