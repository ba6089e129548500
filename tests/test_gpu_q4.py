"""The cache in 4 bits on the GPU: rows written and read back, attention over it, each against plain float64.

Tolerances, from the arithmetic:
 * codes and pairs: equal; the kernel and the plain form take the same float32 steps with IEEE roundings.
 * attention, bfloat16: the result is rounded once (half a step: 2^-8 of the value), and so are the probabilities where they
   enter a product of bfloat16 (2^-8 of the row's sum of |p v|, itself at most the largest |v|); everything else is float32 over
   at most a few thousand keys (2^-24 of the same, times the number of terms).  Together 2^-8 |o| + 2^-8 max|v|, and the float32
   part well below a tenth of it.
 * attention, float32: sums of at most n + hd float32 terms, relative to scores' and values' largest products: 4 (n + hd) 2^-24
   of max|v| times one plus the largest |score| (an error of a score multiplies its probability).
"""
import math
import types

import pytest
import torch

import plain_q4 as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def K():
    from kvcm.kernels import library
    return library


def angles(T, rotary, seed):
    g = torch.Generator().manual_seed(seed)
    pos = torch.randint(0, 9000, (T,), generator=g).double()
    a = pos[:, None] * 10000.0 ** (-torch.arange(0, rotary, 2).double() / rotary)
    return a.cos().float(), a.sin().float()


def make_cache(pages, nkv, B, hd, seed, offset=0.0):
    """A pool of quantised random rows (every row of every page) on the CPU."""
    g = torch.Generator().manual_seed(seed)
    cache = torch.zeros((pages, nkv, P.page_bytes(B, hd)), dtype=torch.uint8)
    x = torch.randn((pages, B, nkv, hd), generator=g) + offset
    for p in range(pages):
        for o in range(B):
            P.write(cache, B, p, o, x[p, o])
    return cache


def make_step(spans, B, seed, pad=0, extra_pages=2, width_extra=1):
    """Page tables (shuffled ids) and the step's arrays of requests (start, rows); ``pad`` padded single-row entries behind them."""
    g = torch.Generator().manual_seed(seed)
    blocks = [-(-(s + n) // B) for s, n in spans]
    pages = sum(blocks) + extra_pages
    ids = torch.randperm(pages, generator=g).int()
    tables = torch.full((len(spans) + pad, max(blocks) + width_extra), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(blocks):
        tables[i, :n] = ids[at:at + n]
        at += n
    single = [i for i, (_, n) in enumerate(spans) if n == 1]
    assert single == list(range(len(single))), "entries of one row come first"
    q_start, tiles, row = [], [], 0
    for i, (_, n) in enumerate(spans):
        q_start.append(row)
        row += n
        if n > 1:
            tiles += [(i, q) for q in range(0, n, 64)]
    assert not pad or not tiles
    i32 = dict(dtype=torch.int32, device=DEV)
    ends = [s + n for s, n in spans] + [0] * pad
    ctx = types.SimpleNamespace(
        rows=row + pad, seqs=len(spans) + pad, decode_seqs=len(single) + pad, prefill_rows=row - len(single), prefill_tiles=len(tiles),
        tile_rows=64, max_ctx=max(ends), max_decode_ctx=max([ends[i] for i in single] + [0]), max_q_len=max(n for _, n in spans),
        positions=torch.tensor([s + r for s, n in spans for r in range(n)] + [-1] * pad, **i32),
        row_seq=torch.tensor([i for i, (_, n) in enumerate(spans) for _ in range(n)] + [len(spans) + j for j in range(pad)], **i32),
        seq_q_start=torch.tensor(q_start + [row + j for j in range(pad)], **i32),
        seq_q_len=torch.tensor([n for _, n in spans] + [1] * pad, **i32), seq_ctx_len=torch.tensor(ends, **i32),
        tile_seq=torch.tensor([t for t, _ in tiles], **i32), tile_q0=torch.tensor([q for _, q in tiles], **i32), options={})
    return tables, pages, ctx


# ------------------------------------------------------------------------------------------- write and read

@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("nh,nkv,hd,B,rotary,interleaved", [
    (4, 2, 64, 16, 64, False), (3, 1, 128, 16, 64, False), (2, 2, 16, 4, 16, False), (5, 5, 96, 7, 10, True), (1, 1, 8, 1, 0, False),
    (2, 1, 256, 8, 256, True), (6, 3, 40, 5, 32, False)])
def test_rows_written_and_read_back(dtype, nh, nkv, hd, B, rotary, interleaved):
    dt, T = DT[dtype], 37
    g = torch.Generator().manual_seed(hd + T)
    wide = torch.randn((T, (nh + 2 * nkv) * hd + 16), generator=g).to(dt)        # rows with a stride of their own
    pages = -(-T // B) + 3
    slots = torch.randperm(pages * B, generator=g)[:T].int()
    slots[5], slots[11] = -1, pages * B                                          # nowhere, and beyond the pool
    cos, sin = angles(T, max(rotary, 2), 3)
    table = torch.cat((cos, sin), 1).contiguous().to(DEV) if rotary else None
    before = torch.randint(0, 256, (2, pages, nkv, P.page_bytes(B, hd)), generator=g, dtype=torch.uint8)
    kc, vc = before[0].to(DEV), before[1].to(DEV)
    rows = wide.to(DEV)[:, :(nh + 2 * nkv) * hd]
    q = torch.empty((T, nh * hd), dtype=dt, device=DEV)
    K().rope_cache_q4(rows, table, interleaved, slots.to(DEV), kc, vc, q, nh, nkv, hd, B)
    x = wide[:, :(nh + 2 * nkv) * hd].float().view(T, nh + 2 * nkv, hd)
    qk = P.rotated(x[:, :nh + nkv], cos, sin, interleaved) if rotary else x[:, :nh + nkv]
    assert torch.equal(q.cpu(), qk[:, :nh].reshape(T, nh * hd).to(dt))
    assert torch.equal(rows.cpu(), wide[:, :(nh + 2 * nkv) * hd])                # the fused rows stay
    want_k, want_v = before[0].clone(), before[1].clone()
    for t in range(T):
        if 0 <= slots[t] < pages * B:
            P.write(want_k, B, int(slots[t]) // B, int(slots[t]) % B, qk[t, nh:])
            P.write(want_v, B, int(slots[t]) // B, int(slots[t]) % B, x[t, nh + nkv:])
    assert torch.equal(kc.cpu(), want_k) and torch.equal(vc.cpu(), want_v)       # every other byte too
    for back in (torch.float32, torch.bfloat16):
        k_rows = torch.full((T, nkv * hd), 7.0, dtype=back, device=DEV)
        v_rows = torch.full((T, nkv * hd), 7.0, dtype=back, device=DEV)
        K().read_cache_q4(kc, vc, slots.to(DEV), k_rows, v_rows, nkv, hd, B)
        for got, cache in ((k_rows, want_k), (v_rows, want_v)):
            values = P.read(cache, hd, B)
            for t in range(T):
                s = int(slots[t])
                want = values[s // B, :, s % B].reshape(-1) if 0 <= s < pages * B else torch.full((nkv * hd,), 7.0)
                assert torch.equal(got[t].cpu(), want.float().to(back))
    # in place: the q columns of the fused rows themselves
    kc2, vc2 = before[0].to(DEV), before[1].to(DEV)
    K().rope_cache_q4(rows, table, interleaved, slots.to(DEV), kc2, vc2, rows[:, :nh * hd], nh, nkv, hd, B)
    assert torch.equal(rows[:, :nh * hd], q) and torch.equal(kc2, kc) and torch.equal(vc2, vc)


def test_half_a_step_of_error_and_odd_rows():
    """|x - read back| <= scale / 2 + what the pair's own roundings move: 2^-9 of |zero| and 15 * 2^-9 of the scale."""
    hd, B, T = 64, 16, 32
    g = torch.Generator().manual_seed(2)
    x = torch.randn((T, 3, hd), generator=g) * torch.logspace(-30, 30, T)[:, None, None]
    x[3] = 0.0
    x[4] = -2.5                                                     # equal elements: scale 0
    x[5, 1, 7] = math.inf
    x[6, 2, 0] = math.nan
    x[7, 1, 3], x[7, 1, 4] = 3e38, -3e38                            # a range beyond float32
    rows = x.view(T, -1).to(DEV)
    kc = torch.zeros((2, 1, P.page_bytes(B, hd)), dtype=torch.uint8, device=DEV)
    vc, q = torch.zeros_like(kc), torch.empty((T, hd), device=DEV)
    slots = torch.arange(T, dtype=torch.int32, device=DEV)
    K().rope_cache_q4(rows, None, False, slots, kc, vc, q, 1, 1, hd, B)
    k, v = torch.empty((T, hd), device=DEV), torch.empty((T, hd), device=DEV)
    K().read_cache_q4(kc, vc, slots, k, v, 1, hd, B)
    k, v = k.cpu().double(), v.cpu().double()
    assert k[5].isnan().all() and k[7].isnan().all() and v[6].isnan().all() and v[5].isfinite().all() and k[6].isfinite().all()
    for got, col in ((k, 1), (v, 2)):
        for t in range(T):
            want = x[t, col].double()
            if not want.isfinite().all() or t == 7:
                continue
            step = (want.max() - want.min()) / 15
            room = step * (0.5 + 15 * 2.0 ** -9) * (1 + 2.0 ** -8) + want.min().abs() * 2.0 ** -9
            assert (got[t] - want).abs().max() <= room, (t, col)
    assert torch.equal(k[4], torch.full((hd,), -2.5).double()) and not k[3].any()


# ------------------------------------------------------------------------------------------- attention

def check_attention(got, want, v_max, dtype, terms, top=0.0):
    got, want = got.double().cpu(), want.double()
    assert torch.isfinite(got).all()
    if dtype == "bfloat16":
        room = (2.0 ** -8 * want.abs() + 2.0 ** -8 * v_max) * 1.1
    else:
        room = torch.full_like(want, 4 * terms * 2.0 ** -24 * v_max * (1 + top))
    over = ((got - want).abs() - room).max().item()
    assert over <= 0, over


def run_attention(call, spans, nh, nkv, hd, B, dtype, seed=0, pad=0, q_scale=1.0, **opts):
    tables, pages, ctx = make_step(spans, B, seed, pad)
    kc, vc = make_cache(pages, nkv, B, hd, seed + 1, 0.5), make_cache(pages, nkv, B, hd, seed + 2, -0.25)
    g = torch.Generator().manual_seed(seed + 3)
    q = (q_scale * torch.randn((ctx.rows, nh * hd + 8), generator=g)).to(DT[dtype]).to(DEV)[:, :nh * hd]
    sink = opts.pop("sink", None)
    sink_t = torch.linspace(-1.0, 3.0, nh) if sink else None
    out = torch.full((ctx.rows + 2, nh * hd), 9.0, dtype=DT[dtype], device=DEV)
    scale = hd ** -0.5
    call(q, out[:ctx.rows], kc.to(DEV), vc.to(DEV), tables.to(DEV), ctx, nh, nkv, hd, B, scale, sink=sink_t.to(DEV) if sink else None, **opts)
    torch.cuda.synchronize()
    K().check_errors()
    rows = sum(n for _, n in spans)
    assert (out[ctx.rows:] == 9).all()                              # rows behind the last one
    assert not out[rows:ctx.rows].any()                             # padded entries see nothing
    k, v = P.read(kc, hd, B), P.read(vc, hd, B)
    want = P.attention(q.cpu().double().view(-1, nh, hd)[:rows], k, v, tables, spans, nh, nkv, B, scale, sink=sink_t, **opts)
    top = (q.abs().max() * k.abs().max() * hd ** 0.5).item()
    check_attention(out[:rows].view(-1, nh, hd), want, v.abs().max().item(), dtype, ctx.max_ctx + hd, top)
    return out[:rows]


def plain(q, out, kc, vc, tables, ctx, *args, **kw):
    K().attention_plain_q4(q, out, kc, vc, tables, ctx.row_seq, ctx.positions, *args, **kw)


OPTIONS = [{}, {"window": 7}, {"softcap": 4.0}, {"sink": True}, {"window": 33, "softcap": 2.0, "sink": True}]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("opts", OPTIONS, ids=str)
@pytest.mark.parametrize("nh,nkv,hd,B", [(4, 2, 16, 16), (3, 1, 40, 7), (2, 2, 256, 8), (8, 1, 64, 16)])
def test_plain_attention(dtype, opts, nh, nkv, hd, B):
    run_attention(plain, [(0, 1), (1, 1), (B - 1, 1), (63, 1), (40, 5), (0, 3)], nh, nkv, hd, B, dtype, **dict(opts))


def test_plain_attention_of_more_keys_than_a_chunk():
    run_attention(plain, [(511, 1), (512, 1), (1300, 1)], 2, 1, 32, 16, "float32")


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_a_step_of_single_rows_and_portions(dtype):
    for hd, B in ((16, 16), (64, 16), (128, 8)):
        run_attention(K().paged_attention_q4, [(0, 1), (30, 1), (77, 1), (0, 2), (19, 40), (0, 70)], 4, 2, hd, B, dtype)


# ------------------------------------------------------------------------------------------- single rows on the tensor cores

def decode(force=0, merge="cluster"):
    def call(q, out, kc, vc, tables, ctx, *args, **kw):
        ctx.options = {"attn_parts": force, "attn_merge": merge}
        K().attention_decode_q4(q, out, kc, vc, tables, ctx, *args, **kw)
    return call


@pytest.mark.parametrize("nh,nkv,hd,B", [(2, 2, 32, 16), (8, 1, 64, 16), (4, 2, 96, 8), (6, 1, 128, 16), (3, 3, 160, 4), (18, 2, 192, 16), (4, 2, 224, 5),
                                         (17, 1, 256, 32), (12, 1, 64, 1), (5, 5, 128, 100)])
@pytest.mark.parametrize("force,merge", [(0, "cluster"), (1, "cluster"), (3, "cluster"), (3, "kernel"), (-1, "kernel")])
def test_single_rows(nh, nkv, hd, B, force, merge):
    spans = [(0, 1), (1, 1), (30, 1), (31, 1), (32, 1), (127, 1), (128, 1), (129, 1), (300, 1), (399, 1)]
    run_attention(decode(force, merge), spans, nh, nkv, hd, B, "bfloat16", seed=hd, pad=3)


@pytest.mark.parametrize("opts", OPTIONS[1:], ids=str)
@pytest.mark.parametrize("nh,nkv,hd,B", [(8, 1, 64, 16), (6, 1, 128, 7), (2, 2, 96, 16), (2, 1, 256, 16)])
@pytest.mark.parametrize("force", [0, 2, -1])
def test_single_rows_with_masks(opts, nh, nkv, hd, B, force):
    run_attention(decode(force), [(0, 1), (6, 1), (7, 1), (45, 1), (200, 1), (385, 1)], nh, nkv, hd, B, "bfloat16", seed=7, pad=1, **dict(opts))


def test_more_partitions_than_a_cluster_and_more_pages_than_the_slice():
    run_attention(decode(12), [(1500, 1), (2, 1), (1535, 1)], 2, 1, 64, 16, "bfloat16")
    for force in (1, -1):
        run_attention(decode(force), [(600, 1), (1100, 1)], 2, 1, 64, 1, "bfloat16")      # 601 pages of one key each


def test_shares_of_many_requests():
    """More tiles than blocks at once, shares that begin and end inside requests, empty requests among them."""
    spans = [(int(700 * abs(math.sin(3 * i))), 1) for i in range(40)]
    run_attention(decode(-1), spans, 16, 8, 64, 16, "bfloat16", pad=7)
    run_attention(decode(-1), [(5000, 1), (0, 1), (3, 1)], 12, 4, 128, 16, "bfloat16")


def test_large_scores_and_one_key_that_counts():
    """Scores of a few hundred: one key has all the weight, and its value comes back."""
    run_attention(decode(), [(700, 1), (65, 1)], 4, 2, 128, 16, "bfloat16", q_scale=60.0)
    run_attention(decode(2), [(700, 1), (65, 1)], 4, 2, 64, 16, "bfloat16", q_scale=60.0)


def test_a_key_behind_the_context_does_not_count():
    """Pages end inside a step: what lies behind the context (not-a-number among it) is not seen; inside it is."""
    hd, B, nh, nkv = 64, 16, 4, 1
    tables, pages, ctx = make_step([(40, 1), (20, 1)], B, 3)
    kc, vc = make_cache(pages, nkv, B, hd, 1), make_cache(pages, nkv, B, hd, 2)
    q = torch.randn(2, nh * hd).to(torch.bfloat16).to(DEV)

    def run(k, v):
        out = torch.empty_like(q)
        K().attention_decode_q4(q, out, k.to(DEV), v.to(DEV), tables.to(DEV), ctx, nh, nkv, hd, B, 0.125)
        return out
    clean = run(kc, vc)
    for key, seen in ((41, False), (47, False), (40, True), (0, True)):
        for which in (0, 1):
            bad = [kc.clone(), vc.clone()]
            page, off = int(tables[0, key // B]), key % B
            bad[which][page, 0, B * hd // 2 + 4 * off:B * hd // 2 + 4 * off + 4] = torch.tensor([0xc0, 0x7f, 0xc0, 0x7f], dtype=torch.uint8)
            got = run(*bad)
            assert torch.equal(got[1], clean[1])
            assert bool(got[0].isnan().all()) if seen else torch.equal(got[0], clean[0]), (key, which)


# ------------------------------------------------------------------------------------------- portions

@pytest.mark.parametrize("opts", OPTIONS, ids=str)
@pytest.mark.parametrize("nh,nkv,hd,B", [(4, 2, 32, 16), (8, 1, 64, 16), (2, 2, 96, 8), (6, 1, 128, 16), (4, 2, 64, 64), (4, 4, 128, 8), (2, 1, 256, 16),
                                         (3, 1, 64, 7)])
@pytest.mark.parametrize("how", ["auto", "unpack"])
def test_portions(opts, nh, nkv, hd, B, how):
    if how == "unpack" and hd not in (64, 128):
        pytest.skip("the only way for this head size")

    def call(q, out, kc, vc, tables, ctx, *args, **kw):
        ctx.options = {"attn_prefill": how}
        K().attention_prefill_q4(q, out, kc, vc, tables, ctx, *args, **kw)
    spans = [(0, 2), (0, 65), (7, 64), (131, 130), (64, 3), (0, 300)]
    run_attention(call, spans, nh, nkv, hd, B, "bfloat16", seed=hd + B, **dict(opts))


@pytest.mark.parametrize("spans", [[(0, 127)], [(0, 128)], [(1, 129)], [(63, 255)], [(64, 256)], [(0, 257)], [(700, 513)], [(2, 2), (900, 30), (0, 600)]],
                         ids=str)
@pytest.mark.parametrize("hd", [64, 128])
def test_groups_and_tiles_of_portions(spans, hd):
    run_attention(K().attention_prefill_q4, spans, 2, 1, hd, 16, "bfloat16", seed=len(spans))


def test_portions_with_large_scores_and_tiles_that_are_none():
    def call(q, out, kc, vc, tables, ctx, *args, **kw):
        none = torch.full((3,), -1, dtype=torch.int32, device=DEV)
        ctx.tile_seq, ctx.tile_q0 = torch.cat((ctx.tile_seq, none)), torch.cat((ctx.tile_q0, none))
        ctx.prefill_tiles += 3
        K().attention_prefill_q4(q, out, kc, vc, tables, ctx, *args, **kw)
    for hd in (64, 128):
        run_attention(call, [(300, 90), (0, 200)], 4, 2, hd, 16, "bfloat16", q_scale=40.0)


def test_single_rows_before_portions():
    for hd, B in ((64, 16), (128, 32)):
        run_attention(K().paged_attention_q4, [(200, 1), (0, 1), (5, 1), (90, 140), (0, 20)], 8, 2, hd, B, "bfloat16", seed=hd)
