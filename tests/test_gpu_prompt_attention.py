"""Whole prompts over their own rows on the GPU, within bounds that follow from the kernel's roundings (plain_q8.py)."""
import types

import pytest
import torch

import plain_q8 as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def K():
    from kvcm.kernels import library
    return library


def make_ctx(lengths, pad=0, gap=0):
    """Prompts one behind another (``gap`` rows of nobody before the first), those of one row first; ``pad`` empty tiles."""
    singles = [n for n in lengths if n == 1]
    assert lengths[:len(singles)] == singles
    starts, tiles, at = [], [], gap
    for i, n in enumerate(lengths):
        starts.append(at)
        if n > 1:
            tiles += [(i, q) for q in range(0, n, 64)]
        at += n
    tiles += [(-1, -1)] * pad
    i32 = dict(dtype=torch.int32, device=DEV)
    return types.SimpleNamespace(
        rows=at, seqs=len(lengths), decode_seqs=len(singles), prefill_tiles=len(tiles), tile_rows=64, seq_q_start=torch.tensor(starts, **i32),
        seq_q_len=torch.tensor(lengths, **i32), tile_seq=torch.tensor([t for t, _ in tiles], **i32),
        tile_q0=torch.tensor([q for _, q in tiles], **i32), options={}), starts, at


def check(lengths, nh, nkv, hd, window=0, softcap=0.0, sink=False, dtype=torch.bfloat16, options=None, behind=3, pad=0, gap=0, q_size=1.5, poison=None,
          kind=None, exponential=2.0 ** -21):
    g = torch.Generator().manual_seed(hd + sum(lengths))
    ctx, starts, rows = make_ctx(lengths, pad, gap)
    ctx.options = options or {}
    T = rows + behind
    width = (nh + 2 * nkv) * hd
    qkv = torch.randn((T, width + 8), generator=g)
    qkv[:, :nh * hd] *= q_size
    qkv = qkv.to(dtype)
    qkv[rows:] = float("nan")                                      # rows of nobody may hold anything
    qkv[:gap] = float("inf")
    if poison:
        poison(qkv, starts)
    dev = qkv.to(DEV)
    q, k, v = dev[:, :nh * hd], dev[:, nh * hd:(nh + nkv) * hd], dev[:, (nh + nkv) * hd:width]
    s = torch.randn((nh,), generator=g) if sink else None
    out = torch.full((T, nh * hd + 8), 7.0, dtype=dtype, device=DEV)
    K().prompt_attention(q, k, v, out[:, :nh * hd], ctx, nh, nkv, hd, hd ** -0.5, window, softcap, s.to(DEV) if sink else None)
    got = out.cpu().double()
    assert bool((got[:, nh * hd:] == 7.0).all()) and bool((got[rows:] == 7.0).all()) and bool((got[:gap] == 7.0).all())
    x = qkv.double()
    wants = []
    for a, n in zip(starts, lengths):
        qq, kk, vv = (x[a:a + n, lo * hd:hi * hd].view(n, -1, hd) for lo, hi in ((0, nh), (nh, nh + nkv), (nh + nkv, nh + 2 * nkv)))
        want, room = P.attend(kind or ("prompt" if dtype == torch.bfloat16 and hd <= 128 and not options else "plain float32" if dtype == torch.float32 else "plain bfloat16"),
                              qq, torch.nan_to_num(kk.transpose(0, 1)), torch.nan_to_num(vv.transpose(0, 1)), torch.arange(n), hd ** -0.5, window,
                              softcap, s, exponential=exponential)
        wants.append((a, n, got[a:a + n, :nh * hd].view(n, nh, hd), want, room))
        if poison is None:
            far = (wants[-1][2] - want).abs()
            assert bool((far <= room).all()), (a, n, float((far / room).max()))
    K().check_errors()
    return wants


@pytest.mark.parametrize("lengths", [[1], [1, 1, 1], [2], [1, 16, 17], [128], [129], [256], [257], [300, 5, 64], [1, 1, 2, 127, 128, 255, 513]])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 1, 64), (4, 2, 128), (3, 3, 128), (2, 1, 96), (4, 2, 32), (2, 2, 8), (2, 1, 72)])
def test_prompts(lengths, nh, nkv, hd):
    check(lengths, nh, nkv, hd)


@pytest.mark.parametrize("masks", [dict(window=100), dict(window=1), dict(window=128), dict(window=300), dict(softcap=20.0), dict(sink=True),
                                   dict(window=77, softcap=5.0, sink=True)])
@pytest.mark.parametrize("hd", [64, 128])
def test_prompts_with_masks(masks, hd):
    check([1, 700, 130, 3], 4, 2, hd, **masks)


def test_a_long_prompt():
    check([2100], 2, 1, 128)
    check([1, 1500], 2, 1, 64, window=700)


@pytest.mark.parametrize("masks", [dict(), dict(window=90), dict(softcap=20.0, sink=True)])
@pytest.mark.parametrize("nh,nkv,hd", [(32, 4, 64), (40, 8, 128)])
def test_more_blocks_than_the_gpu_holds(nh, nkv, hd, masks):
    """Blocks of one and of two groups of rows, whole and with zeros behind the last row, in any order behind one another."""
    check([1, 1, 300, 128, 17, 257, 2, 400, 129, 64, 500, 16, 200], nh, nkv, hd, pad=3, gap=2, **masks)
    check([1] * 9, nh, nkv, hd, **masks)


@pytest.mark.parametrize("q_size", [1e-3, 60.0])
def test_prompts_of_other_sizes(q_size):
    check([400], 4, 2, 128, q_size=q_size)


def test_tiles_of_nobody_and_rows_before_the_first():
    check([1, 200, 70], 4, 2, 128, pad=5, gap=9)


@pytest.mark.parametrize("dtype,hd,options", [(torch.float32, 64, None), (torch.float32, 40, None), (torch.bfloat16, 256, None), (torch.bfloat16, 128, dict(attention="plain"))])
def test_plain_prompts(dtype, hd, options):
    check([1, 130, 9], 4, 2, hd, dtype=dtype, options=options, window=60, softcap=9.0, sink=True, kind=None)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window", [0, 90])
def test_what_a_row_does_not_see_may_be_anything(hd, window):
    """A value that is not a number reaches the rows that see it, and no other; neither does an infinite key."""
    nh, nkv, at = 4, 2, 200

    def poison(qkv, starts):
        a = starts[1]
        qkv[a + at, (nh + nkv) * hd:(nh + nkv) * hd + hd:5] = float("nan")      # one value head
        qkv[a + at, (nh + nkv) * hd + 1] = float("inf")
        qkv[a + at + 30, nh * hd:(nh + nkv) * hd] = float("nan")                # a key
    wants = check([40, 420, 130], nh, nkv, hd, window=window, poison=poison)
    for i, (a, n, got, want, room) in enumerate(wants):
        clear = torch.ones((n, nh), dtype=torch.bool)
        if i == 1:
            row = torch.arange(n)
            sees = lambda key: (row >= key) & ((row < key + window) if window else torch.ones(n, dtype=torch.bool))
            clear &= ~sees(at)[:, None] | torch.tensor([False, False, True, True])      # (heads 0 and 1 read the first KV head)
            clear &= ~sees(at + 30)[:, None]
            assert bool(torch.isnan(got[~clear]).any(-1).all())
        assert bool(((got - want).abs() <= room)[clear].all())


@pytest.mark.parametrize("levels", [(0.0, -90.0), (-90.0, 0.0), (-60.0, -200.0), (30.0, 5.0), (0.0, 250.0), (-200.0, -200.0)])
@pytest.mark.parametrize("at", [1, 70, 150, 300])
def test_scores_far_from_zero(levels, at):
    """Scores of about one level up to row ``at`` and another behind it: references that have to be looked for, and such that must not come down."""
    nh, nkv, hd = 2, 1, 64
    wide = 8.0                                                      # q is (8, noise), k (level, noise): a score is about the level

    def shape(qkv, starts):
        a = starts[0]
        qkv[:, :nh * hd:hd] = wide
        n = qkv.shape[0]
        level = torch.where(torch.arange(n) < a + at, torch.tensor(levels[0]), torch.tensor(levels[1]))
        qkv[:, nh * hd] = (level * hd ** 0.5 / wide).to(qkv.dtype)
    for a, n, got, want, room in check([420], nh, nkv, hd, q_size=0.3, poison=shape, behind=0):
        far = (got - want).abs()
        assert bool((far <= room).all()), float((far / room).max())


def test_agrees_with_pages():
    """The same rows through bfloat16 pages: as far apart as both may be from the definition."""
    nh, nkv, hd, B, n = 4, 2, 128, 16, 333
    wants = check([n], nh, nkv, hd)
    g = torch.Generator().manual_seed(hd + n)
    qkv = torch.randn((n + 3, (nh + 2 * nkv) * hd + 8), generator=g)
    qkv[:, :nh * hd] *= 1.5
    qkv = qkv.bfloat16()[:n, :(nh + 2 * nkv) * hd]
    ctx, _, _ = make_ctx([n])
    ctx.seq_ctx_len, ctx.positions, ctx.row_seq = ctx.seq_q_len, torch.arange(n, dtype=torch.int32, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV)
    blocks = -(-n // B)
    cache = torch.zeros((2, blocks, nkv, B, hd), dtype=torch.bfloat16)
    for j, lo in ((0, nh), (1, nh + nkv)):
        x = torch.zeros((blocks * B, nkv, hd), dtype=torch.bfloat16)
        x[:n] = qkv[:, lo * hd:(lo + nkv) * hd].reshape(n, nkv, hd)
        cache[j] = x.view(blocks, B, nkv, hd).transpose(1, 2)
    cache = cache.to(DEV)
    out = torch.empty((n, nh * hd), dtype=torch.bfloat16, device=DEV)
    K().paged_attention(qkv[:, :nh * hd].contiguous().to(DEV), out, cache[0], cache[1], torch.arange(blocks, dtype=torch.int32, device=DEV)[None].contiguous(),
                        ctx, nh, nkv, hd, hd ** -0.5)
    _, _, got, want, room = wants[0]
    assert bool(((out.cpu().double().view(n, nh, hd) - got).abs() <= 2 * room).all())


@pytest.mark.parametrize("hd", [64, 96, 128])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_a_row_of_one_key_is_its_value(hd, softcap):
    """Weights enter the sum as they were rounded: p v / p is off by two roundings of 2^-24, less than half a step of the result."""
    for _, _, got, want, _ in check([1, 2, 130, 300], 4, 2, hd, window=1, softcap=softcap):
        assert torch.equal(got, want)
    for _, _, got, want, _ in check([5, 257], 4, 2, hd, softcap=softcap):
        assert torch.equal(got[:1], want[:1])
