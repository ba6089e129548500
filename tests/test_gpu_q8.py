"""The cache in 8 bits on the GPU: rows written and read back bit by bit, attention over it within bounds that follow from its roundings
(plain_q8.py)."""
import pytest
import torch

import plain_q4
import plain_q8 as P
from test_gpu_q4 import angles, make_step

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def K():
    from kvcm.kernels import library
    return library


def gpu_pool(codes, scale):
    return codes.to(DEV).view(P.FP8), scale.to(DEV)


def same(codes, want):
    """Codes alike; two not-a-numbers are."""
    a, b = codes.cpu().view(torch.uint8), want
    return bool(((a == b) | ((a & 127 == 127) & (b & 127 == 127))).all())


# ------------------------------------------------------------------------------------------- write and read

def neighbours(spans, B, seed, extra=3):
    """Slots of requests (start, rows) one behind another, pages in any order."""
    g = torch.Generator().manual_seed(seed)
    firsts = [s // B for s, _ in spans]
    counts = [-(-(s + n) // B) - f for (s, n), f in zip(spans, firsts)]
    ids = torch.randperm(sum(counts) + extra, generator=g).tolist()
    slots, at = [], 0
    for (s, n), f, c in zip(spans, firsts, counts):
        mine = ids[at:at + c]
        at += c
        slots += [mine[(s + i) // B - f] * B + (s + i) % B for i in range(n)]
    return torch.tensor(slots, dtype=torch.int32), len(ids)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("nh,nkv,hd,B,rotary,interleaved,spans", [
    (4, 2, 64, 16, 64, False, [(5, 40), (0, 1), (31, 1), (16, 16), (7, 3)]),
    (3, 1, 128, 16, 64, False, [(3, 1)] * 9),
    (2, 2, 16, 4, 16, False, [(0, 23), (2, 11)]),
    (5, 5, 96, 7, 10, True, [(6, 30), (0, 7)]),
    (1, 1, 8, 1, 0, False, [(0, 20)]),
    (2, 1, 256, 8, 256, True, [(1, 30), (4, 2)]),
    (6, 3, 40, 5, 32, False, [(0, 14), (4, 1), (3, 9)]),
    (2, 1, 64, 64, 64, False, [(10, 200), (63, 70)]),               # runs of more rows than a warp keeps
    (1, 1, 32, 100, 32, False, [(40, 59), (0, 100), (1, 150)]),
    (2, 1, 32, 16, 32, False, [(9, 700), (5, 1), (6, 1), (0, 90)]),    # windows of sixteen rows
    (1, 1, 16, 3000, 16, False, [(100, 1200), (2999, 2)])])
def test_rows_written_and_read_back(dtype, nh, nkv, hd, B, rotary, interleaved, spans):
    dt, T = DT[dtype], sum(n for _, n in spans)
    g = torch.Generator().manual_seed(hd + T)
    wide = torch.randn((T, (nh + 2 * nkv) * hd + 16), generator=g) * 2.0 ** torch.randint(-4, 5, (T, 1), generator=g).float()
    wide = wide.to(dt)                                              # rows with a stride of their own
    slots, pages = neighbours(spans, B, T)
    slots[0], slots[-1] = -1, pages * B                             # nowhere, and beyond the pool
    cos, sin = angles(T, max(rotary, 2), 3)
    table = torch.cat((cos, sin), 1).contiguous().to(DEV) if rotary else None
    (kc, ks), (vc, vs) = P.pool(pages, nkv, B, hd, 1, spread=6), P.pool(pages, nkv, B, hd, 2, size=0.01)
    k, k_scale = gpu_pool(kc, ks)
    v, v_scale = gpu_pool(vc, vs)
    rows = wide.to(DEV)[:, :(nh + 2 * nkv) * hd]
    q = torch.empty((T, nh * hd), dtype=dt, device=DEV)
    K().rope_cache_q8(rows, table, interleaved, slots.to(DEV), k, v, k_scale, v_scale, q, nh, nkv, hd)
    x = wide[:, :(nh + 2 * nkv) * hd].float().view(T, nh + 2 * nkv, hd)
    qk = plain_q4.rotated(x[:, :nh + nkv], cos, sin, interleaved) if rotary else x[:, :nh + nkv]
    assert torch.equal(q.cpu(), qk[:, :nh].reshape(T, nh * hd).to(dt))
    assert torch.equal(rows.cpu(), wide[:, :(nh + 2 * nkv) * hd])
    # (a page that begins anew keeps what lies behind its rows, as bytes that stand for nothing)
    P.write(kc, ks, slots, qk[:, nh:])
    P.write(vc, vs, slots, x[:, nh + nkv:])
    assert torch.equal(k_scale.cpu(), ks) and torch.equal(v_scale.cpu(), vs)
    assert same(k, kc) and same(v, vc)
    for back in (torch.float32, torch.bfloat16):
        k_rows = torch.full((T, nkv * hd), 7.0, dtype=back, device=DEV)
        v_rows = torch.full((T, nkv * hd), 7.0, dtype=back, device=DEV)
        K().read_cache_q8(k, v, k_scale, v_scale, slots.to(DEV), k_rows, v_rows)
        for got, codes, scale in ((k_rows, kc, ks), (v_rows, vc, vs)):
            s = slots.long()
            real = (s >= 0) & (s < pages * B)
            want = torch.full((T, nkv * hd), 7.0)
            want[real] = P.values(codes, scale)[s[real] // B, :, s[real] % B].reshape(-1, nkv * hd)
            assert torch.equal(got.cpu(), want.to(back))


def test_extreme_elements():
    """Zeros, the largest and smallest floats, numbers on a step's border, infinities and not-a-number."""
    nh, nkv, hd, B, T = 1, 1, 32, 8, 16
    x = torch.zeros((T, 3 * hd))
    x[0] = 3.4e38
    x[1, :40] = torch.tensor([1e-45, 1e-38, -1e-30, 448.0, 449.0, -448.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9, 464.0] * 4)
    x[8, hd:2 * hd] = 448.0 * 2.0 ** -60                            # the smallest scale's largest element
    x[8, 2 * hd:] = 2.0 ** -80
    x[9, hd], x[9, hd + 1], x[9, 2 * hd + 3] = float("inf"), float("nan"), -float("inf")
    slots = torch.arange(T, dtype=torch.int32)
    (kc, ks), (vc, vs) = P.pool(3, nkv, B, hd, 1), P.pool(3, nkv, B, hd, 2)
    k, k_scale = gpu_pool(kc, ks)
    v, v_scale = gpu_pool(vc, vs)
    q = torch.empty((T, hd), device=DEV)
    K().rope_cache_q8(x.to(DEV), None, False, slots.to(DEV), k, v, k_scale, v_scale, q, nh, nkv, hd)
    rows = x.view(T, 3, hd)
    P.write(kc, ks, slots, rows[:, 1:2])
    P.write(vc, vs, slots, rows[:, 2:])
    assert torch.equal(k_scale.cpu(), ks) and torch.equal(v_scale.cpu(), vs)
    assert same(k, kc) and same(v, vc)
    got = torch.empty((T, hd), device=DEV), torch.empty((T, hd), device=DEV)
    K().read_cache_q8(k, v, k_scale, v_scale, slots.to(DEV), *got)
    assert torch.equal(torch.isnan(got[0].cpu()), ~torch.isfinite(rows[:, 1])) and torch.equal(torch.isnan(got[1].cpu()), ~torch.isfinite(rows[:, 2]))


def test_a_page_filled_row_by_row_keeps_to_its_largest_element():
    """Appending rows of growing size one call at a time: old rows follow the scale, and each is off by a step of the final one at most."""
    nkv, hd, B = 2, 64, 16
    g = torch.Generator().manual_seed(5)
    x = torch.randn((B, 3 * nkv, hd), generator=g) * 2.0 ** torch.arange(B).view(B, 1, 1).float() * 0.01
    k = torch.zeros((2, nkv, B, hd), dtype=torch.uint8, device=DEV).view(P.FP8)
    v, ks, vs = torch.zeros_like(k.view(torch.uint8)).view(P.FP8), torch.zeros((2, nkv), device=DEV), torch.zeros((2, nkv), device=DEV)
    kc, vc, kss, vss = torch.zeros((2, nkv, B, hd), dtype=torch.uint8), torch.zeros((2, nkv, B, hd), dtype=torch.uint8), torch.zeros((2, nkv)), torch.zeros((2, nkv))
    q = torch.empty((1, nkv * hd), device=DEV)
    for t in range(B):
        slot = torch.tensor([B + t], dtype=torch.int32)
        K().rope_cache_q8(x[t].reshape(1, -1).to(DEV), None, False, slot.to(DEV), k, v, ks, vs, q, nkv, nkv, hd)
        P.write(kc, kss, slot, x[t:t + 1, nkv:2 * nkv])
        P.write(vc, vss, slot, x[t:t + 1, 2 * nkv:])
        assert same(k, kc) and same(v, vc) and torch.equal(ks.cpu(), kss) and torch.equal(vs.cpu(), vss)
    got = P.values(kc, kss)[1].transpose(0, 1)                     # [B, nkv, hd]
    want = x[:, nkv:2 * nkv]
    # each rounding: 2^-4 of the value, or half of 2^-9 of the scale of its day; scales double, so all the smaller ones add up to the last
    room = 2.0 ** -4 * want.abs() + 2.0 ** -4 * (1 + 2.0 ** -4) * want.abs() + 2 * 2.0 ** -10 * kss[1][None, :, None]
    assert bool(((got - want).abs() <= room).all())


# ------------------------------------------------------------------------------------------- attention

def check(kind, spans, nh, nkv, hd, B, seed, pad=0, window=0, softcap=0.0, sink=False, dtype="bfloat16", options=None, spread=2, q_size=1.5,
          k_size=1.0, stride=0, climb=False, exponential=2.0 ** -21):
    dt = DT[dtype]
    g = torch.Generator().manual_seed(seed)
    tables, pages, ctx = make_step(spans, B, seed, pad)
    ctx.options = options or {}
    (kc, ks), (vc, vs) = P.pool(pages, nkv, B, hd, seed + 1, k_size, spread), P.pool(pages, nkv, B, hd, seed + 2, 1.0, spread)
    k, k_scale = gpu_pool(kc, ks)
    v, v_scale = gpu_pool(vc, vs)
    T = ctx.rows
    q = (q_size * torch.randn((T, nh * hd + stride), generator=g)).to(dt)
    s = torch.randn((nh,), generator=g) if sink else None
    out = torch.full((T, nh * hd + stride), 7.0, dtype=dt, device=DEV)
    scale = hd ** -0.5
    K().paged_attention_q8(q.to(DEV)[:, :nh * hd], out[:, :nh * hd], k, v, k_scale, v_scale, tables.to(DEV), ctx, nh, nkv, hd, scale, window, softcap,
                           s.to(DEV) if sink else None)
    got = out.cpu().double()
    assert bool((got[:, nh * hd:] == 7.0).all())
    got = got[:, :nh * hd].view(T, nh, hd)
    row = 0
    for i, (start, n) in enumerate(spans):
        end = start + n
        kk, vv = P.gathered(kc, ks, tables[i], end), P.gathered(vc, vs, tables[i], end)
        want, room = P.attend(kind, q[row:row + n, :nh * hd].double().view(n, nh, hd), kk, vv, torch.arange(start, end), scale, window, softcap, s,
                              exponential=exponential)
        far = (got[row:row + n] - want).abs()
        assert bool((far <= room).all()), (i, float((far / room).max()))
        row += n
    assert bool((got[row:] == 0).all())
    K().check_errors()


SINGLES = [[(0, 1)], [(147, 1)], [(0, 1), (1, 1), (15, 1), (16, 1), (127, 1), (128, 1), (500, 1)], [(2000, 1), (3, 1), (1999, 1)]]


@pytest.mark.parametrize("spans", SINGLES)
@pytest.mark.parametrize("nh,nkv,hd,B", [(8, 1, 64, 16), (8, 2, 128, 16), (4, 4, 128, 8), (12, 1, 64, 32), (6, 2, 96, 7), (2, 1, 256, 16), (4, 2, 32, 64),
                                         (4, 2, 160, 5), (3, 1, 40, 16)])
def test_single_rows(spans, nh, nkv, hd, B):
    check("single" if hd % 32 == 0 else "plain bfloat16", spans, nh, nkv, hd, B, 11, pad=2)


@pytest.mark.parametrize("masks", [dict(window=100), dict(window=1), dict(softcap=20.0), dict(sink=True), dict(window=333, softcap=5.0, sink=True)])
@pytest.mark.parametrize("hd,B", [(64, 16), (128, 8), (96, 9)])
def test_single_rows_with_masks(masks, hd, B):
    check("single", [(700, 1), (50, 1), (0, 1), (99, 1), (100, 1)], 8, 2, hd, B, 12, pad=1, **masks)


@pytest.mark.parametrize("options", [dict(attn_parts=1), dict(attn_parts=3), dict(attn_parts=8), dict(attn_parts=13), dict(attn_parts=-1),
                                     dict(attn_parts=5, attn_merge="kernel")])
def test_single_rows_in_parts(options):
    check("single", [(4000, 1), (5, 1), (1700, 1), (128, 1)], 8, 2, 128, 16, 13, pad=1, options=options)


def test_single_rows_of_long_and_many_requests():
    check("single", [(20000, 1)], 4, 1, 64, 16, 14)
    check("single", [(int(37 * i) % 900, 1) for i in range(70)], 4, 2, 64, 16, 15, pad=3)


@pytest.mark.parametrize("spread,q_size,k_size", [(30, 1.5, 1.0), (0, 100.0, 1.0), (0, 1e-3, 1.0), (12, 1.5, 30.0), (0, 1e30, 1e-30)])
def test_single_rows_of_other_sizes(spread, q_size, k_size):
    check("single", [(900, 1), (40, 1)], 8, 2, 128, 16, 16, spread=spread, q_size=q_size, k_size=k_size)


PORTIONS = [[(0, 2)], [(0, 148)], [(0, 300)], [(130, 257), (5, 64)], [(1000, 17), (0, 128), (127, 129)], [(64, 512)]]


@pytest.mark.parametrize("spans", PORTIONS)
@pytest.mark.parametrize("nh,nkv,hd,B", [(4, 1, 64, 16), (4, 2, 128, 16), (2, 2, 128, 8), (2, 1, 64, 64), (4, 2, 128, 24)])
def test_portions(spans, nh, nkv, hd, B):
    check("portion", spans, nh, nkv, hd, B, 21)


@pytest.mark.parametrize("nh,nkv,hd,B", [(4, 2, 96, 16), (2, 1, 256, 16), (4, 2, 32, 8), (4, 2, 128, 7), (4, 2, 64, 20)])
def test_portions_through_laid_out_pages(nh, nkv, hd, B):
    check("laid out", [(0, 148), (130, 70)], nh, nkv, hd, B, 22)


@pytest.mark.parametrize("masks", [dict(window=100), dict(window=1), dict(window=300), dict(softcap=20.0), dict(sink=True), dict(window=77, softcap=5.0, sink=True)])
@pytest.mark.parametrize("hd", [64, 128])
def test_portions_with_masks(masks, hd):
    check("portion", [(700, 200), (0, 300), (3, 40)], 4, 2, hd, 16, 23, **masks)


@pytest.mark.parametrize("spread,q_size,k_size", [(30, 1.5, 1.0), (0, 100.0, 1.0), (0, 1e-3, 1.0), (12, 1.5, 30.0), (0, 1e30, 1e-30)])
def test_portions_of_other_sizes(spread, q_size, k_size):
    check("portion", [(500, 200)], 4, 2, 128, 16, 24, spread=spread, q_size=q_size, k_size=k_size)


def test_single_rows_before_portions_in_rows_of_their_own_stride():
    check("portion", [(300, 1), (0, 1), (20, 200), (0, 65)], 4, 2, 128, 16, 25, stride=24)


@pytest.mark.parametrize("hd,B", [(64, 16), (40, 7)])
def test_plain_rows(hd, B):
    check("plain float32", [(300, 1), (0, 30)], 4, 2, hd, B, 26, dtype="float32")
    check("plain bfloat16", [(300, 1), (0, 30)], 4, 2, hd, B, 27, options=dict(attention="plain"), window=50, softcap=9.0, sink=True)


@pytest.mark.parametrize("single", [True, False])
def test_pages_of_zeros_and_of_large_values_in_one_request(single):
    """A page whose values are all zero has the smallest scale, one of 1e6 a large one: sums must not lose the zeros' probabilities."""
    nh, nkv, hd, B, end = 2, 1, 128, 16, 320
    g = torch.Generator().manual_seed(3)
    n = 1 if single else 40
    tables, pages, ctx = make_step([(end - n, n)], B, 3)
    kx, vx = torch.randn((pages, nkv, B, hd), generator=g), torch.randn((pages, nkv, B, hd), generator=g)
    vx[::2] = 0.0
    vx[1::4] *= 1e6
    kx[5] = 0.0
    ks, vs = P.scale_for(kx.abs().amax((-1, -2))), P.scale_for(vx.abs().amax((-1, -2)))
    kc, vc = P.coded(kx, ks[..., None, None]), P.coded(vx, vs[..., None, None])
    q = torch.randn((n, nh * hd), generator=g).bfloat16()
    out = torch.empty_like(q, device=DEV)
    k, k_scale = gpu_pool(kc, ks)
    v, v_scale = gpu_pool(vc, vs)
    K().paged_attention_q8(q.to(DEV), out, k, v, k_scale, v_scale, tables.to(DEV), ctx, nh, nkv, hd, hd ** -0.5)
    want, room = P.attend("single" if single else "portion", q.double().view(n, nh, hd), P.gathered(kc, ks, tables[0], end),
                          P.gathered(vc, vs, tables[0], end), torch.arange(end - n, end), hd ** -0.5)
    far = (out.cpu().double().view(n, nh, hd) - want).abs()
    assert bool((far <= room).all()), float((far / room).max())


@pytest.mark.parametrize("single", [True, False])
def test_what_a_row_does_not_see_may_be_anything(single):
    """Not-a-number and infinite keys and values behind a row, behind the context and below the window do not reach it."""
    nh, nkv, hd, B, n = 4, 2, 128, 16, 1 if single else 150
    start, window = 200, 100
    g = torch.Generator().manual_seed(4)
    tables, pages, ctx = make_step([(start, n)], B, 4)
    (kc, ks), (vc, vs) = P.pool(pages, nkv, B, hd, 5), P.pool(pages, nkv, B, hd, 6)
    end = start + n

    def poison(key):
        page = int(tables[0, key // B])
        kc[page, :, key % B, ::3] = 127
        vc[page, :, key % B, ::3] = 255
    hidden = [0, start - window] + [key for key in range(end, tables.shape[1] * B) if int(tables[0, key // B]) >= 0]
    seen_later = [] if single else [start + 70, end - 1]
    for key in hidden + seen_later:
        poison(key)
    q = torch.randn((n, nh * hd), generator=g).bfloat16()
    out = torch.empty_like(q, device=DEV)
    k, k_scale = gpu_pool(kc, ks)
    v, v_scale = gpu_pool(vc, vs)
    K().paged_attention_q8(q.to(DEV), out, k, v, k_scale, v_scale, tables.to(DEV), ctx, nh, nkv, hd, hd ** -0.5, window)
    got = out.cpu().double().view(n, nh, hd)
    want, room = P.attend("single" if single else "portion", q.double().view(n, nh, hd), torch.nan_to_num(P.gathered(kc, ks, tables[0], end)),
                          torch.nan_to_num(P.gathered(vc, vs, tables[0], end)), torch.arange(start, end), hd ** -0.5, window)
    first = n if single else 70                                    # rows before see none of it
    assert bool(((got[:first] - want[:first]).abs() <= room[:first]).all())
    assert bool(torch.isnan(got[first:]).any(-1).all())


def test_no_key_lost():
    """The bounds are narrow enough that eight keys that get lost would leave them."""
    nh, nkv, hd, B, end = 4, 1, 128, 16, 600
    g = torch.Generator().manual_seed(9)
    (kc, ks), (vc, vs) = P.pool(40, nkv, B, hd, 5), P.pool(40, nkv, B, hd, 6)
    q, table = torch.randn((1, nh, hd), generator=g).double(), torch.arange(40)
    k, v = P.gathered(kc, ks, table, end), P.gathered(vc, vs, table, end)
    want, room = P.attend("portion", q, k, v, torch.tensor([end - 1]), hd ** -0.5)
    off, _ = P.attend("portion", q, k, v, torch.tensor([end - 1]), hd ** -0.5, lost=(128, 136))
    assert bool(((off - want).abs() > room).any())
