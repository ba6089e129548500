"""Values near the ends of their types' range, on the GPU: finite values whose definition is finite stay finite and exact."""
import pytest
import torch

import plain_q8 as P
from test_gpu_prompt_attention import check as check_prompts
from test_gpu_q4 import make_step
from test_gpu_q8 import DEV, K, gpu_pool

pytestmark = pytest.mark.gpu


def near(wants):
    for a, n, got, want, room in wants:
        far = (got - want).abs()
        assert bool((far <= room).all()), (a, float((far - room).max()), float(want.abs().max()))


@pytest.mark.parametrize("exponent", [60, 100, 118, 125])
@pytest.mark.parametrize("level", [0.0, 13.0])
@pytest.mark.parametrize("hd,masks", [(64, dict()), (128, dict()), (128, dict(window=100)), (128, dict(softcap=30.0, sink=True))])
def test_prompts_of_large_values(hd, masks, level, exponent):
    """Scores up to e^13, near which weights are largest before a row's reference is renewed, times values up to 2^127."""
    nh, nkv = 4, 2

    def shape(qkv, starts):
        qkv[:, :nh * hd:hd] = 8.0
        qkv[:, nh * hd:(nh + nkv) * hd:hd] = level * hd ** 0.5 / 8.0
        v = qkv[:, (nh + nkv) * hd:(nh + 2 * nkv) * hd]
        v.copy_((v.float().clamp(-3.9, 3.9) * 2.0 ** exponent).to(v.dtype))
    near(check_prompts([1, 40, 700], nh, nkv, hd, q_size=0.3, poison=shape, behind=0, **masks))


def test_large_values_beside_infinite_ones():
    """A value that is infinite reaches its own column of the rows that see it; large ones beside it stay finite."""
    nh, nkv, hd, at = 2, 1, 64, 500

    def shape(qkv, starts):
        qkv[:, :nh * hd:hd] = 8.0
        qkv[:, nh * hd] = 13.0 * hd ** 0.5 / 8.0
        v = qkv[:, (nh + nkv) * hd:(nh + 2 * nkv) * hd]
        v.copy_((v.float().clamp(-3.9, 3.9) * 2.0 ** 125).to(v.dtype))
        v[starts[0] + at, 5] = float("inf")
    for a, n, got, want, room in check_prompts([700], nh, nkv, hd, q_size=0.3, poison=shape, behind=0):
        keep = torch.ones_like(got, dtype=torch.bool)
        keep[at:, :, 5] = False
        assert bool(((got - want).abs() <= room)[keep].all())
        assert not bool(torch.isfinite(got[~keep]).any())


@pytest.mark.parametrize("single", [True, False])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("first,second", [(-60, 70), (-60, 100), (100, -50), (80, -60), (-10, 90)])
def test_pages_of_values_far_apart(first, second, hd, single):
    """Pages whose scales are more powers of two apart than float32 has: the small pages' probabilities still count."""
    nh, nkv, B, end = 4, 2, 16, 320
    n = 1 if single else 60
    g = torch.Generator().manual_seed(3)
    tables, pages, ctx = make_step([(end - n, n)], B, 3)
    kx, normal = torch.randn((pages, nkv, B, hd), generator=g), torch.randn((pages, nkv, B, hd), generator=g)
    vx = normal * 2.0 ** first
    for j in (3, 4, 11):
        vx[int(tables[0, j])] = normal[int(tables[0, j])] * 2.0 ** second
    ks, vs = P.scale_for(kx.abs().amax((-1, -2))), P.scale_for(vx.abs().amax((-1, -2)))
    kc, vc = P.coded(kx, ks[..., None, None]), P.coded(vx, vs[..., None, None])
    q = torch.randn((n, nh * hd), generator=g).bfloat16()
    out = torch.empty_like(q, device=DEV)
    k, k_scale = gpu_pool(kc, ks)
    v, v_scale = gpu_pool(vc, vs)
    K().paged_attention_q8(q.to(DEV), out, k, v, k_scale, v_scale, tables.to(DEV), ctx, nh, nkv, hd, hd ** -0.5)
    K().check_errors()
    want, room = P.attend("single" if single else "portion", q.double().view(n, nh, hd), P.gathered(kc, ks, tables[0], end),
                          P.gathered(vc, vs, tables[0], end), torch.arange(end - n, end), hd ** -0.5)
    far = (out.cpu().double().view(n, nh, hd) - want).abs()
    assert bool((far <= room).all()), float((far / room).max())


def test_pages_far_apart_that_only_some_rows_see():
    """The groups of 128 rows of a block decide for themselves, alike in every call."""
    nh, nkv, hd, B, start, n = 2, 1, 128, 16, 100, 256
    end = start + n
    g = torch.Generator().manual_seed(6)
    tables, pages, ctx = make_step([(start, n)], B, 6)
    kx, vx = torch.randn((pages, nkv, B, hd), generator=g), torch.randn((pages, nkv, B, hd), generator=g)
    vx[int(tables[0, end // B - 1])] *= 2.0 ** -60                  # seen by the second group alone, and not with the next
    vx[int(tables[0, end // B])] *= 2.0 ** 90
    ks, vs = P.scale_for(kx.abs().amax((-1, -2))), P.scale_for(vx.abs().amax((-1, -2)))
    kc, vc = P.coded(kx, ks[..., None, None]), P.coded(vx, vs[..., None, None])
    q = torch.randn((n, nh * hd), generator=g).bfloat16()
    k, k_scale = gpu_pool(kc, ks)
    v, v_scale = gpu_pool(vc, vs)
    outs = []
    for _ in range(5):
        out = torch.empty_like(q, device=DEV)
        K().paged_attention_q8(q.to(DEV), out, k, v, k_scale, v_scale, tables.to(DEV), ctx, nh, nkv, hd, hd ** -0.5)
        K().check_errors()
        outs.append(out.cpu())
    want, room = P.attend("portion", q.double().view(n, nh, hd), P.gathered(kc, ks, tables[0], end), P.gathered(vc, vs, tables[0], end),
                          torch.arange(start, end), hd ** -0.5)
    far = (outs[0].double().view(n, nh, hd) - want).abs()
    assert bool((far <= room).all()), float((far / room).max())
    assert all(torch.equal(outs[0], out) for out in outs)
