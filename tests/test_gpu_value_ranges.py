"""Values near the ends of their types' range, on the GPU: finite values whose definition is finite stay finite and exact."""
import pytest
import torch

from test_gpu_prompt_attention import check as check_prompts

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
