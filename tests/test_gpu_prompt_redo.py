"""Rows of a very long prompt that are attended once more, because a value that they do not see is not a number: that takes longer than the
kernel's waits for one another allow for, and is no reason to give up."""
import pytest
import torch

import plain_q8 as P
from test_gpu_prompt_attention import DEV, K, make_ctx

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,hd", [(5003, 128), (450_003, 64)])
def test_rows_before_a_value_that_is_not_a_number(n, hd):
    g = torch.Generator().manual_seed(n)
    ctx, starts, rows = make_ctx([n, 700])
    x = torch.randn((rows, 3 * hd), generator=g).bfloat16()
    x[n - 1, 2 * hd:] = float("nan")                                # the last row's value
    dev = x.to(DEV)
    out = torch.full((rows, hd), 7.0, dtype=torch.bfloat16, device=DEV)
    K().prompt_attention(dev[:, :hd], dev[:, hd:2 * hd], dev[:, 2 * hd:], out, ctx, 1, 1, hd, hd ** -0.5)
    torch.cuda.synchronize()
    K().check_errors()
    got = out.cpu().double()
    assert bool(torch.isnan(got[n - 1]).all()) and bool(torch.isfinite(got[:n - 1]).all()) and bool(torch.isfinite(got[n:]).all())
    for a, end, first in ((0, n, n - 41), (0, n, 0), (n, 700, 500)):      # the last rows of the prompt, its first, another prompt's
        at = torch.arange(first, min(first + 40, end - 1))
        keys = int(at[-1]) + 1
        q, k, v = (x[a:a + keys, i * hd:(i + 1) * hd].double() for i in range(3))
        want, room = P.attend("prompt", q[first:, None], k[None], v[None], at, hd ** -0.5)
        assert bool(((got[a + first:a + first + len(at)] - want[:, 0]).abs() <= room[:, 0]).all())
