"""The bounds of bounds_q4.py on the CPU: they hold around the definition, and no 128 keys can be missing without leaving them."""
import pytest
import torch

import bounds_q4 as bounds
import plain_q4 as P


def test_pages_are_those_of_the_rows_one_by_one():
    x = torch.randn((3, 2, 7, 40), generator=torch.Generator().manual_seed(1))
    cache = torch.zeros((3, 2, P.page_bytes(7, 40)), dtype=torch.uint8)
    for p in range(3):
        for o in range(7):
            P.write(cache, 7, p, o, x[p, :, o])
    assert torch.equal(bounds.cache_of(x), cache)
    code, scale, zero = bounds.parts(cache, 40, 7)
    assert torch.equal(zero + scale * code, P.read(cache, 40, 7)) and code.min() >= 0 and code.max() <= 15


def test_the_result_is_that_of_the_plain_form():
    spans, nh, nkv, hd, B = [(40, 1), (7, 20)], 4, 2, 32, 16
    q, kc, vc, tables = bounds.inputs(spans, nh, nkv, hd, B, torch.bfloat16)
    q = q.double().view(-1, nh, hd)
    for window in (0, 9):
        want, room = bounds.attention("plain float32", q, kc, vc, tables, spans, nh, nkv, hd, B, 0.2, window)
        plain = P.attention(q, P.read(kc, hd, B), P.read(vc, hd, B), tables, spans, nh, nkv, B, 0.2, window)
        bounds.check(plain, want, room)
        assert (plain - want).abs().max() < 1e-12


@pytest.mark.parametrize("kind,spans,nh,nkv,hd,B,options", bounds.CASES, ids=str)
def test_a_lost_piece_leaves_the_bounds(kind, spans, nh, nkv, hd, B, options):
    q, kc, vc, tables = bounds.inputs(spans, nh, nkv, hd, B, torch.float32 if kind == "plain float32" else torch.bfloat16)
    q = q.double().view(-1, nh, hd)
    row = 0
    for i, (start, n) in enumerate(spans):
        args = kind, q[row:row + n], kc, vc, tables[i:i + 1], [(start, n)], nh, nkv, hd, B, hd ** -0.5
        want, room = bounds.attention(*args)
        pieces = range(0, start + n, 128)
        for first in pieces if len(pieces) < 20 else list(pieces)[::len(pieces) // 8]:
            if start + n <= 128:
                continue                                            # nothing would be left
            lost, _ = bounds.attention(*args, lost=(first, min(first + 128, start + n)))
            sees = torch.arange(start, start + n) >= first + 20     # rows that see enough of it
            off = ((lost - want).abs() / room).amax(-1)             # of every row and head
            assert (off[sees] > 1).all(), (i, first, off[sees].min().item())
        row += n
