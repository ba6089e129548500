"""Numbers beyond 32 bits in the calls around the cache in 4 bits, on the CPU: refused or bounded before they reach a kernel."""
import types

import pytest
import torch

from kvcm.kernels import library as K
from test_q4_refusals import B, HD, NH, NKV, T, attend, i32, pools, refused


@pytest.mark.parametrize("window", [2 ** 31, 2 ** 32 + 5, 2 ** 40])
@pytest.mark.parametrize("plain", [False, True])
def test_windows_beyond_32_bits(window, plain):
    refused(attend, "32 bits", window=window, **({"dtype": torch.float32} if plain else {}))


@pytest.mark.parametrize("longest", [64, 65, 2 ** 31 + 128, 2 ** 32 + 128, 2 ** 40 + 128])
@pytest.mark.parametrize("parts", [0, 1, 3, -1])
@pytest.mark.parametrize("window", [0, 40, 2 ** 31 - 1])
def test_partitions_cover_a_table_whatever_the_longest_context_is_said_to_be(monkeypatch, longest, parts, window):
    """Tables of four pages of 16 keys: the partitions that a call asks for cover them in 32 bits."""
    calls = []
    monkeypatch.setattr(K, "_DECODE_Q4", lambda device, *args: calls.append(args) or 0)
    monkeypatch.setattr(K, "_one_device", lambda *a: 0)
    monkeypatch.setattr(K, "_q4_resident_blocks", lambda *a: 592)
    k, v = pools()
    ctx = types.SimpleNamespace(max_decode_ctx=longest, seq_ctx_len=i32(T), options={"attn_parts": parts})
    q = torch.zeros((T, NH * HD), dtype=torch.bfloat16)
    K.attention_decode_q4(q, torch.zeros_like(q), k, v, i32(T, 4), ctx, NH, NKV, HD, B, 0.125, window)
    size, count = calls[0][17:19]
    assert 0 < size < 2 ** 31 and 0 <= count < 2 ** 31
    assert count == 0 or size * count >= min(64, window + 31 if window else 64)
