"""What the calls around the cache in 4 bits and the step's tables refuse, on the CPU: every check comes before the device is touched,
and a call without a fault is refused because its tensors are not on a CUDA device."""
import types

import pytest
import torch

from kvcm.kernels import library as K

NH, NKV, HD, B, T, PAGES = 4, 2, 64, 16, 5, 3


def pools(pages=PAGES, nkv=NKV, hd=HD, block=B, dtype=torch.uint8):
    shape = (pages, nkv, K.q4_page_bytes(block, hd))
    return torch.zeros(shape, dtype=dtype), torch.zeros(shape, dtype=dtype)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def store(**c):
    k, v = c.pop("pools", None) or pools()
    dt = c.pop("dtype", torch.bfloat16)
    a = dict(qkv=torch.zeros((T, (NH + 2 * NKV) * HD), dtype=dt), table=torch.zeros(T, HD), interleaved=False, slot_mapping=i32(T), k_cache=k,
             v_cache=v, q_out=torch.zeros((T, NH * HD), dtype=dt), nh=NH, nkv=NKV, hd=HD, block_size=B)
    a.update(c)
    K.rope_cache_q4(**a)


def read(**c):
    k, v = c.pop("pools", None) or pools()
    a = dict(k_cache=k, v_cache=v, slot_mapping=i32(T), k_rows=torch.zeros(T, NKV * HD), v_rows=torch.zeros(T, NKV * HD), nkv=NKV, hd=HD,
             block_size=B)
    a.update(c)
    K.read_cache_q4(**a)


def attend(**c):
    k, v = c.pop("pools", None) or pools()
    dt = c.pop("dtype", torch.bfloat16)
    ctx = types.SimpleNamespace(rows=T, decode_seqs=T, prefill_tiles=0, tile_rows=64, max_decode_ctx=40, max_ctx=40, options={}, row_seq=i32(T),
                                positions=i32(T), seq_q_start=i32(T), seq_q_len=i32(T), seq_ctx_len=i32(T), tile_seq=i32(0), tile_q0=i32(0))
    a = dict(q=torch.zeros((T, NH * HD), dtype=dt), out=torch.zeros((T, NH * HD), dtype=dt), k_cache=k, v_cache=v, block_tables=i32(T, 4),
             ctx=ctx, nh=NH, nkv=NKV, hd=HD, block_size=B, scale=0.125)
    a.update(c)
    K.paged_attention_q4(**a)


def tables(**c):
    S = c.pop("S", 3)
    a = dict(seq_start=i32(S), seq_q_len=i32(S), block_tables=i32(S, 4), free_pages=i32(9), free_count=i32(1), block_size=B, seq_q_start=i32(S),
             seq_ctx_len=i32(S), positions=i32(T), row_seq=i32(T), slot_mapping=i32(T), free_left=i32(1), status=i32(4), tile_seq=i32(2),
             tile_q0=i32(2))
    a.update(c)
    K.step_tables(**a)


def refused(call, match, **c):
    with pytest.raises(K.KernelError, match=match):
        call(**c)


@pytest.mark.parametrize("call", [store, read, attend, tables])
def test_calls_without_a_fault_want_a_device(call):
    refused(call, "not on a CUDA device")


@pytest.mark.parametrize("call", [store, read, attend])
@pytest.mark.parametrize("change,match", [
    (dict(hd=60), "multiples of 8"), (dict(hd=264), "multiples of 8"), (dict(block_size=0), "block_size"), (dict(block_size=8), "caches must be"),
    (dict(pools=pools(dtype=torch.int8)), "caches must be"), (dict(pools=(pools()[0][..., ::2], pools()[1])), "caches must be"),
    (dict(pools=(pools(4)[0], pools(3)[1])), "number of pages"), (dict(pools=(pools()[0], pools(nkv=1)[1])), "caches must be")])
def test_pools(call, change, match):
    refused(call, match, **change)


@pytest.mark.parametrize("change,match", [
    (dict(dtype=torch.float16), "float32 and bfloat16"), (dict(qkv=torch.zeros((T, 7 * HD), dtype=torch.bfloat16)), "qkv"),
    (dict(qkv=torch.zeros((T, 8 * HD + 1), dtype=torch.bfloat16)), "16-byte"), (dict(q_out=torch.zeros((T, NH * HD))), "q_out"),
    (dict(q_out=torch.zeros((T, 2 * NH * HD), dtype=torch.bfloat16)[:, ::2]), "q_out"), (dict(slot_mapping=i32(T - 1)), "slot_mapping"),
    (dict(slot_mapping=torch.zeros(T, dtype=torch.int64)), "slot_mapping"), (dict(table=torch.zeros(T, 24)), "rotary_dim"),
    (dict(table=torch.zeros(T, HD + 16)), "rotary_dim"), (dict(table=torch.zeros(T, 3), interleaved=True), "rotary_dim"),
    (dict(table=torch.zeros(T - 1, HD)), "table"), (dict(table=torch.zeros(T, HD, dtype=torch.bfloat16)), "table")])
def test_rows_that_cannot_be_written(change, match):
    refused(store, match, **change)


@pytest.mark.parametrize("change,match", [
    (dict(k_rows=torch.zeros(T, NKV * HD, dtype=torch.float16)), "float32 and bfloat16"), (dict(v_rows=torch.zeros(T, NKV * HD - 8)), "v_rows"),
    (dict(v_rows=torch.zeros((T, NKV * HD), dtype=torch.bfloat16)), "v_rows"), (dict(slot_mapping=i32(2)), "slot_mapping")])
def test_rows_that_cannot_be_read(change, match):
    refused(read, match, **change)


@pytest.mark.parametrize("change,match", [
    (dict(nh=3), "multiple"), (dict(dtype=torch.float16), "bfloat16 or float32"), (dict(out=torch.zeros(T, NH * HD)), "q and out"),
    (dict(out=torch.zeros((T - 1, NH * HD), dtype=torch.bfloat16)), "q and out"), (dict(window=-1), "negative"), (dict(softcap=-2.0), "negative"),
    (dict(sink=torch.zeros(NH - 1)), "sink"), (dict(sink=torch.zeros(NH, dtype=torch.bfloat16)), "sink"), (dict(block_tables=i32(T * 4)), "block_tables"),
    (dict(block_tables=torch.zeros((T, 4), dtype=torch.int64)), "block_tables"), (dict(block_tables=i32(T, 0)), "block_tables")])
def test_attention_that_cannot_be(change, match):
    refused(attend, match, **change)


@pytest.mark.parametrize("change,match", [
    (dict(S=8193), "8192"), (dict(seq_start=i32(2)), "per-request"), (dict(block_tables=i32(2, 4)), "block_tables"), (dict(row_seq=i32(T + 1)), "per-row"),
    (dict(tile_q0=None), "go together"), (dict(tile_q0=i32(3)), "go together"), (dict(free_count=i32(2)), "free_count"), (dict(status=i32(3)), "status"),
    (dict(block_size=0), "positive"), (dict(tile_rows=0), "positive"), (dict(positions=torch.zeros(T)), "int32"),
    (dict(seq_q_len=torch.zeros(3, dtype=torch.int64)), "int32"), (dict(block_tables=i32(4, 3).t()), "int32")])
def test_tables_that_cannot_be(change, match):
    refused(tables, match, **change)


def test_the_status_of_a_refused_step_is_an_error():
    K.raise_on_step_tables([0, 0, 5, 1])
    for code in K.STEP_TABLE_ERRORS:
        with pytest.raises(K.KernelError, match="step_tables.* 17"):
            K.raise_on_step_tables(torch.tensor([code, 17, 0, 0]))
