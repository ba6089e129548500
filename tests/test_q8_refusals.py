"""What the calls around the cache in 8 bits, prompts and shared pages refuse, on the CPU: every check comes before the device is touched,
and a call without a fault is refused because its tensors are not on a CUDA device."""
import types

import pytest
import torch

from kvcm.kernels import library as K

NH, NKV, HD, B, T, PAGES = 4, 2, 64, 16, 5, 3
FP8 = torch.float8_e4m3fn


def pools(pages=PAGES, nkv=NKV, hd=HD, block=B, dtype=FP8):
    z = lambda: torch.zeros((pages, nkv, block, hd), dtype=torch.uint8).view(dtype) if dtype == FP8 else torch.zeros((pages, nkv, block, hd), dtype=dtype)
    return dict(k_cache=z(), v_cache=z(), k_scale=torch.zeros(pages, nkv), v_scale=torch.zeros(pages, nkv))


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def context(**c):
    ctx = types.SimpleNamespace(rows=T, decode_seqs=T, prefill_tiles=0, tile_rows=64, max_decode_ctx=40, max_ctx=40, options={}, row_seq=i32(T),
                                positions=i32(T), seq_q_start=i32(T), seq_q_len=i32(T), seq_ctx_len=i32(T), tile_seq=i32(0), tile_q0=i32(0))
    for name, v in c.items():
        setattr(ctx, name, v)
    return ctx


def store(**c):
    dt = c.pop("dtype", torch.bfloat16)
    a = dict(qkv=torch.zeros((T, (NH + 2 * NKV) * HD), dtype=dt), table=torch.zeros(T, HD), interleaved=False, slot_mapping=i32(T),
             q_out=torch.zeros((T, NH * HD), dtype=dt), nh=NH, nkv=NKV, hd=HD, **pools())
    a.update(c)
    K.rope_cache_q8(**a)


def read(**c):
    a = dict(slot_mapping=i32(T), k_rows=torch.zeros(T, NKV * HD), v_rows=torch.zeros(T, NKV * HD), **pools())
    a.update(c)
    K.read_cache_q8(**a)


def attend(**c):
    dt = c.pop("dtype", torch.bfloat16)
    ctx = context(**c.pop("step", {}))
    a = dict(q=torch.zeros((T, NH * HD), dtype=dt), out=torch.zeros((T, NH * HD), dtype=dt), block_tables=i32(T, 4), ctx=ctx, nh=NH, nkv=NKV, hd=HD,
             scale=0.125, **pools())
    a.update(c)
    K.paged_attention_q8(**a)


def portions(**c):
    attend(**{"step": dict(decode_seqs=0, prefill_tiles=1, tile_seq=i32(1), tile_q0=i32(1)), **c})


def prompt(**c):
    dt = c.pop("dtype", torch.bfloat16)
    ctx = context(**{**dict(decode_seqs=0, prefill_tiles=1, tile_seq=i32(1), tile_q0=i32(1)), **c.pop("step", {})})
    a = dict(q=torch.zeros((T, NH * HD), dtype=dt), k=torch.zeros((T, NKV * HD), dtype=dt), v=torch.zeros((T, NKV * HD), dtype=dt),
             out=torch.zeros((T, NH * HD), dtype=dt), ctx=ctx, nh=NH, nkv=NKV, hd=HD, scale=0.125)
    a.update(c)
    K.prompt_attention(**a)


def state(S=3, N=9):
    return dict(seq_len=i32(S), block_tables=i32(S, 4), shared=i32(N), free_pages=i32(N), free_count=i32(1), block_size=B, status=i32(4))


def fork(**c):
    a = dict(parents=i32(2), children=i32(2), pools=[torch.zeros(2, 9, 7)], seq_len_out=i32(3), shared_out=i32(9), free_left=i32(1), **state())
    a.update(c)
    K.fork_requests(**a)


def release(**c):
    a = dict(requests=i32(2), seq_len_out=i32(3), shared_out=i32(9), free_left=i32(1), **state())
    a.update(c)
    K.release_requests(**a)


def compact(**c):
    a = dict(pools=[torch.zeros(2, 9, 7)], tables_out=i32(3, 4), shared_out=i32(9), free_out=i32(9), page_map=i32(9), **state())
    a.update(c)
    K.compact_pages(**a)


def copy(**c):
    a = dict(pools=[torch.zeros(2, 9, 7)], src=i32(2), dst=i32(2))
    a.update(c)
    K.copy_pages(**a)


@pytest.mark.parametrize("call", [store, read, attend, portions, prompt, fork, release, compact, copy])
def test_tensors_not_on_a_gpu(call):
    with pytest.raises(K.KernelError, match="not on a CUDA device"):
        call()


OTHER = pools(nkv=1)
REFUSALS = [
    (store, "float8", dict(k_cache=torch.zeros((PAGES, NKV, B, HD), dtype=torch.uint8))),
    (store, "caches must be", dict(k_cache=OTHER["k_cache"])),
    (store, "caches must be", dict(v_cache=pools(block=8)["v_cache"])),
    (store, "caches must be", dict(k_cache=pools(pages=6)["k_cache"][::2])),
    (store, "scales must be", dict(k_scale=torch.zeros(PAGES, NKV, dtype=torch.bfloat16))),
    (store, "scales must be", dict(v_scale=torch.zeros(PAGES))),
    (store, "head sizes", dict(hd=60)),
    (store, "head sizes", dict(hd=264)),
    (store, "storage", dict(dtype=torch.float16)),
    (store, "qkv must be", dict(qkv=torch.zeros((T, 100), dtype=torch.bfloat16))),
    (store, "16-byte", dict(qkv=torch.zeros((T, (NH + 2 * NKV) * HD + 1), dtype=torch.bfloat16)[:, 1:])),
    (store, "q_out must be", dict(q_out=torch.zeros((T - 1, NH * HD), dtype=torch.bfloat16))),
    (store, "slot_mapping", dict(slot_mapping=torch.zeros(T, dtype=torch.int64))),
    (store, "slot_mapping", dict(slot_mapping=i32(T - 1))),
    (store, "table float32", dict(table=torch.zeros(T - 1, HD))),
    (store, "rotary_dim", dict(table=torch.zeros(T, 24))),
    (store, "rotary_dim", dict(table=torch.zeros(T, 2 * HD))),
    (read, "k_rows must be", dict(k_rows=torch.zeros(T, HD))),
    (read, "v_rows must be", dict(v_rows=torch.zeros(T, NKV * HD, dtype=torch.bfloat16))),
    (read, "slot_mapping", dict(slot_mapping=i32(2))),
    (read, "caches must be", dict(k_cache=torch.zeros(4, 4))),
    (attend, "not a multiple", dict(nh=3)),
    (attend, "not be negative", dict(window=-1)),
    (attend, "not be negative", dict(softcap=-1.0)),
    (attend, "32 bits", dict(window=1 << 31)),
    (attend, "one type", dict(out=torch.zeros((T, NH * HD)))),
    (attend, "rows of", dict(q=torch.zeros((T, NH * HD - 8), dtype=torch.bfloat16))),
    (attend, "dense", dict(q=torch.zeros((T, 2 * NH * HD), dtype=torch.bfloat16)[:, ::2])),
    (attend, "block_tables", dict(block_tables=i32(T, 0))),
    (attend, "block_tables", dict(block_tables=torch.zeros((T, 4)))),
    (attend, "sink", dict(sink=torch.zeros(NH - 1))),
    (attend, "scales must be", dict(k_scale=torch.zeros(PAGES, NKV + 1))),
    (prompt, "k must be", dict(k=torch.zeros((T - 1, NKV * HD), dtype=torch.bfloat16))),
    (prompt, "v must be", dict(v=torch.zeros((T, NKV * HD)))),
    (prompt, "k must be", dict(k=torch.zeros((T, 8), dtype=torch.bfloat16))),
    (prompt, "64 query rows", dict(step=dict(tile_rows=32))),
    (prompt, "tile_seq", dict(step=dict(prefill_tiles=3))),
    (prompt, "prompts of one row", dict(step=dict(decode_seqs=T + 1))),
    (prompt, "not a multiple", dict(nkv=3)),
    (prompt, "32 bits", dict(window=1 << 40)),
    (prompt, "sink", dict(sink=torch.zeros(NH, dtype=torch.bfloat16))),
    (fork, "int32", dict(parents=torch.zeros(2, dtype=torch.int64))),
    (fork, "as many children", dict(children=i32(3))),
    (fork, "8192 parents", dict(parents=i32(8193), children=i32(8193))),
    (fork, "block_tables", dict(block_tables=i32(2, 4))),
    (fork, "block_size", dict(block_size=0)),
    (fork, "fit 32 bits", dict(block_size=1 << 30)),
    (fork, "status", dict(status=i32(3))),
    (fork, "seq_len_out", dict(shared_out=i32(8))),
    (fork, "pools must be", dict(pools=[torch.zeros(2, 8, 7)])),
    (fork, "pools must be", dict(pools=[torch.zeros(9, 7)])),
    (fork, "pools must be", dict(pools=[torch.zeros(2, 9, 14)[:, :, ::2]])),
    (fork, "64 pools", dict(pools=[torch.zeros(1, 9, 1)] * 65)),
    (release, "8192 requests", dict(requests=i32(8193))),
    (release, "free_left", dict(free_left=i32(2))),
    (compact, "page_map", dict(page_map=i32(8))),
    (compact, "tables_out", dict(tables_out=i32(3, 5))),
    (compact, "int32", dict(page_map=torch.zeros(9))),
    (copy, "as many targets", dict(dst=i32(3))),
    (copy, "at least one", dict(pools=[])),
    (copy, "src", dict(src=torch.zeros(2, dtype=torch.int64)))]


@pytest.mark.parametrize("call,match,change", REFUSALS)
def test_refusals(call, match, change):
    with pytest.raises(K.KernelError, match=match):
        call(**change)
