"""Capped scores, s <- cap tanh(scale q.k / cap), with a scale of any sign, on the GPU: every path of attention over pages and over prompts' own
rows.  A negative scale is the positive one of -q, which is how the bounds of plain_q8.py take it; a scale of zero gives every key the same
weight, and so does one so small that its quotient with the cap leaves float32."""
import pytest
import torch

import plain_q8 as P
from test_gpu_prompt_attention import make_ctx
from test_gpu_q4 import make_step
from test_gpu_q8 import DEV, K, gpu_pool

pytestmark = pytest.mark.gpu
SCALES = [-0.09, 0.0, 1e-44, 0.09]


def bounded(kind, got, q, k, v, at, scale, softcap, sink=None):
    want, room = P.attend(kind, -q if scale < 0 else q, k, v, at, abs(scale), 0, softcap, sink)
    far = (got - want).abs()
    assert bool((far <= room).all()), float((far - room).max())


@pytest.mark.parametrize("softcap", [0.0, 7.0])
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("kind,spans,hd,options", [
    ("single", [(300, 1), (0, 1)], 128, {}), ("single", [(2000, 1)], 64, dict(attn_parts=-1)),
    ("portion", [(130, 150)], 128, {}), ("portion", [(0, 300)], 64, {}),
    ("laid out", [(130, 150)], 128, dict(attn_prefill="unpack")), ("laid out", [(20, 70)], 96, {}),
    ("plain bfloat16", [(130, 20)], 40, {})])
def test_pages_in_8_bits(kind, spans, hd, options, scale, softcap):
    nh, nkv, B = 4, 2, 16
    g = torch.Generator().manual_seed(5)
    tables, pages, ctx = make_step(spans, B, 5)
    ctx.options = options
    (kc, ks), (vc, vs) = P.pool(pages, nkv, B, hd, 6, spread=2), P.pool(pages, nkv, B, hd, 7, spread=2)
    k, k_scale = gpu_pool(kc, ks)
    v, v_scale = gpu_pool(vc, vs)
    q = (1.5 * torch.randn((ctx.rows, nh * hd), generator=g)).bfloat16()
    out = torch.full((ctx.rows, nh * hd), 7.0, dtype=torch.bfloat16, device=DEV)
    K().paged_attention_q8(q.to(DEV), out, k, v, k_scale, v_scale, tables.to(DEV), ctx, nh, nkv, hd, scale, 0, softcap)
    K().check_errors()
    row = 0
    for i, (start, n) in enumerate(spans):
        end = start + n
        bounded(kind, out[row:row + n].cpu().double().view(n, nh, hd), q[row:row + n].double().view(n, nh, hd), P.gathered(kc, ks, tables[i], end),
                P.gathered(vc, vs, tables[i], end), torch.arange(start, end), scale, softcap)
        row += n


@pytest.mark.parametrize("softcap", [0.0, 7.0])
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("hd,options", [(64, {}), (128, {}), (128, dict(attention="plain"))])
def test_prompts(hd, options, scale, softcap):
    nh, nkv, lengths = 4, 2, [1, 300, 40]
    g = torch.Generator().manual_seed(8)
    ctx, starts, T = make_ctx(lengths)
    ctx.options = options
    x = torch.randn((T, (nh + 2 * nkv) * hd), generator=g).bfloat16()
    q, k, v = x.to(DEV).split([nh * hd, nkv * hd, nkv * hd], 1)
    sink = torch.randn((nh,), generator=g)
    out = torch.empty((T, nh * hd), dtype=torch.bfloat16, device=DEV)
    K().prompt_attention(q, k, v, out, ctx, nh, nkv, hd, scale, 0, softcap, sink.to(DEV))
    K().check_errors()
    for a, n in zip(starts, lengths):
        rows = x[a:a + n].double().view(n, nh + 2 * nkv, hd)
        bounded("plain bfloat16" if options else "prompt", out[a:a + n].cpu().double().view(n, nh, hd), rows[:, :nh], rows[:, nh:nh + nkv].transpose(0, 1),
                rows[:, nh + nkv:].transpose(0, 1), torch.arange(n), scale, softcap, sink)


@pytest.mark.parametrize("softcap", [0.0, 7.0])
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("start,n,options", [(300, 1, {}), (70, 150, {}), (70, 150, dict(attn_prefill="tcgen05")), (70, 150, dict(attn_prefill="mma"))])
def test_pages_in_bfloat16(start, n, options, scale, softcap):
    nh, nkv, hd, B, end = 4, 2, 128, 16, start + n
    g = torch.Generator().manual_seed(9)
    tables, pages, ctx = make_step([(start, n)], B, 9)
    ctx.options = options
    kv = torch.randn((2, pages, nkv, B, hd), generator=g).bfloat16()
    q = torch.randn((n, nh * hd), generator=g).bfloat16()
    out = torch.empty((n, nh * hd), dtype=torch.bfloat16, device=DEV)
    cache = kv.to(DEV)
    if options.get("attn_prefill") == "tcgen05" and scale < 0 and not softcap:      # refused where it is asked for by name
        with pytest.raises(K().KernelError):
            K().paged_attention(q.to(DEV), out, cache[0], cache[1], tables.to(DEV), ctx, nh, nkv, hd, scale)
        return
    K().paged_attention(q.to(DEV), out, cache[0], cache[1], tables.to(DEV), ctx, nh, nkv, hd, scale, 0, softcap)
    K().check_errors()
    rows = [x[tables[0, :-(-end // B)].long()].double().transpose(0, 1).flatten(1, 2)[:, :end] for x in kv]
    bounded("laid out", out.cpu().double().view(n, nh, hd), q.double().view(n, nh, hd), *rows, torch.arange(start, end), scale, softcap)
