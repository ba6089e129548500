"""The operators as a program uses them: prompts attended over their own rows while their keys and values go into the cache in 8 bits, then steps
that are recorded once and replayed: single rows appended and attended, requests forked in between, ended, their pages given back and the pool
compacted, all lengths and pages on the device."""
import types

import pytest
import torch

import plain_q4
import plain_q8 as P

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NH, NKV, HD, B, S, MB, PAGES = 4, 2, 64, 16, 8, 12, 60
WIDTH = (NH + 2 * NKV) * HD


def K():
    from kvcm.kernels import library
    return library


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Host:
    """The same in loops on the CPU: what every request's keys and values are by now, page by page."""

    def __init__(self):
        z = lambda: (torch.zeros((PAGES, NKV, B, HD), dtype=torch.uint8), torch.zeros((PAGES, NKV)))
        (self.k, self.ks), (self.v, self.vs) = z(), z()
        self.inv = 10000.0 ** (-torch.arange(0, HD, 2).double() / HD)


def test_a_life_of_requests():
    lib = K()
    g = torch.Generator().manual_seed(11)
    host = Host()
    k = torch.zeros((PAGES, NKV, B, HD), dtype=torch.uint8, device=DEV).view(P.FP8)
    v = torch.zeros((PAGES, NKV, B, HD), dtype=torch.uint8, device=DEV).view(P.FP8)
    ks, vs = torch.zeros((PAGES, NKV), device=DEV), torch.zeros((PAGES, NKV), device=DEV)
    pools = [k.view(torch.uint8)[None], v.view(torch.uint8)[None], ks[None], vs[None]]
    inv = host.inv.float().to(DEV)
    length, tables = i32([0] * S), torch.full((S, MB), -1, dtype=torch.int32, device=DEV)
    stack, count, shared = torch.arange(PAGES - 1, -1, -1, dtype=torch.int32, device=DEV), i32([PAGES]), i32([0] * PAGES)
    status = i32([0] * 4)

    def arrays(rows, tiles):
        room = lambda n: torch.empty(n, dtype=torch.int32, device=DEV)
        return dict(seq_q_start=room(S), positions=room(rows), row_seq=room(rows), slot_mapping=room(rows), tile_seq=room(tiles), tile_q0=room(tiles))

    def step(a, n, qkv, out, prompt, decode_seqs, longest):
        """The launches of one step of one layer."""
        rows = a["positions"].numel()
        lib.step_tables(length, n, tables, stack, count, B, seq_ctx_len=length, free_left=count, status=status, **a)
        angles = torch.empty((rows, HD), device=DEV)
        lib.rope_table(a["positions"], inv, angles)
        q = torch.empty((rows, NH * HD), dtype=torch.bfloat16, device=DEV)
        lib.rope_cache_q8(qkv, angles, False, a["slot_mapping"], k, v, ks, vs, q, NH, NKV, HD)
        ctx = types.SimpleNamespace(rows=rows, decode_seqs=decode_seqs, prefill_tiles=a["tile_seq"].numel() if prompt else 0, tile_rows=64,
                                    max_ctx=longest, max_decode_ctx=longest, seq_q_start=a["seq_q_start"], seq_q_len=n, seq_ctx_len=length,
                                    positions=a["positions"], row_seq=a["row_seq"], tile_seq=a["tile_seq"], tile_q0=a["tile_q0"], options={})
        if prompt:
            both = torch.cat((q, qkv[:, NH * HD:]), 1)              # (keys unturned: a layer without positions for the prompt's sake)
            lib.prompt_attention(q, both[:, NH * HD:(NH + NKV) * HD], both[:, (NH + NKV) * HD:], out, ctx, NH, NKV, HD, HD ** -0.5)
        else:
            lib.paged_attention_q8(q, out, k, v, ks, vs, tables, ctx, NH, NKV, HD, HD ** -0.5)
        return q, angles

    def keep(qkv, a, angles):
        """The rows of a step into the host's cache, from the step's own arrays."""
        x = qkv.cpu().float().view(-1, NH + 2 * NKV, HD)
        t = angles.cpu()
        turned = plain_q4.rotated(x[:, :NH + NKV], t[:, :HD // 2], t[:, HD // 2:], False)
        P.write(host.k, host.ks, a["slot_mapping"].cpu(), turned[:, NH:])
        P.write(host.v, host.vs, a["slot_mapping"].cpu(), x[:, NH + NKV:])

    def same_cache():
        for i in range(S):
            n = int(length[i])
            for page in tables[i, :-(-n // B)].tolist():
                assert torch.equal(ks[page].cpu(), host.ks[page]) and torch.equal(vs[page].cpu(), host.vs[page])
            if n:
                for dev, codes, scale in ((k, host.k, host.ks), (v, host.v, host.vs)):
                    got = P.gathered(dev.cpu().view(torch.uint8), scale, tables[i].cpu(), n)
                    assert torch.equal(got, P.gathered(codes, scale, tables[i].cpu(), n))

    # ---- two prompts, of 70 and 33 rows
    prompt = arrays(103, 3)
    n = i32([70, 33] + [0] * (S - 2))
    qkv = torch.randn((103, WIDTH), generator=g).bfloat16().to(DEV)
    out = torch.empty((103, NH * HD), dtype=torch.bfloat16, device=DEV)
    q, angles = step(prompt, n, qkv, out, True, 0, 0)
    keep(qkv, prompt, angles)
    lib.raise_on_step_tables(status.cpu())
    same_cache()
    x = qkv.cpu().double()
    at = 0
    for rows in (70, 33):
        kk, vv = (x[at:at + rows, lo * HD:(lo + NKV) * HD].view(rows, NKV, HD).transpose(0, 1) for lo in (NH, NH + NKV))
        want, room = P.attend("prompt", q[at:at + rows].cpu().double().view(rows, NH, HD), kk, vv, torch.arange(rows), HD ** -0.5)
        assert bool(((out[at:at + rows].cpu().double().view(rows, NH, HD) - want).abs() <= room).all())
        at += rows

    # ---- request 0 into three more, 1 into one more; every one goes on by itself
    def fork(parents, children):
        lib.fork_requests(i32(parents), i32(children), length, tables, shared, stack, count, B, pools, seq_len_out=length, shared_out=shared,
                          free_left=count, status=status)
        lib.raise_on_pages(status.cpu())
        for p, c in zip(parents, children):                        # (the host's pages: whole ones are the same, the last was copied)
            L = int(length[p])
            if L % B:
                a, b = int(tables[p, L // B]), int(tables[c, L // B])
                for t in (host.k, host.v, host.ks, host.vs):
                    t[b] = t[a]
    fork([0, 0, 0, 1], [2, 3, 4, 5])
    assert length.tolist() == [70, 33, 70, 70, 70, 33, 0, 0]
    same_cache()

    live = 6
    single = arrays(live, 1)
    ones = i32([1] * live + [0] * (S - live))
    row = torch.zeros((live, WIDTH), dtype=torch.bfloat16, device=DEV)
    got = torch.empty((live, NH * HD), dtype=torch.bfloat16, device=DEV)
    states = [t.clone() for t in (length, count, tables, stack, shared, k.view(torch.uint8), v.view(torch.uint8), ks, vs)]
    step(single, ones, row, got, False, live, 120)                  # (loads what there is to load; taken back)
    for t, s in zip((length, count, tables, stack, shared, k.view(torch.uint8), v.view(torch.uint8), ks, vs), states):
        t.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q_row, angles_row = step(single, ones, row, got, False, live, 120)
    for turn in range(14):
        row.copy_((torch.randn((live, WIDTH), generator=g) * (1.0 + 0.3 * turn)).bfloat16())        # (rows grow: scales do)
        graph.replay()
        keep(row, single, angles_row)
        same_cache()
        ends = length.tolist()
        for i in range(live):
            kk, vv = P.gathered(host.k, host.ks, tables[i].cpu(), ends[i]), P.gathered(host.v, host.vs, tables[i].cpu(), ends[i])
            want, room = P.attend("single", q_row[i:i + 1].cpu().double().view(1, NH, HD), kk, vv, torch.tensor([ends[i] - 1]), HD ** -0.5)
            assert bool(((got[i:i + 1].cpu().double().view(1, NH, HD) - want).abs() <= room).all())
    lib.raise_on_step_tables(status.cpu())

    # ---- four end; what they shared stays with the others; the pool moves to the front
    before = [P.gathered(host.k, host.ks, tables[i].cpu(), int(length[i])) for i in (3, 5)]
    lib.release_requests(i32([0, 1, 2, 4]), length, tables, shared, stack, count, B, seq_len_out=length, shared_out=shared, free_left=count, status=status)
    lib.raise_on_pages(status.cpu())
    page_map = torch.empty_like(shared)
    lib.compact_pages(length, tables, shared, stack, count, B, pools, tables_out=tables, shared_out=shared, free_out=stack, page_map=page_map, status=status)
    lib.raise_on_pages(status.cpu())
    used = PAGES - int(count)
    assert used == -(-84 // B) + -(-47 // B) and shared.tolist() == [0] * PAGES
    assert int(max(tables[3, :-(-84 // B)].max(), tables[5, :-(-47 // B)].max())) < used
    for i, want in zip((3, 5), before):
        scale = ks.cpu()
        assert torch.equal(P.gathered(k.cpu().view(torch.uint8), scale, tables[i].cpu(), int(length[i])), want)
    lib.check_errors()


def test_two_recorded_steps_and_another_stream():
    """Two graphs over one pool replayed in turn on a stream of their own give what calls give."""
    lib = K()
    g = torch.Generator().manual_seed(3)
    (kc, ks_), (vc, vs_) = P.pool(40, NKV, B, HD, 1), P.pool(40, NKV, B, HD, 2)
    k, v, ks, vs = kc.to(DEV).view(P.FP8), vc.to(DEV).view(P.FP8), ks_.to(DEV), vs_.to(DEV)
    tables = torch.randperm(40, generator=g).int().view(2, 20).to(DEV)
    ctx = lambda n: types.SimpleNamespace(rows=2, decode_seqs=2, prefill_tiles=0, tile_rows=64, max_ctx=n, max_decode_ctx=n, seq_ctx_len=i32([n, n // 2]), options={})
    q = torch.randn((2, NH * HD), generator=g).bfloat16().to(DEV)
    outs, wants, graphs = [], [], []
    for n in (300, 90):
        c = ctx(n)
        want = torch.empty_like(q)
        lib.paged_attention_q8(q, want, k, v, ks, vs, tables, c, NH, NKV, HD, HD ** -0.5)
        out = torch.empty_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            lib.paged_attention_q8(q, out, k, v, ks, vs, tables, c, NH, NKV, HD, HD ** -0.5)
        outs.append(out); wants.append(want); graphs.append((graph, c))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(3):
            for graph, _ in graphs:
                graph.replay()
    side.synchronize()
    for out, want in zip(outs, wants):
        assert torch.equal(out, want)
    with torch.cuda.stream(side):
        late = torch.empty_like(q)
        lib.paged_attention_q8(q, late, k, v, ks, vs, tables, graphs[0][1], NH, NKV, HD, HD ** -0.5)
    side.synchronize()
    assert torch.equal(late, wants[0])
