"""A step's arrays from lengths on the GPU against the host's batch builder and a plain loop: whole numbers, so everything is equal."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def K():
    from kvcm.kernels import library
    return library


def plain(starts, ns, tables, free, count, B, rows, tiles, tile_rows):
    """The definition, request by request; None where the step cannot be."""
    tables, left = [list(t) for t in tables], count
    out = dict(q_start=[], ctx=[], pos=[], seq=[], slot=[], tiles=[])
    for i, (s, n) in enumerate(zip(starts, ns)):
        out["q_start"].append(len(out["pos"]))
        out["ctx"].append(s + n)
        for j in range(-(-s // B), -(-(s + n) // B)):
            left -= 1
            tables[i][j] = free[left]
        for p in range(s, s + n):
            out["pos"].append(p)
            out["seq"].append(i)
            out["slot"].append(tables[i][p // B] * B + p % B)
        if n > 1:
            out["tiles"] += [(i, q) for q in range(0, n, tile_rows)]
    pad = rows - len(out["pos"])
    out["pos"] += [-1] * pad
    out["seq"] += [0] * pad
    out["slot"] += [-1] * pad
    out["tiles"] += [(-1, -1)] * (tiles - len(out["tiles"]))
    return out, tables, left


class Step:
    def __init__(self, starts, ns, B, width, rows, tiles, seed=0, spare=5):
        r = random.Random(seed)
        held = [-(-s // B) for s in starts]
        need = sum(-(-(s + n) // B) for s, n in zip(starts, ns)) + spare
        ids = list(range(need))
        r.shuffle(ids)
        self.tables, at = [], 0
        for h in held:
            self.tables.append(ids[at:at + h] + [-1] * (width - h))
            at += h
        self.free, self.count = ids[at:], need - at
        self.starts, self.ns, self.B = starts, ns, B
        i32 = dict(dtype=torch.int32, device=DEV)
        self.d = dict(start=torch.tensor(starts, **i32), n=torch.tensor(ns, **i32), tables=torch.tensor(self.tables, **i32),
                      free=torch.tensor(self.free + [-7] * 3, **i32), count=torch.tensor([self.count], **i32))
        S = len(starts)
        self.o = dict(seq_q_start=torch.full((S,), 77, **i32), seq_ctx_len=torch.full((S,), 77, **i32), positions=torch.full((rows,), 77, **i32),
                      row_seq=torch.full((rows,), 77, **i32), slot_mapping=torch.full((rows,), 77, **i32), free_left=torch.full((1,), 77, **i32),
                      status=torch.full((4,), 77, **i32), tile_seq=torch.full((tiles,), 77, **i32), tile_q0=torch.full((tiles,), 77, **i32))

    def run(self, tile_rows=64, **more):
        d = self.d
        K().step_tables(d["start"], d["n"], d["tables"], d["free"], d["count"], self.B, tile_rows=tile_rows, **{**self.o, **more})

    def check(self, tile_rows=64):
        o, rows, tiles = self.o, self.o["positions"].numel(), self.o["tile_seq"].numel()
        want, tables, left = plain(self.starts, self.ns, self.tables, self.free, self.count, self.B, rows, tiles, tile_rows)
        assert o["status"].tolist() == [0, 0, sum(self.ns), sum(-(-n // tile_rows) for n in self.ns if n > 1)]
        assert o["seq_q_start"].tolist() == want["q_start"] and o["seq_ctx_len"].tolist() == want["ctx"]
        assert o["positions"].tolist() == want["pos"] and o["row_seq"].tolist() == want["seq"] and o["slot_mapping"].tolist() == want["slot"]
        assert list(zip(o["tile_seq"].tolist(), o["tile_q0"].tolist())) == want["tiles"]
        assert self.d["tables"].tolist() == tables and o["free_left"].tolist() == [left]


@pytest.mark.parametrize("starts,ns,B,width,rows,tiles,tile_rows", [
    ([0], [1], 16, 4, 1, 0, 64), ([0], [1], 1, 4, 3, 1, 64), ([15, 16, 17, 31], [1, 1, 1, 1], 16, 3, 8, 0, 64),
    ([0, 5, 0, 64, 3], [0, 0, 0, 0, 0], 8, 9, 4, 2, 64), ([0, 5, 0, 64, 3, 9], [0, 7, 0, 65, 1, 200], 8, 40, 300, 9, 64),
    ([0, 3], [130, 64], 7, 30, 194, 20, 13)])
def test_small_steps(starts, ns, B, width, rows, tiles, tile_rows):
    s = Step(starts, ns, B, width, rows, tiles)
    s.run(tile_rows)
    s.check(tile_rows)


@pytest.mark.parametrize("S,most,B,seed", [(33, 3, 16, 1), (1024, 1, 16, 2), (1025, 2, 8, 3), (8192, 1, 16, 4), (64, 400, 16, 5), (3, 9000, 32, 6),
                                           (2500, 5, 3, 7)])
def test_random_steps(S, most, B, seed):
    r = random.Random(seed)
    starts = [r.randrange(0, 500) for _ in range(S)]
    ns = [r.randrange(0 if most > 1 else 1, most + 1) for _ in range(S)]
    rows = sum(ns) + r.randrange(0, 30)
    s = Step(starts, ns, B, max(-(-(a + n) // B) for a, n in zip(starts, ns)) + 1, rows, sum(-(-n // 64) for n in ns if n > 1) + 3, seed)
    s.run()
    s.check()


@pytest.mark.parametrize("S,most", [(5, 1), (40, 300)])
def test_in_place_and_without_tiles(S, most):
    r = random.Random(S)
    starts, ns = [r.randrange(0, 90) for _ in range(S)], [r.randrange(1, most + 1) for _ in range(S)]
    s = Step(starts, ns, 16, 40, sum(ns) + 2, 0)
    s.run(seq_ctx_len=s.d["start"], free_left=s.d["count"], tile_seq=None, tile_q0=None)
    want, tables, left = plain(starts, ns, s.tables, s.free, s.count, 16, sum(ns) + 2, 0, 64)
    assert s.d["start"].tolist() == want["ctx"] and s.d["count"].tolist() == [left] and s.d["tables"].tolist() == tables
    assert s.o["slot_mapping"].tolist() == want["slot"]


def test_a_replayed_graph_goes_on_from_step_to_step():
    S, B, steps = 6, 4, 11
    starts = [0, 3, 4, 7, 12, 1]
    s = Step(starts, [1] * S, B, 12, S, 0, spare=60)
    args = dict(seq_ctx_len=s.d["start"], free_left=s.d["count"], tile_seq=None, tile_q0=None)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.run(**args)
    at, tables, count = list(starts), [list(t) for t in s.tables], s.count
    for _ in range(steps):
        g.replay()
        want, tables, count = plain(at, [1] * S, tables, s.free, count, B, S, 0, 64)
        at = want["ctx"]
        assert s.o["slot_mapping"].tolist() == want["slot"] and s.o["positions"].tolist() == want["pos"]
    assert s.d["tables"].tolist() == tables and s.d["count"].tolist() == [count] and s.d["start"].tolist() == at


@pytest.mark.parametrize("change,code,number", [
    (dict(n=[1, -1, 2]), 1, 1), (dict(start=[0, 5, -3]), 1, 2), (dict(start=[0, 63, 9], n=[1, 2, 1]), 2, 1), (dict(n=[3, 4, 4]), 3, 11),
    (dict(n=[1, 11, 1]), 3, 11), (dict(n=[2, 2, 2], tiles=2), 4, 3), (dict(count=0, n=[1, 1, 1]), 5, 1), (dict(count=99), 6, 99), (dict(count=-1), 6, -1),
    (dict(n=[1, 2 ** 31 - 1, 1]), 2, 1)])
def test_a_step_that_cannot_be_changes_nothing(change, code, number):
    """10 rows of room, tables of 64 positions, requests of 16, 5 and 9 positions."""
    start, n = change.get("start", [16, 5, 9]), change.get("n", [1, 2, 3])
    s = Step([16, 5, 9], [1, 2, 3], 16, 4, 10, change.get("tiles", 3))
    i32 = dict(dtype=torch.int32, device=DEV)
    s.d["start"], s.d["n"] = torch.tensor(start, **i32), torch.tensor(n, **i32)
    if "count" in change:
        s.d["count"].fill_(change["count"])
    before = s.d["count"].tolist()
    s.run()
    o = s.o
    status = o["status"].tolist()
    assert status == [code, number, 0, 0]
    assert s.d["tables"].tolist() == s.tables and o["free_left"].tolist() == before and o["seq_ctx_len"].tolist() == start
    assert set(o["positions"].tolist()) == {-1} and set(o["slot_mapping"].tolist()) == {-1} and set(o["row_seq"].tolist()) == {0}
    assert set(o["tile_seq"].tolist()) == {-1} and set(o["tile_q0"].tolist()) == {-1}
    with pytest.raises(K().KernelError, match="step_tables"):
        K().raise_on_step_tables(status)


def test_the_arrays_of_the_batch_builder():
    """The same requests through the host's builder: rows, slots, tables, tiles."""
    from kvcm.cache import core, manager_from_config
    from kvcm.config import KVManagerConfig
    B, width, spans = 8, 16, [(9, 1), (16, 1), (0, 70), (24, 30)]
    kv = manager_from_config(KVManagerConfig(num_blocks=64, block_size=B, max_seq_len=B * width, watermark_blocks=0))
    entries = []
    for i, (a, n) in enumerate(spans):
        q = core.Sequence()
        q.id, q.tokens, q.prompt_len = i, [1] * (a + n), a + n
        assert kv.can_admit(q)
        kv.admit(q)
        assert kv.ensure(q, a + n)
        entries.append((q, a, n, []))
    b = core.BatchBuilder(B, width, 1, 64)
    host = torch.zeros(int(b.capacity_for(200, 8, 8)), dtype=torch.int32)
    L = b.build(entries, host.data_ptr(), host.numel(), 0, 0)
    view = lambda off, n: host[off:off + n].tolist()            # noqa: E731
    T, S, NT = L.rows, L.seqs, L.prefill_tiles
    tables = host[L.off_block_tables:L.off_block_tables + S * width].view(S, width)
    # the device starts from the pages held before the step and takes the new ones, in order, from a stack that holds them
    start, n = [a for a, _ in spans], [m for _, m in spans]
    held = [-(-a // B) for a in start]
    new = [int(tables[i, j]) for i in range(S) for j in range(held[i], -(-(start[i] + n[i]) // B))]
    s = Step(start, n, B, width, T, NT)
    i32 = dict(dtype=torch.int32, device=DEV)
    first = tables.clone()
    for i in range(S):
        first[i, held[i]:] = -1
    s.d.update(tables=first.to(DEV), free=torch.tensor(new[::-1], **i32), count=torch.tensor([len(new)], **i32))
    s.run()
    o = s.o
    assert s.d["tables"].cpu().tolist() == tables.tolist()
    for name, off, k in (("positions", L.off_positions, T), ("row_seq", L.off_row_seq, T), ("slot_mapping", L.off_slot_mapping, T),
                         ("seq_q_start", L.off_seq_q_start, S), ("seq_ctx_len", L.off_seq_ctx_len, S), ("tile_seq", L.off_tile_seq, NT),
                         ("tile_q0", L.off_tile_q0, NT)):
        assert o[name].tolist() == view(off, k), name
