"""Pages that requests share, on the GPU, against plain loops: whole numbers and bytes, so everything is equal."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def K():
    from kvcm.kernels import library
    return library


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


class World:
    """Requests with pages in any order, some of them shared already, a stack of free ones, and pools of three types."""

    def __init__(self, lengths, B, width, free, seed=0, share=0):
        r = random.Random(seed)
        S = len(lengths)
        self.B, self.width, self.lengths = B, width, list(lengths)
        held = [-(-n // B) for n in lengths]
        self.N = sum(held) + free
        ids = list(range(self.N))
        r.shuffle(ids)
        self.tables, at = [], 0
        for h in held:
            self.tables.append(ids[at:at + h] + [-1] * (width - h))
            at += h
        self.stack = ids[at:] + [-1] * (self.N - free)
        self.count, self.shared = free, [0] * self.N
        # whole pages of some requests given to others in place of theirs; theirs are free then
        for _ in range(share):
            a, b = r.randrange(S), r.randrange(S)
            if a == b or lengths[a] // B == 0 or lengths[b] // B == 0 or self.tables[a][0] in self.tables[b]:
                continue
            old, new = self.tables[b][0], self.tables[a][0]
            if self.shared[old]:
                continue
            self.tables[b][0] = new
            self.shared[new] += 1
            self.stack[self.count] = old
            self.count += 1
        g = torch.Generator().manual_seed(seed)
        self.pools = [torch.randint(0, 256, (3, self.N, 2, B, 24), generator=g, dtype=torch.uint8), torch.randn((1, self.N, 5), generator=g),
                      torch.randn((2, self.N, 3, B, 16), generator=g).bfloat16(), torch.randint(0, 256, (2, self.N, 7), generator=g, dtype=torch.uint8)]

    def device(self):
        """The arrays on the GPU."""
        self.d = dict(seq_len=i32(self.lengths), block_tables=i32(self.tables), shared=i32(self.shared), free_pages=i32(self.stack),
                      free_count=i32([self.count]))
        self.dp = [p.to(DEV) for p in self.pools]
        self.status = i32([9] * 4)
        return self.d

    def snapshot(self):
        return [list(map(list, self.tables)), list(self.lengths), list(self.shared), list(self.stack), self.count, [p.clone() for p in self.pools]]

    # ---- the definitions
    def fork(self, parents, children):
        for p, c in zip(parents, children):
            if p < 0:
                continue
            L = self.lengths[p]
            full = L // self.B
            for j in range(full):
                self.tables[c][j] = self.tables[p][j]
                self.shared[self.tables[p][j]] += 1
            if L % self.B:
                self.count -= 1
                new = self.stack[self.count]
                self.tables[c][full] = new
                for pool in self.pools:
                    pool[:, new] = pool[:, self.tables[p][full]]
            self.lengths[c] = L

    def release(self, requests):
        freed = []
        for r in requests:
            if r < 0:
                continue
            for j in range(-(-self.lengths[r] // self.B)):
                page = self.tables[r][j]
                self.shared[page] -= 1
                if self.shared[page] < 0:
                    freed.append(page)
                    self.shared[page] = 0
            self.lengths[r] = 0
        freed.sort(reverse=True)
        self.stack[self.count:self.count + len(freed)] = freed
        self.count += len(freed)
        return len(freed)

    def compact(self):
        free = set(self.stack[:self.count])
        used = self.N - self.count
        holes = sorted(p for p in free if p < used)
        movers = sorted(p for p in range(used, self.N) if p not in free)
        where = {p: (-1 if p in free else p) for p in range(self.N)}
        where.update(zip(movers, holes))
        shared = list(self.shared)
        for a, b in zip(movers, holes):
            shared[b] = self.shared[a]
            for pool in self.pools:
                pool[:, b] = pool[:, a]
        for p in range(used, self.N):
            shared[p] = 0
        self.shared = shared
        for i, L in enumerate(self.lengths):
            for j in range(-(-L // self.B)):
                self.tables[i][j] = where[self.tables[i][j]]
        self.stack[:self.count] = list(range(self.N - 1, used - 1, -1))
        return [where[p] for p in range(self.N)], len(movers)

    def same(self, d, pools=True):
        assert d["seq_len"].tolist() == self.lengths
        assert d["block_tables"].tolist() == self.tables
        assert d["shared"].tolist() == self.shared
        assert d["free_count"].tolist() == [self.count]
        assert d["free_pages"].tolist()[:self.count] == self.stack[:self.count]
        if pools:
            for a, b in zip(self.dp, self.pools):
                assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))


def outs(d, separate):
    fresh = (lambda k: torch.full_like(d[k], 77)) if separate else (lambda k: d[k])
    return dict(seq_len_out=fresh("seq_len"), shared_out=fresh("shared"), free_left=fresh("free_count"))


def after(d, o):
    return dict(d, seq_len=o["seq_len_out"], shared=o["shared_out"], free_count=o["free_left"])


CASES = [([33, 0, 0, 16, 0], 16, 4, 3, 0), ([5, 0], 8, 1, 2, 0), ([64, 0, 7, 0, 0, 0, 63], 16, 9, 40, 3),
         ([int(37 * i) % 200 if i % 3 else 0 for i in range(90)], 8, 30, 200, 20), ([1000, 0, 2500, 0, 0], 16, 200, 30, 0)]


@pytest.mark.parametrize("separate", [False, True])
@pytest.mark.parametrize("lengths,B,width,free,share", CASES)
def test_fork(lengths, B, width, free, share, separate):
    w = World(lengths, B, width, free, seed=len(lengths), share=share)
    held = [i for i, n in enumerate(lengths) if n]
    empty = [i for i, n in enumerate(lengths) if not n]
    r = random.Random(1)
    parents = [r.choice(held) for _ in empty] + [-1, -1]
    children = empty + [-1, 0]
    d = w.device()
    o = outs(d, separate)
    K().fork_requests(i32(parents), i32(children), **d, block_size=B, pools=w.dp, **o, status=w.status)
    before = w.count
    w.fork(parents, children)
    assert w.status.tolist() == [0, 0, before - w.count, 0]
    w.same(after(d, o))
    if separate:                                                    # the same call again: the same
        K().fork_requests(i32(parents), i32(children), **d, block_size=B, pools=w.dp, **o, status=w.status)
        w.same(after(d, o))
    K().raise_on_pages(w.status.cpu())


@pytest.mark.parametrize("separate", [False, True])
@pytest.mark.parametrize("lengths,B,width,free,share", CASES)
@pytest.mark.parametrize("part", [0.0, 0.5, 1.0])
def test_release_and_compact(lengths, B, width, free, share, part, separate):
    w = World(lengths, B, width, free, seed=len(lengths) + 1, share=share)
    r = random.Random(2)
    gone = [i for i in range(len(lengths)) if r.random() < part]
    r.shuffle(gone)
    gone = gone + [-1]
    d = w.device()
    o = outs(d, separate)
    K().release_requests(i32(gone), **d, block_size=B, **o, status=w.status)
    n = w.release(gone)
    assert w.status.tolist() == [0, 0, n, 0]
    d = after(d, o)
    w.same(d)
    c = dict(tables_out=torch.full_like(d["block_tables"], 77) if separate else d["block_tables"],
             shared_out=torch.full_like(d["shared"], 77) if separate else d["shared"],
             free_out=torch.full_like(d["free_pages"], 77) if separate else d["free_pages"], page_map=torch.empty_like(d["shared"]))
    K().compact_pages(**d, block_size=B, pools=w.dp, **c, status=w.status)
    where, moved = w.compact()
    assert w.status.tolist() == [0, 0, moved, 0] and c["page_map"].tolist() == where
    d = dict(d, block_tables=c["tables_out"], shared=c["shared_out"], free_pages=c["free_out"])
    w.same(d)
    K().compact_pages(**d, block_size=B, pools=w.dp, tables_out=d["block_tables"], shared_out=d["shared"], free_out=d["free_pages"],
                      page_map=c["page_map"], status=w.status)     # once more: nothing moves
    assert w.status.tolist() == [0, 0, 0, 0]
    w.same(d)


def test_a_life_of_many_steps_in_place():
    """Forks, ends and compactions one behind another, never read back in between."""
    r = random.Random(7)
    w = World([r.randrange(1, 90) for _ in range(6)] + [0] * 20, 8, 12, 300, seed=5)
    d = w.device()
    o = outs(d, False)
    for step in range(12):
        live = [i for i, n in enumerate(w.lengths) if n]
        empty = [i for i, n in enumerate(w.lengths) if not n]
        children = r.sample(empty, min(len(empty), r.randrange(1, 9)))
        parents = [r.choice(live) for _ in children]
        K().fork_requests(i32(parents), i32(children), **d, block_size=8, pools=w.dp, **o, status=w.status)
        w.fork(parents, children)
        live = [i for i, n in enumerate(w.lengths) if n]
        gone = r.sample(live, r.randrange(0, len(live)))
        K().release_requests(i32(gone), **d, block_size=8, **o, status=w.status)
        w.release(gone)
        if step % 3 == 2:
            K().compact_pages(**d, block_size=8, pools=w.dp, tables_out=d["block_tables"], shared_out=d["shared"], free_out=d["free_pages"],
                              page_map=torch.empty_like(d["shared"]), status=w.status)
            w.compact()
    w.same(d)


REFUSED = [
    ("fork", dict(parents=[9], children=[1]), (1, 0)),
    ("fork", dict(parents=[0, 0], children=[1, -1]), (1, 1)),
    ("fork", dict(parents=[0, 2], children=[1, 1]), (2, 1)),
    ("fork", dict(parents=[0], children=[2]), (3, 2)),             # holds pages
    ("fork", dict(parents=[0], children=[0]), (3, 0)),
    ("fork", dict(parents=[0, 1], children=[1, 3]), (3, 1)),       # begins in the call
    ("fork", dict(parents=[0], children=[1], lengths={0: 65}), (4, 0)),
    ("fork", dict(parents=[0], children=[1], lengths={0: -1}), (4, 0)),
    ("fork", dict(parents=[0], children=[1], tables={(0, 1): 500}), (5, 500)),
    ("fork", dict(parents=[0, 2, 0], children=[1, 3, 4]), (6, 1)),
    ("fork", dict(parents=[0], children=[1], count=99), (7, 99)),
    ("release", dict(requests=[8]), (1, 0)),
    ("release", dict(requests=[0, 2, 0]), (2, 0)),
    ("release", dict(requests=[0], lengths={0: 65}), (4, 0)),
    ("release", dict(requests=[0], count=-3), (7, None)),
    ("release", dict(requests=[0], tables={(0, 0): -1}), (5, None)),
    ("release", dict(requests=[0, 2], tables={(0, 0): "same"}), (8, "same")),      # both hold it, nobody says that it is shared
    ("compact", dict(tables={(0, 0): "free"}), (5, "free")),
    ("compact", dict(tables={(2, 0): 1000}), (5, 1000)),
    ("compact", dict(stack={1: "first"}), (2, "first")),
    ("compact", dict(stack={0: 4000}), (5, 4000)),
    ("compact", dict(count=4000), (7, 4000)),
    ("compact", dict(lengths={2: 100}), (4, 2))]


@pytest.mark.parametrize("separate", [False, True])
@pytest.mark.parametrize("call,change,want", REFUSED)
def test_refusals_leave_everything_as_it_was(call, change, want, separate):
    w = World([40, 0, 21, 0, 0], 16, 4, 2, seed=3)
    names = {"same": w.tables[2][0], "free": w.stack[0], "first": w.stack[0]}
    val = lambda x: names.get(x, x)
    for i, n in change.get("lengths", {}).items():
        w.lengths[i] = n
    for (i, j), n in change.get("tables", {}).items():
        w.tables[i][j] = val(n)
    for i, n in change.get("stack", {}).items():
        w.stack[i] = val(n)
    w.count = change.get("count", w.count)
    d = w.device()
    o = outs(d, separate)
    if call == "fork":
        K().fork_requests(i32(change["parents"]), i32(change["children"]), **d, block_size=16, pools=w.dp, **o, status=w.status)
        d = after(d, o)
    elif call == "release":
        K().release_requests(i32(change["requests"]), **d, block_size=16, **o, status=w.status)
        d = after(d, o)
    else:
        c = dict(tables_out=torch.full_like(d["block_tables"], 77) if separate else d["block_tables"],
                 shared_out=torch.full_like(d["shared"], 77) if separate else d["shared"],
                 free_out=d["free_pages"], page_map=torch.empty_like(d["shared"]))
        K().compact_pages(**d, block_size=16, pools=w.dp, **c, status=w.status)
        assert c["page_map"].tolist() == list(range(w.N))
        d = dict(d, block_tables=c["tables_out"], shared=c["shared_out"])
    code, number = want
    got = w.status.tolist()
    assert got[0] == code and (number is None or got[1] == val(number)) and got[2:] == [0, 0]
    assert d["free_pages"].tolist() == w.stack
    stack, w.stack = w.stack, w.stack[:max(0, min(w.count, len(w.stack)))]
    if 0 <= w.count <= len(stack):
        w.same(d)
    else:
        assert d["seq_len"].tolist() == w.lengths and d["block_tables"].tolist() == w.tables and d["shared"].tolist() == w.shared
    with pytest.raises(K().KernelError, match="pages"):
        K().raise_on_pages(w.status.cpu())


def test_copy_pages():
    w = World([100], 16, 8, 60, seed=4)
    w.device()
    src, dst = [1, 5, -1, 7, 9, 200, 3], [20, 21, 22, -5, 400, 23, 3]
    K().copy_pages(w.dp, i32(src), i32(dst))
    for pool in w.pools:
        for a, b in zip(src[:2], dst[:2]):
            pool[:, b] = pool[:, a]
    for a, b in zip(w.dp, w.pools):
        assert torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8))
    big = torch.randint(0, 256, (2, 30, 3, 40000), dtype=torch.uint8, device=DEV)      # pages of many pieces; layers with a stride of their own
    want = big.clone()
    K().copy_pages([big[:, :, 1:2].squeeze(2)[:, :, None][:1].contiguous(), big], i32([3, 4]), i32([10, 11]))
    want[:, [10, 11]] = want[:, [3, 4]]
    assert torch.equal(big, want)


def test_a_step_of_a_beam_in_a_graph():
    """Recorded once, replayed: losers end, winners fork, in place; the host never looks in between."""
    w = World([50, 50, 50, 50], 16, 8, 40, seed=6)
    w.lengths = [50, 50, 0, 0]
    w.stack[w.count:w.count + 8] = w.tables[2][:4] + w.tables[3][:4]
    w.count += 8
    d = w.device()
    o = outs(d, False)
    gone, parents, children = i32([-1, -1]), i32([0, 1]), i32([2, 3])

    def step():
        K().release_requests(gone, **d, block_size=16, **o, status=w.status)
        K().fork_requests(parents, children, **d, block_size=16, pools=w.dp, **o, status=w.status)
    K().copy_pages(w.dp, i32([-1]), i32([-1]))                      # (loads the library's kernels before the capture)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    plans = [([-1, -1], [0, 1], [2, 3]), ([0, 3], [2, 1], [3, 0]), ([1, 2], [3, 3], [1, 2])]
    for g_, p_, c_ in plans:
        gone.copy_(i32(g_))
        parents.copy_(i32(p_))
        children.copy_(i32(c_))
        graph.replay()
        w.release(g_)
        w.fork(p_, c_)
        assert w.status.tolist()[0] == 0
    w.same(d)
