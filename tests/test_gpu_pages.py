"""The page pool's operations on the GPU against a model of lists: tables,
lengths, counts and the pools' contents, which have to be equal."""
import random

import pytest
import torch

from gdnx_amd import attention, pages
from oracle import attention as oa

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Both:
    """A pool on the GPU and its model on the CPU."""

    def __init__(self, n_pages, page, rows, width, layers=2, Hkv=2, D=64, dtype=torch.bfloat16, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.k, self.v = (torch.randn(layers, n_pages, Hkv, page, D, generator=g).to(dtype) for _ in range(2))
        self.kp, self.vp = self.k.to(DEV), self.v.to(DEV)
        self.model = oa.Pages(n_pages, page, rows, width)
        i = dict(dtype=torch.int32, device=DEV)
        self.table, self.lengths = torch.full((rows, width), -1, **i), torch.zeros(rows, **i)
        self.refs, self.status = torch.zeros(n_pages, **i), torch.zeros(2, **i)
        self.page, self.g, self.dtype = page, g, dtype

    def ints(self, xs):
        return torch.tensor(xs, dtype=torch.int32, device=DEV)

    def same(self):
        m = self.model
        assert self.refs.tolist() == m.refs and self.lengths.tolist() == m.lens
        got = self.table.tolist()
        for r, row in enumerate(m.table()):
            n = len(m.rows[r])
            assert got[r][:n] == row[:n], r
        assert torch.equal(self.kp.cpu(), self.k) and torch.equal(self.vp.cpu(), self.v)

    def reserve(self, slots, n):
        start = pages.pages_reserve(self.table, self.lengths, self.refs, self.ints(slots), n, self.page, self.status)
        want = self.model.reserve(slots, n)
        assert start.tolist() == ([-1] * len(slots) if want is None else want)
        return start, want

    def write(self, slots, start, want, T):
        L, _, Hkv, _, D = self.k.shape
        new = [torch.randn(L, len(slots), T, Hkv, D, generator=self.g).to(self.dtype) for _ in range(2)]
        pages.pages_write(new[0].to(DEV), new[1].to(DEV), self.kp, self.vp, self.table, self.ints(slots), start)
        for i, s in enumerate(slots):
            for t in range(T if want is not None and want[i] >= 0 else 0):
                p = want[i] + t
                pg = self.model.rows[s][p // self.page]
                for pool, x in ((self.k, new[0]), (self.v, new[1])):
                    pool[:, pg, :, p % self.page] = x[:, i, t]

    def fork(self, parents, children):
        pages.pages_fork(self.kp, self.vp, self.table, self.lengths, self.refs, self.ints(parents),
                         self.ints(children), self.status)
        for a, b in self.model.fork(parents, children) or ():
            self.k[:, b], self.v[:, b] = self.k[:, a], self.v[:, a]

    def free(self, slots):
        pages.pages_free(self.table, self.lengths, self.refs, self.ints(slots))
        self.model.free(set(slots))

    def trim(self, slots, window, sinks):
        pages.pages_trim(self.table, self.lengths, self.refs, self.ints(slots), window, sinks, self.page)
        self.model.trim(slots, window, sinks)

    def compact(self, out=False):
        o = (torch.empty_like(self.table), torch.empty_like(self.refs)) if out else None
        before = self.table.clone(), self.refs.clone()
        t, r = pages.pages_compact(self.kp, self.vp, self.table, self.refs, out=o)
        if out:
            assert torch.equal(self.table, before[0]) and torch.equal(self.refs, before[1])
            self.table, self.refs = t, r
        for a, b in self.model.compact():
            self.k[:, b], self.v[:, b] = self.k[:, a], self.v[:, a]


@pytest.mark.parametrize("n_pages,page,rows,width,layers,Hkv,D,dtype", [
    (40, 4, 9, 12, 1, 1, 64, torch.bfloat16), (300, 16, 30, 20, 3, 2, 64, torch.bfloat16),
    (5000, 1, 40, 200, 1, 1, 64, torch.float32), (70, 64, 12, 9, 2, 3, 128, torch.float32)])
def test_a_life_of_the_pool(gpu_lib, n_pages, page, rows, width, layers, Hkv, D, dtype):
    b, rng = Both(n_pages, page, rows, width, layers, Hkv, D, dtype), random.Random(5)
    empty, live = list(range(rows)), []
    refused = 0
    for turn in range(60):
        op = rng.choice(("grow", "grow", "new", "fork", "free", "trim", "compact"))
        if op == "new" and empty:
            live.append(empty.pop(rng.randrange(len(empty))))
            op = "grow"
        if op == "grow" and live:
            slots = rng.sample(live, rng.randint(1, len(live)))
            if rng.random() < 0.3:
                slots.insert(rng.randint(0, len(slots)), rng.choice((-1, rows, 10 ** 6)))
            T = rng.choice((1, 1, 2, page, page + 1, 3 * page - 1))
            start, want = b.reserve(slots, T)
            refused += want is None
            b.write(slots, start, want, T)
        elif op == "fork" and live and empty:
            parents = [rng.choice(live) for _ in range(rng.randint(1, len(empty)))]
            children = [empty.pop() for _ in parents]
            before = list(b.model.lens)
            b.fork(parents, children)
            live += children
        elif op == "free" and live:
            gone = rng.sample(live, rng.randint(1, len(live)))
            b.free(gone + gone[:1])                       # (a row named twice is freed once)
            live, empty = [r for r in live if r not in gone], empty + gone
        elif op == "trim" and live:
            b.trim(rng.sample(live, rng.randint(1, len(live))), rng.choice((1, page, 5 * page)), rng.choice((0, 1, page + 1)))
        elif op == "compact":
            b.compact(out=rng.random() < 0.5)
        b.same()


def test_nothing_changes_when_the_pool_is_too_small(gpu_lib):
    b = Both(10, 8, 6, 4)
    start, want = b.reserve([0, 1], 20)                   # 6 pages
    b.write([0, 1], start, want, 20)
    assert b.reserve([2, 3], 24)[1] is None and b.status.tolist() == [2, 0]
    assert b.reserve([0], 13)[1] is None and b.status.tolist() == [0, 1]
    start, _ = b.reserve([2, 3], 9)                       # the rest
    b.fork([0, 1], [4, 5])
    assert b.status.tolist() == [2, 0] and b.lengths.tolist() == [20, 20, 9, 9, 0, 0]
    b.same()
    b.free([3])
    b.fork([0, 1], [4, 5])
    b.same()


def test_fork_leaves_out_what_is_no_pair(gpu_lib):
    b = Both(20, 8, 6, 4)
    b.reserve([0, 1], 12)
    pages.pages_fork(b.kp, b.vp, b.table, b.lengths, b.refs, b.ints([0, 0, -1, 7, 0, 2]), b.ints([1, 6, 3, 3, 0, 4]), b.status)
    b.same()                                              # (an empty parent gives an empty child)
    b.fork([0], [5])
    b.same()


def test_copy(gpu_lib):
    b = Both(12, 32, 1, 1, layers=3, Hkv=3, D=128)
    pages.pages_copy(b.kp, b.vp, b.ints([3, -1, 5, 99, 3]), b.ints([0, 1, 11, 2, 12]))
    for s, d in ((3, 0), (5, 11)):
        b.k[:, d], b.v[:, d] = b.k[:, s], b.v[:, s]
    b.same()
    pages.pages_copy(b.kp[1], b.vp[1], b.ints([7]), b.ints([8]))
    b.k[1, 8], b.v[1, 8] = b.k[1, 7], b.v[1, 7]
    b.same()


def test_a_pool_beyond_32_bits(gpu_lib):
    """Pages past 4 GB: written, forked and compacted."""
    n_pages, page, Hkv, D = 20000, 128, 8, 128            # 5.2 GB a pool
    kp = torch.zeros(1, n_pages, Hkv, page, D, dtype=torch.bfloat16, device=DEV)
    vp = torch.zeros_like(kp)
    i = dict(dtype=torch.int32, device=DEV)
    table, lengths, status = torch.full((4, 4), -1, **i), torch.zeros(4, **i), torch.zeros(2, **i)
    refs = torch.ones(n_pages, **i)
    refs[19990:] = 0                                      # the free ones are the last
    new = torch.randn(1, 1, 200, Hkv, D, device=DEV).bfloat16()
    slots = torch.tensor([1], **i)
    start = pages.pages_reserve(table, lengths, refs, slots, 200, page, status)
    pages.pages_write(new, 2 * new, kp, vp, table, slots, start)
    pages.pages_fork(kp, vp, table, lengths, refs, slots, torch.tensor([3], **i), status)
    assert table.tolist()[1][:2] == [19990, 19991] and table.tolist()[3][:2] == [19990, 19992]
    flat = lambda pool, r: pool[0][table[r, :2].long()].permute(0, 2, 1, 3).reshape(-1, Hkv, D)[:200]
    for r in (1, 3):
        assert torch.equal(flat(kp, r), new[0, 0]) and torch.equal(flat(vp, r), 2 * new[0, 0])
    refs[:10000] = 0
    pages.pages_compact(kp, vp, table, refs)
    assert table.max() < 9993 + 3 and int((refs != 0).sum()) == 9993
    for r in (1, 3):
        assert torch.equal(flat(kp, r), new[0, 0]) and torch.equal(flat(vp, r), 2 * new[0, 0])


def test_cache_serves_forked_rows(gpu_lib):
    """PagedKVCache: prompts, samples of them, steps with a window, trimming and compaction, against the oracle."""
    torch.manual_seed(0)
    Hq, Hkv, D, L, W, S = 4, 2, 64, 2, 40, 3
    c = pages.PagedKVCache(60, 16, Hkv, D, 8, 400, layers=L)
    rows = c.alloc(2)
    rt = c.rows_tensor(rows)
    hist = {}
    T = 90
    k, v = (torch.randn(L, 2, T, Hkv, D, device=DEV).bfloat16() for _ in range(2))
    c.write(rt, c.reserve(rows, T), k, v)
    for i, r in enumerate(rows):
        hist[r] = [k[:, i].cpu(), v[:, i].cpu()]
    kids = c.fork([rows[0], rows[0], rows[1]])
    for p, x in zip((rows[0], rows[0], rows[1]), kids):
        hist[x] = [t.clone() for t in hist[p]]
    rows = rows + kids
    rt = c.rows_tensor(rows)
    for turn in range(20):
        c.reserve(rows, 1)
        q = torch.randn(L, len(rows), Hq, D, device=DEV).bfloat16()
        k, v = (torch.randn(L, len(rows), Hkv, D, device=DEV).bfloat16() for _ in range(2))
        for i, r in enumerate(rows):
            hist[r] = [torch.cat([h, x[:, i:i + 1].cpu()], 1) for h, x in zip(hist[r], (k, v))]
        for layer in range(L):
            y = c.step(layer, rt, q[layer], k[layer], v[layer], window=W, sinks=S)
            ref = torch.stack([oa.attention(q[layer, i][None, None], hist[r][0][layer][None], hist[r][1][layer][None], W,
                                            S)[0][0, 0] for i, r in enumerate(rows)])
            err = (y.cpu().double() - ref).norm() / ref.norm()
            assert err <= 4e-3, (turn, layer, err)
        if turn % 5 == 4:
            c.trim(rows, W, S)
            c.compact()
            used = c.pages_in_use()
            assert int((c.refs[:used] != 0).sum()) == used
    c.free(rows)
    assert c.pages_in_use() == 0 and (c.lengths == 0).all() and (c.table == -1).all()
    assert len(c.alloc(8)) == 8


def test_graph_of_a_serving_step(gpu_lib):
    """reserve, step and trim captured together; every replay equals the eager calls, with other work in between."""
    Hq, Hkv, D, page = 4, 2, 64, 16
    def state():
        g = torch.Generator(device=DEV).manual_seed(1)
        i = dict(dtype=torch.int32, device=DEV)
        s = dict(kp=torch.randn(40, Hkv, page, D, device=DEV, generator=g).bfloat16(),
                 vp=torch.randn(40, Hkv, page, D, device=DEV, generator=g).bfloat16(), table=torch.full((4, 16), -1, **i),
                 lengths=torch.zeros(4, **i), refs=torch.zeros(40, **i), status=torch.zeros(2, **i),
                 slots=torch.tensor([2, 0, -1], **i), y=torch.zeros(3, Hq, D, device=DEV).bfloat16())
        pages.pages_reserve(s["table"], s["lengths"], s["refs"], torch.tensor([0, 2], **i), 60, page, s["status"])
        return s
    ins = [torch.zeros(3, h, D, device=DEV).bfloat16() for h in (Hq, Hkv, Hkv)]
    def step(s):
        pages.pages_reserve(s["table"], s["lengths"], s["refs"], s["slots"], 1, page, s["status"])
        attention.paged_attention_step(*ins, s["kp"], s["vp"], s["table"], s["lengths"], slots=s["slots"], window=30,
                                       sinks=2, out=s["y"])
        pages.pages_trim(s["table"], s["lengths"], s["refs"], s["slots"], 30, 2, page)
    a, b = state(), state()
    warm = state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(b)
    for turn in range(12):
        for x in ins:
            x.copy_(torch.randn(x.shape, device=DEV))
        step(a)
        graph.replay()
        torch.cuda.synchronize()
        for n in a:
            assert torch.equal(a[n], b[n]), (turn, n)
