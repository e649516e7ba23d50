"""Packed rows over the page cache on the GPU against the 64-bit oracle.

Tolerances (relative L2), as for windowed attention: float32 1e-5 (a score is
a sum of D products, wrong by about sqrt(D) 2^-24 of its terms, and P and the
second product follow).  bfloat16: the output is rounded once (at most 2^-8 of the
value, 1.7e-3 rms) and P, where it is an operand of the second product, once
more: sqrt(2) * 1.7e-3 with head room, 4e-3.  A vector of D values: five times as
much, against its own size and the mean one.
"""
import pytest
import torch

from gdnx_amd import attention, pages
from oracle import attention as oa

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = {torch.float32: 1e-5, torch.bfloat16: 4e-3}


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def close(got, want, dtype):
    got = got.double().cpu()
    d = (got - want).flatten(0, 1).norm(dim=1)
    size = want.flatten(0, 1).norm(dim=1)
    mean = float(want.norm()) / max(1, size.numel()) ** 0.5
    assert torch.isfinite(got).all()
    assert float((got - want).norm()) <= TOL[dtype] * float(want.norm()) and (d <= 5 * TOL[dtype] * (size + mean)).all()


class Batch:
    """Rows with `past` cached and `counts` new tokens in a pool whose pages lie anywhere; what no row holds is NaN."""

    def __init__(self, past, counts, Hq, Hkv, D, page, dtype, seed=0, extra_rows=2):
        g = torch.Generator().manual_seed(seed)
        n = len(past)
        self.lens = [p + c for p, c in zip(past, counts)]
        need = [-(-l // page) for l in self.lens]
        n_pages, width = sum(need) + 3, max(need) + 1
        order = torch.randperm(n_pages, generator=g).tolist()
        self.slots = torch.randperm(n + extra_rows, generator=g).tolist()[:n]
        self.table = [[-1] * width for _ in range(n + extra_rows)]
        self.lengths = [0] * (n + extra_rows)
        self.kp, self.vp = (torch.full((n_pages, Hkv, page, D), float("nan")) for _ in range(2))
        for b, r in enumerate(self.slots):
            self.lengths[r] = self.lens[b]
            for c in range(need[b]):
                pg = self.table[r][c] = order.pop()
                m = min(page, self.lens[b] - c * page)
                for pool in (self.kp, self.vp):
                    pool[pg, :, :m] = torch.randn(Hkv, m, D, generator=g)
        self.kp, self.vp = self.kp.to(dtype), self.vp.to(dtype)
        self.offsets = [sum(counts[:i]) for i in range(n + 1)]
        self.q = torch.randn(sum(counts), Hq, D, generator=g).to(dtype)

    def run(self, q=None, **kw):
        return attention.paged_attention_chunk(self.q.to(DEV) if q is None else q, self.kp.to(DEV), self.vp.to(DEV),
                                               i32(self.table), i32(self.lengths), i32(self.offsets),
                                               slots=i32(self.slots), **kw)

    def want(self, **kw):
        return oa.paged_chunk(self.q, self.kp, self.vp, self.table, self.lengths, self.offsets, self.slots, **kw)


CASES = [
    # past, counts, query heads, key heads, page, window, sinks
    ([0], [1], 1, 1, 16, None, 0),
    ([40], [1], 4, 2, 16, None, 0),
    ([0, 5, 100], [70, 0, 1], 4, 2, 16, None, 0),
    ([63, 64, 65, 1], [1, 1, 1, 1], 4, 1, 64, None, 0),
    ([200, 0, 31], [5, 5, 5], 16, 4, 32, None, 0),
    ([130, 77], [33, 200], 6, 2, 16, 40, 3),
    ([300, 3], [100, 140], 8, 2, 128, 64, 70),
    ([30, 500, 0], [1, 2, 300], 2, 2, 1, None, 0),           # a page for every token
    ([100, 2], [20, 50], 6, 3, 2, 7, 1),
    ([90, 0], [260, 17], 20, 1, 4, None, 0),                 # a group that is no power of two
    ([10], [3], 150, 1, 16, None, 0),                        # a group longer than a tile's rows
    ([1000] * 3, [1, 130, 9], 8, 1, 16, None, 0),
    ([5, 17], [40, 40], 2, 1, 8, 1, 0),                      # every token sees itself alone
    ([700], [40], 4, 1, 16, 100, 500),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[2:])))
def test_chunk(gpu_lib, case, D, dtype):
    past, counts, Hq, Hkv, page, window, sinks = case
    b = Batch(past, counts, Hq, Hkv, D, page, dtype)
    y = b.run(window=window, sinks=sinks)
    assert y.dtype == dtype
    close(y, b.want(window=window, sinks=sinks), dtype)
    assert torch.equal(y, b.run(window=window, sinks=sinks))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scale_views_and_the_rows_behind(gpu_lib, dtype):
    """Queries of a fused projection; tokens of nobody stay as they were; scales of either sign."""
    b = Batch([50, 9], [30, 70], 4, 2, 64, 16, dtype)
    N = b.q.shape[0]
    wide = torch.full((N + 8, 4 + 2 + 2, 64), float("nan"), device=DEV).to(dtype)
    wide[:N, :4] = b.q.to(DEV)
    for scale in (0.3, -0.2, 0.0):
        out = torch.full((N + 8, 4, 64), 5.0, device=DEV).to(dtype)
        y = b.run(wide[:, :4], scale=scale, out=out)
        assert y is out and (out[N:] == 5).all()
        close(out[:N], b.want(scale=scale), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_see_nothing(gpu_lib, dtype):
    """Rows outside the table, more new tokens than the row's length, lengths that do not fit, missing pages."""
    b = Batch([20, 30, 40, 50], [6, 40, 5, 33], 4, 2, 64, 16, dtype)
    lens, slots = list(b.lengths), list(b.slots)
    b.slots[0] = -1
    b.lengths[slots[1]] = 25                       # 40 new tokens end at position 24: the first 15 stand before 0
    b.lengths[slots[2]] = 16 * len(b.table[0]) + 1
    b.table[slots[3]][1] = b.table[slots[3]][4] = -1
    b.table[slots[3]][2] = 1 << 20
    y, want = b.run(), b.want()
    assert (y[:6] == 0).all() and (y[6:21] == 0).all() and (y[46:51] == 0).all()
    close(y, want, dtype)
    b.table[slots[3]] = [-1] * len(b.table[0])
    assert (b.run()[51:] == 0).all()
    b.lengths, b.slots = lens, [1 << 30, -7, 99, 6]
    assert (b.run()[:51] == 0).all()
    b.lengths[slots[1]] = -5
    b.slots = slots
    assert (b.run()[6:46] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_values_that_are_not_finite_reach_those_that_see_them(gpu_lib, dtype, value):
    """In the cached tokens, in the new ones (later tokens see them, earlier ones do not), behind the window."""
    for window, sinks, at in ((None, 0, 70), (None, 0, 130), (24, 2, 60), (24, 2, 1)):
        b = Batch([64, 3], [90, 20], 4, 2, 64, 16, dtype)
        plain = b.run(window=window, sinks=sinks)
        r = b.slots[0]
        b.vp[b.table[r][at // 16], 1, at % 16, 5] = value
        y = b.run(window=window, sinks=sinks)
        p = torch.arange(64, 154, device=DEV)
        sees = (at <= p) & ((p - at < (window or 1 << 20)) | (at < sinks))
        hit = torch.zeros(110, 4, 64, dtype=torch.bool, device=DEV)
        hit[:90][sees, 2:, 5] = True
        assert torch.equal(~torch.isfinite(y), hit)
        # rows of the tile may be formed in another order: they agree to the type's accuracy
        close(torch.where(hit, plain, y), plain.double().cpu(), dtype)


def test_long_row_past_32_bits(gpu_lib):
    """A pool whose last pages lie beyond 2^31 elements; few queries against many keys."""
    Hkv, D, page, n_pages = 2, 128, 128, 70000              # 2.3e9 elements
    kp = torch.zeros(n_pages, Hkv, page, D, dtype=torch.bfloat16, device=DEV)
    vp = torch.zeros_like(kp)
    g = torch.Generator().manual_seed(3)
    used = [n_pages - 1, 0, n_pages - 3, 66000, 5]
    for pg in used:
        kp[pg], vp[pg] = (torch.randn(Hkv, page, D, generator=g).bfloat16().to(DEV) for _ in range(2))
    q = torch.randn(9, 4, D, generator=g).bfloat16()
    table = [[used[i] for i in range(5)]]
    y = attention.paged_attention_chunk(q.to(DEV), kp, vp, i32(table), i32([600]), i32([0, 9]))
    small = torch.stack([kp[p].cpu() for p in used]), torch.stack([vp[p].cpu() for p in used])
    close(y, oa.paged_chunk(q, *small, [[0, 1, 2, 3, 4]], [600], [0, 9]), torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_rows(gpu_lib, dtype):
    """More rows than a wave looks at in one go, empty ones among them, against the single-token step."""
    n = 300
    past = [(37 * i) % 90 for i in range(n)]
    counts = [0 if i % 5 == 3 else 1 for i in range(n)]
    b = Batch(past, counts, 4, 2, 64, 16, dtype)
    y = b.run()
    named = [s for s, c in zip(b.slots, counts) if c]
    step = attention.paged_attention_step(b.q.to(DEV), None, None, b.kp.to(DEV), b.vp.to(DEV), i32(b.table),
                                          i32(b.lengths), slots=i32(named))
    close(y, step.double().cpu(), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [130, 1100])
def test_long_rows_among_many(gpu_lib, n, dtype):
    """Long rows first, last and between short and empty ones, of one tile, of several and of a pair more than a tile."""
    past, counts = [(11 * i) % 40 for i in range(n)], [(0, 1, 2, 1)[i % 4] for i in range(n)]
    for i, c in ((0, 70), (63, 33), (64, 129), (n // 2, 17), (n - 1, 65)):
        counts[i] = c
    b = Batch(past, counts, 4, 2, 64, 16, dtype)
    close(b.run(), b.want(), dtype)
    close(b.run(window=20, sinks=2), b.want(window=20, sinks=2), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 3)])
def test_prompt_in_pieces_is_the_whole(gpu_lib, dtype, window, sinks):
    """Two prompts of unlike lengths taken in by pieces beside each other, against windowed attention over each."""
    Hq, Hkv, D, page, lens = 8, 2, 64, 16, (230, 97)
    c = pages.PagedKVCache(64, page, Hkv, D, 4, 256, layers=2, dtype=dtype)
    qkv = [torch.randn(1, n, Hq + 2 * Hkv, D, device=DEV).to(dtype) for n in lens]
    rows, at, ys = c.alloc(2), [0, 0], [[], []]
    for take in ((100, 1), (1, 60), (0, 30), (129, 6)):
        packed = torch.cat([x[0, a:a + n] for x, a, n in zip(qkv, at, take)])
        q, k, v = packed.split([Hq, Hkv, Hkv], 1)
        plan = c.reserve_packed(rows, take, tokens=packed.shape[0])
        c.write_packed(plan, k, v, layer=1)
        y = c.chunk(1, rows, plan, q, window=window, sinks=sinks)
        for i, part in enumerate(y.split(list(take))):
            ys[i].append(part)
        at = [a + n for a, n in zip(at, take)]
    for i, x in enumerate(qkv):
        want = attention.window_attention(*x.split([Hq, Hkv, Hkv], 2), window, sinks)[0]
        close(torch.cat(ys[i]), want.double().cpu(), dtype)
    assert c.lens[rows[0]] == 230 and c.lens[rows[1]] == 97


def test_malformed_offsets_stay_in_the_batch(gpu_lib):
    b = Batch([30, 20, 10], [20, 30, 10], 4, 2, 64, 16, torch.bfloat16)
    guard = torch.full((64, 4, 64), 3.0, device=DEV).bfloat16()
    for off in ([50, 3, 1000, -9], [-5, 1 << 30, 0, 60], [60, 60, 60, 60], [7, 7, 7, 7]):
        b.offsets = off
        b.run(out=guard[:60])
        assert (guard[60:] == 3).all()


# ---- the bookkeeping ----
def _state(n_pages, rows, width):
    i = dict(dtype=torch.int32, device=DEV)
    return (torch.full((rows, width), -1, **i), torch.zeros(rows, **i), torch.zeros(n_pages, **i)), torch.zeros(2, **i)


@pytest.mark.parametrize("page", [1, 16, 64])
def test_reserve_packed(gpu_lib, page):
    """Several calls in a row, empty rows, rows without tokens, a batch larger than its tokens."""
    n_pages, rows, width = 400 if page < 64 else 40, 9, 90
    (table, lengths, refs), status = _state(n_pages, rows, width)
    o = oa.Pages(n_pages, page, rows, width)
    refs[[3, 4, 17]] = 1
    for p in (3, 4, 17):
        o.refs[p] = 1
    for slots, n_new, tokens in (([2, 0, 5], [30, 1, 0], 31), ([0, -1, 7, 2], [16, 5, 17, 1], 45), ([8], [64], 64),
                                 ([1, 99, 3, 4], [0, 0, -4, 0], 0), ([0, 2], [1, 1], 300)):
        plan = pages.pages_reserve_packed(table, lengths, refs, i32(slots), i32(n_new), page, status, tokens)
        want = o.reserve_packed(slots, n_new, tokens)
        assert [t.tolist() for t in plan] == [list(w) for w in want]
        assert table.tolist() == o.table() and lengths.tolist() == o.lens and refs.tolist() == o.refs
    assert status.tolist() == [0, 0]


@pytest.mark.parametrize("why", ["pool", "table", "batch"])
def test_reserve_packed_that_cannot_be_served(gpu_lib, why):
    (table, lengths, refs), status = _state(6, 4, 5)
    pages.pages_reserve_packed(table, lengths, refs, i32([1]), i32([20]), 16, status, 20)
    before = table.clone(), lengths.clone(), refs.clone()
    slots, n_new, tokens = {"pool": ([0, 2, 3], [40, 30, 1], 90), "table": ([0, 1], [3, 61], 90),
                            "batch": ([0, 2, 3], [10, 5, 5], 14)}[why]
    plan = pages.pages_reserve_packed(table, lengths, refs, i32(slots), i32(n_new), 16, status, tokens)
    assert status.tolist() == {"pool": [2, 0], "table": [0, 1], "batch": [0, 2]}[why]
    assert all(torch.equal(a, b) for a, b in zip(before, (table, lengths, refs)))
    assert (plan.offsets == 0).all() and all((t == -1).all() for t in plan[1:])
    # what follows such a plan does nothing
    kp, vp = torch.ones(6, 1, 16, 64, device=DEV), torch.ones(6, 1, 16, 64, device=DEV)
    pages.pages_write_packed(torch.zeros(tokens, 1, 64, device=DEV), torch.zeros(tokens, 1, 64, device=DEV), kp, vp, plan.places)
    out = torch.full((tokens, 1, 64), 4.0, device=DEV)
    attention.paged_attention_chunk(torch.ones(tokens, 1, 64, device=DEV), kp, vp, table, lengths, plan.offsets,
                                    slots=i32(slots), out=out)
    assert (kp == 1).all() and (vp == 1).all() and (out == 4).all()


def test_reserve_packed_many_rows(gpu_lib):
    """More rows than the bookkeeping takes in one step, more pages than it looks through in one."""
    n, page, n_pages, width = 2500, 16, 20000, 12
    g = torch.Generator().manual_seed(7)
    n_new = torch.randint(0, 150, (n,), generator=g).tolist()
    (table, lengths, refs), status = _state(n_pages, n + 5, width)
    o = oa.Pages(n_pages, page, n + 5, width)
    o.refs = torch.randint(0, 3, (n_pages,), generator=g).clamp(max=1).tolist()
    refs.copy_(i32(o.refs))
    slots = torch.randperm(n + 5, generator=g).tolist()[:n]
    n_new = [c if i % 3 else c // 30 for i, c in enumerate(n_new)]
    tokens = sum(n_new) + 11
    free = o.refs.count(0)
    need = sum(-(-c // page) for c in n_new)
    plan = pages.pages_reserve_packed(table, lengths, refs, i32(slots), i32(n_new), page, status, tokens)
    assert need > free and status.tolist() == [need - free, 0]
    n_new = [c // 3 for c in n_new]
    plan = pages.pages_reserve_packed(table, lengths, refs, i32(slots), i32(n_new), page, status, tokens)
    o._free = lambda free=[p for p, c in enumerate(o.refs) if c == 0]: list(free)
    want = o.reserve_packed(slots, n_new, tokens)
    assert [t.tolist() for t in plan] == [list(w) for w in want]
    assert table.tolist() == o.table() and refs.tolist() == o.refs and lengths.tolist() == o.lens


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layers", [None, 1, 3])
@pytest.mark.parametrize("N,Hkv,D,page", [(1, 1, 64, 1), (77, 3, 64, 16), (300, 2, 128, 32)])
def test_write_packed(gpu_lib, N, Hkv, D, page, layers, dtype):
    lead, n_pages = () if layers is None else (layers,), -(-N // page) + 9
    g = torch.Generator(device=DEV).manual_seed(N)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)  # noqa: E731
    kp, vp = r(*lead, n_pages, Hkv, page, D), r(*lead, n_pages, Hkv, page, D)
    k, v = r(*lead, N, 3 * Hkv, D)[..., Hkv:2 * Hkv, :], r(*lead, N, Hkv, D)
    places = torch.randperm(n_pages * page, generator=g, device=DEV)[:N].int()
    if N > 5:
        places[3], places[5] = -1, n_pages * page + 2
    want = kp.clone(), vp.clone()
    for t, p in enumerate(places.tolist()):
        if 0 <= p < n_pages * page:
            for pool, x in zip(want, (k, v)):
                pool[..., p // page, :, p % page, :] = x[..., t, :, :]
    pages.pages_write_packed(k, v, kp, vp, places)
    assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])


def test_cache_refuses_before_it_changes(gpu_lib):
    c = pages.PagedKVCache(8, 16, 1, 64, 3, 64)
    rows = c.alloc(2)
    with pytest.raises(ValueError, match="the table holds"):
        c.reserve_packed(rows, [3, 65])
    with pytest.raises(ValueError, match="tokens in a batch"):
        c.reserve_packed(rows, [3, 4], tokens=6)
    with pytest.raises(ValueError, match="every row"):
        c.reserve_packed(rows, [3])
    with pytest.raises(ValueError, match="every row"):
        c.reserve_packed(rows, [3, -1])
    plan = c.reserve_packed(rows, [64, 60])
    assert c.lens[rows[0]] == 64 and plan.places.numel() == 124 and c.pages_in_use() == 8
    other = c.alloc(1)
    with pytest.raises(RuntimeError, match="page cache full"):
        c.reserve_packed(other, [1])
    assert c.lens[other[0]] == 0 and c.pages_in_use() == 8


def test_graph_of_a_mixed_step(gpu_lib):
    """reserve, write and attention of a packed batch captured together; every replay equals the eager calls."""
    Hq, Hkv, D, page, N = 4, 2, 64, 16, 24
    def state():
        (table, lengths, refs), status = _state(90, 5, 20)
        g = torch.Generator(device=DEV).manual_seed(2)
        pools = [torch.randn(90, Hkv, page, D, generator=g, device=DEV).bfloat16() for _ in range(2)]
        return dict(table=table, lengths=lengths, refs=refs, status=status, kp=pools[0], vp=pools[1],
                    y=torch.zeros(N, Hq, D, device=DEV).bfloat16())
    qkv, n_new, slots = torch.zeros(N, Hq + 2 * Hkv, D, device=DEV).bfloat16(), i32([0, 0, 0, 0]), i32([3, 0, -1, 4])
    def step(s):
        plan = pages.pages_reserve_packed(s["table"], s["lengths"], s["refs"], slots, n_new, page, s["status"], N)
        q, k, v = qkv.split([Hq, Hkv, Hkv], 1)
        pages.pages_write_packed(k, v, s["kp"], s["vp"], plan.places)
        attention.paged_attention_chunk(q, s["kp"], s["vp"], s["table"], s["lengths"], plan.offsets, slots=slots,
                                        window=60, sinks=2, out=s["y"])
        return plan
    a, b = state(), state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(state())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(b)
    for turn in range(8):
        qkv.copy_(torch.randn(qkv.shape, device=DEV))
        n_new.copy_(i32([(5 * turn) % 13, 1, 2, 0 if turn == 3 else 8]))
        want = step(a)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, got)), turn
        assert all(torch.equal(a[n], b[n]) for n in a), turn
