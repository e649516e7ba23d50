"""Drafts tried and taken back: by lowering a row's length, whose pages are not lost then, and on a fork."""
import pytest
import torch

from gdnx_amd import attention, pages

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def consistent(table, refs):
    """Every page's count is the number of entries that name it."""
    named = torch.zeros_like(refs)
    at = table[(table >= 0) & (table < refs.numel())].long()
    named.index_add_(0, at, torch.ones_like(at, dtype=torch.int32))
    return torch.equal(named, refs)


def state(n_pages, rows, width):
    i = dict(dtype=torch.int32, device=DEV)
    return torch.full((rows, width), -1, **i), torch.zeros(rows, **i), torch.zeros(n_pages, **i), torch.zeros(2, **i)


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("page", [1, 4, 16])
def test_lengths_may_be_lowered(gpu_lib, page, packed):
    """The pool holds what three rows of 160 tokens and 40 new ones take: a page lost at a time would soon be missing."""
    n_pages = 600 // page + 8
    table, lengths, refs, status = state(n_pages, 6, 16 * 16 // page)
    slots, g = i32([4, 0, 3]), torch.Generator().manual_seed(page)
    want = [0, 0, 0]
    for turn in range(60):
        new = torch.randint(0, 40, (3,), generator=g).tolist() if packed else [int(torch.randint(1, 40, (1,), generator=g))] * 3
        if packed:
            plan = pages.pages_reserve_packed(table, lengths, refs, slots, i32(new), page, status, sum(new))
            assert (plan.places >= 0).all() and plan.start.tolist() == want
        else:
            assert pages.pages_reserve(table, lengths, refs, slots, new[0], page, status).tolist() == want
        assert status.tolist() == [0, 0] and consistent(table, refs)
        for r, w, c in zip((4, 0, 3), want, new):        # every token has a page of its own row
            assert (table[r, :-(-(w + c) // page)] >= 0).all()
        # a few of the new tokens stay; now and then some older ones go too
        want = [max(0, min(w + c, w + int(torch.randint(-9, 12, (1,), generator=g)), 120)) for w, c in zip(want, new)]
        lengths[[4, 0, 3]] = i32(want)
    pages.pages_free(table, lengths, refs, slots)
    assert not refs.any() and (table == -1).all()


def test_a_lowered_row_as_a_forks_child(gpu_lib):
    table, lengths, refs, status = state(40, 4, 8)
    kp, vp = torch.zeros(40, 1, 16, 64, device=DEV), torch.zeros(40, 1, 16, 64, device=DEV)
    pages.pages_reserve_packed(table, lengths, refs, i32([0, 1, 2]), i32([70, 100, 33]), 16, status, 203)
    lengths[[1, 2]] = 0                                  # emptied, but not freed
    pages.pages_fork(kp, vp, table, lengths, refs, i32([0, 0]), i32([1, 2]), status)
    assert lengths.tolist()[:3] == [70] * 3 and status.tolist() == [0, 0]
    assert consistent(table, refs)
    pages.pages_free(table, lengths, refs, i32([0, 1, 2]))
    assert not refs.any()


def alike(a, b):
    """The same keys seen, beside other tokens: both rounded once (2^-8 and 2^-24 of the value at most), after float32 sums of
    up to 150 terms whose maxima may differ."""
    return torch.allclose(a.float(), b.float(), rtol=2.0 ** -6 if a.dtype == torch.bfloat16 else 1e-4, atol=1e-4)


def _chunk(kp, vp, table, lengths, refs, status, slots, parts):
    """The packed tokens q, k, v [n,3,64] of every row, reserved, written and attended over."""
    x = torch.cat(parts)
    plan = pages.pages_reserve_packed(table, lengths, refs, slots, i32([len(p) for p in parts]), 16, status, len(x))
    pages.pages_write_packed(x[:, 1:2], x[:, 2:], kp, vp, plan.places)
    return attention.paged_attention_chunk(x[:, :1], kp, vp, table, lengths, plan.offsets, slots=slots).split([len(p) for p in parts])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_drafts_over_page_ends(gpu_lib, dtype):
    """Drafts of seven tokens, of which some stay: what they attend over is the sequence without those that went."""
    g = torch.Generator(device=DEV).manual_seed(1)
    r = lambda n: torch.randn(n, 3, 64, generator=g, device=DEV).to(dtype)  # noqa: E731
    st, ref = state(24, 3, 10), state(24, 3, 10)
    pools = [torch.zeros(24, 1, 16, 64, dtype=dtype, device=DEV) for _ in range(4)]
    slots = i32([2, 0])
    start = [r(13), r(30)]
    _chunk(*pools[:2], *st, slots, start)
    _chunk(*pools[2:], *ref, slots, start)
    for turn in range(20):
        draft, keep = [r(7), r(7)], [turn % 4 + 1, (turn * 3) % 5]
        got = _chunk(*pools[:2], *st, slots, draft)
        st[1][[2, 0]] -= i32([7 - k for k in keep])
        want = _chunk(*pools[2:], *ref, slots, [d[:k] for d, k in zip(draft, keep)])
        assert all(alike(a[:k], b) for a, b, k in zip(got, want, keep))
        assert consistent(st[0], st[2]) and torch.equal(st[1], ref[1])
    pages.pages_free(*st[:3], slots)
    assert not st[2].any()


def test_drafts_on_a_fork(gpu_lib):
    """The cache that keeps lengths on the host: a draft is tried on a fork, and what stays is written to the row."""
    c = pages.PagedKVCache(14, 16, 1, 64, 4, 160)
    g = torch.Generator(device=DEV).manual_seed(2)
    r = lambda n: torch.randn(n, 3, 64, generator=g, device=DEV).bfloat16()  # noqa: E731
    row = c.alloc(1)
    def put(rows, x):
        plan = c.reserve_packed(rows, [len(x)])
        c.write_packed(plan, x[:, 1:2], x[:, 2:], layer=0)
        return c.chunk(0, rows, plan, x[:, :1])
    put(row, r(14))
    for turn in range(30):
        draft, keep = r(9), turn % 4 + 1
        kid = c.fork(row)
        tried = put(kid, draft)
        c.free(kid)
        kept = put(row, draft[:keep])
        assert alike(kept, tried[:keep])
        assert c.pages_in_use() == -(-c.lens[row[0]] // 16) and consistent(c.table, c.refs)
    assert c.lens[row[0]] == 14 + sum(t % 4 + 1 for t in range(30))
