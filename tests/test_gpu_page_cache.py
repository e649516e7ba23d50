"""PagedKVCache's calls beside the device: which of them wait for it, and which rows they name."""
import pytest
import torch

from gdnx_amd import pages

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture
def no_waits():
    """Any wait for the device raises."""
    torch.zeros(1, device=DEV).sum().item()
    torch.cuda.set_sync_debug_mode("error")
    yield
    torch.cuda.set_sync_debug_mode("default")


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_serving_does_not_wait_for_the_device(gpu_lib, no_waits, mode):
    with mode():
        serve()


def serve():
    c = pages.PagedKVCache(64, 16, 2, 64, 8, 256)
    rows = c.alloc(3)
    x = lambda *s: torch.zeros(*s, 64, dtype=torch.bfloat16, device=DEV)
    c.write(rows, c.reserve(rows, 20), x(1, 3, 20, 2), x(1, 3, 20, 2))
    rows += c.fork([rows[0], rows[0]])
    rt = c.rows_tensor(rows)
    for named in (rows, rt, tuple(rows), rt):
        c.reserve(named)
        c.step(0, named, x(5, 4), x(5, 2), x(5, 2), window=8)
        c.trim(named, 8)
    c.compact()
    c.free(rt)
    torch.cuda.set_sync_debug_mode("default")
    assert c.lens == [0] * 8 and (c.lengths == 0).all() and c.pages_in_use() == 0


def test_rows_arrive_in_order(gpu_lib):
    """Many uploads behind work that is still queued: each call gets its own rows."""
    n, turns = 64, 40
    c = pages.PagedKVCache(n * 3, 16, 1, 64, n, 48)
    rows = c.alloc(n)
    big = torch.zeros(1 << 28, device=DEV)
    g = torch.Generator().manual_seed(0)
    want = [0] * n
    for _ in range(turns):
        big.add_(1.0)
        some = [rows[i] for i in torch.randperm(n, generator=g)[:7].tolist()]
        c.reserve(some)
        for r in some:
            want[r] += 1
    assert c.lengths.tolist() == want == c.lens


def test_rows_by_any_tensor(gpu_lib):
    c = pages.PagedKVCache(16, 16, 1, 64, 4, 64)
    rows = c.alloc(2)
    rt = c.rows_tensor(rows)
    c.reserve(rt, 3)
    c.reserve(torch.tensor(rows[:1]), 2)                 # read back, and taken in 64 bits too
    assert c.lens[rows[0]] == 5 and c.lens[rows[1]] == 3 and c.lengths.tolist() == c.lens
    c.reserve(rt.repeat_interleave(2)[::2])              # a view with gaps
    assert c.lengths.tolist() == c.lens == [6, 4, 0, 0]
    rt[0] = rt[1]                                        # changed since: what it was made of no longer holds
    with pytest.raises(ValueError, match="twice"):
        c.reserve(rt)
    rt[0] = 3
    with pytest.raises(ValueError, match="not allocated"):
        c.free(rt)
    c.free(rows)
    with pytest.raises(ValueError, match="not allocated"):
        c.reserve(c.rows_tensor(rows))


def test_rows_named_as_ints_are_not_captured(gpu_lib):
    """Their upload would be of memory that is used again by the next one."""
    c = pages.PagedKVCache(16, 16, 1, 64, 4, 64)
    rows = c.alloc(2)
    rt = c.rows_tensor(rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.reserve(rt)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pages.pages_reserve(c.table, c.lengths, c.refs, rt, 1, c.page, c.status)
        with pytest.raises(RuntimeError, match="captured"):
            c.reserve(rows)
        with pytest.raises(RuntimeError, match="captured"):
            c.fork(rows)
    assert len(c.alloc(2)) == 2 and c.lens == [1, 1, 0, 0]      # (nothing was taken)
    for n in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert [c.lengths.tolist()[r] for r in rows] == [n + 2] * 2
