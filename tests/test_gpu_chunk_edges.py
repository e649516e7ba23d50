"""Packed rows over the page cache: values that are not finite in rows of both kinds, whole and cut into parts and spans."""
import pytest
import torch

from test_gpu_chunk import DEV, Batch, close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what,value", [("v", float("nan")), ("v", float("inf")), ("k", float("nan"))])
@pytest.mark.parametrize("past,counts", [([64, 3], [5, 4]), ([1500, 900], [5, 4]), ([1500, 900], [1, 5]),
                                         ([1500, 3], [90, 20]), ([1500, 900], [90, 5])],
                         ids=["short", "spans", "single", "parts", "both"])
def test_what_is_not_finite_reaches_those_that_see_it(gpu_lib, past, counts, what, value, D, dtype):
    """Among the cached tokens, the new ones, and where the window leaves it behind between one new token and the next."""
    for window, sinks, back in ((None, 0, 40), (None, 0, 0), (None, 0, -1), (None, 0, 1 - counts[0]), (24, 2, 22), (24, 2, 30),
                                (24, 2, past[0] - 1)):
        at = past[0] - back                                # its position in the first row
        b = Batch(past, counts, 4, 2, D, 16, dtype)
        if at >= b.lens[0]:
            continue
        plain = b.run(window=window, sinks=sinks)
        pool = b.vp if what == "v" else b.kp
        pool[b.table[b.slots[0]][at // 16], 1, at % 16, 5] = value
        y = b.run(window=window, sinks=sinks)
        p = torch.arange(past[0], past[0] + counts[0], device=DEV)
        sees = (at <= p) & ((p - at < (window or 1 << 20)) | (at < sinks))
        hit = torch.zeros(sum(counts), 4, D, dtype=torch.bool, device=DEV)
        columns = slice(5, 6) if what == "v" else slice(None)
        hit[:counts[0]][sees, 2:, columns] = True
        assert torch.equal(~torch.isfinite(y), hit), (window, back)
        close(torch.where(hit, plain, y), plain.double().cpu(), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Hq", [1, 3])
def test_odd_parts_before_spans(gpu_lib, Hq, dtype):
    """An odd number of tokens, heads and parts of long rows, beside short rows in several spans."""
    for past in (800, 1100):
        b = Batch([past, past - 30, past - 7], [41, 1, 1], Hq, Hq, 64, 16, dtype)
        close(b.run(), b.want(), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("window,sinks", [(None, 0), (300, 5)])
@pytest.mark.parametrize("past,count", [(1500, 1), (0, 1), (2000, 4), (40, 3)])
def test_a_short_row_in_a_batch_of_a_fixed_size(gpu_lib, past, count, window, sinks, dtype):
    """Alone or before tokens of nobody it is the same row, served the same way: equal bit for bit."""
    b = Batch([past], [count], 4, 2, 64, 16, dtype)
    alone = b.run(window=window, sinks=sinks)
    close(alone, b.want(window=window, sinks=sinks), dtype)
    for N in (17, 300, 2048):
        q = torch.full((N, 4, 64), float("nan"), device=DEV).to(dtype)
        q[:count] = b.q.to(DEV)
        out = torch.full((N, 4, 64), 5.0, device=DEV).to(dtype)
        y = b.run(q, window=window, sinks=sinks, out=out)
        assert torch.equal(y[:count], alone) and (y[count:] == 5).all(), N


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [3, 400])
def test_a_batch_whose_first_tokens_are_nobodys(gpu_lib, n, dtype):
    """Offsets may begin anywhere: long, short and empty rows behind 37 tokens that no row has."""
    past, counts = [(11 * i) % 40 for i in range(n)], [(1, 0, 2)[i % 3] for i in range(n)]
    counts[0], counts[n // 2] = 70, 19
    b = Batch(past, counts, 4, 2, 64, 16, dtype)
    want, N = b.want(window=30, sinks=2), b.q.shape[0]
    b.offsets = [37 + o for o in b.offsets]
    q = torch.full((37 + N + 5, 4, 64), float("nan"), device=DEV).to(dtype)
    q[37:37 + N] = b.q.to(DEV)
    out = torch.full_like(q, 5.0)
    b.run(q, window=30, sinks=2, out=out)
    assert (out[:37] == 5).all() and (out[37 + N:] == 5).all()
    close(out[37:37 + N], want, dtype)
