"""The attention oracle on the CPU: against torch's own differentiation and
differences, and its special cases."""
import pytest
import torch

from oracle import attention as oa


def _x(B, Tq, Tk, Hq, Hkv, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    return r(B, Tq, Hq, D), r(B, Tk, Hkv, D), r(B, Tk, Hkv, D), r(B, Tq, Hq, D)


@pytest.mark.parametrize("Tq,Tk,window,sinks,lengths", [
    (7, 7, None, 0, None), (7, 7, 3, 0, None), (7, 7, 3, 2, [7, 4]), (3, 9, 2, 1, [9, 0]), (9, 5, 4, 1, [5, 2])])
def test_gradients_by_formula_and_by_differences(Tq, Tk, window, sinks, lengths):
    q, k, v, dy = _x(2, Tq, Tk, 4, 2, 3)
    _, _, dq, dk, dv = oa.attention(q, k, v, window, sinks, None, lengths, dy)
    f = lambda a, b, c: float((oa.attention(a, b, c, window, sinks, None, lengths)[0] * dy).sum())
    g = torch.Generator().manual_seed(1)
    for i, (x, dx) in enumerate(((q, dq), (k, dk), (v, dv))):
        d = torch.randn(x.shape, generator=g, dtype=torch.float64)
        step = lambda h: [a + h * d if n == i else a for n, a in enumerate((q, k, v))]
        # central differences in 64 bits: an error of order h^2 = 1e-10 beside values of order 1 to 10
        num = (f(*step(1e-5)) - f(*step(-1e-5))) / 2e-5
        assert abs(num - float((dx * d).sum())) < 1e-7 * max(1.0, abs(num))


def test_hidden_places_may_hold_anything():
    q, k, v, dy = _x(1, 6, 6, 1, 1, 4)
    a = oa.attention(q, k, v, 3, 1, None, [4], dy)
    k2, v2, q2 = k.clone(), v.clone(), q.clone()
    k2[0, 4:], v2[0, 4:], q2[0, 4:] = float("nan"), float("inf"), float("nan")
    b = oa.attention(q2, k2, v2, 3, 1, None, [4], dy)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert (a[0][0, 4:] == 0).all() and torch.isinf(a[1][0, 0, 4:]).all()


def test_matches_a_softmax_over_everything():
    q, k, v, _ = _x(1, 5, 5, 2, 1, 4)
    y, lse = oa.attention(q, k, v)
    s = torch.einsum("ihd,jd->hij", q[0], k[0, :, 0]) / 2.0
    s = s.masked_fill(~torch.tril(torch.ones(5, 5, dtype=torch.bool)), float("-inf"))
    assert torch.allclose(y[0], torch.einsum("hij,jd->ihd", s.softmax(-1), v[0, :, 0]), atol=1e-14)
    assert torch.allclose(lse[0], s.logsumexp(-1), atol=1e-14)


def test_page_lists():
    c = oa.Pages(6, 4, 3, 4)
    assert c.reserve([0, 1], 5) == [0, 0] and c.rows[:2] == [[0, 1], [2, 3]]
    assert c.fork([0], [2]) == [(1, 4)] and c.rows[2] == [0, 4] and c.refs == [2, 1, 1, 1, 1, 0]
    assert c.reserve([0], 8) is None
    c.free([1])
    assert c.compact() == [(4, 2)] and c.rows == [[0, 1], [], [0, 2]] and c.refs == [2, 1, 1, 0, 0, 0]
