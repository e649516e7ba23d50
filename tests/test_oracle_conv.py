"""The 64-bit statement of the short convolution: against a library convolution, and its gradients against differences."""
import torch
import torch.nn.functional as F

from oracle import conv as oc


def test_against_a_library_convolution():
    g = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((2, 9, 5), (5, 4), (5,)))
    y, last = oc.causal_conv(x, w, b)
    want = F.silu(F.conv1d(F.pad(x.transpose(1, 2), (3, 0)), w[:, None], b, groups=5)).transpose(1, 2)
    assert torch.allclose(y, want, atol=1e-12) and torch.equal(last, x[:, -3:])


def test_a_sequence_in_pieces_is_the_whole():
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(1, 11, 3, generator=g, dtype=torch.float64), torch.randn(3, 4, generator=g, dtype=torch.float64)
    whole, last = oc.causal_conv(x, w)
    state, ys = torch.zeros(1, 3, 3, dtype=torch.float64), []
    for a, b in ((0, 1), (1, 3), (3, 3), (3, 11)):
        y, state = oc.causal_conv(x[:, a:b], w, state=state)
        ys.append(y)
    assert torch.allclose(torch.cat(ys, 1), whole, atol=1e-14) and torch.equal(state, last)
    y, pool = oc.causal_conv_packed(x[0], [0, 4, 4, 11], torch.zeros(3, 3, 3, dtype=torch.float64), w, slots=[2, 0, 7])
    assert torch.equal(y[:4], whole[0, :4]) and (y[4:] == 0).all() and torch.equal(pool[2], x[0, 1:4])


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64, requires_grad=True)  # noqa: E731
    ins = r(2, 5, 3), r(3, 4), r(3), r(2, 3, 3)
    for lengths in (None, [5, 2], [0, 1]):
        assert torch.autograd.gradcheck(lambda *a: oc.causal_conv(*a, lengths), ins)


def test_gradients_against_the_formulas():
    g = torch.Generator().manual_seed(3)
    T, C, W = 7, 2, 3
    x, w, dy = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((1, T, C), (C, W), (1, T, C)))
    leaves = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y, _ = oc.causal_conv(*leaves)
    dx, dw = torch.autograd.grad(y, leaves, dy)
    pad = torch.cat([torch.zeros(1, W - 1, C, dtype=torch.float64), x], 1)
    u = sum(pad[:, j:j + T] * w[:, j] for j in range(W))
    s = torch.sigmoid(u)
    du = dy * s * (1 + u * (1 - s))
    after = torch.cat([du, torch.zeros(1, W - 1, C, dtype=torch.float64)], 1)
    assert torch.allclose(dx, sum(after[:, k:k + T] * w[:, W - 1 - k] for k in range(W)), atol=1e-13)
    assert torch.allclose(dw, torch.stack([(du * pad[:, j:j + T]).sum((0, 1)) for j in range(W)], 1), atol=1e-13)
