"""The short causal convolution on the GPU against the 64-bit oracle.

Tolerances.  Inputs, filters and biases are of unit size.  A float32 u is a sum
of W + 1 products, wrong by (W + 1) 2^-24 of the sum S of their sizes at most;
its exponential by (|u| + 4) 2^-24 of itself, |u| <= S; the activation and its
derivative are at most S and 1.1 and change by at most 1.1 and 0.5 for a unit of
u, so y and du are wrong by (W + 1 + S + 8) 2^-24 S, and with W <= 8 and S of
up to 30 by 47 * 2^-24 of S at worst: 3e-6 S, 30 times smaller in the mean.  dx sums W such
terms.  Relative L2: 3e-6 for y and dx in float32.  A filter's gradient is a sum
of n terms of random sign in spans of 64, rows and blocks: at most (64 + 32 +
blocks) 2^-24 of the terms' sizes, whose sum is about sqrt(n) the gradient's: with
n to 2000 and blocks to 40, 136 * 45 * 2^-24 = 4e-4 at the very worst, and about
the square root of the additions, 12 * 2^-24 * 45 / 12, in the mean: 2e-5.
bfloat16 outputs are rounded once, by at most 2^-8 of the value: 2^-8 of it and the float32 error
above.  States are moved, not computed.
"""
import pytest
import torch

from gdnx_amd import conv
from oracle import conv as oc

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = 2.0 ** -8


def rel(got, want):
    got, want = got.detach().double().cpu(), want.detach()
    return float((got - want).norm() / want.norm()) if want.norm() > 0 else float(got.norm())


def tol(dtype, f32):
    return f32 + (HALF if dtype == torch.bfloat16 else 0.0)


def make(B, T, C, W, dtype, wdtype=torch.float32, bias=True, state=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return dict(x=r(B, T, C).to(dtype), weight=r(C, W).to(wdtype), bias=r(C).to(wdtype) if bias else None,
                state=r(B, W - 1, C).to(dtype) if state else None)


def check(ins, lengths=None, silu=True, seed=5, put=lambda n, t: t.to(DEV)):
    leaves = {n: put(n, t).requires_grad_(True) for n, t in ins.items() if t is not None}
    ref = {n: t.double().requires_grad_(True) for n, t in ins.items() if t is not None}
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    y, last = conv.causal_conv(leaves["x"], leaves["weight"], leaves.get("bias"), activation="silu" if silu else None,
                               state=leaves.get("state"), lengths=ln, return_state=True)
    want, wlast = oc.causal_conv(ref["x"], ref["weight"], ref.get("bias"), ref.get("state"), lengths, silu)
    g = torch.Generator().manual_seed(seed)
    dy, dlast = (torch.randn(t.shape, generator=g).to(y.dtype) for t in (want, wlast))
    got = torch.autograd.grad((y, last), list(leaves.values()), (dy.to(DEV), dlast.to(DEV)))
    exact = torch.autograd.grad((want, wlast), list(ref.values()), (dy.double(), dlast.double()), allow_unused=True)
    assert torch.equal(last.detach().double().cpu(), wlast.detach())
    assert rel(y, want) <= tol(y.dtype, 3e-6)
    assert ((y.detach().double().cpu() - want.detach()).abs() <= tol(y.dtype, 0) * want.detach().abs() + 1e-4).all()
    for (n, t), a, b in zip(leaves.items(), got, exact):
        assert a.shape == t.shape and a.dtype == t.dtype
        b = torch.zeros_like(ref[n]) if b is None else b
        assert rel(a, b) <= tol(a.dtype, 2e-5 if n in ("weight", "bias") else 3e-6), n
    with torch.no_grad():
        y2 = conv.causal_conv(leaves["x"], leaves["weight"], leaves.get("bias"), activation="silu" if silu else None,
                              state=leaves.get("state"), lengths=ln)
    assert torch.equal(y, y2)
    again = torch.autograd.grad(conv.causal_conv(leaves["x"], leaves["weight"], leaves.get("bias"),
                                                 activation="silu" if silu else None, state=leaves.get("state"),
                                                 lengths=ln, return_state=True),
                                list(leaves.values()), (dy.to(DEV), dlast.to(DEV)))
    assert all(torch.equal(a, b) for a, b in zip(got, again))            # (no sum depends on timing)
    return leaves, y, got


SHAPES = [
    # B, T, C, W, lengths
    (1, 1, 1, 2, None),
    (1, 1, 8, 4, None),
    (2, 2, 7, 4, None),                    # fewer tokens than taps
    (1, 3, 64, 8, None),
    (3, 9, 33, 5, [9, 0, 4]),
    (2, 64, 512, 4, None),                 # a span exactly
    (2, 65, 513, 3, [65, 1]),
    (4, 130, 100, 6, [130, 129, 2, 7]),
    (1, 700, 24, 7, None),
    (2, 515, 768, 4, [515, 300]),
    (5, 8, 1030, 4, [8, -3, 99, 3, 2]),    # lengths beyond both ends
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[:4])))
def test_causal_conv(gpu_lib, shape, dtype):
    B, T, C, W, lengths = shape
    check(make(B, T, C, W, dtype), lengths)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("silu", [False, True])
def test_options(gpu_lib, bias, state, silu):
    check(make(2, 37, 48, 4, torch.bfloat16, torch.bfloat16, bias, state), [37, 20], silu)
    check(make(2, 37, 48, 3, torch.float32, torch.float32, bias, state), None, silu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views(gpu_lib, dtype):
    """A slice of a fused projection, at an odd place; transposed tokens; a filter kept [C,1,W]."""
    ins = make(2, 70, 40, 4, dtype)
    def slice_of(n, t):
        if n == "x":
            wide = torch.randn(2, 70, 40 + 23, device=DEV).to(dtype)
            wide[..., 3:43] = t.to(DEV)
            return wide[..., 3:43].detach()
        return t.to(DEV)
    def transposed(n, t):
        if n == "x":
            return t.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
        if n == "state":
            return t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
        return t.to(DEV)
    a, b, c = check(ins), check(ins, put=slice_of), check(ins, put=transposed)
    assert torch.equal(a[1], b[1]) and torch.equal(a[1], c[1])
    assert all(torch.equal(p, q) and torch.equal(p, r) for p, q, r in zip(a[2], b[2], c[2]))
    channels_first = ins["x"].transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    with torch.no_grad():
        y = conv.causal_conv(channels_first, ins["weight"].to(DEV)[:, None], ins["bias"].to(DEV), state=ins["state"].to(DEV))
        one = conv.causal_conv(ins["x"][:1].to(DEV).expand(3, 70, 40), ins["weight"].to(DEV))       # a broadcast row
    assert torch.equal(a[1], y) and torch.equal(one[0], one[2])
    w3 = ins["weight"].to(DEV)[:, None].requires_grad_(True)
    assert torch.autograd.grad(conv.causal_conv(channels_first, w3).float().sum(), w3)[0].shape == w3.shape


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_padding_may_hold_anything(gpu_lib, dtype):
    ins = make(2, 50, 24, 4, dtype)
    a = check(ins, [31, 0])
    bad = dict(ins, x=ins["x"].clone())
    bad["x"][0, 31:], bad["x"][1] = float("nan"), float("inf")
    leaves = {n: t.to(DEV).requires_grad_(True) for n, t in bad.items()}
    ln = torch.tensor([31, 0], dtype=torch.int32, device=DEV)
    y, last = conv.causal_conv(leaves["x"], leaves["weight"], leaves["bias"], state=leaves["state"], lengths=ln,
                               return_state=True)
    g = torch.Generator().manual_seed(5)
    dy = torch.randn(y.shape, generator=g).to(dtype).to(DEV)
    dlast = torch.randn(last.shape, generator=g).to(dtype).to(DEV)
    dy[0, 31:], dy[1] = float("nan"), float("-inf")
    got = torch.autograd.grad((y, last), list(leaves.values()), (dy, dlast))
    assert torch.equal(y, a[1]) and all(torch.equal(p, q) for p, q in zip(got, a[2]))
    assert (y[0, 31:] == 0).all() and (y[1] == 0).all() and (got[0][0, 31:] == 0).all() and (got[0][1] == 0).all()


def test_large_values(gpu_lib):
    """Where sigmoid is 0 or 1 in float32: y = 0 and u, derivatives 0 and 1; a value that is not finite reaches W tokens."""
    x = torch.tensor([-3e4, 3e4, -200.0, 200.0, 90.0, -90.0], device=DEV).view(1, 6, 1).requires_grad_(True)
    w = torch.tensor([[0.0, 1.0]], device=DEV)
    y = conv.causal_conv(x, w)
    dx, = torch.autograd.grad(y.sum(), x)
    assert torch.allclose(y.flatten(), torch.tensor([0, 3e4, 0, 200, 90, 0.0], device=DEV), atol=1e-30)
    assert torch.allclose(dx.flatten(), torch.tensor([0, 1, 0, 1, 1, 0.0], device=DEV), atol=1e-30)
    x = torch.ones(1, 9, 3, device=DEV)
    x[0, 4, 1] = float("nan")
    y = conv.causal_conv(x, torch.ones(3, 4, device=DEV))
    bad = torch.isnan(y)
    assert bad[0, 4:8, 1].all() and int(bad.sum()) == 4


def test_empty_and_unused_gradients(gpu_lib):
    w = torch.randn(6, 4, device=DEV, requires_grad=True)
    st = torch.randn(2, 3, 6, device=DEV, requires_grad=True)
    x = torch.randn(2, 0, 6, device=DEV, requires_grad=True)
    y, last = conv.causal_conv(x, w, state=st, return_state=True)
    assert y.shape == (2, 0, 6) and torch.equal(last, st)
    gx, gw, gs = torch.autograd.grad(y.sum() + last.sum(), (x, w, st))
    assert gx.shape == x.shape and (gw == 0).all() and (gs == 1).all()
    assert conv.causal_conv(torch.randn(0, 5, 6, device=DEV), w.detach()).shape == (0, 5, 6)
    x = torch.randn(2, 5, 6, device=DEV, requires_grad=True)
    y, last = conv.causal_conv(x, w, state=st, return_state=True)
    g1 = torch.autograd.grad(last.sum(), (x, w, st), retain_graph=True)          # the state alone
    assert (g1[0][:, 2:] == 1).all() and (g1[0][:, :2] == 0).all() and (g1[1] == 0).all() and (g1[2] == 0).all()
    g2 = torch.autograd.grad(y.sum(), (x, w, st))
    assert all(torch.isfinite(t).all() for t in g2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("counts", [[1], [0], [5, 0, 1, 17, 1], [1] * 70, [0, 0, 3, 0], [40, 300, 2], [2, 3, 4, 8, 9]],
                         ids=lambda c: "-".join(map(str, c[:5])))
def test_packed(gpu_lib, counts, dtype):
    n, N, C, W, tail = len(counts), sum(counts), 43, 4, 6
    g = torch.Generator().manual_seed(n)
    x, pool = torch.randn(N + tail, C, generator=g).to(dtype), torch.randn(2 * n + 3, W - 1, C, generator=g).to(dtype)
    w, b = torch.randn(C, W, generator=g), torch.randn(C, generator=g)
    off = [sum(counts[:i]) for i in range(n + 1)]
    perm = torch.randperm(2 * n + 3, generator=g).tolist()
    slots, to = perm[:n], perm[n:2 * n]
    if n > 4:
        slots[1], to[4], slots[3] = -1, 1 << 20, 1 << 30        # empty rows, a state that goes nowhere
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    for dst in (None, to):
        want, wpool = oc.causal_conv_packed(x.double(), off, pool.double(), w.double(), b.double(), slots, dst)
        p = pool.to(DEV)
        out = torch.full((N + tail, C), 7.0, device=DEV).to(dtype)
        y = conv.causal_conv_packed(x.to(DEV), i32(off), p, w.to(DEV), b.to(DEV), slots=i32(slots),
                                    to_slots=None if dst is None else i32(dst), out=out)
        assert y is out and (y[N:] == 7).all()
        assert torch.equal(p.double().cpu(), wpool)
        if N:
            assert rel(y[:N], want[:N]) <= tol(dtype, 3e-6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pieces_and_steps_are_the_whole(gpu_lib, dtype):
    """A sequence taken in by pieces and single tokens gives what one call gives, bit for bit."""
    C, W, T = 520, 4, 50
    x, w = torch.randn(2, T, C, device=DEV).to(dtype), torch.randn(C, W, device=DEV)
    whole, last = conv.causal_conv(x, w, return_state=True)
    pool, ys = torch.zeros(2, W - 1, C, device=DEV, dtype=dtype), []
    at = 0
    for n in (3, 1, 20, 2):
        part = x[:, at:at + n].reshape(2 * n, C)
        off = torch.tensor([0, n, 2 * n], dtype=torch.int32, device=DEV)
        ys.append(conv.causal_conv_packed(part, off, pool, w).view(2, n, C))
        at += n
    for t in range(at, T):
        ys.append(conv.causal_conv_step(x[:, t], pool, w)[:, None])
    assert torch.equal(torch.cat(ys, 1), whole) and torch.equal(pool, last)


def test_malformed_offsets_stay_in_the_batch(gpu_lib):
    """Offsets that fall or leave the batch: some answer, nothing outside touched."""
    x, pool = torch.randn(40, 16, device=DEV), torch.randn(4, 3, 16, device=DEV)
    w = torch.randn(16, 4, device=DEV)
    guard = torch.full((48, 16), 3.0, device=DEV)
    for off in ([5, 2, 90, -7, 40], [-100, 1 << 30, 0, 0, 0], [7, 7, 7, 7, 7]):
        conv.causal_conv_packed(x, torch.tensor(off, dtype=torch.int32, device=DEV), pool, w, out=guard[:40])
        assert (guard[40:] == 3).all()


def test_graph_and_other_stream(gpu_lib):
    """A training step and a serving step captured; every replay equals the eager calls, with other work in between."""
    C, W = 96, 4
    xs, dys = torch.zeros(2, 33, C, device=DEV).bfloat16(), torch.zeros(2, 33, C, device=DEV).bfloat16()
    w, tok, off = torch.randn(C, W, device=DEV), torch.zeros(9, C, device=DEV), torch.tensor([0, 5, 5, 9], dtype=torch.int32, device=DEV)
    pools = [torch.randn(3, W - 1, C, device=DEV)]
    pools.append(pools[0].clone())
    def step(pool):
        x = xs.detach().requires_grad_(True)
        wl = w.detach().requires_grad_(True)
        y = conv.causal_conv(x, wl)
        return (y.detach(), *torch.autograd.grad(y, (x, wl), dys), conv.causal_conv_packed(tok, off, pool, w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(torch.zeros_like(pools[0]))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(pools[1])
    for turn in range(6):
        for t in (xs, dys, tok):
            t.copy_(torch.randn(t.shape, device=DEV))
        graph.replay()
        want = step(pools[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)) and torch.equal(*pools), turn


@pytest.mark.parametrize("C", [4096, 37])
def test_more_than_2_to_the_31_elements(gpu_lib, C):
    """Forward, backward and a packed call whose last rows lie beyond 32-bit offsets, against the same rows alone."""
    T, W = (1 << 31) // C + 1000, 4
    x = torch.zeros(1, T, C, dtype=torch.bfloat16, device=DEV)
    tail = torch.randn(1, 300, C, device=DEV).bfloat16()
    x[:, -300:] = tail
    w = torch.randn(C, W, device=DEV)
    x.requires_grad_(True)
    y = conv.causal_conv(x, w)
    dy = torch.zeros_like(y)
    dy[:, -300:] = torch.randn(1, 300, C, device=DEV).bfloat16()
    dx, = torch.autograd.grad(y, x, dy)
    small = tail.clone().requires_grad_(True)
    ys = conv.causal_conv(small, w)
    dxs, = torch.autograd.grad(ys, small, dy[:, -300:].contiguous())
    assert torch.equal(y[:, -300:], ys) and torch.equal(dx[:, -300:], dxs) and not dx[:, -400:-303].any()
    del dx, dy, y
    pool = torch.zeros(3, W - 1, C, dtype=torch.bfloat16, device=DEV)
    off = torch.tensor([0, 5, T - 200, T], dtype=torch.int32, device=DEV)
    y = conv.causal_conv_packed(x.detach()[0], off, pool, w)
    assert torch.equal(y[T - 300:T - 200], ys[0, :100])
    assert torch.equal(y[T - 200:], conv.causal_conv(tail[:, 100:], w)[0]) and torch.equal(pool[2], tail[0, -3:])


def test_refuses_what_it_has_no_derivative_for(gpu_lib):
    x, w = torch.randn(1, 5, 8, device=DEV, requires_grad=True), torch.randn(8, 4, device=DEV)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ValueError, match="the convolution has no forward-mode derivative"):
            conv.causal_conv(torch.autograd.forward_ad.make_dual(x.detach(), x.detach()), w)
    g, = torch.autograd.grad(conv.causal_conv(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
    with pytest.raises(ValueError, match="and not x"):
        p = torch.zeros(5, 3, 8, device=DEV)
        conv.causal_conv_step(x.detach()[0], p, w, out=x.detach()[0])
