"""Windowed attention and the paged step on the GPU against the 64-bit oracle.

Tolerances (relative L2).  float32: a score is a sum of D products, wrong by
about sqrt(D) 2^-24 of its terms, a few 1e-6 for scores of a few units, and P
and every later sum follow: 1e-5 for y, 3e-5 for the gradients (two more
products).  bfloat16: the output is rounded once (2^-9 at most, 1.1e-3 rms)
and P and dS are operands of a further product (1.1e-3 rms each):
sqrt(2..5) x 1.1e-3 with head room: 4e-3 for y and 8e-3 for the gradients.  lse is float32 in both: 1e-5 and, of bf16 inputs, the same.
"""
import pytest
import torch

from gdnx_amd import attention
from oracle import attention as oa

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = {torch.float32: (1e-5, 3e-5), torch.bfloat16: (4e-3, 8e-3)}


def rel(a, b):
    a, b = a.detach().double().cpu(), b.detach().double()
    return float((a - b).norm() / b.norm().clamp(min=1e-30)) if b.norm() > 0 else float(a.norm())


def cancels(want, dy):
    """Whether a gradient is zero in exact arithmetic (queries that see one key: dP and delta are equal): its
    error is then that of the terms that cancel, of dy's size, and is measured against it."""
    return float(want.norm()) < 1e-6 * float(dy.double().norm())


def rows_rel(a, b):
    """The worst vector of D values, against its own size and the tensor's mean size."""
    a, b = a.double().cpu().flatten(0, -2), b.double().flatten(0, -2)
    return float(((a - b).norm(dim=1) / (b.norm(dim=1) + b.norm() / b.shape[0] ** 0.5).clamp(min=1e-30)).max())


def make(B, Tq, Tk, Hq, Hkv, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)
    return r(B, Tq, Hq, D), r(B, Tk, Hkv, D), r(B, Tk, Hkv, D), r(B, Tq, Hq, D)


def check(q, k, v, dy, window, sinks, lengths, scale=None):
    ins = [x.to(DEV).requires_grad_(True) for x in (q, k, v)]
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    y, lse = attention.window_attention(*ins, window=window, sinks=sinks, lengths=ln, scale=scale, return_lse=True)
    grads = torch.autograd.grad(y, ins, grad_outputs=dy.to(DEV))
    ref = oa.attention(q, k, v, window, sinks, scale, lengths, dy)
    ty, tg = TOL[q.dtype]
    seen = torch.isfinite(ref[1])
    assert torch.equal(torch.isfinite(lse).cpu(), seen) and (lse.cpu()[~seen] == float("-inf")).all()
    errs = {"lse": float((lse.cpu().double() - ref[1])[seen].abs().max()) if seen.any() else 0.0}
    assert errs["lse"] <= 1e-4, errs          # absolute: scores of a few units
    for name, got, want, tol in (("y", y, ref[0], ty), ("dq", grads[0], ref[2], tg), ("dk", grads[1], ref[3], tg),
                                 ("dv", grads[2], ref[4], tg)):
        assert got.dtype == q.dtype and got.shape == want.shape
        if name != "y" and cancels(want, dy):
            errs[name] = float(got.double().norm()) / float(dy.double().norm())
            assert errs[name] <= tol, (name, errs)
            continue
        errs[name] = (rel(got, want), rows_rel(got, want))
        assert errs[name][0] <= tol and errs[name][1] <= 5 * tol, (name, errs)
    with torch.no_grad():                      # the same without a gradient
        y2 = attention.window_attention(*ins, window=window, sinks=sinks, lengths=ln, scale=scale)
    assert torch.equal(y, y2)
    return y, grads


SHAPES = [
    # B, Tq, Tk, Hq, Hkv, window, sinks, lengths
    (1, 1, 1, 1, 1, None, 0, None),
    (2, 1, 65, 4, 2, None, 0, None),
    (1, 17, 17, 3, 1, None, 0, None),
    (2, 64, 64, 2, 2, 1, 0, None),               # every query sees itself alone
    (1, 130, 130, 4, 1, 33, 0, None),
    (1, 257, 257, 6, 2, 40, 3, None),
    (2, 300, 300, 2, 1, 64, 70, None),           # more sinks than a tile
    (1, 200, 200, 2, 1, 16, 500, None),          # all tokens are sinks
    (3, 150, 150, 2, 1, 50, 5, [150, 0, 1]),     # an empty row, a row of one token
    (2, 33, 290, 4, 2, 100, 4, [290, 260]),      # the next piece of a prompt
    (2, 90, 40, 2, 1, 20, 2, [40, 13]),          # queries before position 0
    (1, 515, 515, 8, 1, None, 0, [450]),
    (1, 1030, 1030, 4, 2, 200, 130, None),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[:7])) + ("-len" if s[7] else ""))
def test_window_attention(gpu_lib, shape, D, dtype):
    B, Tq, Tk, Hq, Hkv, window, sinks, lengths = shape
    check(*make(B, Tq, Tk, Hq, Hkv, D, dtype), window, sinks, lengths)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 40, 40, 20, 1, 9, 2, None), (2, 9, 300, 150, 1, 60, 0, [300, 295]),
                                   (1, 70, 70, 34, 2, None, 0, [66]), (1, 3, 20, 400, 2, None, 0, None)],
                         ids=lambda s: "-".join(map(str, s[:7])))
def test_large_groups(gpu_lib, shape, dtype):
    """Groups that are no power of two, longer than a tile's rows, or the size of several tiles."""
    B, Tq, Tk, Hq, Hkv, window, sinks, lengths = shape
    check(*make(B, Tq, Tk, Hq, Hkv, 64, dtype), window, sinks, lengths)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_padding_may_hold_anything(gpu_lib, dtype):
    q, k, v, dy = make(2, 100, 100, 4, 2, 64, dtype)
    lengths = [61, 0]
    a = check(q, k, v, dy, 30, 4, lengths)
    for b, n in enumerate(lengths):
        q[b, n:], k[b, n:], v[b, n:], dy[b, n:] = float("inf"), float("nan"), float("-inf"), float("nan")
    b = check(q, k, v, dy, 30, 4, lengths)
    assert torch.equal(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[1], b[1]))
    assert all((x[0, 61:] == 0).all() and (x[1] == 0).all() for x in (b[0], *b[1]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_token_that_is_not_finite_reaches_only_who_sees_it(gpu_lib, bad, D, dtype):
    """Keys and values of inner tokens: later than some queries of their tile, or left behind by its window."""
    T, W, S, at = 300, 50, 3, (1, 100, 163, 250)
    q, k, v, _ = make(1, T, T, 4, 2, D, dtype, seed=6)
    hide = oa.visible(T, T, W, S, T)[:, list(at)].any(1)            # queries that see one of them
    clean = oa.attention(q, k, v, W, S)[0]
    y0 = attention.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), window=W, sinks=S)
    for what in "kv":
        k2, v2 = k.clone(), v.clone()
        for j in at:
            (k2 if what == "k" else v2)[0, j, :, 3] = bad
        y = attention.window_attention(q.to(DEV), k2.to(DEV), v2.to(DEV), window=W, sinks=S)
        assert torch.isfinite(y[0, ~hide]).all()
        assert rel(y[0, ~hide], clean[0, ~hide]) <= TOL[dtype][0]
        if what == "v":
            assert not torch.isfinite(y[0, hide][..., 3].float()).any()      # and who sees it gets it, in its column
            assert rel(y[0, hide][..., 4:], clean[0, hide][..., 4:]) <= TOL[dtype][0]
    assert rel(y0, clean) <= TOL[dtype][0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_scores_of_all_sizes(gpu_lib, dtype, scale):
    """A scale of 1: scores to +-40, where the running maximum does all the work.  Rounding scores of that
    size costs P |s| 2^-24 a score in float32, so its bound is the scores' size (8 rms) times as wide."""
    q, k, v, dy = make(1, 190, 190, 2, 1, 64, dtype, seed=3)
    ins = [x.to(DEV).requires_grad_(True) for x in (q, k, v)]
    y = attention.window_attention(*ins, window=70, sinks=2, scale=scale)
    grads = torch.autograd.grad(y, ins, grad_outputs=dy.to(DEV))
    ref = oa.attention(q, k, v, 70, 2, scale, None, dy)
    ty, tg = TOL[dtype]
    grow = 8 if scale == 1.0 and dtype == torch.float32 else 1
    assert rel(y, ref[0]) <= ty * grow
    for g, r in zip(grads, ref[2:]):
        assert rel(g, r) <= tg * grow


def test_large_scores_do_not_overflow(gpu_lib):
    q, k, v, dy = make(1, 80, 80, 2, 2, 64, torch.float32, seed=4)
    y, lse = attention.window_attention((q * 1e3).to(DEV), (k * 1e3).to(DEV), v.to(DEV), window=40, return_lse=True)
    assert torch.isfinite(y).all() and torch.isfinite(lse).all()
    ref = oa.attention(q * 1e3, k * 1e3, v, 40)
    # scores of 1e6 carry float32 errors near 0.1: all but a few rows still have one key that takes all
    assert (y.double().cpu() - ref[0]).norm(dim=-1).median() < 1e-5


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides(gpu_lib, dtype):
    """Views of a fused projection, heads before tokens, a broadcast batch; a last axis that is not contiguous."""
    B, T, Hq, Hkv, D = 2, 77, 4, 2, 64
    g = torch.Generator().manual_seed(5)
    fused = torch.randn(B, T, (Hq + 2 * Hkv) * D, generator=g).to(dtype)
    dy = torch.randn(B, T, Hq, D, generator=g).to(dtype)
    x = fused.to(DEV).requires_grad_(True)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in x.split([Hq * D, Hkv * D, Hkv * D], -1))
    assert attention._rows16(q) is q and attention._rows16(v) is v
    y = attention.window_attention(q, k, v, window=20, sinks=3)
    dx, = torch.autograd.grad(y, x, grad_outputs=dy.to(DEV))
    qc, kc, vc = (t.unflatten(-1, (-1, D)) for t in fused.split([Hq * D, Hkv * D, Hkv * D], -1))
    ref = oa.attention(qc, kc, vc, 20, 3, None, None, dy)
    ty, tg = TOL[dtype]
    assert rel(y, ref[0]) <= ty and rel(dx, torch.cat([r.flatten(2) for r in ref[2:]], -1)) <= tg
    heads_first = [t.to(DEV).transpose(1, 2).contiguous().transpose(1, 2) for t in (qc, kc, vc)]
    assert torch.equal(attention.window_attention(*heads_first, window=20, sinks=3), y)
    last = [t.to(DEV).transpose(2, 3).contiguous().transpose(2, 3) for t in (qc, kc, vc)]
    assert torch.equal(attention.window_attention(*last, window=20, sinks=3), y)
    one = [t[:1].to(DEV).requires_grad_(True) for t in (kc, vc)]          # one cache for both rows
    y2 = attention.window_attention(qc.to(DEV), *(t.expand(B, -1, -1, -1) for t in one), window=20, sinks=3)
    d1 = torch.autograd.grad(y2, one, grad_outputs=dy.to(DEV))
    r2 = oa.attention(qc, *(t.expand(B, -1, -1, -1) for t in (kc[:1], vc[:1])), 20, 3, None, None, dy)
    assert rel(y2, r2[0]) <= ty
    for a, b in zip(d1, r2[3:]):
        assert a.shape[0] == 1 and rel(a, b.sum(0, keepdim=True)) <= tg
    unaligned = torch.randn(B * T * Hq * D + 1, generator=g).to(dtype).to(DEV)[1:].view(B, T, Hq, D)
    y3 = attention.window_attention(unaligned, *heads_first[1:], window=20, sinks=3)
    assert torch.equal(y3, attention.window_attention(unaligned.clone(), *heads_first[1:], window=20, sinks=3))


@pytest.mark.parametrize("need", ["q", "k", "v", "kv"])
def test_some_gradients_only(gpu_lib, need):
    q, k, v, dy = make(1, 50, 50, 2, 1, 64, torch.float32)
    ins = {n: t.to(DEV).requires_grad_(n in need) for n, t in zip("qkv", (q, k, v))}
    y = attention.window_attention(ins["q"], ins["k"], ins["v"], window=9)
    grads = torch.autograd.grad(y, [ins[n] for n in need], grad_outputs=dy.to(DEV))
    ref = dict(zip("qkv", oa.attention(q, k, v, 9, dy=dy)[2:]))
    for n, g in zip(need, grads):
        assert rel(g, ref[n]) <= 3e-5


def test_gradient_against_differences(gpu_lib):
    """The float32 gradient along a direction against central differences of the 64-bit oracle's output."""
    q, k, v, dy = make(1, 70, 70, 4, 2, 64, torch.float32, seed=8)
    ins = [x.to(DEV).requires_grad_(True) for x in (q, k, v)]
    y = attention.window_attention(*ins, window=25, sinks=2)
    grads = torch.autograd.grad(y, ins, grad_outputs=dy.to(DEV))
    g = torch.Generator().manual_seed(9)
    for i in range(3):
        d = torch.randn(ins[i].shape, generator=g)
        xs = lambda h: [x.double() + (h * d.double() if n == i else 0.0) for n, x in enumerate((q, k, v))]
        f = lambda h: float((oa.attention(*xs(h), 25, 2)[0] * dy.double()).sum())
        num = (f(1e-4) - f(-1e-4)) / 2e-4
        # the gradient's own 3e-5, over a sum of independent terms of the size of |g| |d| / sqrt(n)
        size = float(grads[i].norm()) * float(d.norm()) / d.numel() ** 0.5
        assert abs(float((grads[i].cpu().double() * d.double()).sum()) - num) <= 1e-4 * size


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_same_bits_every_time_and_on_another_stream(gpu_lib, dtype):
    q, k, v, dy = (x.to(DEV) for x in make(2, 700, 700, 8, 2, 128, dtype))
    def once():
        ins = [x.detach().requires_grad_(True) for x in (q, k, v)]
        y = attention.window_attention(*ins, window=128, sinks=20)
        return (y, *torch.autograd.grad(y, ins, grad_outputs=dy))
    a, b = once(), once()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c = once()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(a, b, c))


def test_empty_calls(gpu_lib):
    x = lambda B, T, H: torch.randn(B, T, H, 64, device=DEV, requires_grad=True)
    for q, k, v in ((x(0, 4, 2), x(0, 4, 2), x(0, 4, 2)), (x(2, 0, 2), x(2, 4, 1), x(2, 4, 1)),
                    (x(2, 3, 2), x(2, 0, 1), x(2, 0, 1))):
        y = attention.window_attention(q, k, v, window=3)
        assert y.shape == q.shape and (y == 0).all()
        for g, t in zip(torch.autograd.grad(y.sum(), (q, k, v)), (q, k, v)):
            assert g.shape == t.shape and (g == 0).all()


def test_a_row_beyond_32_bits(gpu_lib):
    """Rows far apart: offsets of more than 4 GB within the batch and within a row."""
    D, T = 64, 200
    big = torch.zeros(2, T, 1 << 24, dtype=torch.bfloat16, device=DEV)      # 32 MB a token, 6.7 GB a row
    g = torch.Generator().manual_seed(2)
    parts = [torch.randn(2, T, 1, D, generator=g).bfloat16() for _ in range(3)]
    views = []
    for n, p in enumerate(parts):
        w = big[:, :, n * D:(n + 1) * D].unflatten(-1, (1, D))
        w.copy_(p)
        views.append(w)
    assert all(attention._rows16(w) is w for w in views)
    y = attention.window_attention(*views, window=11, sinks=1)
    assert rel(y, oa.attention(*parts, 11, 1)[0]) <= 4e-3


# ---------------------------------------------------------------------------
# one token over the page cache
# ---------------------------------------------------------------------------
def paged(lens, Hq, Hkv, D, page, dtype, width=None, n_pages=None, seed=0, fill=None):
    """A cache of random pages in random places; returns device tensors and the rows' own keys and values."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    n_pages = n_pages or sum(need) + 3
    width = width or max(need + [1])
    order, table, at = torch.randperm(n_pages, generator=g), torch.full((len(lens), width), -1, dtype=torch.int32), 0
    kp = torch.randn(n_pages, Hkv, page, D, generator=g).to(dtype)
    vp = torch.randn(n_pages, Hkv, page, D, generator=g).to(dtype)
    ks, vs = [], []
    for r, n in enumerate(lens):
        own = order[at:at + need[r]]
        at += need[r]
        table[r, :need[r]] = own.int()
        rows = lambda t: t[own].permute(0, 2, 1, 3).reshape(-1, Hkv, D)[:n].clone()
        ks.append(rows(kp))
        vs.append(rows(vp))
        if fill is not None and n % page:
            kp[own[-1], :, n % page:] = fill
            vp[own[-1], :, n % page:] = fill
    for p in order[at:].tolist():
        if fill is not None:
            kp[p], vp[p] = fill, fill
    q = torch.randn(len(lens), Hq, D, generator=g).to(dtype)
    return q, kp, vp, table, torch.tensor(lens, dtype=torch.int32), ks, vs


def step_ref(q, ks, vs, window, sinks, scale=None):
    ys = [oa.attention(q[r][None, None], ks[r][None], vs[r][None], window, sinks, scale)[0][0, 0] if len(ks[r]) else
          torch.zeros(q.shape[1:], dtype=torch.float64) for r in range(len(ks))]
    return torch.stack(ys)


STEPS = [
    # lens, Hq, Hkv, page, window, sinks
    ([1], 1, 1, 16, None, 0), ([0, 1, 2, 17], 4, 2, 16, None, 0), ([33, 200, 0, 129], 6, 2, 32, None, 0),
    ([1000, 37], 16, 1, 1, None, 0), ([700, 64], 20, 1, 64, None, 0),          # more than 16 query heads a key head
    ([5000, 3, 4097], 8, 8, 128, None, 0), ([900, 31, 64, 65], 4, 4, 16, 64, 0), ([900, 31, 64, 65], 4, 2, 16, 50, 7),
    ([2500, 90], 4, 1, 256, 1, 1), ([300, 10], 8, 2, 8, 20, 400), ([20000], 3, 1, 16, None, 0),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("case", STEPS, ids=lambda c: "-".join(str(x) for x in (max(c[0]), *c[1:])))
def test_paged_step(gpu_lib, case, D, dtype):
    lens, Hq, Hkv, page, window, sinks = case
    q, kp, vp, table, ln, ks, vs = paged(lens, Hq, Hkv, D, page, dtype, fill=float("nan"))
    dev = [t.to(DEV) for t in (q, kp, vp, table, ln)]
    y = attention.paged_attention_step(dev[0], None, None, *dev[1:], window=window, sinks=sinks)
    ref = step_ref(q, ks, vs, window, sinks)
    tol = TOL[dtype][0]
    assert rel(y, ref) <= tol and rows_rel(y, ref) <= 5 * tol
    for r, n in enumerate(lens):
        assert n or (y[r] == 0).all()
    assert torch.equal(dev[1].cpu().nan_to_num(7.0), kp.nan_to_num(7.0))             # nothing written
    # the last token handed over with the call: the same result, and its page holds it afterwards
    new_k, new_v = (torch.stack([x[-1] if len(x) else torch.zeros(Hkv, D, dtype=dtype) for x in xs]) for xs in (ks, vs))
    dev2 = [t.to(DEV) for t in (q, kp, vp, table, ln)]
    for r, n in enumerate(lens):
        if n:
            at = (table[r, (n - 1) // page].item(), slice(None), (n - 1) % page)
            dev2[1][at], dev2[2][at] = float("nan"), float("nan")
    y2 = attention.paged_attention_step(dev2[0], new_k.to(DEV), new_v.to(DEV), *dev2[1:], window=window, sinks=sinks)
    assert torch.equal(y, y2)
    assert torch.equal(dev2[1].cpu().nan_to_num(7.0), kp.nan_to_num(7.0))
    assert torch.equal(dev2[2].cpu().nan_to_num(7.0), vp.nan_to_num(7.0))


@pytest.mark.parametrize("lens,Hq,Hkv,window", [([3000] * 40, 8, 8, None), ([2000 + 700 * r for r in range(16)], 4, 4, 1500),
                                                ([1, 9000, 0, 40] * 8, 16, 8, None)])
def test_paged_step_spans(gpu_lib, lens, Hq, Hkv, window):
    """Enough rows and heads for one span or a few, whose number the table's width and not the row decides."""
    q, kp, vp, table, ln, ks, vs = paged(lens, Hq, Hkv, 64, 64, torch.bfloat16, fill=float("nan"))
    y = attention.paged_attention_step(q.to(DEV), None, None, *(t.to(DEV) for t in (kp, vp, table, ln)),
                                       window=window, sinks=5)
    ref = step_ref(q, ks, vs, window, 5)
    tol = TOL[torch.bfloat16][0]
    assert rel(y, ref) <= tol and rows_rel(y, ref) <= 5 * tol


def test_paged_step_slots_missing_pages_and_odd_tables(gpu_lib):
    lens, dtype = [100, 50, 75], torch.bfloat16
    q, kp, vp, table, ln, ks, vs = paged(lens, 4, 2, 64, 16, dtype, width=4096)      # a table far wider than its rows
    dev = [t.to(DEV) for t in (kp, vp, table, ln)]
    slots = torch.tensor([2, -1, 0, 9, 1], dtype=torch.int32, device=DEV)
    qs = q[[2, 0, 0, 0, 1]].to(DEV)
    out = torch.full((5, 4, 64), 5.0, dtype=dtype, device=DEV)
    y = attention.paged_attention_step(qs, None, None, *dev, slots=slots, window=30, sinks=3, out=out)
    ref = step_ref(q, ks, vs, 30, 3)
    assert y is out and (y[1] == 0).all() and (y[3] == 0).all()
    assert rel(y[[0, 2, 4]], ref[[2, 0, 1]]) <= 4e-3
    # a page that is not there: its tokens are not seen, wherever the entry points
    for bad in (-1, 10 ** 9):
        t2 = table.clone()
        t2[0, 3] = bad
        y = attention.paged_attention_step(q.to(DEV), None, None, dev[0], dev[1], t2.to(DEV), dev[3])
        keep = torch.tensor([j for j in range(100) if j // 16 != 3])
        ref = step_ref(q, [ks[0][keep], *ks[1:]], [vs[0][keep], *vs[1:]], None, 0)
        assert rel(y, ref) <= 4e-3
    # lengths beyond the table are cut to it, negative ones are empty
    y = attention.paged_attention_step(q.to(DEV), None, None, dev[0], dev[1], table[:, :3].contiguous().to(DEV),
                                       torch.tensor([100, -5, 48], dtype=torch.int32, device=DEV))
    ref = step_ref(q, [ks[0][:48], ks[1][:0], ks[2][:48]], [vs[0][:48], vs[1][:0], vs[2][:48]], None, 0)
    assert rel(y, ref) <= 4e-3 and (y[1] == 0).all()


def test_paged_step_matches_the_prompt_form(gpu_lib):
    q, kp, vp, table, ln, ks, vs = paged([333], 8, 2, 128, 32, torch.bfloat16)
    y = attention.paged_attention_step(q.to(DEV), None, None, *(t.to(DEV) for t in (kp, vp, table, ln)),
                                       window=100, sinks=5)
    z = attention.window_attention(q[None].to(DEV), ks[0][None].to(DEV), vs[0][None].to(DEV), window=100, sinks=5)
    assert rel(y, z[0].cpu()) <= 4e-3


def test_paged_step_in_a_pool_beyond_32_bits(gpu_lib):
    """Pages past 4 GB (and past 2^31 elements) of the pool."""
    Hkv, page, D, n_pages = 8, 128, 128, 20000            # 5.2 GB for the keys
    kp = torch.zeros(n_pages, Hkv, page, D, dtype=torch.bfloat16, device=DEV)
    vp = torch.zeros_like(kp)
    g = torch.Generator().manual_seed(3)
    at = [19999, 17001, 5, 16500]
    ks, vs = (torch.randn(4, Hkv, page, D, generator=g).bfloat16() for _ in range(2))
    for i, p in enumerate(at):
        kp[p], vp[p] = ks[i].to(DEV), vs[i].to(DEV)
    table = torch.tensor([at], dtype=torch.int32, device=DEV)
    n = 3 * page + 50
    q = torch.randn(1, 16, D, generator=g).bfloat16()
    flat = lambda t: t.permute(0, 2, 1, 3).reshape(-1, Hkv, D)[:n]
    y = attention.paged_attention_step(q.to(DEV), None, None, kp, vp, table, torch.tensor([n], dtype=torch.int32, device=DEV))
    assert rel(y, step_ref(q, [flat(ks)], [flat(vs)], None, 0)) <= 4e-3


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_paged_step_same_bits(gpu_lib, dtype):
    q, kp, vp, table, ln, _, _ = paged([3000, 17, 900], 8, 2, 64, 16, dtype)
    dev = [t.to(DEV) for t in (kp, vp, table, ln)]
    a = attention.paged_attention_step(q.to(DEV), None, None, *dev)
    b = attention.paged_attention_step(q.to(DEV), None, None, *dev)
    assert torch.equal(a, b)
    one = attention.paged_attention_step(q[:1].to(DEV), None, None, *dev)     # fewer rows: other spans
    assert rel(one, a[:1].double().cpu()) <= TOL[dtype][0]
