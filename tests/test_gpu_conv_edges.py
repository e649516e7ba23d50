"""The short convolution where its kernels' forms part: every number of taps, lanes on whole and on split channels, packed
rows with and without an activation, filters of either type; and beside values that are not finite.  Tolerances as in
test_gpu_conv.py, whose bounds hold for up to eight taps."""
import pytest
import torch

from gdnx_amd import conv
from oracle import conv as oc
from test_gpu_conv import DEV, check, make, rel, tol

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [
    # B, T, C, W, lengths: spans of 8 to 64 tokens, whose edges W - 1 tokens reach over
    (2, 130, 520, 2, [130, 65]),
    (3, 70, 36, 2, None),
    (2, 90, 260, 3, [0, 90]),
    (2, 200, 264, 5, [200, 131]),
    (2, 140, 136, 6, [140, 9]),
    (1, 131, 1032, 7, None),
    (1, 150, 70, 8, [150]),
    (2, 97, 520, 8, [97, 96]),
], ids=lambda s: "-".join(map(str, s[:4])))
def test_every_number_of_taps(gpu_lib, shape, dtype):
    B, T, C, W, lengths = shape
    check(make(B, T, C, W, dtype), lengths)
    check(make(B, T, C, W, dtype, dtype, bias=False, state=False), lengths, silu=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("silu", [True, False])
@pytest.mark.parametrize("C", [43, 528])
@pytest.mark.parametrize("W", [2, 3, 4, 5, 6, 7, 8])
def test_packed_forms(gpu_lib, W, C, silu, dtype):
    counts = [5, 0, 1, 40, 9, 7, 1]
    n, N = len(counts), sum(counts)
    off = [sum(counts[:i]) for i in range(n + 1)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    for wdtype, bias in ((torch.float32, True), (dtype, False)):
        g = torch.Generator().manual_seed(W)
        x, pool = torch.randn(N, C, generator=g).to(dtype), torch.randn(2 * n + 1, W - 1, C, generator=g).to(dtype)
        w, b = torch.randn(C, W, generator=g).to(wdtype), torch.randn(C, generator=g).to(wdtype)
        slots, to = torch.randperm(2 * n + 1, generator=g).tolist()[:n], None
        want, wpool = oc.causal_conv_packed(x.double(), off, pool.double(), w.double(), b.double() if bias else None, slots,
                                            to, silu)
        p = pool.to(DEV)
        kw = dict(slots=i32(slots), activation="silu" if silu else None)
        y = conv.causal_conv_packed(x.to(DEV), i32(off), p, w.to(DEV), b.to(DEV) if bias else None, **kw)
        assert torch.equal(p.double().cpu(), wpool)
        assert rel(y, want) <= tol(dtype, 3e-6)
        # a token a row is the same row by row, bit for bit
        p1, p2 = pool.to(DEV), pool.to(DEV)
        args = w.to(DEV), b.to(DEV) if bias else None
        one = conv.causal_conv_step(x[:n].to(DEV), p1, *args, **kw)
        assert torch.equal(one, conv.causal_conv_packed(x[:n].to(DEV), i32(list(range(n + 1))), p2, *args, **kw))
        assert torch.equal(p1, p2)


def _grads(ins, lengths, silu):
    leaves = {n: t.to(DEV).requires_grad_(True) for n, t in ins.items()}
    y, last = conv.causal_conv(leaves["x"], leaves["weight"], leaves["bias"], activation="silu" if silu else None,
                               state=leaves["state"], lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV),
                               return_state=True)
    g = torch.Generator().manual_seed(5)
    dy, dlast = (torch.randn(t.shape, generator=g).to(t.dtype).to(DEV) for t in (y, last))
    return dict(zip(leaves, torch.autograd.grad((y, last), list(leaves.values()), (dy, dlast)))), dlast


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("C", [24, 520])
def test_gradients_take_nothing_from_behind_a_rows_end(gpu_lib, C, dtype):
    """Beside inputs, states and filters that are not finite: a token behind the end adds nothing, not zero times something."""
    lengths, end = [40, 0, 21], 21
    ins = make(3, 40, C, 4, dtype)
    for silu in (False, True):
        plain, dlast = _grads(ins, lengths, silu)
        bad = dict(ins, state=ins["state"].clone())
        bad["state"][1] = float("nan")                       # of a row without tokens: it is handed on, and that is all
        got, _ = _grads(bad, lengths, silu)
        assert all(torch.equal(got[n], plain[n]) for n in plain)
        assert torch.equal(got["state"][1], dlast[1])
    plain, _ = _grads(ins, lengths, False)
    bad = dict(ins, x=ins["x"].clone())
    bad["x"][2, end - 1] = float("inf")                      # a row's last token meets the newest tap alone
    got, _ = _grads(bad, lengths, False)
    assert torch.equal(got["weight"][:, :3], plain["weight"][:, :3]) and not torch.isfinite(got["weight"][:, 3]).any()
    assert all(torch.equal(got[n], plain[n]) for n in ("x", "bias", "state"))
    bad = dict(ins, weight=ins["weight"].clone())
    bad["weight"][:, 0] = float("inf")                       # the oldest tap reaches the tokens W - 1 before another
    got, _ = _grads(bad, lengths, False)
    for b, n in enumerate(lengths):
        assert (got["x"][b, n:] == 0).all()
        assert torch.equal(got["x"][b, max(n - 3, 0):n], plain["x"][b, max(n - 3, 0):n])
        assert not torch.isfinite(got["x"][b, :max(n - 3, 0)]).any()


def test_pool_without_slots(gpu_lib):
    """All rows are empty ones: y = 0 for their tokens, and what lies behind the last row's stays."""
    x, w = torch.randn(6, 8, device=DEV), torch.randn(8, 4, device=DEV)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    pool, slots = torch.zeros(0, 3, 8, device=DEV), i32([0, -1, 5])
    for to in (None, i32([0, 0, 1])):
        out = torch.full((6, 8), 7.0, device=DEV)
        y = conv.causal_conv_packed(x, i32([0, 2, 2, 4]), pool, w, slots=slots, to_slots=to, out=out)
        assert y is out and (out[:4] == 0).all() and (out[4:] == 7).all()
        assert (conv.causal_conv_step(x[:3], pool, w, slots=slots, to_slots=to) == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_batch_whose_first_tokens_are_nobodys(gpu_lib, dtype):
    counts, C, lead = [5, 0, 1, 70, 9], 520, 37
    n, N = len(counts), sum(counts)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    off = [sum(counts[:i]) for i in range(n + 1)]
    x, w, pool = torch.randn(lead + N + 3, C, device=DEV).to(dtype), torch.randn(C, 4, device=DEV), torch.randn(n, 3, C, device=DEV)
    p1, p2 = pool.to(dtype, copy=True), pool.to(dtype, copy=True)
    want = conv.causal_conv_packed(x[lead:lead + N], i32(off), p1, w)
    out = torch.full_like(x, 5.0)
    conv.causal_conv_packed(x, i32([lead + o for o in off]), p2, w, out=out)
    assert torch.equal(out[lead:lead + N], want) and torch.equal(p1, p2)
    assert (out[:lead] == 5).all() and (out[lead + N:] == 5).all()
