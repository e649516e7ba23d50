"""Attention beside values that are not finite, padding, split keys, odd strides and the ends of the arguments' ranges.

Tolerances are those of test_gpu_attention, where they are derived.
"""
import pytest
import torch

from gdnx_amd import _lib, attention
from oracle import attention as oa
from test_gpu_attention import DEV, TOL, check, make, paged, rel, step_ref

pytestmark = pytest.mark.gpu
DTYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
HEADS = pytest.mark.parametrize("D", [64, 128])


def ints(xs):
    return torch.tensor(xs, dtype=torch.int32, device=DEV)


# B, Tq, Tk, Hq, Hkv, window, sinks, lengths, tokens that are not finite (each within every row's length)
UNSEEN = [
    (2, 100, 100, 4, 2, 30, 4, [61, 90], (3, 59)),               # padded queries beside them
    (2, 100, 100, 3, 1, None, 0, [70, 97], (1, 69)),
    (1, 90, 40, 2, 1, 20, 2, None, (0, 5)),                      # queries before position 0
    (2, 100, 3000, 4, 2, None, 0, [2950, 2925], (7, 2920)),      # keys split over several workgroups
]


def unseeing(case, what, bad, D, dtype):
    """The case's inputs, k or v not finite at its tokens, and which queries see nothing."""
    B, Tq, Tk, Hq, Hkv, _, _, lengths, at = case
    q, k, v, dy = make(B, Tq, Tk, Hq, Hkv, D, dtype, seed=11)
    (k if what == "k" else v)[:, list(at), :, 3] = bad
    p = torch.arange(Tq) + Tk - Tq
    none = (p < 0) | (p >= torch.tensor(lengths or [Tk] * B)[:, None])
    assert none.any(1).all()
    return [x.to(DEV).requires_grad_(True) for x in (q, k, v)], dy.to(DEV), none.to(DEV)


@DTYPES
@HEADS
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("case", UNSEEN, ids=lambda c: "-".join(map(str, c[:7])))
def test_queries_that_see_nothing_give_zero_beside_what_is_not_finite(gpu_lib, case, what, bad, D, dtype):
    W, S, lengths = case[5:8]
    ins, _, none = unseeing(case, what, bad, D, dtype)
    y, lse = attention.window_attention(*ins, window=W, sinks=S, lengths=None if lengths is None else ints(lengths),
                                        return_lse=True)
    assert (y[none] == 0).all() and (lse.transpose(1, 2)[none] == float("-inf")).all()


@DTYPES
@HEADS
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("case", UNSEEN, ids=lambda c: "-".join(map(str, c[:7])))
def test_queries_that_see_nothing_have_no_gradient(gpu_lib, case, what, bad, D, dtype):
    W, S, lengths = case[5:8]
    ins, dy, none = unseeing(case, what, bad, D, dtype)
    y = attention.window_attention(*ins, window=W, sinks=S, lengths=None if lengths is None else ints(lengths))
    dq, = torch.autograd.grad(y, ins[:1], grad_outputs=dy)
    assert (dq[none] == 0).all()


@DTYPES
@HEADS
@pytest.mark.parametrize("case", [(2, 100, 100, 4, 2, 30, 0, [61, 90], 55),       # tokens beyond the length
                                  (1, 200, 200, 2, 1, 40, 2, [150], 149),
                                  (1, 20, 300, 4, 1, 50, 3, None, 10)],           # tokens that no query reaches
                         ids=lambda c: "-".join(map(str, c[:7])))
def test_tokens_that_nobody_sees_have_no_gradient(gpu_lib, case, D, dtype):
    """Whatever a query of their tile holds."""
    B, Tq, Tk, Hq, Hkv, W, S, lengths, at = case
    q, k, v, dy = make(B, Tq, Tk, Hq, Hkv, D, dtype, seed=12)
    seen = torch.stack([oa.visible(Tq, Tk, W, S, n).any(0) for n in lengths or [Tk] * B])
    seen &= torch.arange(Tk) < torch.tensor(lengths or [Tk] * B)[:, None]
    for what in ("q", "dy"):
        q2, g2 = q.clone(), dy.clone()
        (q2 if what == "q" else g2)[:, at, :, 5] = float("inf")
        ins = [x.to(DEV).requires_grad_(True) for x in (q2, k, v)]
        y = attention.window_attention(*ins, window=W, sinks=S, lengths=None if lengths is None else ints(lengths))
        _, dk, dv = torch.autograd.grad(y, ins, grad_outputs=g2.to(DEV))
        assert not seen.all() and (dk[~seen.to(DEV)] == 0).all() and (dv[~seen.to(DEV)] == 0).all()


@DTYPES
def test_axes_of_one_element_may_have_any_stride(gpu_lib, dtype):
    """The last token of a fused projection whose width is no multiple of 16 bytes, aligned and not; one head
    whose stride is that of a transposed axis."""
    T, D, width = 40, 64, 6 * 64 + 6
    g = torch.Generator().manual_seed(13)
    k, v = (torch.randn(1, T, 1, D, generator=g).to(dtype) for _ in range(2))
    fused = torch.randn(1, T, width, generator=g).to(dtype)
    for first in (0, 2):
        x = fused.to(DEV)[..., first:first + 4 * D].unflatten(-1, (4, D))[:, -1:]
        assert x.is_contiguous() and x.stride(1) == width
        x.requires_grad_(True)
        y = attention.window_attention(x, k.to(DEV), v.to(DEV), window=20, sinks=3)
        dx, = torch.autograd.grad(y.float().sum(), x)
        want = oa.attention(fused[..., first:first + 4 * D].unflatten(-1, (4, D))[:, -1:], k, v, 20, 3,
                            dy=torch.ones(1, 1, 4, D))
        assert rel(y, want[0]) <= TOL[dtype][0] and rel(dx, want[2]) <= TOL[dtype][1]
    one = torch.randn(1, T, D, 1, generator=g).to(dtype)
    x = one.to(DEV).transpose(2, 3)
    assert x.is_contiguous() and x.stride(2) == 1
    y = attention.window_attention(x, k.to(DEV), v.to(DEV), window=20, sinks=3)
    assert rel(y, oa.attention(one.transpose(2, 3), k, v, 20, 3)[0]) <= TOL[dtype][0]
    far = torch.randn(1, 2, (1 << 24) + 8, generator=g).to(dtype).to(DEV)[:, :1, 8:8 + D].unflatten(-1, (1, D))
    attention.window_attention(far, k.to(DEV), v.to(DEV))      # (a stride that no token needs)


@DTYPES
def test_sinks_to_the_end_of_an_int(gpu_lib, dtype):
    """All tokens are sinks, in a C caller's natural words for it."""
    B, T, Hq, Hkv, D, W = 1, 150, 4, 2, 64, 20
    q, k, v, dy = (x.to(DEV) for x in make(B, T, T, Hq, Hkv, D, dtype, seed=16))
    code = _lib.dtype_code(dtype)
    def run(sinks):
        y, dq, low = torch.empty_like(q), torch.empty_like(q), torch.empty_like(q)
        dk, dv = torch.empty_like(k), torch.empty_like(v)
        lse = torch.empty(B, Hq, T, device=DEV)
        sizes = (B, T, T, Hq, Hkv, D, W, sinks)
        ws = [torch.empty(max(16, getattr(gpu_lib, f"gdnx_win_attn_{d}_workspace_bytes")(*sizes, code)),
                          dtype=torch.uint8, device=DEV) for d in ("fwd", "bwd")]
        st = [*q.stride()[:3], *k.stride()[:3], *v.stride()[:3]]
        p = lambda *ts: [t.data_ptr() for t in ts]
        _lib.call("gdnx_win_attn_fwd", q.device, *p(q, k, v), None, *p(y, low, lse, ws[0]), *st, *sizes, 0.125, code)
        _lib.call("gdnx_win_attn_bwd", q.device, *p(q, k, v), None, *p(y, low, lse, dy, dq, dk, dv, ws[1]), *st, *sizes,
                  0.125, code)
        return y, lse, dq, dk, dv
    want = run(T)
    for sinks in (1 << 30, (1 << 31) - 64, (1 << 31) - 1):
        assert all(torch.equal(a, b) for a, b in zip(run(sinks), want)), sinks
    assert rel(want[0], oa.attention(q, k, v)[0]) <= TOL[dtype][0]


def test_a_backward_of_many_rows_and_heads(gpu_lib):
    """526 thousand workgroups and 2^32 elements a tensor; all rows of the batch are alike."""
    B, T, H, D, W = 64, 32769, 32, 64, 40
    g = torch.Generator(device=DEV).manual_seed(20)
    one = [torch.randn(1, T, H, D, generator=g, device=DEV).bfloat16() for _ in range(4)]
    def run(B):
        ins = [x.expand(B, -1, -1, -1).detach().requires_grad_(True) for x in one[:3]]
        y = attention.window_attention(*ins, window=W)
        return (y, *torch.autograd.grad(y, ins, grad_outputs=one[3].expand(B, -1, -1, -1).contiguous()))
    for got, want in zip(run(B), run(1)):
        assert rel(got[0], want[0].cpu()) <= 1e-3            # (other spans, which are summed in another order)
        assert all(torch.equal(x, got[0]) for x in got)


@DTYPES
def test_a_scale_that_is_no_number(gpu_lib, dtype):
    """Gives no number, in both types, in the prompt's form and the served token's."""
    q, k, v, _ = (x.to(DEV) for x in make(1, 40, 40, 2, 1, 64, dtype, seed=17))
    y = attention.window_attention(q, k, v, window=9, scale=float("nan"))
    assert torch.isnan(y).all()
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    pool = [x[0].transpose(0, 1).unsqueeze(0).contiguous() for x in (k[:, :32], v[:, :32])]
    y = attention.paged_attention_step(q[:, 0], None, None, *pool, table, ints([32]), scale=float("nan"))
    assert torch.isnan(y).all()


def test_empty_lse_is_float32(gpu_lib):
    x = lambda T: torch.randn(2, T, 2, 64, device=DEV)
    q, k = x(3), x(0)
    torch.set_default_dtype(torch.float64)
    try:
        _, lse = attention.window_attention(q, k, k, return_lse=True)
    finally:
        torch.set_default_dtype(torch.float32)
    assert lse.dtype == torch.float32 and lse.shape == (2, 2, 3) and (lse == float("-inf")).all()


def test_forward_mode_is_refused(gpu_lib):
    """There is no forward-mode derivative: an error, not a result without its tangent."""
    q, k, v, t = make(1, 8, 8, 2, 2, 64, torch.float32, seed=18)
    q, k, v, t = (x.to(DEV) for x in (q, k, v, t))
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    with torch.autograd.forward_ad.dual_level():
        attention.window_attention(q, k, v)                          # (no tangent: as ever)
        for n in range(3):
            ins = [torch.autograd.forward_ad.make_dual(x, t) if i == n else x for i, x in enumerate((q, k, v))]
            with pytest.raises(ValueError, match="forward-mode"):
                attention.window_attention(*ins)
        q1 = torch.autograd.forward_ad.make_dual(q[:, 0], t[:, 0])
        with pytest.raises(ValueError, match="forward-mode"):
            attention.paged_attention_step(q1, None, None, *(x.transpose(1, 2).contiguous() for x in (k, v)), table, ints([8]))


@DTYPES
def test_a_new_token_without_a_place(gpu_lib, dtype):
    """Neither written nor seen: the call does what it does of a cache alone, and no cached token is lost."""
    q, kp, vp, table, _, ks, vs = paged([48, 40], 4, 2, 64, 16, dtype, seed=19)
    new = [torch.randn(2, 2, 64, generator=torch.Generator().manual_seed(n)).to(dtype).to(DEV) for n in (1, 2)]
    gone = table.clone()
    gone[0, 2] = -1
    gone[1, 2] = 10 ** 6
    for tab, lens in ((table, [49, 1000]), (gone, [48, 40])):        # longer than its table row; its page is not there
        kd, vd, td = kp.to(DEV), vp.to(DEV), tab.to(DEV)
        alone = attention.paged_attention_step(q.to(DEV), None, None, kd, vd, td, ints(lens))
        y = attention.paged_attention_step(q.to(DEV), *new, kd, vd, td, ints(lens))
        assert torch.equal(kd.cpu(), kp) and torch.equal(vd.cpu(), vp)
        assert torch.equal(y, alone) and torch.isfinite(y).all()


def parts(q, k, window, sinks):
    """Workspace bytes of the forward: more than none where its keys are split."""
    code = _lib.dtype_code(q.dtype)
    return _lib.load().gdnx_win_attn_fwd_workspace_bytes(*q.shape[:2], k.shape[1], q.shape[2], k.shape[2], q.shape[3],
                                                         window or 0, sinks, code)


@DTYPES
@HEADS
@pytest.mark.parametrize("shape", [
    (2, 33, 1500, 4, 2, None, 0, [1500, 1481]), (2, 33, 1500, 4, 2, None, 0, [1499, 70]),     # fewer tiles than parts
    (1, 40, 2500, 6, 2, 1500, 70, None), (4, 130, 1200, 16, 4, None, 0, [1200, 1070, 0, 1100]),
    (1, 1, 2000, 3, 1, None, 0, [2000])], ids=lambda s: "-".join(map(str, s[:7])) + f"-{s[7]}")
def test_split_keys(gpu_lib, shape, D, dtype):
    B, Tq, Tk, Hq, Hkv, window, sinks, lengths = shape
    x = make(B, Tq, Tk, Hq, Hkv, D, dtype, seed=14)
    assert parts(x[0], x[1], window, sinks) > 0
    check(*x, window, sinks, lengths)


@DTYPES
@HEADS
@pytest.mark.parametrize("bad", [float("nan"), float("-inf")])
def test_split_keys_beside_what_is_not_finite(gpu_lib, bad, D, dtype):
    """Inner tokens that some queries of their tile do not see: later ones, and those the window has left behind."""
    Tq, Tk, W, S, at = 100, 2600, 2200, 3, (310, 2550)
    q, k, v, _ = make(1, Tq, Tk, 4, 2, D, dtype, seed=15)
    assert parts(q, k, W, S) > 0
    hide = oa.visible(Tq, Tk, W, S, Tk)[:, list(at)].any(1)
    want, want_lse = oa.attention(q, k, v, W, S)
    assert hide.any() and not hide.all()
    for what in "kv":
        k2, v2 = k.clone(), v.clone()
        (k2 if what == "k" else v2)[0, list(at), :, 3] = bad
        y, lse = attention.window_attention(q.to(DEV), k2.to(DEV), v2.to(DEV), window=W, sinks=S, return_lse=True)
        assert rel(y[0, ~hide], want[0, ~hide]) <= TOL[dtype][0]
        assert float((lse[0][:, ~hide].cpu().double() - want_lse[0][:, ~hide]).abs().max()) <= 1e-4
        if what == "v":
            assert not torch.isfinite(y[0, hide][..., 3].float()).any()
            assert rel(y[0, hide][..., 4:], want[0, hide][..., 4:]) <= TOL[dtype][0]


@HEADS
@pytest.mark.parametrize("lens,Hq,Hkv,window", [([3000, 17, 900, 2000], 16, 4, None), ([5000], 32, 8, 700),
                                                ([100] * 20, 8, 2, None)])
def test_a_served_token_is_rounded_once(gpu_lib, lens, Hq, Hkv, window, D):
    """bf16: half a unit in the last place is 2^-8 of a power of two, so rounding a value m 2^e, 1 <= m < 2, is off by
    2^-8 / sqrt(3) / m of it, in the mean over a Gaussian's values 1.66e-3; a tenth more for a sample of some thousand.
    A probability rounded to bf16 before its product would add as much again in squares: 2.2e-3."""
    q, kp, vp, table, _, ks, vs = paged(lens, Hq, Hkv, D, 16, torch.bfloat16, seed=21)
    y = attention.paged_attention_step(q.to(DEV), None, None, kp.to(DEV), vp.to(DEV), table.to(DEV), ints(lens),
                                       window=window, sinks=4)
    assert rel(y, step_ref(q, ks, vs, window, 4)) <= 1.83e-3


@DTYPES
def test_scores_that_are_all_minus_infinity(gpu_lib, dtype):
    q, k, v, _ = (x.to(DEV) for x in make(1, 40, 40, 2, 1, 64, dtype, seed=22))
    q[..., 0], k[:, :20, :, 0] = 1.0, float("-inf")
    y, lse = attention.window_attention(q, k, v, window=9, return_lse=True)
    assert (y[:, :20] == 0).all() and (lse[..., :20] == float("-inf")).all()
    want = oa.attention(q[:, 20:], k[:, 20:], v[:, 20:], 9)           # the others see finite ones
    assert rel(y[:, 20:], want[0]) <= TOL[dtype][0] and torch.isfinite(lse[..., 20:]).all()
    pool = [x[0].transpose(0, 1).unsqueeze(0).contiguous() for x in (k[:, :32], v[:, :32])]
    y = attention.paged_attention_step(q[:, 0], None, None, *pool, torch.zeros(1, 1, dtype=torch.int32, device=DEV), ints([20]))
    assert (y == 0).all()
