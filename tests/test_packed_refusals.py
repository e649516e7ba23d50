"""Arguments that the convolution and the packed entry points refuse, before they touch a GPU."""
import ctypes

import pytest
import torch

from gdnx_amd import _lib, attention, conv, pages

VP = lambda x: None if x is None else ctypes.c_void_p(x)  # noqa: E731
BF16, F32 = _lib.DTYPE_BF16, _lib.DTYPE_F32


def err():
    return _lib.load().gdnx_last_error().decode()


def _conv(over, bwd=False):
    a = dict(x=64, weight=64, bias=None, state=None, lengths=None, y=64, last=None, dy=64, dlast=None, dx=64, dw=64,
             db=None, dstate=None, ws=64, xb=80, xt=8, B=2, T=10, C=8, W=4, silu=1, wdt=F32, dt=BF16)
    a.update(over)
    names = ("x", "weight", "bias", "state", "lengths") + (
        ("dy", "dlast", "dx", "dw", "db", "dstate", "ws") if bwd else ("y", "last"))
    fn = _lib.load().gdnx_conv_bwd if bwd else _lib.load().gdnx_conv_fwd
    return fn(*(VP(a[n]) for n in names), a["xb"], a["xt"],
              *(a[n] for n in ("B", "T", "C", "W", "silu", "wdt", "dt")), None), err()


@pytest.mark.parametrize("bwd", [False, True])
@pytest.mark.parametrize("over,code,msg", [
    (dict(x=None), -1, "non-null"), (dict(weight=None), -1, "non-null"), (dict(dt=2), -1, "dtype"), (dict(wdt=7), -1, "dtype"),
    (dict(W=1), -2, "taps"), (dict(W=9), -2, "taps"), (dict(T=0), -2, "sizes"), (dict(B=0), -2, "sizes"),
    (dict(C=0), -2, "sizes"), (dict(C=1 << 25), -2, "sizes"), (dict(T=1 << 30), -2, "sizes"),
    (dict(B=1 << 20, T=1 << 20, C=1 << 10), -2, "too many"), (dict(B=1 << 25, T=1, C=1), -2, "too many"),
    (dict(xt=-8), -2, "strides"), (dict(xb=-1), -2, "strides")])
def test_conv_refuses(over, code, msg, bwd):
    rc, e = _conv(over, bwd)
    assert rc == code and msg in e


def test_conv_needs_outputs_and_workspace():
    assert _conv(dict(y=None))[0] == -1
    for n in ("dy", "dx", "dw"):
        assert _conv({n: None}, True)[0] == -1
    rc, e = _conv(dict(ws=None), True)
    assert rc == -3 and "workspace" in e
    assert _conv(dict(ws=66), True)[0] == -1
    size = _lib.load().gdnx_conv_bwd_workspace_bytes
    assert size(2, 10, 8, 4, BF16) >= 5 * 8 * 4 and size(2, 10, 8, 9, BF16) == -1 and size(0, 10, 8, 4, BF16) == -1
    assert size(4, 4096, 6144, 4, BF16) < 4 * 4096 * 6144 * 2 // 10          # beside x


def _packed(over):
    a = dict(x=64, off=64, weight=64, bias=None, pool=64, slots=64, to=None, y=64, xt=8, N=5, n=3, ns=4, C=8, W=4, silu=1,
             wdt=F32, dt=F32)
    a.update(over)
    v = list(a.values())
    return _lib.load().gdnx_conv_packed(*map(VP, v[:8]), *v[8:], None), err()


@pytest.mark.parametrize("over,code,msg", [
    (dict(x=None), -1, "non-null"), (dict(pool=None), -1, "non-null"), (dict(y=None), -1, "non-null"), (dict(dt=2), -1, "dtype"),
    (dict(W=1), -2, "taps"), (dict(n=0), -2, "sizes"), (dict(N=-1), -2, "sizes"), (dict(N=1 << 30), -2, "sizes"),
    (dict(ns=0), -2, "slots"), (dict(slots=None, n=5), -2, "slots"), (dict(off=None), -2, "one token"),
    (dict(xt=-1), -2, "strides"), (dict(C=1 << 24, N=1 << 26), -2, "too many")])
def test_conv_packed_refuses(over, code, msg):
    rc, e = _packed(over)
    assert rc == code and msg in e


def _chunk(over):
    a = dict(q=64, kp=64, vp=64, table=64, lengths=64, off=64, slots=None, y=64, ws=64, qt=128, qh=64, N=20, n=2, rows=2,
             width=4, n_pages=8, page=16, Hq=2, Hkv=1, D=64, window=0, sinks=0, scale=0.125, dt=BF16)
    a.update(over)
    v = list(a.values())
    return _lib.load().gdnx_chunk_attn(*map(VP, v[:9]), *v[9:], None), err()


@pytest.mark.parametrize("over,code,msg", [
    (dict(q=None), -1, "non-null"), (dict(off=None), -1, "non-null"), (dict(vp=72), -1, "aligned"), (dict(y=8), -1, "aligned"),
    (dict(dt=9), -1, "dtype"), (dict(D=80), -2, "head_dim"), (dict(page=24), -2, "power of two"), (dict(n=3), -2, "rows"),
    (dict(n=0), -2, "sizes"), (dict(N=-1), -2, "sizes"), (dict(n_pages=0), -2, "sizes"), (dict(width=1 << 27), -2, "sizes"),
    (dict(Hq=5, Hkv=2), -2, "multiple"), (dict(qt=100), -2, "strides"), (dict(qh=-64), -2, "strides"),
    (dict(window=-1), -2, "negative"), (dict(N=1 << 29, Hq=64, Hkv=64), -2, "too many")])
def test_chunk_refuses(over, code, msg):
    rc, e = _chunk(over)
    assert rc == code and msg in e


def test_packed_page_operations_refuse():
    lib, p = _lib.load(), VP(64)
    res = lambda *a: lib.gdnx_pages_reserve_packed(*a, None)  # noqa: E731
    assert res(*[p] * 11, 0, 5, 1, 1, 1, 16) == -2 and res(*[p] * 11, 1, -1, 1, 1, 1, 16) == -2
    assert res(*[p] * 10, None, 1, 5, 1, 1, 1, 16) == -3 and "workspace" in err()
    assert res(*[p] * 4, None, *[p] * 6, 1, 5, 1, 1, 1, 16) == -1
    assert res(*[p] * 8, None, p, p, 1, 5, 1, 1, 1, 16) == -1                  # tokens without places
    assert res(*[p] * 11, 1, 5, 1, 1, 1, 24) == -2 and "power of two" in err()
    assert res(*[p] * 11, 1, 5, 1, 1, 1 << 20, 1 << 11) == -2 and "2^31" in err()
    put = lambda *a: lib.gdnx_pages_write_packed(*a, None)  # noqa: E731
    st = [64] * 6
    assert put(p, p, p, p, None, *st, 1, 4, 8, 16, 1, 64, BF16) == -1
    assert put(p, VP(72), p, p, p, *st, 1, 4, 8, 16, 1, 64, BF16) == -1 and "aligned" in err()
    assert put(p, p, p, p, p, *st, 1, 0, 8, 16, 1, 64, BF16) == -2
    assert put(p, p, p, p, p, 64, 4, 64, 64, 64, 64, 1, 4, 8, 16, 1, 64, BF16) == -2 and "strides" in err()
    assert put(p, p, p, p, p, *st, 0, 4, 8, 16, 1, 64, BF16) == -2 and "layers" in err()
    assert lib.gdnx_pages_packed_workspace_bytes(3, 4) >= 32 and lib.gdnx_pages_packed_workspace_bytes(-1, 4) == -1


def test_python_refuses():
    x, w = torch.zeros(2, 5, 8), torch.zeros(8, 4)
    with pytest.raises(ValueError, match="CUDA"):
        conv.causal_conv(x, w)
    with pytest.raises(ValueError, match="CUDA"):
        conv.causal_conv_step(x[0], torch.zeros(5, 3, 8), w)
    with pytest.raises(ValueError, match="offsets"):
        conv.causal_conv_packed(x[0], torch.zeros(3), torch.zeros(5, 3, 8), w)
    with pytest.raises(ValueError, match="taps"):
        conv._weight(x, torch.zeros(8, 9), None)
    with pytest.raises(ValueError, match="weight"):
        conv._weight(x, torch.zeros(7, 4), None)
    with pytest.raises(ValueError, match="bias"):
        conv._weight(x, w, torch.zeros(7))
    with pytest.raises(ValueError, match="float32 or of x's dtype"):
        conv._weight(x, w.half(), None)
    with pytest.raises(ValueError, match="activation"):
        conv._silu("gelu")
    q = torch.zeros(5, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        attention.paged_attention_chunk(q, q, q, q, q, q)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="int32"):
        pages.pages_reserve_packed(i[None], i, i, i, i, 16, i[:2], 4)
    with pytest.raises(ValueError, match="k_pages and v_pages"):
        pages.pages_write_packed(q, q, q, q, i)


@pytest.mark.parametrize("dt", [BF16, F32])
def test_chunk_workspace_is_whole_units_of_16_bytes(dt):
    """Parts of long rows lie before spans of short ones, which are read 16 bytes at a time."""
    size = _lib.load().gdnx_chunk_attn_workspace_bytes
    for N in (43, 45, 129, 2049):
        for n in (1, 2, 3):
            for width in (40, 50, 63, 200):
                for Hq in (1, 3):
                    assert size(N, n, width, 16, Hq, Hq, 64, 0, 0, dt) % 16 == 0
