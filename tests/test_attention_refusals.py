"""Arguments that the attention and page entry points refuse, before they touch a GPU."""
import ctypes

import pytest
import torch

from gdnx_amd import _lib, attention, pages

VP = lambda x: None if x is None else ctypes.c_void_p(x)


def _win(over, bwd=False):
    a = dict(q=64, k=64, v=64, lengths=None, y=64, low=64, lse=64, dy=64, dq=64, dk=64, dv=64, ws=64, st=[128] * 9, B=1, Tq=8,
             Tk=8, Hq=2, Hkv=1, D=64, window=0, sinks=0, scale=0.125, dt=_lib.DTYPE_BF16)
    a.update(over)
    lib = _lib.load()
    ints = [a[n] for n in ("B", "Tq", "Tk", "Hq", "Hkv", "D", "window", "sinks")]
    names = ("q", "k", "v", "lengths", "y", "low", "lse") + (("dy", "dq", "dk", "dv", "ws") if bwd else ("ws",))
    fn = lib.gdnx_win_attn_bwd if bwd else lib.gdnx_win_attn_fwd
    return fn(*(VP(a[n]) for n in names), *a["st"], *ints, a["scale"], a["dt"], None), lib.gdnx_last_error().decode()


@pytest.mark.parametrize("bwd", [False, True])
@pytest.mark.parametrize("over,code,msg", [
    (dict(q=None), -1, "non-null"), (dict(k=72), -1, "aligned"), (dict(dt=2), -1, "dtype"), (dict(D=96), -2, "head_dim"),
    (dict(Hq=3, Hkv=2), -2, "multiple"), (dict(Tq=0), -2, "sizes"), (dict(Tk=1 << 30), -2, "sizes"),
    (dict(B=1 << 20, Hq=64), -2, "too many"), (dict(window=-1), -2, "negative"), (dict(sinks=-1), -2, "negative"),
    (dict(st=[128] * 4 + [100] + [128] * 4), -2, "strides"), (dict(st=[-128] + [128] * 8), -2, "strides")])
def test_window_attention_refuses(over, code, msg, bwd):
    rc, err = _win(over, bwd)
    assert rc == code and msg in err


def test_window_attention_needs_its_workspace():
    rc, err = _win(dict(ws=None), True)
    assert rc == -3 and "workspace" in err
    rc, err = _win(dict(ws=None, Tk=1 << 20))            # few queries, many keys: split over the keys
    assert rc == -3 and "workspace" in err
    lib = _lib.load()
    assert lib.gdnx_win_attn_bwd_workspace_bytes(2, 100, 100, 4, 2, 64, 10, 2, _lib.DTYPE_BF16) >= 2 * 100 * 4 * 4
    assert lib.gdnx_win_attn_bwd_workspace_bytes(2, 100, 100, 4, 3, 64, 10, 2, _lib.DTYPE_BF16) == -1


def _step(over):
    a = dict(q=64, k=64, v=64, kp=64, vp=64, table=64, lengths=64, slots=None, y=64, ws=64, NS=2, rows=2, width=4,
             n_pages=8, page=16, Hq=2, Hkv=1, D=64, window=0, sinks=0, scale=0.125, dt=_lib.DTYPE_BF16)
    a.update(over)
    lib = _lib.load()
    v = list(a.values())
    return lib.gdnx_paged_attn_step(*map(VP, v[:10]), *v[10:], None), lib.gdnx_last_error().decode()


@pytest.mark.parametrize("over,code,msg", [
    (dict(table=None), -1, "non-null"), (dict(k=None), -1, "together"), (dict(vp=72), -1, "aligned"),
    (dict(dt=9), -1, "dtype"), (dict(D=80), -2, "head_dim"), (dict(page=24), -2, "power of two"),
    (dict(page=0), -2, "power of two"), (dict(NS=3), -2, "rows"), (dict(n_pages=0), -2, "sizes"),
    (dict(width=1 << 27), -2, "sizes"), (dict(Hq=5, Hkv=2), -2, "multiple"),
    (dict(ws=None, width=4096), -3, "workspace")])
def test_paged_step_refuses(over, code, msg):
    rc, err = _step(over)
    assert rc == code and msg in err


def test_page_operations_refuse():
    lib, p, err = _lib.load(), VP(64), lambda: lib.gdnx_last_error().decode()
    assert lib.gdnx_pages_reserve(p, p, p, p, p, p, None, 1, 1, 1, 1, 1, 16, None) == -3 and "workspace" in err()
    assert lib.gdnx_pages_reserve(p, p, p, p, p, p, p, 1, -1, 1, 1, 1, 16, None) == -2
    assert lib.gdnx_pages_reserve(p, p, p, p, None, p, p, 1, 1, 1, 1, 1, 16, None) == -1
    assert lib.gdnx_pages_write(p, p, p, p, p, p, p, 1, 1, 0, 1, 1, 1, 16, 1, 64, 1, None) == -2
    assert lib.gdnx_pages_write(p, p, p, VP(72), p, p, p, 1, 1, 1, 1, 1, 1, 16, 1, 64, 1, None) == -1
    assert lib.gdnx_pages_copy(p, p, p, p, 0, 1, 1, 16, 1, 64, 1, None) == -2 and "layers" in err()
    assert lib.gdnx_pages_fork(p, p, p, p, p, p, p, p, None, 1, 1, 1, 1, 1, 16, 1, 64, 1, None) == -3
    assert lib.gdnx_pages_free(p, p, p, p, 0, 1, 1, 1, None) == -2
    assert lib.gdnx_pages_trim(p, p, p, p, 0, 0, 1, 1, 1, 1, 16, None) == -2 and "window" in err()
    assert lib.gdnx_pages_compact(p, p, p, p, p, p, p, 1, 1, 1, 1, 48, 1, 64, 1, None) == -2 and "power" in err()
    assert lib.gdnx_pages_workspace_bytes(-1, 4) == -1 and lib.gdnx_pages_workspace_bytes(3, 4) > 0


def test_python_refuses():
    x = torch.zeros(1, 4, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        attention.window_attention(x, x, x)
    with pytest.raises(ValueError, match="negative"):
        attention.window_attention(x, x, x, window=-3)
    with pytest.raises(ValueError, match="int32"):
        pages.pages_free(torch.zeros(2, 2), torch.zeros(2), torch.zeros(4), torch.zeros(1))
    with pytest.raises(ValueError, match="power of two"):
        pages.PagedKVCache(8, 12, 1, 64, 2, 64, device="cpu")


def test_cache_rows_on_the_host():
    c = pages.PagedKVCache(8, 16, 1, 64, 3, 64, device="cpu")
    a, b = c.alloc(2)
    with pytest.raises(RuntimeError, match="full"):
        c.alloc(2)
    with pytest.raises(ValueError, match="twice"):
        c.reserve([a, a])
    with pytest.raises(ValueError, match="not allocated"):
        c.reserve([a, 2])
    with pytest.raises(ValueError, match="holds"):
        c.reserve([b], 65)
    with pytest.raises(RuntimeError, match="pages asked"):
        c.refs.fill_(1)
        c._free_bound = 0
        c.reserve([a], 1)
