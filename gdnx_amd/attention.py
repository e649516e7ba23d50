"""Softmax attention for the layers of a hybrid model that are not recurrent.

``window_attention`` is differentiable attention over a sliding window of the
last tokens and the first few ones (sinks), for training and prompts;
``paged_attention_step`` serves one token per sequence from a paged key-value
cache (``gdnx_amd.pages``) under the same visibility rule.  Grouped heads:
query head h reads key head h // (Hq // Hkv).  The kernels are
csrc/attn_win.hip and csrc/attn_paged.hip (gdnx_win_attn_*,
gdnx_paged_attn_step in include/gdnx.h).
"""
from __future__ import annotations

import functools

import torch
from torch.autograd import forward_ad

from . import _lib
from .ops import _need, empty_result


def _window(window, sinks):
    window, sinks = 0 if window is None else int(window), int(sinks)
    _need(window >= 0 and sinks >= 0, "window and sinks must not be negative")
    return min(window, 1 << 30), min(sinks, 1 << 30)


@functools.lru_cache(maxsize=4096)
def _bytes(query, *sizes):
    """A workspace's bytes: the library's size query, once per sizes."""
    return getattr(_lib.load(), query)(*sizes)


def _addr(t):
    return None if t is None else t.data_ptr()


def _no_tangents(*ts):
    if forward_ad._current_level >= 0:          # (inside dual_level() only)
        _need(all(t is None or forward_ad.unpack_dual(t).tangent is None for t in ts),
              "attention has no forward-mode derivative")


def _rows16(t):
    """t with D contiguous and every other stride that is used a multiple of 16
    bytes, as the kernels read it (views of a fused projection are taken as they
    are; axes of one element may have any stride)."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():
            return t                    # (D is 64 or 128: every row is whole units)
        unit = 16 // t.element_size()
        if t.stride(-1) == 1 and all(s % unit == 0 or n == 1 for s, n in zip(t.stride()[:-1], t.shape)) and (
                t.stride(1) <= 1 << 24 or t.shape[1] == 1):
            return t
    return t.contiguous() if not t.is_contiguous() else t.clone()


def _strides(t):
    """Batch, token and head stride; none that an axis of one element has of its own."""
    if t.is_contiguous():
        _, T, H, D = t.shape
        return T * H * D, H * D, D
    st = t.stride()
    return st[:3] if 1 not in t.shape else [0 if n == 1 else s for s, n in zip(st[:3], t.shape)]


def _check(q, k, v, lengths):
    _need(q.is_cuda, "gdnx ops need CUDA (HIP) tensors")
    _need(q.dim() == 4 and k.dim() == 4 and k.shape == v.shape, "q must be [B,Tq,Hq,D], k and v [B,Tk,Hkv,D]")
    _need(q.dtype == k.dtype == v.dtype, "q, k, v must share dtype")
    _need(k.device == q.device and v.device == q.device, "inputs must be on one device")
    B, Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[1:3]
    _need(k.shape[0] == B and k.shape[3] == D, "q, k, v must share batch and head dim")
    _need(Hkv > 0 and Hq > 0 and Hq % Hkv == 0, "query heads must be a multiple of key heads")
    if lengths is not None:
        _need(tuple(lengths.shape) == (B,) and lengths.dtype == torch.int32 and lengths.is_contiguous()
              and lengths.device == q.device, "lengths must be contiguous int32 [B] on q's device")
    return B, Tq, Tk, Hq, Hkv, D


def _forward(q, k, v, window, sinks, scale, lengths, want_lse, train=False):
    B, Tq, Tk, Hq, Hkv, D = _check(q, k, v, lengths)
    code = _lib.dtype_code(q.dtype)
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    y = torch.empty(B, Tq, Hq, D, dtype=q.dtype, device=q.device)
    lse = torch.empty(B, Hq, Tq, dtype=torch.float32, device=q.device) if want_lse else None
    low = torch.empty_like(y) if train and q.dtype == torch.bfloat16 else None      # y minus its rounding
    nws = _bytes("gdnx_win_attn_fwd_workspace_bytes", B, Tq, Tk, Hq, Hkv, D, window, sinks, code)
    ws = torch.empty(nws, dtype=torch.uint8, device=q.device) if nws > 0 else None
    _lib.call("gdnx_win_attn_fwd", q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(), _addr(lengths), y.data_ptr(),
              _addr(low), _addr(lse), _addr(ws), *_strides(q), *_strides(k), *_strides(v), B, Tq, Tk, Hq,
              Hkv, D, window, sinks, scale, code)
    return q, k, v, y, lse, low


class WindowAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, scale, lengths):
        q, k, v, y, lse, low = _forward(q, k, v, window, sinks, scale, lengths, True, True)
        ctx.save_for_backward(q, k, v, lengths, y, lse, low)
        ctx.args = (window, sinks, scale)
        ctx.mark_non_differentiable(lse)
        return y, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _):
        q, k, v, lengths, y, lse, low = ctx.saved_tensors
        window, sinks, scale = ctx.args
        B, Tq, Hq, D = q.shape
        Tk, Hkv = k.shape[1:3]
        code = _lib.dtype_code(q.dtype)
        dy = _rows16(dy.to(q.dtype).contiguous())
        dq = torch.empty(B, Tq, Hq, D, dtype=q.dtype, device=q.device)
        dk, dv = (torch.empty(B, Tk, Hkv, D, dtype=q.dtype, device=q.device) for _ in range(2))
        nws = _bytes("gdnx_win_attn_bwd_workspace_bytes", B, Tq, Tk, Hq, Hkv, D, window, sinks, code)
        _need(nws >= 0, "invalid sizes")
        ws = torch.empty(nws, dtype=torch.uint8, device=q.device)
        _lib.call("gdnx_win_attn_bwd", q.device, q.data_ptr(), k.data_ptr(), v.data_ptr(), _addr(lengths),
                  y.data_ptr(), _addr(low), lse.data_ptr(), dy.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                  ws.data_ptr(), *_strides(q), *_strides(k), *_strides(v), B, Tq, Tk, Hq, Hkv, D, window,
                  sinks, scale, code)
        return dq, dk, dv, None, None, None, None


def window_attention(q, k, v, window=None, sinks=0, *, scale=None, lengths=None, return_lse=False):
    """Attention of q [B,Tq,Hq,D] over k, v [B,Tk,Hkv,D] (bfloat16 or float32,
    D 64 or 128, any strides), differentiable in q, k and v.

    Query i stands at position p = i + Tk - Tq and sees key j if j <= p and
    p - j < window or j < sinks (window None or 0: every earlier key).  lengths
    (int32 [B]): tokens at or beyond a row's length are padding, whatever they
    hold; their outputs and gradients are zero, as are those of queries before
    position 0.  A value within the length that is not finite reaches the
    outputs of the queries that see it, and gradients of its tile.  scale
    defaults to 1/sqrt(D).  Returns y [B,Tq,Hq,D], with return_lse also the
    log-sum-exp of each query's scores [B,Hq,Tq] (float32, -inf where nothing
    is seen, not differentiable).  There is no forward-mode derivative and no
    second one."""
    window, sinks = _window(window, sinks)
    _no_tangents(q, k, v)
    B, Tq, Tk, Hq, Hkv, D = _check(q, k, v, lengths)
    if B == 0 or Tq == 0 or Tk == 0:
        y = empty_result((B, Tq, Hq, D), q.dtype, q.device, q, k, v)
        return (y, torch.full((B, Hq, Tq), float("-inf"), dtype=torch.float32, device=q.device)) if return_lse else y
    scale = D ** -0.5 if scale is None else float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        y, lse = WindowAttentionFunction.apply(q, k, v, window, sinks, scale, lengths)
    else:
        y, lse = _forward(q, k, v, window, sinks, scale, lengths, return_lse)[3:5]
    return (y, lse) if return_lse else y


def paged_attention_step(q, k, v, k_pages, v_pages, table, lengths, *, slots=None, window=None, sinks=0, scale=None,
                         out=None):
    """One served token for every row: q [NS,Hq,D] over the row's cached tokens.

    k_pages, v_pages [n_pages,Hkv,page,D], table [rows,width] and lengths
    [rows] (int32) as ``gdnx_amd.pages`` keeps them; row s is table row
    slots[s] (int32 [NS]; outside the table: an empty row, y = 0), or s.  The
    token stands at position length - 1.  k, v [NS,Hkv,D] are its key and
    value, which the call also writes to their page; None where they are there
    already; a token that has no place in the table is neither written nor seen.
    window, sinks and scale as in ``window_attention``.  Returns y
    [NS,Hq,D] (or ``out``), which is not differentiable: no gradient reaches the
    inputs."""
    window, sinks = _window(window, sinks)
    _no_tangents(q, k, v, k_pages, v_pages)
    dev, dtype = q.device, q.dtype
    _need(q.is_cuda and q.dim() == 3, "q must be a CUDA (HIP) tensor [NS,Hq,D]")
    NS, Hq, D = q.shape
    _need(k_pages.dim() == 4 and k_pages.shape == v_pages.shape and k_pages.shape[3] == D,
          "k_pages and v_pages must share shape [n_pages,Hkv,page,D]")
    n_pages, Hkv, page, _ = k_pages.shape
    _need(Hkv > 0 and Hq % Hkv == 0, "query heads must be a multiple of key heads")
    _need(table.dim() == 2 and lengths.dim() == 1 and lengths.shape[0] == table.shape[0],
          "table must be [rows,width], lengths [rows]")
    rows, width = table.shape
    _need((k is None) == (v is None), "k and v must be given together")
    if k is not None:
        _need(k.shape == v.shape == (NS, Hkv, D) and k.dtype == v.dtype == dtype and k.device == v.device == dev,
              "k and v must be [NS,Hkv,D] of q's dtype on q's device")
        k, v = _rows16(k.contiguous()), _rows16(v.contiguous())
    if slots is None:
        _need(NS <= rows, "more rows than the table has: name their slots")
    else:
        _need(slots.shape == (NS,) and slots.dtype == torch.int32 and slots.is_contiguous() and slots.device == dev,
              "slots must be contiguous int32 [NS] on q's device")
    _need(table.dtype == lengths.dtype == torch.int32 and table.is_contiguous() and lengths.is_contiguous()
          and table.device == lengths.device == dev, "table and lengths must be contiguous int32 on q's device")
    _need(k_pages.dtype == v_pages.dtype == dtype and k_pages.device == v_pages.device == dev
          and k_pages.is_contiguous() and v_pages.is_contiguous(),
          "k_pages and v_pages must be contiguous, of q's dtype and device")
    code = _lib.dtype_code(q.dtype)
    if out is None:
        out = torch.empty(NS, Hq, D, dtype=q.dtype, device=q.device)
    else:
        _need(tuple(out.shape) == (NS, Hq, D) and out.dtype == q.dtype and out.is_contiguous()
              and out.device == q.device, "out must be contiguous [NS,Hq,D] of q's dtype")
    if NS == 0:
        return out
    q = _rows16(q.contiguous())
    nws = _bytes("gdnx_paged_attn_workspace_bytes", NS, width, page, Hq, Hkv, D, window, sinks, code)
    ws = torch.empty(nws, dtype=torch.uint8, device=dev) if nws > 0 else None
    _lib.call("gdnx_paged_attn_step", q.device, q.data_ptr(), _addr(k), _addr(v), k_pages.data_ptr(),
              v_pages.data_ptr(), table.data_ptr(), lengths.data_ptr(), _addr(slots), out.data_ptr(), _addr(ws), NS,
              rows, width, n_pages, page, Hq, Hkv, D, window, sinks, D ** -0.5 if scale is None else float(scale), code)
    return out
