"""The short causal convolution that stands before a recurrence, trained and served.

The reference's layers convolve the projected queries, keys and values over the
last few tokens of every channel and apply SiLU (gdn3/gdn3_upgrade.py:760-762,
gdn3/kmd2_native.py:140-141) and keep no state for serving.  ``causal_conv`` is
that operator for padded batches, differentiable; ``causal_conv_packed``
continues packed rows of unlike lengths from the states of a pool, and
``causal_conv_step`` one token a row.  A state is the last W - 1 inputs
[W-1,C], oldest first.  The kernels are csrc/conv.hip (gdnx_conv_* in
include/gdnx.h).
"""
from __future__ import annotations

import torch

from . import _lib
from .attention import _addr, _bytes, _no_tangents
from .ops import _need, empty_result


def _weight(x, weight, bias):
    """(weight [C,W], bias, W, its dtype code), as the kernels read them."""
    C = x.shape[-1]
    if weight.dim() == 3 and weight.shape[1] == 1:      # as a depthwise library convolution keeps it
        weight = weight[:, 0]
    _need(weight.dim() == 2 and weight.shape[0] == C, "weight must be [C,W] (or [C,1,W]), C being x's channels")
    W, dtype = weight.shape[1], weight.dtype
    _need(2 <= W <= 8, "2 to 8 taps are supported")
    _need((dtype == torch.float32 or dtype == x.dtype) and weight.device == x.device,
          "weight must be float32 or of x's dtype, on x's device")
    if bias is not None:
        _need(bias.dim() == 1 and bias.shape[0] == C and bias.dtype == dtype and bias.device == x.device,
              "bias must be [C] of weight's dtype on x's device")
        bias = bias.contiguous()
    return weight.contiguous(), bias, W, _lib.dtype_code(dtype)


def _silu(activation):
    _need(activation == "silu" or activation is None, 'activation must be "silu" or None')
    return int(activation is not None)


def _channels(t):
    """t with its channels side by side (other strides as they are)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _bt_strides(x):
    """Batch and token stride; none that an axis of one element has of its own."""
    B, T, _ = x.shape
    b, t, _ = x.stride()
    return b if B > 1 else 0, t if T > 1 else 0


class CausalConvFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, silu, want_state):
        y, last, kept = _forward(x, weight, bias, state, lengths, silu, want_state)
        ctx.save_for_backward(*kept, lengths)
        ctx.args = silu, weight.shape
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dlast):
        x, w, b, state, lengths = ctx.saved_tensors
        silu, shape = ctx.args
        B, T, C = x.shape
        W, code = w.shape[1], _lib.dtype_code(x.dtype)
        dy = torch.zeros(B, T, C, dtype=x.dtype, device=x.device) if dy is None else dy.contiguous()
        dlast = None if dlast is None else dlast.contiguous()
        dx, dw = torch.empty(B, T, C, dtype=x.dtype, device=x.device), torch.empty_like(w)
        db = None if b is None else torch.empty_like(b)
        dstate = None if state is None else torch.empty_like(state)
        ws = torch.empty(_bytes("gdnx_conv_bwd_workspace_bytes", B, T, C, W, code), dtype=torch.uint8, device=x.device)
        st = _bt_strides(x)
        _lib.call("gdnx_conv_bwd", x.device, x.data_ptr(), w.data_ptr(), _addr(b), _addr(state), _addr(lengths),
                  dy.data_ptr(), _addr(dlast), dx.data_ptr(), dw.data_ptr(), _addr(db), _addr(dstate), ws.data_ptr(),
                  st[0], st[1], B, T, C, W, silu, _lib.dtype_code(w.dtype), code)
        return dx, dw.view(shape), db, dstate, None, None, None


def _forward(x, weight, bias, state, lengths, silu, want_state):
    """y, the state handed on (or None), and the inputs as the kernels read them."""
    weight, bias, W, wcode = _weight(x, weight, bias)
    x = _channels(x)
    B, T, C = x.shape
    state = None if state is None else state.contiguous()
    y = torch.empty(B, T, C, dtype=x.dtype, device=x.device)
    last = torch.empty(B, W - 1, C, dtype=x.dtype, device=x.device) if want_state else None
    st = _bt_strides(x)
    _lib.call("gdnx_conv_fwd", x.device, x.data_ptr(), weight.data_ptr(), _addr(bias), _addr(state), _addr(lengths),
              y.data_ptr(), _addr(last), st[0], st[1], B, T, C, W, silu, wcode, _lib.dtype_code(x.dtype))
    return y, last, (x, weight, bias, state)


def causal_conv(x, weight, bias=None, *, activation="silu", state=None, lengths=None, return_state=False):
    """Causal convolution of x [B,T,C] (bfloat16 or float32, any batch and token
    strides) along the tokens: u_t = bias + sum_j weight[:, j] x_{t-W+1+j}, then
    SiLU (activation None: nothing).  Differentiable in x, weight, bias and state.

    weight [C,W] (or [C,1,W]), W from 2 to 8, and bias [C] are float32 or of x's
    dtype; sums are float32 and rounded once.  state [B,W-1,C], in x's dtype:
    the inputs before token 0 (None: zeros).  lengths (int32 [B]): tokens at
    or beyond a row's length are padding, whatever they hold; their outputs
    and gradients are zero.  Returns y [B,T,C], with return_state also the last
    W - 1 inputs before each row's end [B,W-1,C].  There is no forward-mode
    derivative and no second one.  A step captured in a HIP graph takes leaves
    of its own (detached): autograd waits for the stream of an eager graph that
    still holds the same ones, which a capture does not allow."""
    _no_tangents(x, weight, bias, state, what="the convolution")
    _need(x.is_cuda and x.dim() == 3, "x must be a CUDA (HIP) tensor [B,T,C]")
    _lib.dtype_code(x.dtype)
    silu, (B, T, C) = _silu(activation), x.shape
    W = _weight(x, weight, bias)[2]
    if state is not None:
        _need(tuple(state.shape) == (B, W - 1, C) and state.dtype == x.dtype and state.device == x.device,
              "state must be [B,W-1,C] of x's dtype on x's device")
    if lengths is not None:
        _need(tuple(lengths.shape) == (B,) and lengths.dtype == torch.int32 and lengths.is_contiguous()
              and lengths.device == x.device, "lengths must be contiguous int32 [B] on x's device")
    srcs = (x, weight, bias, state)
    if x.numel() == 0:
        y = empty_result((B, T, C), x.dtype, x.device, *srcs)
        last = state.clone() if state is not None else empty_result((B, W - 1, C), x.dtype, x.device, *srcs)
    elif torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in srcs):
        y, last = CausalConvFunction.apply(x, weight, bias, state, lengths, silu, return_state)
    else:
        y, last, _ = _forward(x, weight, bias, state, lengths, silu, return_state)
    return (y, last) if return_state else y


def _slots(slots, n, x):
    if slots is not None:
        _need(slots.dim() == 1 and slots.shape[0] == n and slots.dtype == torch.int32 and slots.is_contiguous()
              and slots.device == x.device, "slots and to_slots must be contiguous int32 [n] on x's device")


def _packed(x, offsets, n, pool, weight, bias, slots, to_slots, activation, out):
    _no_tangents(x, weight, bias, pool, what="the convolution")
    _need(x.is_cuda and x.dim() == 2, "x must be a CUDA (HIP) tensor [tokens,C]")
    code, silu, (N, C) = _lib.dtype_code(x.dtype), _silu(activation), x.shape
    weight, bias, W, wcode = _weight(x, weight, bias)
    _need(pool.dim() == 3 and pool.shape[1] == W - 1 and pool.shape[2] == C and pool.dtype == x.dtype and pool.device == x.device
          and pool.is_contiguous(), "pool must be contiguous [n_slots,W-1,C] of x's dtype on x's device")
    _slots(slots, n, x)
    _slots(to_slots, n, x)
    _need(slots is not None or n <= pool.shape[0], "more rows than the pool has slots: name their slots")
    if out is None:
        out = torch.empty(N, C, dtype=x.dtype, device=x.device)
    else:
        _need(tuple(out.shape) == (N, C) and out.dtype == x.dtype and out.is_contiguous() and out.device == x.device
              and (N == 0 or out.data_ptr() != x.data_ptr()),
              "out must be contiguous, of x's shape, dtype and device, and not x")
    if n == 0 or C == 0:
        return out
    if pool.shape[0] == 0:                              # every row is an empty one, of a pool that is only looked at
        pool, slots, to_slots = torch.zeros(1, W - 1, C, dtype=x.dtype, device=x.device), torch.full_like(slots, -1), None
    x = _channels(x)
    _lib.call("gdnx_conv_packed", x.device, x.data_ptr(), _addr(offsets), weight.data_ptr(), _addr(bias),
              pool.data_ptr(), _addr(slots), _addr(to_slots), out.data_ptr(), x.stride(0) if N > 1 else 0, N, n, pool.shape[0], C, W,
              silu, wcode, code)
    return out


def causal_conv_packed(x, offsets, pool, weight, bias=None, *, slots=None, to_slots=None, activation="silu", out=None):
    """``causal_conv`` of packed rows, each continuing a state: row i has tokens
    x[offsets[i]:offsets[i+1]] (x [N,C], offsets int32 [n+1]; a row may have
    none) and continues pool[slots[i]] (pool [n_slots,W-1,C] in x's dtype;
    slots int32 [n], None: i; outside the pool: an empty row, y = 0).  Its new
    state goes to pool[to_slots[i]] (None: where the old one was; outside the
    pool: nowhere), so that tokens can be tried and taken back.  No slot that a
    row writes may be read or written by another row.  Returns y [N,C] (or ``out``,
    which keeps what it holds behind the last row's tokens; a new tensor's rows
    there are not initialised), which is not differentiable."""
    _need(offsets.dim() == 1 and offsets.numel() >= 1 and offsets.dtype == torch.int32 and offsets.is_contiguous()
          and offsets.device == x.device, "offsets must be contiguous int32 [n+1] on x's device")
    return _packed(x, offsets, offsets.numel() - 1, pool, weight, bias, slots, to_slots, activation, out)


def causal_conv_step(x, pool, weight, bias=None, *, slots=None, to_slots=None, activation="silu", out=None):
    """``causal_conv_packed`` of one token a row: x [n,C]."""
    return _packed(x, None, x.shape[0], pool, weight, bias, slots, to_slots, activation, out)
