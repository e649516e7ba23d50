"""A plain statement, in 64 bits, of the short causal convolution with its
activation and state, for the tests of the convolution kernels."""
from __future__ import annotations

import torch


def _row(line, weight, bias, silu):
    """[n + W - 1, C] inputs -> [n, C]: u_t = bias + sum_j weight[:, j] line[t + j]."""
    W = weight.shape[1]
    n = line.shape[0] - (W - 1)
    u = bias + sum(line[j:j + n] * weight[:, j] for j in range(W))
    return u / (1 + torch.exp(-u)) if silu else u


def causal_conv(x, weight, bias=None, state=None, lengths=None, silu=True):
    """y [B,T,C] and the state handed on [B,W-1,C], in float64, differentiable.
    What is padding does not enter."""
    B, T, C = x.shape
    W = weight.shape[1]
    bias = torch.zeros(C, dtype=torch.float64) if bias is None else bias
    ys, lasts = [], []
    for b in range(B):
        n = T if lengths is None else min(max(int(lengths[b]), 0), T)
        before = torch.zeros(W - 1, C, dtype=torch.float64) if state is None else state[b]
        line = torch.cat([before, x[b, :n]])
        ys.append(torch.cat([_row(line, weight, bias, silu), torch.zeros(T - n, C, dtype=torch.float64)]))
        lasts.append(line[n:])
    return torch.stack(ys), torch.stack(lasts)


def causal_conv_packed(x, offsets, pool, weight, bias=None, slots=None, to_slots=None, silu=True):
    """(y [N,C], pool) in float64 from offsets, slots and to_slots as lists; an
    empty row gives zeros, tokens behind the last row NaN."""
    y, new = torch.full_like(x, float("nan")), pool.clone()
    bias = torch.zeros(x.shape[1], dtype=torch.float64) if bias is None else bias
    for i in range(len(offsets) - 1):
        s = i if slots is None else slots[i]
        t = s if to_slots is None else to_slots[i]
        rows = slice(offsets[i], offsets[i + 1])
        if not 0 <= s < pool.shape[0]:
            y[rows] = 0
            continue
        line = torch.cat([pool[s], x[rows]])
        y[rows] = _row(line, weight, bias, silu)
        if 0 <= t < pool.shape[0]:
            new[t] = line[line.shape[0] - (weight.shape[1] - 1):]
    return y, new
