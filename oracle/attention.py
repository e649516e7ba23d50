"""Plain statements, in 64 bits, of windowed attention with sinks, its
gradients, and the bookkeeping of a paged key-value cache (a few lines of
lists), for the tests of the attention kernels."""
from __future__ import annotations

import torch


def visible(Tq, Tk, window, sinks, length):
    """[Tq,Tk]: query i at position p = i + Tk - Tq sees key j if j <= p, p < length and
    (p - j < window or j < sinks); window None: every earlier key."""
    p = torch.arange(Tq)[:, None] + Tk - Tq
    j = torch.arange(Tk)[None]
    ok = (j <= p) & (p < length)
    if window is not None:
        ok = ok & ((p - j < window) | (j < sinks))
    return ok


def attention(q, k, v, window=None, sinks=0, scale=None, lengths=None, dy=None):
    """y [B,Tq,Hq,D] and lse [B,Hq,Tq] in float64; with dy also (dq, dk, dv).
    What a pair's mask hides does not enter (keys and values of hidden places
    may be anything)."""
    B, Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    dy = None if dy is None else dy.detach().cpu().double()
    y, lse = torch.zeros_like(q), torch.full((B, Hq, Tq), float("-inf"), dtype=torch.float64)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        n = Tk if lengths is None else int(lengths[b])
        ok = visible(Tq, Tk, window, sinks, n)
        some = ok.any(1)
        kb, vb = (torch.where((torch.arange(Tk) < n)[:, None, None], x[b], 0.0) for x in (k, v))
        qb = torch.where(some[:, None, None], q[b], 0.0)
        for h in range(Hq):
            kh, vh = kb[:, h // (Hq // Hkv)], vb[:, h // (Hq // Hkv)]
            s = (qb[:, h] @ kh.T * scale).masked_fill(~ok, float("-inf"))
            L = torch.logsumexp(s, 1)
            p = torch.exp(s - torch.where(some, L, 0.0)[:, None])
            y[b, :, h], lse[b, h] = p @ vh, L
            if dy is not None:
                g = torch.where(some[:, None], dy[b, :, h], 0.0)
                dp = g @ vh.T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
                dq[b, :, h] = ds @ kh
                dk[b, :, h // (Hq // Hkv)] += ds.T @ qb[:, h]
                dv[b, :, h // (Hq // Hkv)] += p.T @ g
    return (y, lse) if dy is None else (y, lse, dq, dk, dv)


def paged_chunk(q, k_pages, v_pages, table, lengths, offsets, slots=None, window=None, sinks=0, scale=None):
    """y [N,Hq,D] in float64 of packed new tokens over a paged cache; table, lengths, offsets and slots are
    lists.  Tokens behind the last row are NaN."""
    N, Hq, D = q.shape
    n_pages, Hkv, page, _ = k_pages.shape
    scale = D ** -0.5 if scale is None else scale
    q, k_pages, v_pages = (x.detach().cpu().double() for x in (q, k_pages, v_pages))
    y = torch.full_like(q, float("nan"))
    for i in range(len(offsets) - 1):
        t0, c = offsets[i], offsets[i + 1] - offsets[i]
        r = i if slots is None else slots[i]
        n = lengths[r] if 0 <= r < len(table) else 0
        if n > len(table[0]) * page:
            n = 0
        for t in range(c):
            p = n - c + t
            seen = [j for j in range(p + 1) if (window is None or p - j < window or j < sinks)
                    and 0 <= table[r][j // page] < n_pages] if n else []
            y[t0 + t] = 0
            if not seen:
                continue
            at = torch.tensor([table[r][j // page] for j in seen])
            place = torch.tensor([j % page for j in seen])
            for h in range(Hkv):
                k, v = k_pages[at, h, place], v_pages[at, h, place]
                g = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
                y[t0 + t, g] = torch.softmax(q[t0 + t, g] @ k.T * scale, 1) @ v
    return y


class Pages:
    """The cache as lists: ``rows[r]`` is the row's page numbers (None where
    trimmed), ``lens[r]`` its tokens, ``refs`` the counts, ``data[page]`` any value."""

    def __init__(self, n_pages, page, rows, width):
        self.page, self.width = page, width
        self.rows, self.lens, self.refs = [[] for _ in range(rows)], [0] * rows, [0] * n_pages

    def _free(self):
        return [p for p, c in enumerate(self.refs) if c == 0]

    def reserve(self, slots, n_new):
        need = [-(-(self.lens[s] + n_new) // self.page) - -(-self.lens[s] // self.page)
                if 0 <= s < len(self.rows) else 0 for s in slots]
        short = sum(0 <= s < len(self.rows) and self.lens[s] + n_new > self.width * self.page for s in slots)
        if short or sum(need) > len(self._free()):
            return None
        free, start = self._free(), []
        for s, n in zip(slots, need):
            if not 0 <= s < len(self.rows):
                start.append(-1)
                continue
            for _ in range(n):
                p = free.pop(0)
                self.rows[s].append(p)
                self.refs[p] = 1
            start.append(self.lens[s])
            self.lens[s] += n_new
        return start

    def reserve_packed(self, slots, n_new, tokens):
        """(offsets, start, positions, places), or None where a row, the pool or the batch is too small."""
        n_new, here = [max(c, 0) for c in n_new], [0 <= s < len(self.rows) for s in slots]
        need = [-(-(self.lens[s] + c) // self.page) - -(-self.lens[s] // self.page) if ok else 0
                for s, c, ok in zip(slots, n_new, here)]
        short = any(ok and self.lens[s] + c > self.width * self.page for s, c, ok in zip(slots, n_new, here))
        if short or sum(need) > len(self._free()) or sum(n_new) > tokens:
            return None
        free, offsets, start, positions, places = self._free(), [0], [], [], []
        for s, c, n, ok in zip(slots, n_new, need, here):
            offsets.append(offsets[-1] + c)
            start.append(self.lens[s] if ok else -1)
            if not ok:
                positions += [-1] * c
                places += [-1] * c
                continue
            for _ in range(n):
                self.rows[s].append(free.pop(0))
                self.refs[self.rows[s][-1]] = 1
            for p in range(self.lens[s], self.lens[s] + c):
                pg = self.rows[s][p // self.page]
                positions.append(p)
                places.append(-1 if pg is None else pg * self.page + p % self.page)
            self.lens[s] += c
        more = [-1] * (tokens - offsets[-1])
        return offsets, start, positions + more, places + more

    def fork(self, parents, children):
        """(page, copy) pairs, or None where pages are missing."""
        free, moves = self._free(), []
        if sum(self.lens[p] % self.page != 0 for p in parents) > len(free):
            return None
        for p, c in zip(parents, children):
            row = list(self.rows[p])
            if self.lens[p] % self.page:
                new = free.pop(0)
                self.refs[new] = 1
                moves.append((row[-1], new))
                row[-1] = new
                shared = row[:-1]
            else:
                shared = row
            for x in shared:
                if x is not None:
                    self.refs[x] += 1
            self.rows[c], self.lens[c] = row, self.lens[p]
        return moves

    def free(self, slots):
        for s in slots:
            for p in self.rows[s]:
                if p is not None:
                    self.refs[p] -= 1
            self.rows[s], self.lens[s] = [], 0

    def trim(self, slots, window, sinks):
        for s in slots:
            for c, p in enumerate(self.rows[s]):
                if p is not None and c * self.page >= sinks and (c + 1) * self.page <= self.lens[s] - window:
                    self.refs[p] -= 1
                    self.rows[s][c] = None

    def compact(self):
        used = sum(c > 0 for c in self.refs)
        src = [p for p, c in enumerate(self.refs) if c > 0 and p >= used]
        dst = [p for p, c in enumerate(self.refs) if c == 0 and p < used]
        to = dict(zip(src, dst))
        for s, d in to.items():
            self.refs[d], self.refs[s] = self.refs[s], 0
        self.rows = [[to.get(p, p) for p in r] for r in self.rows]
        return list(to.items())

    def table(self):
        return [[-1 if p is None else p for p in r] + [-1] * (self.width - len(r)) for r in self.rows]
