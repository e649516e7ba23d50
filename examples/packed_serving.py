"""A hybrid block with a short convolution, served in packed steps: prompts taken in by pieces beside single tokens.

    python examples/packed_serving.py

The block is the one of hybrid.py with a causal convolution over the projected
queries, keys and values of its recurrent layer.  A training step runs it over
a padded batch.  The server then gets, at every step, the next tokens of any of
its sequences, as many as it likes of each, packed without padding: the
convolution continues every sequence's last inputs (DecodeStateCache.convolve),
the attention layer reserves and fills pages for all of them at once and attends
over them (PagedKVCache.reserve_packed, write_packed, chunk).  What was served is
checked against the whole sequences run at once.
"""
from __future__ import annotations

import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

from hybrid import HybridBlock, train_step  # noqa: E402

from gdnx_amd import conv, gdn3  # noqa: E402
from gdnx_amd.decode_cache import DecodeStateCache  # noqa: E402
from gdnx_amd.pages import PagedKVCache  # noqa: E402


class ConvHybridBlock(HybridBlock):
    def __init__(self, taps=4, **kw):
        super().__init__(**kw)
        self.taps = taps
        self.filter = torch.nn.Parameter(torch.randn(3 * self.H * self.D, taps, device="cuda") * taps ** -0.5)

    def recurrent_inputs(self, x, qkv=None):
        """As HybridBlock's, from the convolved projection ``qkv`` (None: that of the whole sequences x)."""
        if qkv is None:
            qkv = conv.causal_conv(self.rec_in(x), self.filter)
        q, k, v = qkv.unflatten(-1, (3, self.H, self.D)).unbind(-3)
        beta, decay = self.rec_gates(x).float().unflatten(-1, (2, self.H, 1)).unbind(-3)
        q, k = F.normalize(q.float(), dim=-1).bfloat16(), F.normalize(k.float(), dim=-1).bfloat16()
        return q, k, v, beta.sigmoid(), -0.1 * decay.sigmoid()


class PackedServer:
    """Sequences of a ConvHybridBlock; a sequence is named by its (state slot, cache row)."""

    def __init__(self, block, rows=16, max_len=4096, n_pages=512, page=16):
        self.block = block
        self.states = DecodeStateCache(rows, block.H, 1, block.D, conv=(3 * block.H * block.D, block.taps))
        self.pages = PagedKVCache(n_pages, page, block.Hkv, block.D, rows, max_len)

    def start(self, n):
        return list(zip(self.states.alloc(n), self.pages.alloc(n)))

    def _recurrence(self, slots, counts, q, k, v, beta, g):
        """Single tokens in one call, each piece of several by itself."""
        at = [sum(counts[:i]) for i in range(len(counts))]
        y = torch.empty_like(v)
        a = gdn3.gdn3_coeff(k[None].contiguous(), beta[None].contiguous())[0]
        ones = [i for i, c in enumerate(counts) if c == 1]
        if ones:
            t = torch.tensor([at[i] for i in ones], device=v.device)
            y[t] = self.states.step([slots[i] for i in ones], q[t], k[t], v[t], a[t], a[t], g[t])[:, :, 0]
        for i, c in enumerate(counts):
            if c > 1:
                t = slice(at[i], at[i] + c)
                y[t] = self.states.prefill([slots[i]], *(z[None, t] for z in (q, k, v, a, a, g)))[0, :, :, 0]
        return y

    @torch.no_grad()
    def step(self, seqs, counts, x):
        """The next counts[i] tokens of every sequence, packed x [sum(counts),width]; returns their outputs."""
        b = self.block
        slots, rows = [s for s, _ in seqs], self.pages.rows_tensor([r for _, r in seqs])
        plan = self.pages.reserve_packed(rows, counts)
        qkv = self.states.convolve(slots, b.rec_in(x), b.filter, offsets=plan.offsets)
        x = x + b.rec_out(self._recurrence(slots, counts, *b.recurrent_inputs(x, qkv)).flatten(1))
        q, k, v = b.attention_inputs(x)
        self.pages.write_packed(plan, k, v, layer=0)
        y = self.pages.chunk(0, rows, plan, q, window=b.window, sinks=b.sinks)
        return x + b.att_out(y.flatten(1))

    def end(self, seqs):
        self.states.free([s for s, _ in seqs])
        self.pages.free([r for _, r in seqs])


def main(lengths=(300, 70, 181), piece=64, steps=20):
    torch.manual_seed(0)
    block = ConvHybridBlock()
    width = block.rec_out.out_features
    x = torch.randn(2, 300, width, device="cuda").bfloat16()
    grads = train_step(block, x, torch.randn_like(x), torch.tensor([300, 150], dtype=torch.int32, device="cuda"))
    assert all(torch.isfinite(g).all() for g in grads)
    print("training step: gradient norms", " ".join(f"{float(g.float().norm()):.1f}" for g in grads))

    server = PackedServer(block)
    seqs = server.start(len(lengths))
    whole = [torch.randn(n + steps, width, device="cuda").bfloat16() for n in lengths]
    at, out, turns = [0] * len(lengths), [[] for _ in lengths], 0
    while any(a < len(w) for a, w in zip(at, whole)):
        # a piece of every prompt that is not in yet, one token of every other sequence that still runs
        counts = [min(piece, n - a) if a < n else int(a < len(w)) for a, n, w in zip(at, lengths, whole)]
        packed = torch.cat([w[a:a + c] for w, a, c in zip(whole, at, counts)])
        for o, y in zip(out, server.step(seqs, counts, packed).split(counts)):
            o.append(y)
        at = [a + c for a, c in zip(at, counts)]
        turns += 1
    print(f"{sum(at)} tokens of {len(lengths)} sequences in {turns} packed steps")
    errs = []
    with torch.no_grad():
        for w, o in zip(whole, out):
            want = block(w[None])[0].float()
            errs.append(float((torch.cat(o).float() - want).norm() / want.norm()))
    print("served against the whole sequences:", " ".join(f"{e:.1e}" for e in errs))
    assert max(errs) < 1e-2
    server.end(seqs)
    assert server.pages.pages_in_use() == 0
    return max(errs)


if __name__ == "__main__":
    main()
