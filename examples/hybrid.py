"""A hybrid block trained and served: a gated delta-rule layer and a softmax-attention layer with a window and sinks.

    python examples/hybrid.py

The recurrent layer keeps one state per sequence (DecodeStateCache), the
attention layer its last keys and values in pages (PagedKVCache).  A training
step runs both layers forward and backward; then two prompts are taken in,
each is continued in three ways (the rows fork: full pages are shared, the
state is copied), tokens are served one at a time, pages that the window has
left behind are dropped and the pool is compacted.  What was served is checked
against the whole sequences run at once.
"""
from __future__ import annotations

import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from gdnx_amd import attention, gdn3  # noqa: E402
from gdnx_amd.decode_cache import DecodeStateCache  # noqa: E402
from gdnx_amd.pages import PagedKVCache  # noqa: E402


class HybridBlock(torch.nn.Module):
    def __init__(self, width=512, heads=4, q_heads=8, kv_heads=2, D=64, window=96, sinks=4):
        super().__init__()
        self.H, self.Hq, self.Hkv, self.D, self.window, self.sinks = heads, q_heads, kv_heads, D, window, sinks
        lin = lambda i, o: torch.nn.Linear(i, o, bias=False, dtype=torch.bfloat16, device="cuda")
        self.rec_in, self.rec_gates, self.rec_out = lin(width, 3 * heads * D), lin(width, 2 * heads), lin(heads * D, width)
        self.att_in, self.att_out = lin(width, (q_heads + 2 * kv_heads) * D), lin(q_heads * D, width)

    def recurrent_inputs(self, x):
        """q, k, v [..,H,D] and the write strength and log-decay [..,H,1] of the recurrent layer."""
        q, k, v = self.rec_in(x).unflatten(-1, (3, self.H, self.D)).unbind(-3)
        beta, decay = self.rec_gates(x).float().unflatten(-1, (2, self.H, 1)).unbind(-3)
        q, k = F.normalize(q.float(), dim=-1).bfloat16(), F.normalize(k.float(), dim=-1).bfloat16()
        return q, k, v, beta.sigmoid(), -0.1 * decay.sigmoid()

    def attention_inputs(self, x):
        return self.att_in(x).unflatten(-1, (-1, self.D)).split([self.Hq, self.Hkv, self.Hkv], -2)

    def forward(self, x, lengths=None):
        """[B,T,width] -> [B,T,width]; lengths (int32 [B]): what lies behind a row's length is padding."""
        q, k, v, beta, g = self.recurrent_inputs(x)
        y = gdn3.gdn3_scan(q.contiguous(), k.contiguous(), v.contiguous(), beta.contiguous(), g.contiguous())
        x = x + self.rec_out(y.flatten(2))
        q, k, v = self.attention_inputs(x)
        y = attention.window_attention(q, k, v, self.window, self.sinks, lengths=lengths)
        return x + self.att_out(y.flatten(2))


class Server:
    """Sequences of a HybridBlock, one token at a time."""

    def __init__(self, block, rows=16, max_len=4096, n_pages=512, page=16):
        self.block = block
        self.states = DecodeStateCache(rows, block.H, 1, block.D)
        self.pages = PagedKVCache(n_pages, page, block.Hkv, block.D, rows, max_len)

    @torch.no_grad()
    def prompt(self, x):
        """Takes in prompts x [n,T,width]; returns (sequences, their last outputs)."""
        b, (n, T, _) = self.block, x.shape
        slots, rows = self.states.alloc(n), self.pages.alloc(n)
        q, k, v, beta, g = b.recurrent_inputs(x)
        a = gdn3.gdn3_coeff(k.contiguous(), beta.contiguous())
        x = x + b.rec_out(self.states.prefill(slots, q, k, v, a, a, g).flatten(2))
        q, k, v = b.attention_inputs(x)
        y = attention.window_attention(q, k, v, b.window, b.sinks)
        self.pages.write(rows, self.pages.reserve(rows, T), k.contiguous(), v.contiguous(), layer=0)
        return list(zip(slots, rows)), (x + b.att_out(y.flatten(2)))[:, -1]

    def fork(self, seqs, ways):
        """Every sequence continued in `ways` ways: itself and ways - 1 copies."""
        more = [s for s in seqs for _ in range(ways - 1)]
        slots, rows = self.states.alloc(len(more)), self.pages.fork([r for _, r in more])
        self.states.pool[slots] = self.states.pool[[s for s, _ in more]]
        new = list(zip(slots, rows))
        return [s for i, q in enumerate(seqs) for s in (q, *new[i * (ways - 1):(i + 1) * (ways - 1)])]

    @torch.no_grad()
    def step(self, seqs, x):
        """One token x [n,width] for every sequence; returns the outputs [n,width]."""
        b = self.block
        slots, rows = [s for s, _ in seqs], [r for _, r in seqs]
        q, k, v, beta, g = b.recurrent_inputs(x)
        a = gdn3.gdn3_coeff(k.contiguous().unsqueeze(1), beta.contiguous().unsqueeze(1)).squeeze(1)
        x = x + b.rec_out(self.states.step(slots, q, k, v, a, a, g).flatten(1))
        q, k, v = b.attention_inputs(x)
        self.pages.reserve(rows, 1)
        y = self.pages.step(0, rows, q, k, v, window=b.window, sinks=b.sinks)
        return x + b.att_out(y.flatten(1))

    def tidy(self, seqs):
        """Drops the pages that the window has left behind and gathers the rest."""
        self.pages.trim([r for _, r in seqs], self.block.window, self.block.sinks)
        self.pages.compact()

    def end(self, seqs):
        self.states.free([s for s, _ in seqs])
        self.pages.free([r for _, r in seqs])


def train_step(block, x, dy, lengths=None):
    """Loss <y, dy>; returns the gradient of every weight."""
    y = block(x, lengths)
    return torch.autograd.grad((y.float() * dy.float()).sum(), tuple(block.parameters()))


def main(T=300, steps=40, ways=3):
    torch.manual_seed(0)
    block = HybridBlock()
    width = block.rec_out.out_features
    x = torch.randn(2, T, width, device="cuda").bfloat16()
    lengths = torch.tensor([T, T // 2], dtype=torch.int32, device="cuda")
    grads = train_step(block, x, torch.randn_like(x), lengths)
    assert all(torch.isfinite(g).all() for g in grads)
    print("training step: gradient norms", " ".join(f"{float(g.float().norm()):.1f}" for g in grads))

    server = Server(block)
    seqs, _ = server.prompt(x)
    seqs = server.fork(seqs, ways)
    print(f"prompts of {T} tokens, {len(seqs)} sequences: {server.pages.pages_in_use()} pages")
    fed, out = [], []
    for t in range(steps):
        tok = torch.randn(len(seqs), width, device="cuda").bfloat16()
        fed.append(tok)
        out.append(server.step(seqs, tok))
        if t % 16 == 15:
            server.tidy(seqs)
    used = server.pages.pages_in_use()
    print(f"after {steps} tokens each: {used} pages, all among the pool's first {used}")
    with torch.no_grad():
        whole = block(torch.cat([x.repeat_interleave(ways, 0), torch.stack(fed, 1)], 1))[:, T:]
    err = float((torch.stack(out, 1).float() - whole.float()).norm() / whole.float().norm())
    print(f"served tokens against the whole sequences: {err:.1e}")
    assert err < 1e-2
    server.end(seqs)
    assert server.pages.pages_in_use() == 0
    return err


if __name__ == "__main__":
    main()
