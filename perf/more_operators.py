"""Performance cases of the operators that take in tokens: the short convolution before a recurrence, and batches of prompts' pieces, drafts and single tokens over a page cache.

A recurrent layer convolves its queries, keys and values over the last few
tokens of every channel before the recurrence; a server hands a model, at every
step, the next piece of some prompts beside one token of every running
sequence, packed without padding.

  kind     operator                                        in real use
  conv     conv.causal_conv forward + backward             a training step of the convolution before a recurrence
  tokens   conv.causal_conv_packed                         the same convolution served: packed rows of unlike lengths,
                                                           each continuing its own state
  admit    pages.pages_reserve_packed, pages.pages_free    pages for rows of unlike lengths, every packed token's row
                                                           position and place in the pool; the rows given back again
  write    pages.pages_write_packed                        packed keys and values to their places in every layer
  chunk    attention.paged_attention_chunk                 attention of packed new tokens over their rows' cached ones

With ``own`` false, ``run`` computes an operator from elementary torch
operations in float32; with ``own`` true it calls the package.

Convolution over W taps: u_t = bias + sum_j weight_j x_{t-W+1+j}, y = u sigmoid(u)
(or u); what lies before a row's first token comes from its state, the last
W - 1 inputs.  Attention: the n new tokens of a row of length len (the new ones
included) stand at positions len - n .. len - 1; position p sees key j if
j <= p and p - j < window (0: no window) or j < sinks.

Work counts each input that is needed and each output once; 4 D operations for
every visible pair of an attention.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the training step before the 16-head recurrent layer: its batch and length, the queries, keys and values of one
        # fused projection whose last columns are the output gate's
        dict(name="conv_layer", kind="conv", B=4, T=4096, C=6144, extra=2048, W=4, silu=True, bias=False, state=False,
             ragged=False, dtype="bf16"),
        # sequences continued from their states in one padded batch (one of them empty), float32, odd sizes everywhere
        dict(name="conv_continued_f32", kind="conv", B=5, T=519, C=771, extra=0, W=3, silu=True, bias=True, state=True,
             ragged=True, dtype="f32"),
        # a serving step: pieces of three prompts beside one token of every other sequence
        dict(name="tokens_mixed", kind="tokens", n=64, pieces=3, longest=1024, C=6144, W=4, silu=True, bias=False,
             dtype="bf16"),
        # a few interactive users: the smallest call, where latency counts
        dict(name="tokens_few", kind="tokens", n=3, pieces=0, longest=1, C=1536, W=4, silu=True, bias=True, dtype="bf16"),
        # prompts of unlike lengths enter a busy cache
        dict(name="admit_few", kind="admit", n=8, pieces=8, longest=300, rows=64, pages=2048, page=16),
        # a night's documents are queued at once
        dict(name="admit_many", kind="admit", n=512, pieces=480, longest=2000, rows=700, pages=65536, page=16),
        # the keys and values of a serving step's tokens, all layers at once
        dict(name="write_step", kind="write", n=64, pieces=3, longest=1024, layers=8, Hkv=4, D=128, page=64, dtype="bf16"),
        # one layer's, straight from its fused projection
        dict(name="write_fused_f32", kind="write", n=9, pieces=5, longest=301, layers=1, Hkv=6, D=64, page=16, dtype="f32"),
        # drafts of five tokens to be checked, for a few users
        dict(name="chunk_drafts", kind="chunk", n=8, pieces=8, longest=5, T=2000, Hq=16, Hkv=4, D=128, page=16, window=0,
             sinks=0, dtype="bf16"),
        # a serving step: pieces of three prompts beside single tokens of sequences at all stages
        dict(name="chunk_mixed", kind="chunk", n=64, pieces=3, longest=1024, T=8192, Hq=16, Hkv=4, D=128, page=64, window=0,
             sinks=0, dtype="bf16"),
        # the last piece of one long prompt
        dict(name="chunk_long", kind="chunk", n=1, pieces=1, longest=2048, T=30001, Hq=16, Hkv=4, D=128, page=128, window=0,
             sinks=0, dtype="bf16"),
        # the windowed layer of the float32 model: pages behind the window are gone already
        dict(name="chunk_window_f32", kind="chunk", n=12, pieces=5, longest=129, T=2999, Hq=6, Hkv=2, D=64, page=16,
             window=512, sinks=4, dtype="f32"),
    ]


def _size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("conv", "conv", "conv", "tokens", "tokens", "admit", "write", "chunk", "chunk", "chunk", "chunk"))
    dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
    if kind == "conv":
        C = rng.choice((_size(rng, 33, 8192), 64 * rng.randint(1, 128), 64 * rng.randint(1, 128)))
        B = rng.randint(1, 5)
        # at most half the listed layer's elements in float32, so that no call moves more bytes
        T = max(1, min(_size(rng, 16, 16384), 16000 * 6144 // (B * C) // (1 if dtype == "bf16" else 2)))
        return dict(kind=kind, B=B, T=T, C=C, extra=rng.choice((0, 0, 64 * rng.randint(1, 16))), W=rng.choice((2, 3, 4, 4, 4)),
                    silu=rng.random() < 0.8, bias=rng.random() < 0.5, state=rng.random() < 0.4, ragged=rng.random() < 0.4,
                    dtype=dtype)
    if kind in ("tokens", "admit"):
        n = _size(rng, 1, 256)
        pieces = rng.choice((0, rng.randint(0, min(n, 8)), n))
        longest = max(1, min(_size(rng, 2, 2048), 16384 // max(pieces, 1)))
        if kind == "tokens":
            return dict(kind=kind, n=n, pieces=pieces, longest=longest, C=64 * rng.randint(1, 96) + rng.choice((0, 0, 0, 7)),
                        W=rng.choice((2, 3, 4, 4, 4)), silu=rng.random() < 0.8, bias=rng.random() < 0.5, dtype=dtype)
        page = rng.choice((16, 32, 64, 128))
        return dict(kind=kind, n=n, pieces=pieces, longest=longest, rows=n + rng.randint(0, 100),
                    pages=2 * (n + pieces * -(-longest // page)) + _size(rng, 10, 30000), page=page)
    Hkv, D = rng.choice((1, 2, 3, 4, 8)), rng.choice((64, 128, 128))
    n = _size(rng, 1, 64)
    pieces = rng.choice((rng.randint(0, min(n, 4)), rng.randint(0, min(n, 4)), n))
    if kind == "write":
        return dict(kind=kind, n=n, pieces=pieces, longest=max(1, min(_size(rng, 2, 2048), 1024 // max(pieces, 1))),
                    layers=rng.choice((1, 1, 3, 8)), Hkv=min(Hkv, 4), D=D, page=rng.choice((16, 32, 64, 128)),
                    dtype="bf16" if dtype == "bf16" else "f32")
    Hq = Hkv * rng.choice([g for g in (1, 2, 3, 4, 8) if g * Hkv <= 16])
    longest = max(1, min(_size(rng, 2, 2048), 2048 // max(pieces, 1)))
    # pairs of queries and keys at most a quarter of the listed long prompt's (of that an eighth in float32)
    most = 16 * 2048 * 32000 // (4 if dtype == "bf16" else 32) // (Hq * (n + pieces * longest))
    T = max(16, min(_size(rng, 64, 32768), most, 500_000 // (n * Hkv)))
    return dict(kind=kind, n=n, pieces=pieces, longest=longest, T=T, Hq=Hq, Hkv=Hkv, D=D, page=rng.choice((16, 32, 64, 128)),
                window=rng.choice((0, 0, _size(rng, 32, 2048))), sinks=rng.choice((0, 4, 64)), dtype=dtype)


def _io(case):
    return torch.bfloat16 if case.get("dtype") == "bf16" else torch.float32


def _row_lengths(case):
    """Valid tokens of each row of a padded batch: unlike lengths, an empty row and a full one among them."""
    B, T = case["B"], case["T"]
    if not case["ragged"]:
        return [T] * B
    return [T if b == 0 else 0 if b == 2 else max(1, T * ((5 * b + 2) % 7 + 1) // 9) for b in range(B)]


def _counts(case):
    """New tokens of each row: pieces of unlike lengths first, then single tokens; of more than eight rows one has none."""
    n, L = case["n"], case["longest"]
    cs = [max(1, L - (L * ((29 * b) % 16)) // 32) if b < case["pieces"] else 1 for b in range(n)]
    if n > 8:
        cs[n // 2] = 0
    return cs


def _past(case):
    """Cached tokens of each row before the new ones: spread over the range; of more than eight rows one has none."""
    n, T = case["n"], case["T"]
    ls = [max(1, T - (T * ((37 * b) % 64)) // 64) for b in range(n)]
    if n > 8:
        ls[1] = 0
    return ls


def _first_kept(case, past):
    """The first cached token behind the sinks that a row still sees."""
    return max(0, past - case["window"] + 1) if case["window"] else 0


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
class _Draws:
    """Values of one seed, drawn on the GPU in a fixed order."""

    def __init__(self, seed):
        self.gen = torch.Generator(device=DEV).manual_seed(int(seed) % (1 << 63))

    def n(self, *shape, dtype=torch.float32):
        return torch.randn(*shape, generator=self.gen, device=DEV).to(dtype)

    def pool(self, *shape, dtype):
        """Cached values (a layer at a time, so that the float32 draws stay small)."""
        out = torch.empty(*shape, dtype=dtype, device=DEV)
        for i in range(shape[0]):
            out[i] = torch.randn(*shape[1:], generator=self.gen, device=DEV)
        return out

    def order(self, n):
        return torch.randperm(n, generator=self.gen, device=DEV)


def _ints(xs):
    return torch.tensor(xs, dtype=torch.int32, device=DEV)


def _offsets(counts):
    return _ints([sum(counts[:i]) for i in range(len(counts) + 1)])


def prepare(case, seed):
    d, io, kind = _Draws(seed), _io(case), case["kind"]
    st = {"case": case}
    if kind in ("conv", "tokens"):
        C, W = case["C"], case["W"]
        # (weights are kept in float32, as a trainer keeps them)
        st["weight"] = d.n(C, W) * W ** -0.5
        st["bias"] = d.n(C) * 0.2 if case["bias"] else None
    if kind == "conv":
        B, T, C, W = (case[n] for n in ("B", "T", "C", "W"))
        st["x"] = d.n(B, T, C + case["extra"], dtype=io)[..., :C]
        st["state"] = d.n(B, W - 1, C, dtype=io) if case["state"] else None
        st["lengths"] = _ints(_row_lengths(case)) if case["ragged"] else None
        st["dy"] = d.n(B, T, C, dtype=io)
        st["dstate"] = d.n(B, W - 1, C, dtype=io) if case["state"] else None
        st["leaves"] = [n for n in ("x", "weight", "bias", "state") if st[n] is not None]
        for n in st["leaves"]:
            st[n] = st[n].detach().requires_grad_(True)
        return st
    counts = _counts(case)
    n, N = case["n"], sum(counts)
    if kind == "tokens":
        st["x"] = d.n(N, C, dtype=io)
        # a row's new state goes to a slot of its own: the old one is kept until its tokens are accepted
        st["pool"] = d.n(2 * n + 3, W - 1, C, dtype=io)
        order = d.order(2 * n + 3).int()
        st["slots"], st["to"] = order[:n].clone(), order[n:2 * n].clone()
        st["offsets"] = _offsets(counts)
        return st
    if kind == "admit":
        rows, pages, page = case["rows"], case["pages"], case["page"]
        width = -(-case["longest"] // page) + 1
        st["table"] = torch.full((rows, width), -1, dtype=torch.int32, device=DEV)
        st["lengths"] = torch.zeros(rows, dtype=torch.int32, device=DEV)
        st["refs"] = torch.zeros(pages, dtype=torch.int32, device=DEV)
        st["refs"][d.order(pages)[:(pages - sum(-(-c // page) for c in counts)) // 2]] = 1      # other rows' pages
        st["slots"] = d.order(rows)[:n].int()
        st["n_new"], st["tokens"] = _ints(counts), N + 5           # (a batch of fixed size: its last tokens are nobody's)
        st["status"] = torch.zeros(2, dtype=torch.int32, device=DEV)
        return st
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    if kind == "write":
        L = case["layers"]
        pages = sum(-(-c // page) + 1 for c in counts) + 5
        pos = [torch.arange(c) + (13 * b) % page for b, c in enumerate(counts)]      # each row goes on inside a page
        base = [sum(-(-x // page) + 1 for x in counts[:b]) for b in range(n)]
        places = torch.cat([p % page + (p // page + base[b]) * page for b, p in enumerate(pos)]).to(DEV)
        order = d.order(pages)
        places = (order[places // page] * page + places % page).int()
        places[N // 2] = -1                                        # a token of an empty row
        st["places"] = places
        st["k_pages"], st["v_pages"] = d.pool(L, pages, Hkv, page, D, dtype=io), d.pool(L, pages, Hkv, page, D, dtype=io)
        qkv = d.n(L, N, 4 * Hkv, D, dtype=io)                      # queries, keys and values of a fused projection
        st["k"], st["v"] = qkv[:, :, 2 * Hkv:3 * Hkv], qkv[:, :, 3 * Hkv:]
        return st
    past = _past(case)
    lens = [p + c for p, c in zip(past, counts)]
    need = [-(-l // page) for l in lens]
    pages, width = sum(need) + 8, max(need) + 1
    order, rows = d.order(pages).int(), n + 2
    slots = d.order(rows)[:n]
    table = torch.full((rows, width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, r in enumerate(slots.tolist()):
        table[r, :need[b]] = order[at:at + need[b]]
        at += need[b]
        # what the window has left behind is gone, but for the sinks
        gone, kept = _first_kept(case, past[b]) // page, -(-case["sinks"] // page)
        table[r, kept:max(gone, kept)] = -1
    st["table"], st["slots"] = table, slots.int()
    st["lengths"] = torch.zeros(rows, dtype=torch.int32, device=DEV)
    st["lengths"][slots] = _ints(lens)
    st["offsets"] = _offsets(counts)
    st["k_pages"], st["v_pages"] = d.pool(pages, Hkv, page, D, dtype=io), d.pool(pages, Hkv, page, D, dtype=io)
    st["q"] = d.n(N, case["Hq"], D, dtype=io)
    st["counts"], st["past"] = counts, past                        # what a scheduler knows on the host
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    return (_RUN_OWN if own else _RUN_PLAIN)[st["case"]["kind"]](st)


def _own_conv(st):
    from gdnx_amd import conv
    res = conv.causal_conv(st["x"], st["weight"], st["bias"], activation="silu" if st["case"]["silu"] else None,
                           state=st["state"], lengths=st["lengths"], return_state=st["case"]["state"])
    outs = res if st["case"]["state"] else (res,)
    grads = torch.autograd.grad(outs, [st[n] for n in st["leaves"]],
                                grad_outputs=(st["dy"], st["dstate"])[:len(outs)])
    return (*(o.detach() for o in outs), *grads)


def _own_tokens(st):
    from gdnx_amd import conv
    y = conv.causal_conv_packed(st["x"], st["offsets"], st["pool"], st["weight"], st["bias"], slots=st["slots"],
                                to_slots=st["to"], activation="silu" if st["case"]["silu"] else None)
    return y, st["pool"]


def _own_admit(st):
    from gdnx_amd import pages
    plan = pages.pages_reserve_packed(st["table"], st["lengths"], st["refs"], st["slots"], st["n_new"],
                                      st["case"]["page"], st["status"], st["tokens"])
    pages.pages_free(st["table"], st["lengths"], st["refs"], st["slots"])
    return plan.offsets, plan.start, plan.positions, plan.places, st["table"], st["lengths"], st["refs"]


def _own_write(st):
    from gdnx_amd import pages
    pages.pages_write_packed(st["k"], st["v"], st["k_pages"], st["v_pages"], st["places"])
    return st["k_pages"], st["v_pages"]


def _own_chunk(st):
    from gdnx_amd import attention
    c = st["case"]
    return attention.paged_attention_chunk(st["q"], st["k_pages"], st["v_pages"], st["table"], st["lengths"],
                                           st["offsets"], slots=st["slots"], window=c["window"] or None,
                                           sinks=c["sinks"])


def _within(st, T):
    """[B,T,1]: the tokens that are not padding (all of them: None)."""
    if st["lengths"] is None:
        return None
    return (torch.arange(T, device=DEV) < st["lengths"].long()[:, None])[..., None]


def _plain_conv(st):
    c, W = st["case"], st["case"]["W"]
    x, io = st["x"].detach(), st["x"].dtype
    B, T, C = x.shape
    valid = _within(st, T)
    w = st["weight"].detach().t()
    before = x.new_zeros(B, W - 1, C) if st["state"] is None else st["state"].detach()
    xs = torch.cat([before, x if valid is None else x.masked_fill(~valid, 0)], 1).float()       # token t at t + W - 1
    dy = st["dy"].float() if valid is None else st["dy"].float().masked_fill(~valid, 0)
    u = sum(xs[:, j:j + T] * w[j] for j in range(W))
    u = u if st["bias"] is None else u + st["bias"].detach()
    s = torch.sigmoid(u)
    y = u * s if c["silu"] else u
    du = dy * s * (1 + u * (1 - s)) if c["silu"] else dy
    dxs = sum(torch.nn.functional.pad(du * w[j], (0, 0, j, W - 1 - j)) for j in range(W))
    dw = torch.stack([(du * xs[:, j:j + T]).sum((0, 1)) for j in range(W)], 1)
    outs = [(y if valid is None else y.masked_fill(~valid, 0)).to(io)]
    last = None
    if c["state"]:
        n = torch.full((B,), T, device=DEV) if st["lengths"] is None else st["lengths"].long()
        last = (n[:, None] + torch.arange(W - 1, device=DEV))[..., None].expand(B, W - 1, C)
        outs.append(xs.gather(1, last).to(io))
        dxs = dxs.scatter_add(1, last, st["dstate"].float())
    grads = {"x": dxs[:, W - 1:].to(io), "weight": dw, "bias": du.sum((0, 1)), "state": dxs[:, :W - 1].to(io)}
    return (*outs, *(grads[n] for n in st["leaves"]))


def _plain_tokens(st):
    c, W = st["case"], st["case"]["W"]
    x, pool, off, slots = st["x"], st["pool"], st["offsets"].long(), st["slots"].long()
    n, N = slots.numel(), x.shape[0]
    counts = off[1:] - off[:-1]
    row = torch.repeat_interleave(torch.arange(n, device=DEV), counts, output_size=N)
    i = torch.arange(N, device=DEV) - off[row]                     # a token's place among its row's new ones
    old = pool[slots]
    tap = lambda k: torch.where((i >= k)[:, None], x[(torch.arange(N, device=DEV) - k).clamp(min=0)],  # noqa: E731
                                old[row, (W - 1 + i - k).clamp(max=W - 2)]).float()
    u = sum(tap(W - 1 - j) * st["weight"][:, j] for j in range(W))
    u = u if st["bias"] is None else u + st["bias"]
    m = counts[:, None] - (W - 1) + torch.arange(W - 1, device=DEV)       # the inputs that the new state holds
    kept = old.gather(1, (m + W - 1).clamp(max=W - 2)[..., None].expand_as(old))
    pool[st["to"].long()] = torch.where((m >= 0)[..., None], x[(off[:-1, None] + m).clamp(0, N - 1)], kept)
    return (u * torch.sigmoid(u) if c["silu"] else u).to(x.dtype), pool


def _plain_admit(st):
    page, N, slots = st["case"]["page"], st["tokens"], st["slots"].long()
    table, lengths, refs, new = st["table"], st["lengths"], st["refs"], st["n_new"].long()
    off = torch.cat([new.new_zeros(1), new.cumsum(0)])
    start = lengths[slots].long()
    had, want = (start + page - 1) // page, (start + new + page - 1) // page
    ends = (want - had).cumsum(0)
    free = (refs == 0).nonzero()[:, 0]
    take = int(ends[-1])
    at = torch.arange(take, device=DEV)
    owner = torch.searchsorted(ends, at, right=True)
    table[slots[owner], had[owner] + at - (ends - (want - had))[owner]] = free[:take].int()
    refs[free[:take]] = 1
    lengths[slots] += new.int()
    t = torch.arange(N, device=DEV)
    row = torch.searchsorted(off[1:], t, right=True)
    some = row < new.numel()
    row = row.clamp(max=new.numel() - 1)
    pos = start[row] + t - off[row]
    place = table[slots[row], (pos // page).clamp(max=table.shape[1] - 1)] * page + pos % page
    out = off.int(), start.int(), torch.where(some, pos, -1).int(), torch.where(some, place, -1).int()
    refs[free[:take]] = 0
    table[slots] = -1
    lengths[slots] = 0
    return (*out, table, lengths, refs)


def _plain_write(st):
    page, at = st["case"]["page"], st["places"].long()
    token = (at >= 0).nonzero()[:, 0]
    at = at[token]
    st["k_pages"][:, at // page, :, at % page] = st["k"][:, token].transpose(0, 1)
    st["v_pages"][:, at // page, :, at % page] = st["v"][:, token].transpose(0, 1)
    return st["k_pages"], st["v_pages"]


def _seen_keys(c, past, count):
    """The cached tokens that some new token of a row sees."""
    j = torch.arange(past + count, device=DEV)
    return j[(j >= _first_kept(c, past)) | (j < c["sinks"])] if c["window"] else j


def _plain_row(st, b, at, past, count):
    c, page = st["case"], st["case"]["page"]
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    j = _seen_keys(c, past, count)
    pages = st["table"][st["slots"][b].long()].long()[j // page]
    k = st["k_pages"][pages, :, j % page].float().transpose(0, 1)                          # [Hkv, keys, D]
    v = st["v_pages"][pages, :, j % page].float().transpose(0, 1)
    q = st["q"][at:at + count].float().view(count, Hkv, Hq // Hkv, D).permute(1, 2, 0, 3).reshape(Hkv, -1, D)
    s = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(D ** -0.5).view(Hkv, Hq // Hkv, count, -1)
    p = (past + torch.arange(count, device=DEV))[:, None]
    hidden = j > p
    if c["window"]:
        hidden = hidden | ((p - j >= c["window"]) & (j >= c["sinks"]))
    s = s.masked_fill_(hidden, -math.inf)
    s = s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    y = torch.matmul(s.view(Hkv, -1, j.numel()), v).view(Hkv, Hq // Hkv, count, D) / total
    return y.permute(2, 0, 1, 3).reshape(count, Hq, D).to(st["q"].dtype)


def _plain_chunk(st):
    counts = st["counts"]
    at = [sum(counts[:b]) for b in range(len(counts))]
    return torch.cat([_plain_row(st, b, at[b], st["past"][b], n) for b, n in enumerate(counts) if n])


_RUN_OWN = {"conv": _own_conv, "tokens": _own_tokens, "admit": _own_admit, "write": _own_write, "chunk": _own_chunk}
_RUN_PLAIN = {"conv": _plain_conv, "tokens": _plain_tokens, "admit": _plain_admit, "write": _plain_write,
              "chunk": _plain_chunk}


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    kind, size = case["kind"], 2 if case.get("dtype") == "bf16" else 4
    if kind == "conv":
        tokens, C, W = sum(_row_lengths(case)), case["C"], case["W"]
        out = case["B"] * case["T"] * C                            # y and dx are written for padding too
        state = 4 * case["B"] * (W - 1) * C if case["state"] else 0
        # x and dy are read, y and dx written, the weights read and their gradients written; a product and a sum each tap
        # forward, two backward, and the activation's
        return {"bytes": size * (2 * tokens * C + 2 * out + state) + 8 * C * (W + case["bias"]),
                "flops": tokens * C * (6 * W + (15 if case["silu"] else 0))}
    counts = _counts(case)
    N = sum(counts)
    if kind == "tokens":
        C, W = case["C"], case["W"]
        return {"bytes": size * (2 * N * C + 2 * case["n"] * (W - 1) * C) + 4 * C * (W + case["bias"]) + 12 * case["n"],
                "flops": N * C * (2 * W + (4 if case["silu"] else 0))}
    if kind == "admit":
        pages = sum(-(-c // case["page"]) for c in counts)
        # reference counts read until enough free ones are found; tables, counts and lengths written twice; the maps
        return {"bytes": 4 * (2 * (N + 5) + 3 * pages + 4 * pages + 8 * case["n"]), "flops": 0}
    Hkv, D = case["Hkv"], case["D"]
    if kind == "write":
        return {"bytes": 4 * size * case["layers"] * (N - 1) * Hkv * D + 4 * N, "flops": 0}
    keys = pairs = 0
    W, S = case["window"], case["sinks"]
    for past, n in zip(_past(case), counts):
        first = _first_kept(case, past)
        keys += past + n - first + min(S, first) if n else 0
        for p in range(past, past + n):
            pairs += min(p + 1, W) + min(S, max(0, p + 1 - W)) if W else p + 1
    return {"bytes": size * (2 * N * case["Hq"] * D + 2 * keys * Hkv * D) + 4 * keys // case["page"],
            "flops": 4 * D * pairs * case["Hq"]}


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    """``run``'s outputs in float64, from the inputs that ``prepare`` makes; what is only moved has no computed numbers."""
    if case["kind"] == "conv":
        return _exact_conv(prepare(case, seed))
    if case["kind"] == "tokens":
        return _exact_tokens(prepare(case, seed))
    if case["kind"] == "chunk":
        return _exact_chunk(prepare(case, seed))
    return None


def _exact_conv(st):
    """Row by row on its valid tokens, in groups of channels: a library convolution in float64 and its autograd."""
    c, W = st["case"], st["case"]["W"]
    B, T, C = st["x"].shape
    lens = [T] * B if st["lengths"] is None else st["lengths"].tolist()
    f64 = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device=DEV)  # noqa: E731
    y, last = f64(B, T, C), f64(B, W - 1, C)
    grads = {"x": f64(B, T, C), "weight": f64(C, W), "bias": f64(C), "state": f64(B, W - 1, C)}
    for c0 in range(0, C, 512):
        ch = slice(c0, min(c0 + 512, C))
        for b in range(B):
            n = lens[b]
            given = {"x": st["x"][b, :n, ch], "weight": st["weight"][ch],
                     "bias": st["bias"][ch] if c["bias"] else f64(ch.stop - c0),
                     "state": st["state"][b, :, ch] if c["state"] else f64(W - 1, ch.stop - c0)}
            leaf = {k: t.detach().double().clone().requires_grad_(True) for k, t in given.items()}
            line = torch.cat([leaf["state"], leaf["x"]])
            u = (line.unfold(0, W, 1) * leaf["weight"]).sum(-1) + leaf["bias"] if n else line[:0]
            out = u / (1 + torch.exp(-u)) if c["silu"] else u
            y[b, :n, ch], last[b, :, ch] = out.detach(), line[n:].detach()
            loss = (out * st["dy"][b, :n, ch].double()).sum()
            if c["state"]:
                loss = loss + (line[n:] * st["dstate"][b, :, ch].double()).sum()
            for (k, t), g in zip(leaf.items(), torch.autograd.grad(loss, list(leaf.values()), allow_unused=True)):
                if g is not None:
                    to = {"x": grads["x"][b, :n, ch], "weight": grads["weight"][ch], "bias": grads["bias"][ch],
                          "state": grads["state"][b, :, ch]}[k]
                    to += g
    return (y, *([last] if c["state"] else []), *(grads[n] for n in st["leaves"]))


def _exact_tokens(st):
    c, W = st["case"], st["case"]["W"]
    off, slots, to = st["offsets"].tolist(), st["slots"].tolist(), st["to"].tolist()
    y, pool = torch.zeros_like(st["x"], dtype=torch.float64), st["pool"].double()
    before = st["pool"].double()
    for b, (s, t) in enumerate(zip(slots, to)):
        line = torch.cat([before[s], st["x"][off[b]:off[b + 1]].double()])
        pool[t] = line[line.shape[0] - (W - 1):]
        if off[b + 1] > off[b]:
            u = (line.unfold(0, W, 1) * st["weight"].double()).sum(-1)
            u = u + st["bias"].double() if c["bias"] else u
            y[off[b]:off[b + 1]] = u / (1 + torch.exp(-u)) if c["silu"] else u
    return y, pool


def _exact_chunk(st):
    """A row and a head at a time."""
    c = st["case"]
    page, G = c["page"], c["Hq"] // c["Hkv"]
    y = torch.zeros(*st["q"].shape, dtype=torch.float64, device=DEV)
    off = st["offsets"].tolist()
    for b, r in enumerate(st["slots"].tolist()):
        n, length = off[b + 1] - off[b], int(st["lengths"][r])
        if n == 0:
            continue
        place = torch.arange(length, device=DEV)
        where = st["table"][r].long()[place // page]
        pos = torch.arange(length - n, length, device=DEV).unsqueeze(1)
        seen = (place <= pos) & (where >= 0)
        if c["window"]:
            seen &= (pos - place < c["window"]) | (place < c["sinks"])
        for h in range(c["Hq"]):
            kh = st["k_pages"][where.clamp(min=0), h // G, place % page].double()
            vh = st["v_pages"][where.clamp(min=0), h // G, place % page].double()
            logit = torch.mm(st["q"][off[b]:off[b + 1], h].double(), kh.t()) / math.sqrt(c["D"])
            y[off[b]:off[b + 1], h] = torch.mm(torch.softmax(logit.masked_fill_(~seen, -math.inf), 1), vh)
    return y
