"""Performance cases of the attention operators that stand beside the recurrences in a hybrid model.

A hybrid model keeps a few layers of softmax attention between its recurrent
layers.  They look at a window of the last tokens and at the first ones
(sinks), or at everything, and are served from a cache of fixed-size pages.

  kind     operator                                       in real use
  train    attention.window_attention forward + backward  a training step of such a layer
  prefill  attention.window_attention, no gradient        a prompt, or the next piece of one, taken in
  step     attention.paged_attention_step                 one served token for every sequence: into the page cache, and
                                                          attention over it
  fork     pages.pages_fork, then pages.pages_free        sequences continued in several ways, the ways dropped again
  compact  pages.pages_compact                            a cache with holes gathered at the front of its pool
  admit    pages.pages_reserve, pages_write, pages_free   a request's pages: taken, filled in every layer, given back

With ``own`` false, ``run`` computes an operator from elementary torch
operations in float32; with ``own`` true it calls the package.

Positions: query i of Tq stands at p = i + Tk - Tq.  It sees key j if j <= p,
p and j lie before the row's length, and p - j < window (0: no window) or
j < sinks.  A query that sees nothing gives zero.

Work counts the visible pairs: 4 D operations each forward and 10 D backward,
and each input that is needed and each output once.
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
        # the training step of an attention layer beside the 16-head recurrent layer: its batch and length, a window
        # of a quarter of it and a few sinks, four query heads to a key head
        dict(name="train_layer", kind="train", B=4, Tq=4096, Tk=4096, Hq=16, Hkv=4, D=128, window=1024, sinks=16,
             ragged=False, dtype="bf16"),
        # fine-tuning on documents of unlike length in one padded batch (one of them empty); odd sizes everywhere
        dict(name="train_ragged", kind="train", B=5, Tq=1999, Tk=1999, Hq=6, Hkv=2, D=64, window=257, sinks=3,
             ragged=True, dtype="bf16"),
        # the small float32 model of experiments and gradient checks
        dict(name="train_f32", kind="train", B=2, Tq=513, Tk=513, Hq=4, Hkv=4, D=64, window=100, sinks=0,
             ragged=False, dtype="f32"),
        # a long prompt in one piece
        dict(name="prefill_long", kind="prefill", B=1, Tq=32768, Tk=32768, Hq=16, Hkv=4, D=128, window=2048, sinks=64,
             ragged=False, dtype="bf16"),
        # the next piece of two prompts: few queries against all the tokens before them
        dict(name="prefill_piece", kind="prefill", B=2, Tq=200, Tk=16584, Hq=16, Hkv=2, D=128, window=0, sinks=0,
             ragged=False, dtype="bf16"),
        # a few interactive users: the smallest call, where latency counts
        dict(name="step_few", kind="step", B=3, T=2000, Hq=16, Hkv=4, D=128, page=16, window=0, sinks=0, dtype="bf16"),
        # a full serving batch of sequences at all stages, empty rows among them
        dict(name="step_batch", kind="step", B=256, T=8192, Hq=16, Hkv=4, D=128, page=64, window=0, sinks=0,
             dtype="bf16"),
        # two very long conversations: few rows, so the length has to be shared out
        dict(name="step_long", kind="step", B=2, T=262143, Hq=32, Hkv=8, D=128, page=128, window=0, sinks=0,
             dtype="bf16"),
        # the windowed layer of the float32 model, served
        dict(name="step_window_f32", kind="step", B=48, T=6000, Hq=12, Hkv=12, D=64, page=32, window=512, sinks=4,
             dtype="f32"),
        # 16 prompts answered four times each: the children share the full pages and copy the last one
        dict(name="fork_samples", kind="fork", rows=128, par=16, ways=4, T=2047, pages=1500, page=64, layers=8, Hkv=4,
             D=128, dtype="bf16"),
        # a cache after a busy hour: less than half of the pages in use, all over the pool
        dict(name="compact_pool", kind="compact", rows=96, T=1000, pages=1024, page=64, layers=8, Hkv=4, D=128,
             dtype="bf16"),
        # eight new prompts enter a cache of small pages
        dict(name="admit_prompts", kind="admit", rows=64, B=8, T=1001, pages=2048, page=16, layers=4, Hkv=4, D=64,
             dtype="bf16"),
    ]


def _size(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return n - 1 if n == 3072 else n


def draw(rng):
    kind = rng.choice(("train", "train", "train", "prefill", "prefill", "step", "step", "step", "fork", "compact",
                       "admit"))
    D = rng.choice((64, 128, 128))
    Hkv = rng.choice((1, 2, 3, 4, 8))
    dtype = rng.choice(("bf16", "bf16", "bf16", "f32"))
    if kind in ("train", "prefill"):
        Hq = Hkv * rng.choice([g for g in (1, 2, 3, 4, 8) if g * Hkv <= 16])
        B = rng.randint(1, 5)
        # at most the tokens and heads of the largest listed steps (an eighth of that in float32)
        cap = (1 if dtype == "bf16" else 8) * B * Hq
        T = _size(rng, 64, 8192)
        T = max(64, min(T, 4 * 4096 * 16 // cap))
        window = rng.choice((0, _size(rng, 32, 2048), _size(rng, 32, 2048), _size(rng, 32, 2048)))
        if window == 0:
            T = min(T, 2048 if dtype == "bf16" else 1024)
        Tq = T
        if kind == "prefill" and rng.random() < 0.5:
            Tq = max(1, T // rng.choice((2, 7, 30)))
        return dict(kind=kind, B=B, Tq=Tq, Tk=T, Hq=Hq, Hkv=Hkv, D=D, window=window,
                    sinks=rng.choice((0, 1, 4, _size(rng, 8, 128))), ragged=rng.random() < 0.4, dtype=dtype)
    if kind == "step":
        B = _size(rng, 1, 256)
        T = max(16, min(_size(rng, 64, 100000), 2_000_000 // (B * Hkv) * (2 if dtype == "bf16" else 1)))
        return dict(kind=kind, B=B, T=T, Hq=Hkv * rng.choice((1, 2, 4, 8)), Hkv=Hkv, D=D,
                    page=rng.choice((16, 32, 64, 128)), window=rng.choice((0, 0, _size(rng, 32, 2048))),
                    sinks=rng.choice((0, 4, 64)), dtype=dtype)
    page = rng.choice((16, 32, 64))
    layers = rng.choice((1, 3, 8))
    if kind == "fork":
        par, ways, T = _size(rng, 1, 24), rng.randint(1, 4), _size(rng, 64, 2048)
        return dict(kind=kind, rows=128, par=par, ways=ways, T=T, pages=par * (-(-T // page) + ways + 1) + 40,
                    page=page, layers=layers, Hkv=Hkv, D=D, dtype=dtype)
    if kind == "compact":
        rows, T = _size(rng, 4, 96), _size(rng, 64, 1000)
        return dict(kind=kind, rows=rows, T=T, pages=max(64, rows * -(-T // page)), page=page, layers=layers, Hkv=Hkv,
                    D=D, dtype=dtype)
    B, T = _size(rng, 1, 12), _size(rng, 1, 2000)
    return dict(kind=kind, rows=64, B=B, T=T, pages=B * (-(-T // page)) + 100, page=page, layers=layers, Hkv=Hkv,
                D=D, dtype=dtype)


def _io(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _row_lengths(case):
    """Valid tokens of each row of a padded batch: unlike lengths, an empty row and a full one among them."""
    B, T = case["B"], case["Tk"]
    if not case["ragged"]:
        return [T] * B
    return [T if b == 0 else 0 if b == 2 else max(1, T * ((5 * b + 2) % 7 + 1) // 9) for b in range(B)]


def _cached_lengths(case):
    """Cached tokens of each served row: spread over the range; of more than eight rows one is empty, one at its first token."""
    B, T = case["B"], case["T"]
    ls = [max(1, T - (T * ((37 * b) % 64)) // 64) for b in range(B)]
    if B > 8:
        ls[3], ls[5] = 0, 1
    return ls


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


def _page_table(d, lengths, page, n_pages, width=None):
    """A table whose rows own ceil(length / page) pages, taken from all over the pool."""
    need = [-(-l // page) for l in lengths]
    table = torch.full((len(lengths), width or max(max(need), 1)), -1, dtype=torch.int32, device=DEV)
    order, at = d.order(n_pages).int(), 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    return table


def _ints(xs):
    return torch.tensor(xs, dtype=torch.int32, device=DEV)


def _refs(table, n_pages):
    used = table[table >= 0].long()
    return torch.zeros(n_pages, dtype=torch.int32, device=DEV).index_add_(0, used, torch.ones_like(used, dtype=torch.int32))


def prepare(case, seed):
    d, io, kind = _Draws(seed), _io(case), case["kind"]
    st = {"case": case}
    if kind in ("train", "prefill"):
        B, Tq, Tk, Hq, Hkv, D = (case[n] for n in ("B", "Tq", "Tk", "Hq", "Hkv", "D"))
        st["q"], st["k"], st["v"] = d.n(B, Tq, Hq, D, dtype=io), d.n(B, Tk, Hkv, D, dtype=io), d.n(B, Tk, Hkv, D, dtype=io)
        st["lengths"] = _ints(_row_lengths(case)) if case["ragged"] else None
        if kind == "train":
            st["dy"] = d.n(B, Tq, Hq, D, dtype=io)
            for n in "qkv":
                st[n].requires_grad_(True)
        return st
    if kind == "step":
        Hkv, D, page = case["Hkv"], case["D"], case["page"]
        ls = _cached_lengths(case)
        n_pages = sum(-(-l // page) for l in ls) + 8
        st["table"] = _page_table(d, ls, page, n_pages)
        st["lengths"] = _ints(ls)
        st["k_pages"] = d.pool(n_pages, Hkv, page, D, dtype=io)
        st["v_pages"] = d.pool(n_pages, Hkv, page, D, dtype=io)
        st["q"] = d.n(case["B"], case["Hq"], D, dtype=io)
        st["k"], st["v"] = d.n(case["B"], Hkv, D, dtype=io), d.n(case["B"], Hkv, D, dtype=io)   # the token at lengths - 1
        return st
    rows, n_pages, page = case["rows"], case["pages"], case["page"]
    shape = (case["layers"], n_pages, case["Hkv"], page, case["D"])
    width = -(-case["T"] // page) + 1
    if kind == "fork":
        ls = [max(1, case["T"] - (31 * r) % page) if r < case["par"] else 0 for r in range(rows)]
        kids = case["par"] * case["ways"]
        st["parents"] = _ints([i // case["ways"] for i in range(kids)])
        st["children"] = _ints([case["par"] + i for i in range(kids)])
    elif kind == "compact":
        ls = [case["T"] if r % 9 else 0 for r in range(rows)]
        ls = [l // (1 + (5 * r) % 4) if r % 3 else l // 2 for r, l in enumerate(ls)]
    else:
        ls = [0] * rows
        st["slots"] = _ints([(7 * b + 3) % rows for b in range(case["B"])])
        st["k"] = d.n(case["layers"], case["B"], case["T"], case["Hkv"], case["D"], dtype=io)
        st["v"] = d.n(case["layers"], case["B"], case["T"], case["Hkv"], case["D"], dtype=io)
    st["table"] = _page_table(d, ls, page, n_pages, width)
    st["lengths"] = _ints(ls)
    st["refs"] = _refs(st["table"], n_pages)
    st["k_pages"], st["v_pages"] = d.pool(*shape, dtype=io), d.pool(*shape, dtype=io)
    st["status"] = torch.zeros(2, dtype=torch.int32, device=DEV)
    if kind == "compact":
        st["out"] = (torch.empty_like(st["table"]), torch.empty_like(st["refs"]))
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(st):
    return (_RUN_OWN if own else _RUN_PLAIN)[st["case"]["kind"]](st)


def _own_attention(st):
    from gdnx_amd import attention
    c = st["case"]
    args = dict(window=c["window"] or None, sinks=c["sinks"], lengths=st["lengths"])
    if c["kind"] == "train":
        y = attention.window_attention(st["q"], st["k"], st["v"], **args)
        return (y.detach(), *torch.autograd.grad(y, (st["q"], st["k"], st["v"]), grad_outputs=st["dy"]))
    with torch.no_grad():
        return attention.window_attention(st["q"], st["k"], st["v"], **args)


def _own_step(st):
    from gdnx_amd import attention
    c = st["case"]
    y = attention.paged_attention_step(st["q"], st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"],
                                       st["lengths"], window=c["window"] or None, sinks=c["sinks"])
    return y, st["k_pages"], st["v_pages"]


def _own_fork(st):
    from gdnx_amd import pages
    pages.pages_fork(st["k_pages"], st["v_pages"], st["table"], st["lengths"], st["refs"], st["parents"],
                     st["children"], st["status"])
    shared = st["table"].clone(), st["lengths"].clone()
    pages.pages_free(st["table"], st["lengths"], st["refs"], st["children"])
    return st["k_pages"], st["v_pages"], *shared, st["table"], st["lengths"], st["refs"]


def _own_compact(st):
    from gdnx_amd import pages
    table, refs = pages.pages_compact(st["k_pages"], st["v_pages"], st["table"], st["refs"], out=st["out"])
    return st["k_pages"], st["v_pages"], table, refs


def _own_admit(st):
    from gdnx_amd import pages
    start = pages.pages_reserve(st["table"], st["lengths"], st["refs"], st["slots"], st["case"]["T"],
                                st["case"]["page"], st["status"])
    pages.pages_write(st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["slots"], start)
    taken = st["table"].clone(), st["lengths"].clone()
    pages.pages_free(st["table"], st["lengths"], st["refs"], st["slots"])
    return st["k_pages"], st["v_pages"], start, *taken, st["table"], st["lengths"], st["refs"]


def _visible(p, j, lengths, window, sinks):
    """[B, len(p), len(j)]: whether the query at position p sees key j."""
    p, j = p[:, None], j[None, :]
    ok = (j <= p) & (p >= 0)
    if window:
        ok = ok & ((p - j < window) | (j < sinks))
    ok = ok[None]
    if lengths is not None:
        n = lengths.long()[:, None, None]
        ok = ok & (p[None] < n) & (j[None] < n)
    return ok


def _plain_attention(st):
    """Blocks of queries against the keys that some of them see: scores, softmax, product; backward by the formulas
    dV = P'dY, dP = dY V', dS = P (dP - rowsum(dY Y)), dQ = s dS K, dK = s dS' Q."""
    c = st["case"]
    q, k, v = (st[n].detach() for n in "qkv")
    B, Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[1], k.shape[2]
    G, scale, train = Hq // Hkv, 1.0 / math.sqrt(D), c["kind"] == "train"
    kf, vf = k.float().transpose(1, 2).contiguous(), v.float().transpose(1, 2).contiguous()   # [B,Hkv,Tk,D]
    y = torch.empty_like(q)
    if train:
        dq, dk, dv = torch.empty_like(q), torch.zeros_like(kf), torch.zeros_like(vf)

    def heads(x):                                  # [B,n,Hq,D] -> [B,Hkv,G*n,D]
        return x.float().view(B, -1, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)

    def rows(x):                                   # and back
        return x.view(B, Hkv, G, -1, D).permute(0, 3, 1, 2, 4).reshape(B, -1, Hq, D).to(q.dtype)

    for i0 in range(0, Tq, 512):
        i1 = min(i0 + 512, Tq)
        p = torch.arange(i0, i1, device=DEV) + Tk - Tq
        lo, hi = 0, max(0, i1 + Tk - Tq)
        if c["window"]:
            lo = min(hi, max(0, i0 + Tk - Tq - c["window"] + 1))
        ns = min(c["sinks"], lo)
        j = torch.cat([torch.arange(0, ns, device=DEV), torch.arange(lo, hi, device=DEV)])
        kb, vb = (torch.cat([x[:, :, :ns], x[:, :, lo:hi]], 2) for x in (kf, vf))
        ok = _visible(p, j, st["lengths"], c["window"], c["sinks"])[:, None, None]
        qb = heads(q[:, i0:i1])
        s = (qb @ kb.transpose(2, 3).contiguous()) * scale
        s = s.view(B, Hkv, G, i1 - i0, -1).masked_fill(~ok, -math.inf)
        top = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_zeros(*s.shape[:-1], 1)
        e = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
        total = e.sum(-1, keepdim=True)
        e = (e / total.masked_fill(total == 0, 1.0)).view(B, Hkv, G * (i1 - i0), -1)
        o = e @ vb
        y[:, i0:i1] = rows(o)
        if train:
            g = heads(st["dy"][:, i0:i1])
            ds = e * (g @ vb.transpose(2, 3).contiguous() - (g * o).sum(-1, keepdim=True)) * scale
            dq[:, i0:i1] = rows(ds @ kb)
            dkb, dvb = ds.transpose(2, 3).contiguous() @ qb, e.transpose(2, 3).contiguous() @ g
            for acc, part in ((dk, dkb), (dv, dvb)):
                acc[:, :, :ns] += part[:, :, :ns]
                acc[:, :, lo:hi] += part[:, :, ns:]
    if not train:
        return y
    return y, dq, dk.transpose(1, 2).to(q.dtype).contiguous(), dv.transpose(1, 2).to(q.dtype).contiguous()


def _plain_step(st):
    """The new token into its page, every row's pages gathered, then scores, softmax and product over the longest row."""
    c = st["case"]
    q, table, n = st["q"], st["table"].long(), st["lengths"].long()
    B, Hq, D = q.shape
    Hkv, page = st["k_pages"].shape[1:3]
    Tk = table.shape[1] * page
    live, last = n > 0, (n - 1).clamp(min=0)
    at, first = torch.gather(table, 1, (last // page)[:, None])[:, 0], live.int().argmax()
    for pool, new in ((st["k_pages"], st["k"]), (st["v_pages"], st["v"])):
        # (an empty row writes what the first live row writes)
        pool[torch.where(live, at, at[first]), :, torch.where(live, last, last[first]) % page] = \
            torch.where(live[:, None, None], new, new[first])
    j = torch.arange(Tk, device=DEV)
    ok = j[None] < n[:, None]
    if c["window"]:
        ok = ok & ((j[None] >= n[:, None] - c["window"]) | (j[None] < c["sinks"]))

    def cached(pool):                              # [B,Hkv,Tk,D]
        return pool[table.clamp(min=0)].float().transpose(1, 2).reshape(B, Hkv, Tk, D)

    qf = q.float().view(B, Hkv, Hq // Hkv, D)
    s = (qf @ cached(st["k_pages"]).transpose(2, 3).contiguous()) / math.sqrt(D)
    s = s.masked_fill(~ok[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
    total = e.sum(-1, keepdim=True)
    e = e / total.masked_fill(total == 0, 1.0)
    return (e @ cached(st["v_pages"])).reshape(B, Hq, D).to(q.dtype), st["k_pages"], st["v_pages"]


def _give_back(table, lengths, refs, slots):
    slots = slots.long()
    gone = table[slots]
    refs.index_add_(0, gone.clamp(min=0).view(-1).long(), -(gone >= 0).int().view(-1))
    table[slots] = -1
    lengths[slots] = 0


def _plain_fork(st):
    """Children take their parents' full pages (a count more) and the lowest free pages, in order, for the started ones."""
    table, lengths, refs = st["table"], st["lengths"], st["refs"]
    par, kid, page = st["parents"].long(), st["children"].long(), st["case"]["page"]
    n, at = lengths[par].long(), torch.arange(par.numel(), device=DEV)
    rows, started = table[par], n % page != 0
    col = (n // page).clamp(max=table.shape[1] - 1)
    free = torch.sort((refs != 0).int(), stable=True)[1]
    new = free[(torch.cumsum(started.int(), 0) - 1).clamp(min=0)]
    src = torch.where(started, rows[at, col], rows[:, 0]).long()    # (a full parent: its first page onto itself)
    dst = torch.where(started, new, src)
    st["k_pages"][:, dst] = st["k_pages"][:, src]
    st["v_pages"][:, dst] = st["v_pages"][:, src]
    rows[at, col] = torch.where(started, new.int(), rows[at, col])
    refs.index_add_(0, rows.clamp(min=0).view(-1).long(), (rows >= 0).int().view(-1))
    table[kid], lengths[kid] = rows, n.int()
    shared = table.clone(), lengths.clone()
    _give_back(table, lengths, refs, st["children"])
    return st["k_pages"], st["v_pages"], *shared, table, lengths, refs


def _plain_compact(st):
    """Used pages beyond the count of used pages move, in order, into the free pages before it."""
    refs, table = st["refs"], st["table"]
    used = refs != 0
    count = used.sum()
    at = torch.arange(refs.numel(), device=DEV)
    src, dst = at[used & (at >= count)], at[~used & (at < count)]
    st["k_pages"][:, dst] = st["k_pages"][:, src]
    st["v_pages"][:, dst] = st["v_pages"][:, src]
    to = at.clone()
    to[src] = dst
    new_refs = refs.clone()
    new_refs[dst] = refs[src]
    new_refs[src] = 0
    return st["k_pages"], st["v_pages"], torch.where(table >= 0, to[table.clamp(min=0).long()].int(), table), new_refs


def _plain_admit(st):
    """The rows' pages are the lowest free ones, row by row; a token goes to its page and place."""
    table, lengths, refs = st["table"], st["lengths"], st["refs"]
    slots, T, page = st["slots"].long(), st["case"]["T"], st["case"]["page"]
    start = lengths[slots].clone()
    have, want = (start + page - 1) // page, (start + T + page - 1) // page
    col = torch.arange(table.shape[1], device=DEV)[None]
    take = (col >= have[:, None]) & (col < want[:, None])
    free = torch.sort((refs != 0).int(), stable=True)[1]
    rank = (torch.cumsum(take.view(-1).int(), 0) - 1).clamp(min=0).view_as(take)
    rows = torch.where(take, free[rank].int(), table[slots])
    refs.index_add_(0, torch.where(take, rows, 0).view(-1).long(), take.int().view(-1))
    table[slots], lengths[slots] = rows, start + T
    pos = start.long()[:, None] + torch.arange(T, device=DEV)
    where = torch.gather(rows.long(), 1, pos // page)
    for pool, new in ((st["k_pages"], st["k"]), (st["v_pages"], st["v"])):
        for layer in range(pool.shape[0]):
            pool[layer][where, :, pos % page] = new[layer]
    taken = table.clone(), lengths.clone()
    _give_back(table, lengths, refs, st["slots"])
    return st["k_pages"], st["v_pages"], start, *taken, table, lengths, refs


_RUN_OWN = {"train": _own_attention, "prefill": _own_attention, "step": _own_step, "fork": _own_fork,
            "compact": _own_compact, "admit": _own_admit}
_RUN_PLAIN = {"train": _plain_attention, "prefill": _plain_attention, "step": _plain_step, "fork": _plain_fork,
              "compact": _plain_compact, "admit": _plain_admit}


# ---------------------------------------------------------------------------
# the work of one pass
# ---------------------------------------------------------------------------
def _pairs(case):
    """Visible (query, key) pairs of one head, and keys that some query sees, over the batch."""
    Tq, Tk, W, S = case["Tq"], case["Tk"], case["window"], case["sinks"]
    pairs = keys = 0
    for n in _row_lengths(case):
        first, end = max(0, Tk - Tq), min(n, Tk)
        for p in range(first, end):
            if W and p + 1 > W:
                pairs += W + min(S, p + 1 - W)
            else:
                pairs += p + 1
        if end > first:
            lo = max(0, first - W + 1) if W else 0
            keys += end - lo + min(S, lo)
    return pairs, keys


def work(case):
    size, D, kind = (2 if case["dtype"] == "bf16" else 4), case["D"], case["kind"]
    if kind in ("train", "prefill"):
        pairs, keys = _pairs(case)
        q, kv = case["B"] * case["Tq"] * case["Hq"] * D, keys * case["Hkv"] * D
        if kind == "prefill":
            return {"bytes": size * (2 * q + 2 * kv), "flops": 4 * D * pairs * case["Hq"]}
        return {"bytes": size * (4 * q + 4 * kv), "flops": 14 * D * pairs * case["Hq"]}
    if kind == "step":
        W, S = case["window"], case["sinks"]
        keys = sum(min(l, W) + min(S, max(0, l - W)) if W else l for l in _cached_lengths(case))
        q = case["B"] * case["Hq"] * D
        new = 2 * case["B"] * case["Hkv"] * D         # the new tokens: written once more than the keys are read
        return {"bytes": size * (2 * q + new + 2 * keys * case["Hkv"] * D), "flops": 4 * D * keys * case["Hq"]}
    page_bytes = 2 * size * case["layers"] * case["Hkv"] * case["page"] * D
    width = -(-case["T"] // case["page"]) + 1
    if kind == "fork":
        kids = case["par"] * case["ways"]
        started = sum(max(1, case["T"] - (31 * r) % case["page"]) % case["page"] != 0 for r in range(case["par"]))
        return {"bytes": 2 * page_bytes * started * case["ways"] + 16 * kids * width, "flops": 0}
    if kind == "compact":
        ls = [case["T"] if r % 9 else 0 for r in range(case["rows"])]
        ls = [l // (1 + (5 * r) % 4) if r % 3 else l // 2 for r, l in enumerate(ls)]
        used = sum(-(-l // case["page"]) for l in ls)
        moved = used * (case["pages"] - used) // case["pages"]      # of pages placed at random
        return {"bytes": 2 * page_bytes * moved + 8 * (case["pages"] + case["rows"] * width), "flops": 0}
    return {"bytes": 4 * size * case["layers"] * case["B"] * case["T"] * case["Hkv"] * D + 16 * case["B"] * width,
            "flops": 0}


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    """``run``'s outputs in float64, from the inputs that ``prepare`` makes; what is only moved has no computed numbers."""
    if case["kind"] in ("train", "prefill"):
        return _exact_attention(prepare(case, seed))
    if case["kind"] == "step":
        return _exact_step(prepare(case, seed))
    return None


def _exact_attention(st):
    """One row and head at a time, 4096 queries against all keys."""
    c = st["case"]
    q, k, v = (st[n].detach().double() for n in "qkv")
    train = c["kind"] == "train"
    B, Tq, Hq, D = q.shape
    Tk, G = k.shape[1], Hq // k.shape[2]
    y = torch.zeros_like(q)
    grads = [torch.zeros_like(x) for x in (q, k, v)] if train else []
    j = torch.arange(Tk, device=DEV)
    lens = [Tk] * B if st["lengths"] is None else st["lengths"].tolist()
    for i0 in range(0, Tq, 4096):
        i = torch.arange(i0, min(i0 + 4096, Tq), device=DEV)
        pos = (i + (Tk - Tq)).unsqueeze(1)
        near = j <= pos
        if c["window"]:
            near &= (j > pos - c["window"]) | (j < c["sinks"])
        for b in range(B):
            seen = near & (j < lens[b]) & (pos < lens[b])
            some = seen.any(1, keepdim=True)
            for h in range(Hq):
                qi, kh, vh = q[b, i, h], k[b, :, h // G], v[b, :, h // G]
                logit = torch.mm(qi, kh.t()).mul_(D ** -0.5)
                logit[~seen] = -math.inf
                prob = torch.softmax(logit, 1).masked_fill_(~some, 0.0)
                y[b, i, h] = torch.mm(prob, vh)
                if train:
                    g = st["dy"][b, i, h].double()
                    back = torch.mm(g, vh.t())
                    back = prob * (back - (prob * back).sum(1, keepdim=True)) * D ** -0.5
                    grads[0][b, i, h] = torch.mm(back, kh)
                    grads[1][b, :, h // G] += torch.mm(back.t(), qi)
                    grads[2][b, :, h // G] += torch.mm(prob.t(), g)
    return (y, *grads) if train else y


def _exact_step(st):
    c = st["case"]
    q = st["q"].double()
    B, Hq, D = q.shape
    Hkv, page = st["k_pages"].shape[1:3]
    y = torch.zeros_like(q)
    for b, n in enumerate(st["lengths"].tolist()):
        if n == 0:
            continue
        j = torch.arange(n, device=DEV)
        if c["window"]:
            j = j[(j >= n - c["window"]) | (j < c["sinks"])]
        at = st["table"][b].long()[j // page]
        for h in range(Hkv):
            kj, vj = st["k_pages"][at, h, j % page].double(), st["v_pages"][at, h, j % page].double()
            kj[-1], vj[-1] = st["k"][b, h].double(), st["v"][b, h].double()
            rows = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
            y[b, rows] = torch.softmax(q[b, rows] @ kj.t() * D ** -0.5, -1) @ vj
    return y, None, None
