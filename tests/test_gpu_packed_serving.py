"""The operators of a packed step together: the example, and the convolution of a decode-state cache."""
import importlib.util
import os
import sys

import pytest
import torch

from gdnx_amd import attention, conv
from gdnx_amd.decode_cache import DecodeStateCache

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_packed_serving_example(gpu_lib):
    spec = importlib.util.spec_from_file_location("packed_serving", os.path.join(ROOT, "examples", "packed_serving.py"))
    ex = importlib.util.module_from_spec(spec)
    try:
        spec.loader.exec_module(ex)
    finally:
        sys.path.remove(os.path.join(ROOT, "examples"))
    # bf16 layers: each rounds its output once (2e-3 relative) and the served form sums in another order
    assert ex.main(lengths=(90, 17, 130), piece=32, steps=9) < 1e-2


@pytest.mark.parametrize("kind,M", [("dense", 1), ("gdn3", 2)])
def test_cache_convolution(gpu_lib, kind, M):
    """Equal prompts, packed pieces and single tokens continue one another; slots come back empty."""
    n, C, W, T = 3, 40, 4, 12
    x, w = torch.randn(n, T, C, device="cuda").bfloat16(), torch.randn(C, W, device="cuda")
    b = torch.randn(C, device="cuda")
    whole = conv.causal_conv(x, w, b)
    cache = DecodeStateCache(5, 2, M, 64, kind=kind, conv=(C, W))
    slots = cache.alloc(n)[::-1]
    got = [cache.convolve(slots, x[:, :5], w, b)]
    off = torch.tensor([0, 2, 4, 6], dtype=torch.int32, device="cuda")
    got.append(cache.convolve(slots, x[:, 5:7].reshape(-1, C), w, b, offsets=off).view(n, 2, C))
    for t in range(7, T):
        got.append(cache.convolve(slots, x[:, t], w, b)[:, None])
    assert torch.equal(torch.cat(got, 1), whole)
    assert (cache.convolve([slots[0], -1], x[:2, 0], w, b)[1] == 0).all()
    assert (cache.conv_pool[slots] != 0).any()
    cache.free(slots)
    cache.alloc(5)
    assert (cache.conv_pool == 0).all()
    with pytest.raises(ValueError, match="twice"):
        cache.convolve([1, 1], x[:2, 0], w, b)
    with pytest.raises(ValueError, match="rows for"):
        cache.convolve([1, 2], x[:, 0], w, b)
    with pytest.raises(ValueError, match="without a convolution"):
        DecodeStateCache(2, 1, 1, 64).convolve([0], x[:1, 0], w, b)


def test_refuses_what_would_be_read_wrongly(gpu_lib):
    """Heads beside the channels of a prompt; attention over its own queries' memory."""
    cache = DecodeStateCache(3, 1, 1, 64, conv=(64, 4))
    x, w = torch.randn(2, 5, 3, 64, device="cuda").bfloat16(), torch.randn(64, 4, device="cuda")
    before = cache.conv_pool.clone()
    with pytest.raises(ValueError, match="x must be"):
        cache.convolve([0, 1], x, w)
    assert torch.equal(cache.conv_pool, before)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q, pool = torch.randn(4, 1, 64, device="cuda").bfloat16(), torch.zeros(2, 1, 16, 64, device="cuda").bfloat16()
    kept = q.clone()
    with pytest.raises(ValueError, match="and not q"):
        attention.paged_attention_chunk(q, pool, pool, i32([[0]]), i32([4]), i32([0, 4]), out=q)
    assert torch.equal(q, kept)


def test_calls_on_two_streams_at_once(gpu_lib):
    """Long and short rows with parts and spans, a training step of the convolution: each call has a workspace of its own."""
    g = torch.Generator().manual_seed(3)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    kp, vp = (torch.randn(80, 2, 64, 64, generator=g).bfloat16().to("cuda") for _ in range(2))
    table, off, lens = i32([list(range(40)), list(range(40, 80))]), i32([0, 3, 203]), i32([2500, 2400])
    qs = [torch.randn(203, 8, 64, generator=g).bfloat16().to("cuda") for _ in range(2)]
    xs = [torch.randn(2, 400, 256, generator=g).bfloat16().to("cuda") for _ in range(2)]
    w = torch.randn(256, 4, generator=g).to("cuda")
    def both(i):
        y = attention.paged_attention_chunk(qs[i], kp, vp, table, lens, off)
        x, wl = xs[i].detach().requires_grad_(True), w.detach().requires_grad_(True)
        z = conv.causal_conv(x, wl)
        return (y, z.detach(), *torch.autograd.grad(z, (x, wl), xs[1 - i]))
    want = [both(0), both(1)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(both(i))
    torch.cuda.synchronize()
    for i in range(2):
        for turn in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(turn, want[i]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_outputs_that_are_not_finite_are_reported(gpu_lib, dtype):
    """With checking on: what the calls wrote, and not what lies behind the last row's tokens."""
    from gdnx_amd import _lib
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    r = lambda *s: torch.randn(*s, device="cuda").to(dtype)  # noqa: E731
    nan = float("nan")
    kp, vp, table, lens = r(8, 1, 16, 64), r(8, 1, 16, 64), i32([[0, 1, 2, 3], [4, 5, 6, 7]]), i32([40, 60])
    w, x = torch.randn(12, 4, device="cuda"), r(2, 9, 12)
    def chunk(counts, v, spare):                         # `spare` tokens of nobody before and behind the rows'
        N, end = sum(counts) + 2 * spare, sum(counts) + spare
        q = torch.full((N, 2, 64), nan, device="cuda").to(dtype)
        q[spare:end] = r(sum(counts), 2, 64)
        return attention.paged_attention_chunk(q, kp, v, table, lens, i32([spare, spare + counts[0], end]),
                                               out=torch.full_like(q, nan))
    def packed(x, spare, pool):
        none = torch.full((spare, 12), nan, device="cuda").to(dtype)
        x = torch.cat([none, x, none])
        return conv.causal_conv_packed(x, i32([spare, spare + 4, spare + 9]), pool, w, out=torch.full_like(x, nan))
    bad_v, bad_x, bad_state = vp.clone(), x.clone(), torch.zeros(2, 3, 12, device="cuda").to(dtype)
    bad_v[6, 0, 11, 3] = nan                             # position 43 of the second row
    bad_x[0, 3, 5] = float("inf")
    bad_state[1, 2, 4] = nan
    pool = lambda: torch.zeros(2, 3, 12, device="cuda").to(dtype)  # noqa: E731
    prev = _lib.set_check_finite(True)
    try:
        for counts in ([1, 1], [3, 20], [40, 30], [0, 5]):
            for spare in (0, 7):
                chunk(counts, vp, spare)
                with pytest.raises(_lib.GdnxNonFinite):
                    chunk(counts, bad_v, spare)
        for spare in (0, 7):
            packed(x[0], spare, pool())
            with pytest.raises(_lib.GdnxNonFinite):
                packed(bad_x[0], spare, pool())
        conv.causal_conv_step(x[:, 0], pool(), w)
        with pytest.raises(_lib.GdnxNonFinite):
            conv.causal_conv_step(bad_x[:, 3], pool(), w)
        lengths = i32([9, 0])                            # a row without tokens hands its state on
        conv.causal_conv(x, w, state=pool(), lengths=lengths, return_state=True)
        conv.causal_conv(x, w, state=bad_state, lengths=lengths)
        with pytest.raises(_lib.GdnxNonFinite):
            conv.causal_conv(x, w, state=bad_state, lengths=lengths, return_state=True)
    finally:
        _lib.set_check_finite(prev)
    chunk([1, 1], bad_v, 0)                              # off: no word of it
    torch.cuda.synchronize()


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
@pytest.mark.parametrize("kind,M", [("dense", 2), ("chan", 1), ("gdn3", 2)])
def test_a_served_step_does_not_wait_for_the_device(gpu_lib, kind, M, mode):
    n, H, D, C = 3, 2, 64, 40
    with mode():
        z = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
        cache = DecodeStateCache(4, H, M, D, kind=kind, conv=(C, 4), P=16)
        x, w, off = z(n, C, t=torch.bfloat16), z(C, 4), z(n + 1, t=torch.int32)
        io = torch.float32 if kind == "chan" else torch.bfloat16
        qkv, gates = [z(n, H, D, t=io) for _ in range(3)], [z(n, H, M) for _ in range(2)]
        decay = z(n, H, M, D) if kind == "chan" else z(n, H, M)
        slots = [2, 0, -1]
        torch.cuda.set_sync_debug_mode("error")              # (a cache may wait while it is made)
        try:
            for named in (slots, tuple(slots), cache.slots_tensor(slots), cache.slots_tensor(slots)):
                cache.convolve(named, x, w)
                cache.convolve(named, x[:, None].expand(n, 5, C), w)
                cache.convolve(named, x, w, offsets=off)
                cache.step(named, *qkv, *gates, decay)
        finally:
            torch.cuda.set_sync_debug_mode("default")
        if kind == "gdn3":
            assert cache.pos == [4, 0, 4, 0]


def test_slots_by_any_tensor(gpu_lib):
    cache = DecodeStateCache(4, 1, 1, 64, conv=(8, 4))
    x, w = torch.randn(2, 8, device="cuda").bfloat16(), torch.randn(8, 4, device="cuda")
    st = cache.slots_tensor([2, 1])
    assert st.tolist() == [2, 1] and st.dtype == torch.int32 and cache.slots_tensor(st) is st
    a = cache.convolve(st, x, w)
    cache.conv_pool.zero_()
    for named in (torch.tensor([2, 1]), torch.tensor([2, 1], device="cuda"), st.repeat_interleave(2)[::2]):
        assert torch.equal(cache.convolve(named, x, w), a)          # read back, and taken in 64 bits too
        cache.conv_pool.zero_()
    st[0] = 1                                                       # written since: what it was made of no longer holds
    with pytest.raises(ValueError, match="twice"):
        cache.convolve(st, x, w)
    own = torch.tensor([0, 3], dtype=torch.int32, device="cuda")    # a caller's buffer is read at every call
    with torch.inference_mode():
        own = own.clone()
        cache.convolve(own, x, w)
        own[0] = 3
        with pytest.raises(ValueError, match="twice"):
            cache.convolve(own, x, w)


@pytest.mark.parametrize("kind", ["dense", "gdn3"])
def test_a_caches_convolution_is_captured(gpu_lib, kind):
    """By the slots' tensor; ints, whose upload would be of memory that is used again, are refused before anything moves."""
    n, C, W = 3, 24, 4
    caches = [DecodeStateCache(5, 1, 1, 64, kind=kind, conv=(C, W)) for _ in range(2)]
    st = [c.slots_tensor([4, 0, 2]) for c in caches]
    x, w = torch.zeros(n, C, device="cuda").bfloat16(), torch.randn(C, W, device="cuda")
    off = torch.tensor([0, 2, 2, 3], dtype=torch.int32, device="cuda")
    step = lambda c, s: (c.convolve(s, x, w, offsets=off), c.convolve(s, x, w), c.convolve(s, x[:, None], w))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(DecodeStateCache(5, 1, 1, 64, kind=kind, conv=(C, W)), st[0])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[1], st[1])
        with pytest.raises(RuntimeError, match="captured"):
            caches[1].convolve([4, 0, 2], x, w)
        if kind == "gdn3":
            z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
            with pytest.raises(RuntimeError, match="captured"):
                caches[1].step(st[1], z(n, 1, 64), z(n, 1, 64), z(n, 1, 64), z(n, 1, 1), z(n, 1, 1), z(n, 1, 1))
    for turn in range(4):
        x.copy_(torch.randn(n, C, device="cuda"))
        graph.replay()
        want = step(caches[0], st[0])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn
        assert torch.equal(caches[0].conv_pool, caches[1].conv_pool)
