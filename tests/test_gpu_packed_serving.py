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
