"""The key/value cache operators where they can go wrong: codes at ties,
factors of any sign, value scales far apart, rows that see nothing of a large
value, workspaces that grow, lists that share blocks.

Expected values come from the formulas in 64 bits (or exact fractions), of the
codes and scales that the cache holds, written apart from the kernels."""
import ctypes
import math
from fractions import Fraction

import numpy as np
import pytest

DTYPES = ("float16", "bfloat16")
STEP = np.float32(1) / np.float32(127)


def magnitudes(dtype):
    """The numbers of the type in [1, 2), as float32, whose product with the float nearest 1/127 is not the float nearest
    to their 127th part."""
    if dtype == "float16":
        x = np.arange(0x3C00, 0x4000, dtype=np.uint16).view(np.float16).astype(np.float32)
    else:
        x = (np.arange(0x3F80, 0x4000, dtype=np.uint32) << 16).view(np.float32)
    return x[x * STEP != x / np.float32(127)]


def int32(a):
    import torch
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def batch_of(table, lens, rows, max_len=None):
    from dance_b200 import kvcache
    off = np.concatenate([[0], np.cumsum(rows)])
    return kvcache.KVBatch(int32(table), int32(lens), int32(off), max(rows), max(lens) if max_len is None else max_len)


# ------------------------------------------------------------------ append
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_rounds_ties_to_even(dance_lib, dtype):
    """Half of a block's largest magnitude lies between two codes, 63.5: the even one is right.  The scale, rounded up
    here, would give the odd one."""
    import torch
    from dance_b200 import kvcache
    most = magnitudes(dtype)
    n = len(most)
    x = np.zeros((16 * n, 1, 64), np.float32)
    x[::16, 0, 0] = most
    x[1::16, 0, 1], x[2::16, 0, 1] = most / 2, -most / 2
    want = round(Fraction(127, 2))
    assert want == 64 and (x[1::16, 0, 1].astype(np.float64) * 2 == most).all()
    cache = kvcache.KVCache.create(n, 1, 64, 16)
    t = torch.tensor(x, device="cuda").to(getattr(torch, dtype))
    assert (t.float().cpu().numpy() == x).all()
    batch = batch_of([list(range(n))], [16 * n], [16 * n])
    for _ in range(2):  # rows written again get the same codes
        kvcache.append(cache, batch, t, t)
        for codes in (cache.k, cache.v):
            c = codes[:, 0].cpu().numpy().astype(int) - 128
            assert (c[:, 0, 0] == 127).all() and (c[:, 1, 1] == want).all() and (c[:, 2, 1] == -want).all()
        b = cache.bounds[:, 0].cpu().numpy().astype(int) - 128
        assert (b[:, 0, 1] == -want).all() and (b[:, 1, 1] == want).all()
        # the scale stays the float nearest to the quotient
        assert (cache.k_scale[:, 0].cpu().numpy() == (most.astype(np.float64) / 127).astype(np.float32)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,bs", [(64, 16), (96, 32), (128, 64)])
def test_append_codes_are_those_of_the_step(dance_lib, dim, bs, dtype):
    """Rows of ordinary sizes, whole and begun blocks: codes and bounds by the step, value by value."""
    import torch
    from dance_b200 import kvcache
    n, h = 64, 4
    g = torch.Generator(device="cuda").manual_seed(dim)
    cache = kvcache.KVCache.create(n, h, dim, bs)
    first, then = bs // 2 + 1, bs * n
    x = (torch.randn((then, h, dim), generator=g, device="cuda") * 1.2).to(getattr(torch, dtype))
    kvcache.append(cache, batch_of([list(range(n))], [first], [first]), x[:first], x[:first])
    kvcache.append(cache, batch_of([list(range(n))], [then], [then - first]), x[first:], x[first:])
    y = x.float().cpu().numpy().reshape(n, bs, h, dim).transpose(0, 2, 1, 3)

    def step(a):
        return np.abs(a).max((-2, -1)).astype(np.float32) * STEP

    def codes(a, s):
        return np.rint(a * (np.float32(1) / s)[..., None, None])

    want = codes(y, step(y))
    for i in range(h):  # the first block was begun by fewer rows
        head, rest = y[0, i, :first], y[0, i, first:]
        s1, s2 = step(head[None])[0], step(rest[None])[0]
        q1, q2 = (np.abs(a).max() / np.float32(127) for a in (head, rest))
        old = np.rint(head * (np.float32(1) / s1))
        s = q1 if q1 > q2 else s2
        want[0, i, :first] = np.rint(old * (q1 / s)) if q2 > q1 else old
        want[0, i, first:] = np.rint(rest * (np.float32(1) / s))
    for t in (cache.k, cache.v):
        assert np.array_equal(t.cpu().numpy().astype(int) - 128, want.astype(int))
    b = cache.bounds.cpu().numpy().astype(int) - 128
    assert np.array_equal(b[:, :, 0], want.min(2)) and np.array_equal(b[:, :, 1], want.max(2))


# ------------------------------------------------------------------ selection
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_selection_rounds_ties_to_even(dance_lib, dtype):
    """Two blocks whose bounds weigh a query's tied channel against its largest one: the code of the tie decides."""
    import torch
    from dance_b200 import kvcache
    most = magnitudes(dtype)
    T = len(most)
    cache = kvcache.KVCache.create(4, 1, 64, 16)
    # scores of blocks 1 and 2: 127 * 63 and 64 * 126 (+ 62 of a channel of code 1), so that code 63 would choose block 1
    cache.bounds[1, 0, :, 0] = 128 + 63
    cache.bounds[2, 0, :, 1] = 128 + 126
    cache.k_scale.fill_(0.5)
    q = np.zeros((T, 1, 64), np.float32)
    q[:, 0, 0], q[:, 0, 1] = most, most / 2
    assert 127 * 63 < 64 * 126 and 127 * 63 > 63 * 126
    t = torch.tensor(q, device="cuda").to(getattr(torch, dtype))
    got = kvcache.select_blocks(cache, batch_of([[0, 1, 2, 3]] * T, [64] * T, [1] * T), t, 3)
    assert np.array_equal(got.cpu().numpy()[:, 0], np.tile([0, 2, 3], (T, 1)))


# ------------------------------------------------------------------ workspaces
def decode_step(tokens, seed=0, heads=8):
    """A call whose splits are joined through the workspace's counters."""
    import torch
    from dance_b200 import kvcache
    n = -(-tokens // 64)
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(1, 256, (2, n, 2, 64, 64), generator=g, device="cuda").to(torch.uint8)
    scale = torch.full((2, n, 2), 0.01, device="cuda")
    cache = kvcache.KVCache(codes[0], codes[1], scale[0], scale[1], codes[0, :, :, :2].contiguous())
    q = torch.randn((1, heads, 64), generator=g, device="cuda").half()
    return cache, batch_of([list(range(n))], [tokens], [1]), q


@pytest.mark.gpu
def test_captured_graph_survives_a_workspace_that_grows(dance_lib):
    import torch
    from dance_b200 import kvcache
    cache, batch, q = decode_step(4000)
    want = kvcache.attention(cache, batch, q)
    ws = kvcache.KVWorkspace()
    ws.reserve(cache, batch, 1, 8)
    kvcache.attention(cache, batch, q, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kvcache.attention(cache, batch, q, workspace=ws)
    small, address = ws._bytes, ws._ptr
    big = decode_step(100000, heads=64)
    large = kvcache.attention(*big, workspace=ws)
    assert ws._bytes > small and ws._ptr != address
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    # what the allocator would hand out of a freed buffer
    other = [torch.full((max(small // 2 ** i, 512),), 255, dtype=torch.uint8, device="cuda") for i in range(8) for _ in range(4)]
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert torch.equal(kvcache.attention(*big, workspace=ws), large)
    assert all((t == 255).all() for t in other)


@pytest.mark.gpu
def test_workspace_does_not_grow_in_a_capture(dance_lib):
    """Its zeroing would be the graph's: the call refuses.  A call without a workspace has one of the graph's own."""
    import torch
    from dance_b200 import kvcache
    cache, batch, q = decode_step(4000)
    want = kvcache.attention(cache, batch, q)
    ws, graph = kvcache.KVWorkspace(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = kvcache.attention(cache, batch, q)
        with pytest.raises(ValueError, match="before the stream capture"):
            kvcache.attention(cache, batch, q, workspace=ws)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert torch.equal(kvcache.attention(cache, batch, q, workspace=ws), want)


@pytest.mark.gpu
def test_workspace_zeroed_on_another_stream(dance_lib):
    """A workspace reserved on a busy stream is used on another one at once."""
    import torch
    from dance_b200 import kvcache
    cache, batch, q = decode_step(4000)
    want = kvcache.attention(cache, batch, q)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        ws = kvcache.KVWorkspace()
        with torch.cuda.stream(a):
            torch.full((64 << 20,), 255, dtype=torch.uint8, device="cuda")  # what the buffer may come out of
            torch.cuda._sleep(20_000_000)
            ws.reserve(cache, batch, 1, 8)
        out = kvcache.attention(cache, batch, q, workspace=ws, stream=b)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
