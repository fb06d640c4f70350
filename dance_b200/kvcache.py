"""Long-context memory next to the index: an 8-bit key/value cache, the
attention over it, and the choice of the blocks that a query reads.

The proximity graphs of this package answer "which stored vectors are near
this one"; a model with a long context asks that of its own keys.  This module
holds those keys and values (8 bits, one scale per block of tokens and head),
writes new tokens into them, reads them back as vectors (what an index build
takes), and attends over all of a sequence or over the blocks that the cheap
block score, or a graph search over the keys, picked:

    cache = KVCache.create(num_blocks, kv_heads=8, head_dim=128, device="cuda")
    batch = KVBatch(block_table, seq_lens, row_offsets, max_rows, max_len)
    append(cache, batch, k_new, v_new)
    out = attention(cache, batch, q)                  # every token
    blocks = select_blocks(cache, batch, q, 64)       # 64 blocks for each row
    out = sparse_attention(cache, batch, q, blocks)   # their tokens

All tensors are CUDA tensors of one device; the calls take ``stream`` (None:
torch's current stream), on which they run and allocate, neither synchronise nor copy to the host, and may be
captured in a CUDA graph; ``status`` tells whether they finished.  The kernels are those of ``dance_kv_*`` in
include/dance_b200.h, where the formulas and the layouts stand.
"""
from __future__ import annotations

import ctypes
import functools
from ctypes import addressof as _address

from . import DANCE_BF16, DANCE_F16, DANCE_F32, DanceKvBatch, DanceKvCache, DanceKvRows, check, load

__all__ = ["KVCache", "KVBatch", "KVWorkspace", "append", "read", "attention", "select_blocks", "sparse_attention",
           "status"]

HEAD_DIMS = (64, 96, 128)
BLOCK_TOKENS = (16, 32, 64, 128)


def _need(ok, message):
    if not ok:
        raise ValueError(message)


def _cuda(name, t, dtype, shape=None):
    import torch
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} is {t.dtype}, {dtype} is needed")
    if shape is not None:
        _need(tuple(t.shape) == tuple(shape), f"{name} has shape {tuple(t.shape)}, {tuple(shape)} is needed")


class KVCache:
    """Keys and values of many sequences in 8 bits.

    k, v: uint8 (num_blocks, kv_heads, block_tokens, head_dim), blocks
    contiguous inside (the first dimension may be strided, as halves of one
    pool are); k_scale, v_scale: float32 (num_blocks, kv_heads); bounds: uint8
    (num_blocks, kv_heads, 2, head_dim), the smallest and largest key code per
    channel.  A code c stands for (c - 128) * scale.  The tensors stay the
    caller's: they are read and written in place.
    """

    def __init__(self, k, v, k_scale, v_scale, bounds):
        import torch
        _need(isinstance(k, torch.Tensor) and k.dim() == 4, "k must be a tensor of four dimensions")
        n, h, bs, d = k.shape
        _cuda("k", k, torch.uint8)
        _cuda("v", v, torch.uint8, k.shape)
        _cuda("k_scale", k_scale, torch.float32, (n, h))
        _cuda("v_scale", v_scale, torch.float32, (n, h))
        _cuda("bounds", bounds, torch.uint8, (n, h, 2, d))
        _need(d in HEAD_DIMS, f"head_dim {d}: one of {HEAD_DIMS} is needed")
        _need(bs in BLOCK_TOKENS, f"block_tokens {bs}: one of {BLOCK_TOKENS} is needed")
        _need(n > 0 and h > 0, "an empty cache")
        for name, t in (("k", k), ("v", v)):
            _need(t.stride()[1:] == (bs * d, d, 1), f"{name}: the blocks must be contiguous inside")
            _need(n == 1 or t.stride(0) >= h * bs * d, f"{name}: the blocks must not overlap")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale), ("bounds", bounds)):
            _need(t.is_contiguous(), f"{name} must be contiguous")
        _need(all(t.device == k.device for t in (v, k_scale, v_scale, bounds)), "the tensors lie on different devices")
        self.k, self.v, self.k_scale, self.v_scale, self.bounds = k, v, k_scale, v_scale, bounds
        self.num_blocks, self.kv_heads, self.block_tokens, self.head_dim = n, h, bs, d
        self.device = k.device
        least = h * bs * d
        self._c = DanceKvCache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), bounds.data_ptr(),
                               max(k.stride(0), least), max(v.stride(0), least), n, h, bs, d)
        self._ptr = ctypes.addressof(self._c)
        self._index = k.get_device()
        self._key = (n, h, bs, d, self._index)

    @classmethod
    def create(cls, num_blocks: int, kv_heads: int, head_dim: int, block_tokens: int = 64, device="cuda"):
        """An empty cache of new tensors."""
        import torch
        code = torch.full((2, num_blocks, kv_heads, block_tokens, head_dim), 128, dtype=torch.uint8, device=device)
        scale = torch.zeros((2, num_blocks, kv_heads), dtype=torch.float32, device=device)
        bounds = torch.full((num_blocks, kv_heads, 2, head_dim), 128, dtype=torch.uint8, device=device)
        return cls(code[0], code[1], scale[0], scale[1], bounds)


class KVBatch:
    """The sequences of a call: which blocks hold them and which rows of the
    call's tensors are theirs.

    block_table: int32 (batch, width), block of every block_tokens tokens, -1
    where there is none; seq_lens: int32 (batch,), tokens of each sequence with
    the call's new rows; row_offsets: int32 (batch + 1,), the rows of sequence
    b being row_offsets[b] .. row_offsets[b + 1], its last row at its last
    token.  max_rows and max_len: bounds of rows and tokens of a sequence, known
    on the host; what lies beyond is not visited.  Rows that belong to no
    sequence, or lie beyond max_rows, are not written: in a new output they hold
    anything.  The tensors may be updated in place between calls.
    """

    def __init__(self, block_table, seq_lens, row_offsets, max_rows: int, max_len: int):
        import torch
        _need(isinstance(seq_lens, torch.Tensor) and seq_lens.dim() == 1 and seq_lens.shape[0] > 0,
              "seq_lens must be a tensor of one dimension")
        n = seq_lens.shape[0]
        _cuda("seq_lens", seq_lens, torch.int32)
        _cuda("row_offsets", row_offsets, torch.int32, (n + 1,))
        _cuda("block_table", block_table, torch.int32)
        _need(block_table.dim() == 2 and block_table.shape[0] == n,
              f"block_table has shape {tuple(block_table.shape)}, ({n}, width) is needed")
        _need(n <= 65535, f"batch of {n} sequences: at most 65535")
        _need(max_rows >= 0 and max_len >= 0, "max_rows and max_len must not be negative")
        for name, t in (("block_table", block_table), ("seq_lens", seq_lens), ("row_offsets", row_offsets)):
            _need(t.is_contiguous(), f"{name} must be contiguous")
            _need(t.device == seq_lens.device, "the tensors lie on different devices")
        self.block_table, self.seq_lens, self.row_offsets = block_table, seq_lens, row_offsets
        self.max_rows, self.max_len, self.batch = int(max_rows), int(max_len), n
        self.device = seq_lens.device
        self._c = DanceKvBatch(block_table.data_ptr(), seq_lens.data_ptr(), row_offsets.data_ptr(),
                               block_table.shape[1], n, self.max_rows, self.max_len)
        self._ptr = ctypes.addressof(self._c)
        self._index = seq_lens.get_device()
        self._key = (n, self.max_rows, self.max_len, block_table.shape[1])


class KVWorkspace:
    """Device scratch of the attention and the selection, grown on demand; it
    serves one call at a time (calls on one stream, or on streams that wait for
    one another).

    Buffers that it outgrew stay allocated as long as it lives: a CUDA graph
    that was captured with one still writes to it, and so may a call in flight.
    Each is at least twice as large as the one before, so that all of them
    together take less than the last one again.
    """

    def __init__(self):
        self._held: dict = {}  # device -> its buffers, the last in use
        self._index = None     # device of the buffer in use
        self._ptr = 0
        self._bytes = 0
        self._known = set()
        self._stream = None    # the stream that last came behind the zeroing
        self._zeroed = None

    def reserve(self, cache: KVCache, batch: KVBatch, rows: int, num_heads: int, select: int = 0) -> None:
        """Room for such a call.  A workspace does not grow in a stream capture, where its zeroing would wait for the
        graph's replay: reserve before, and let that finish."""
        if (cache._key, batch._key, rows, num_heads, select) not in self._known:
            import torch
            self._grow(cache, batch, rows, num_heads, select, not torch.cuda.is_current_stream_capturing())

    def _grow(self, cache, batch, rows, num_heads, select, may_allocate):
        need = load().dance_kv_workspace_bytes(cache._ptr, batch._ptr, rows, num_heads, select)
        if need == 0:
            check(-1, "dance_kv_workspace_bytes")
        if self._index != cache._index:
            self._index, self._bytes, self._stream = cache._index, 0, None
            self._known.clear()
            if self._index in self._held:
                self._set(*self._held[self._index][-1])
        if need > self._bytes:
            import torch
            _need(may_allocate, f"the workspace holds {self._bytes} bytes, {need} are needed: "
                                "reserve them before the stream capture")
            with torch.cuda.device(cache.device):
                t = torch.zeros(max(need, 2 * self._bytes), dtype=torch.uint8, device=cache.device)
                done = torch.cuda.Event()
                done.record()
                self._stream = torch.cuda.current_stream().cuda_stream
            self._held.setdefault(self._index, []).append((t, done))
            self._set(t, done)
        if len(self._known) > 256:
            self._known.clear()
        self._known.add((cache._key, batch._key, rows, num_heads, select))

    def _set(self, t, done):
        self._ptr, self._bytes, self._zeroed = t.data_ptr(), t.numel(), done

    def _follow(self, stream):
        """Lets the current stream, of that handle, wait for the buffer's zeroing."""
        import torch
        if not torch.cuda.is_current_stream_capturing():  # before a capture the caller waits
            torch.cuda.current_stream().wait_event(self._zeroed)
            self._stream = stream


def _scratch(workspace, cache, batch, rows, heads, select, stream):
    """The workspace of a call on the current stream, with room for it; a new one where the caller has none."""
    if workspace is None:
        workspace = KVWorkspace()
        workspace._grow(cache, batch, rows, heads, select, True)  # in a capture it is the graph's, zeroed by each replay
    else:
        workspace.reserve(cache, batch, rows, heads, select)
        if workspace._stream != stream:
            workspace._follow(stream)
    return workspace


# The calls below are short (a decode step calls them once per layer), so what
# they need of torch is bound once, on the first call.
_torch = None
_lib = None
_DTYPES: dict = {}


def _bind():
    global _torch, _lib
    import torch
    _lib = load()
    _DTYPES.update({torch.float16: DANCE_F16, torch.bfloat16: DANCE_BF16, torch.float32: DANCE_F32})
    _torch = torch


def _rows(name, x, cache, heads=None):
    """DanceKvRows of a (rows, heads, head_dim) tensor."""
    try:
        n, h, d = x.shape
        s0, s1, s2 = x.stride()
        code = _DTYPES.get(x.dtype)
        index = x.get_device()
    except (AttributeError, TypeError, ValueError):
        raise ValueError(f"{name} must be a CUDA tensor of three dimensions") from None
    if code is None or code == DANCE_F32:
        raise TypeError(f"{name} is {x.dtype}: float16 or bfloat16 is needed")
    if d != cache.head_dim or (h != heads if heads is not None else h == 0 or h % cache.kv_heads):
        raise ValueError(f"{name} has shape {tuple(x.shape)}: the cache has {cache.kv_heads} heads of {cache.head_dim}")
    if s2 != 1:
        raise ValueError(f"{name}: the channels must be contiguous")
    if index != cache._index:
        raise ValueError(f"{name} lies on {x.device}, the cache on {cache.device}")
    return DanceKvRows(x.data_ptr(), s0, s1, n, code), n, h


def _enter(cache, batch):
    """Checks the devices; torch's current stream, on which outputs and scratch are allocated too."""
    if _torch is None:
        _bind()
    index = cache._index
    if batch._index != index:
        raise ValueError(f"the batch lies on {batch.device}, the cache on {cache.device}")
    if _torch._C._cuda_getDevice() != index:
        raise ValueError(f"the cache lies on {cache.device}, the current device is cuda:{_torch.cuda.current_device()}")
    return _torch._C._cuda_getCurrentRawStream(index)


def _streamed(fn):
    """Adds ``stream``: the call runs, and allocates, with that stream as torch's current one."""
    @functools.wraps(fn)
    def call(*args, stream=None, **kwargs):
        if stream is None:
            return fn(*args, **kwargs)
        import torch
        if not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(int(stream))
        with torch.cuda.stream(stream):
            return fn(*args, **kwargs)
    return call


@_streamed
def append(cache: KVCache, batch: KVBatch, k, v) -> None:
    """Write new tokens' keys and values, (rows, kv_heads, head_dim) each, into
    the cache.  The scales of touched blocks only grow; where one does, the
    block's earlier codes are rounded again.  NaN becomes 0, an infinity the
    largest code."""
    stream = _enter(cache, batch)
    kr, n, _ = _rows("k", k, cache, cache.kv_heads)
    vr, m, _ = _rows("v", v, cache, cache.kv_heads)
    if n != m or k.dtype != v.dtype:
        raise ValueError(f"k is {tuple(k.shape)} {k.dtype}, v {tuple(v.shape)} {v.dtype}")
    rc = _lib.dance_kv_append(cache._ptr, batch._ptr, _address(kr), _address(vr), stream)
    if rc:
        check(rc, "dance_kv_append")


@_streamed
def read(cache: KVCache, batch: KVBatch, rows: int, dtype=None):
    """(keys, values) that the cache holds for the batch's rows, each (rows,
    kv_heads, head_dim) of dtype (float16, bfloat16 or float32; None: float16).
    The keys of a head are a vector store that an index build takes."""
    stream = _enter(cache, batch)
    dtype = dtype or _torch.float16
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"dtype {dtype}: float16, bfloat16 or float32 is needed")
    if rows < 0:
        raise ValueError("rows must not be negative")
    both = _torch.empty((2, rows, cache.kv_heads, cache.head_dim), dtype=dtype, device=cache.device)
    k, v = both.unbind(0)
    rc = _lib.dance_kv_read(cache._ptr, batch._ptr, rows, code, k.data_ptr(), v.data_ptr(), stream)
    if rc:
        check(rc, "dance_kv_read")
    return k, v


def _attend(cache, batch, q, blocks, scale, return_lse, out, workspace):
    stream = _enter(cache, batch)
    qr, rows, heads = _rows("q", q, cache)
    dim = cache.head_dim
    if out is None:
        out = _torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape)
    else:
        _cuda("out", out, q.dtype, q.shape)
        _need(out.is_contiguous() and out.device == cache.device, "out must be contiguous, on the cache's device")
    lse, lse_ptr, select = None, None, 0
    if return_lse:
        lse = _torch.empty((rows, heads), dtype=_torch.float32, device=cache.device)
        lse_ptr = lse.data_ptr()
    if blocks is not None:
        if blocks.dim() != 3 or blocks.shape[0] != rows or blocks.shape[1] != cache.kv_heads:
            raise ValueError(f"blocks has shape {tuple(blocks.shape)}: ({rows}, {cache.kv_heads}, select) is needed")
        if blocks.dtype != _torch.int32:
            raise TypeError(f"blocks is {blocks.dtype}, torch.int32 is needed")
        select = blocks.shape[2]
        if not blocks.is_contiguous() or blocks.get_device() != cache._index:
            raise ValueError("blocks must be contiguous, on the cache's device")
        if not 1 <= select <= 4096:
            raise ValueError(f"{select} blocks per row: 1 to 4096 are supported")
    ws = _scratch(workspace, cache, batch, rows, heads, select, stream)
    if scale is None:
        scale = dim ** -0.5
    if blocks is None:
        rc = _lib.dance_kv_attention(cache._ptr, batch._ptr, _address(qr), heads, scale, out.data_ptr(), lse_ptr,
                                     ws._ptr, ws._bytes, stream)
        if rc:
            check(rc, "dance_kv_attention")
    else:
        rc = _lib.dance_kv_sparse_attention(cache._ptr, batch._ptr, _address(qr), heads, blocks.data_ptr(), select,
                                            scale, out.data_ptr(), lse_ptr, ws._ptr, ws._bytes, stream)
        if rc:
            check(rc, "dance_kv_sparse_attention")
    return (out, lse) if return_lse else out


@_streamed
def attention(cache: KVCache, batch: KVBatch, q, scale: float | None = None, *, return_lse: bool = False, out=None,
              workspace: KVWorkspace | None = None):
    """softmax(scale * q k) v of q (rows, heads, head_dim) over each row's
    sequence up to its own position; heads / kv_heads query heads share a
    key/value head.  scale None: head_dim ** -0.5.  With return_lse also the
    log of the rows' sums (float32, for joining parts): (out, lse).  A row that
    sees nothing gives 0 and -inf."""
    return _attend(cache, batch, q, None, scale, return_lse, out, workspace)


@_streamed
def sparse_attention(cache: KVCache, batch: KVBatch, q, blocks, scale: float | None = None, *,
                     return_lse: bool = False, out=None, workspace: KVWorkspace | None = None):
    """Attention over the tokens, up to each row's position, of the blocks that
    ``blocks`` (int32 (rows, kv_heads, select), positions in the block table,
    negative: none) names for the row and head."""
    _need(blocks is not None and hasattr(blocks, "is_cuda"), "blocks must be a CUDA tensor")
    return _attend(cache, batch, q, blocks, scale, return_lse, out, workspace)


@_streamed
def select_blocks(cache: KVCache, batch: KVBatch, q, select: int, *, first_blocks: int = 1, last_blocks: int = 1,
                  out=None, workspace: KVWorkspace | None = None):
    """The ``select`` blocks that each row of q reads, per key/value head: int32
    (rows, kv_heads, select), ascending, -1 filled.  The row's first
    ``first_blocks`` and last ``last_blocks`` blocks are always among them, the
    others have the largest upper bounds on their logits."""
    stream = _enter(cache, batch)
    qr, rows, heads = _rows("q", q, cache)
    if not 1 <= select <= 4096 or first_blocks < 0 or last_blocks < 0 or first_blocks + last_blocks > select:
        raise ValueError(f"select {select} (1 to 4096) must hold {first_blocks} first and {last_blocks} last blocks")
    if out is None:
        out = _torch.empty((rows, cache.kv_heads, select), dtype=_torch.int32, device=cache.device)
    else:
        _cuda("out", out, _torch.int32, (rows, cache.kv_heads, select))
        _need(out.is_contiguous() and out.device == cache.device, "out must be contiguous, on the cache's device")
    ws = _scratch(workspace, cache, batch, rows, heads, select, stream)
    rc = _lib.dance_kv_select_blocks(cache._ptr, batch._ptr, _address(qr), heads, select, first_blocks, last_blocks,
                                     out.data_ptr(), ws._ptr, ws._bytes, stream)
    if rc:
        check(rc, "dance_kv_select_blocks")
    return out


def status() -> None:
    """Waits for the current device and raises DanceError where blocks of an attention call gave up waiting and left
    not-a-number in their rows.  To be called where results are handed on."""
    check(load().dance_kv_status(), "dance_kv_status")
