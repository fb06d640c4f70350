"""The key/value cache operators against plain restatements: the write and the
selection value by value (they are exact), the attention in 64 bits within the
error that its roundings allow, and what each call refuses.

Tolerance of the attention, per element (fixed before the first run): with
o the result in 64 bits, A = sum_j p_j |v_j| and S the largest
scale * sum_d |q_d k_d| of the row,
    u_out |o| + (2^-11 + 2 (D + 8) 2^-23 S + 2^-19) A + n 2^-39 max|v| + 2^-24:
the output's rounding (u_out = 2^-11 or 2^-8), the weights' (halves, 2^-11),
the logits' (products of D terms in float), 2^x and the sums in float, and
weights below a half's range.
"""
import ctypes
import itertools
import math

import numpy as np
import pytest

DTYPES = ("float16", "bfloat16")


# ------------------------------------------------------------------ plain forms
def plain_scale(x):
    """max finite |x| / 127 in float32, 0 below 2^-126."""
    a = np.abs(x[np.isfinite(x)])
    s = np.float32(a.max() if a.size else 0.0) / np.float32(127.0)
    return np.float32(0.0) if s < np.float32(2.0 ** -126) else s


def plain_codes(x, scale):
    inv = np.float32(1.0) / scale if scale > 0 else np.float32(0.0)
    with np.errstate(over="ignore", invalid="ignore"):
        y = (x * inv).astype(np.float32)
    y = np.where(np.isnan(y), np.float32(0), np.clip(y, -127, 127))
    return np.rint(y).astype(np.int64)


class PlainCache:
    """Codes - 128, scales and bounds on the host, block by block."""

    def __init__(self, n, hkv, bs, dim):
        self.n, self.hkv, self.bs, self.dim = n, hkv, bs, dim
        self.code = {k: np.zeros((n, hkv, bs, dim), np.int64) for k in "kv"}
        self.scale = {k: np.zeros((n, hkv), np.float32) for k in "kv"}
        self.low, self.high = np.zeros((n, hkv, dim), np.int64), np.zeros((n, hkv, dim), np.int64)

    def append(self, table, lens, offsets, k, v):
        for b, n in enumerate(lens):
            rows = offsets[b + 1] - offsets[b]
            first = n - rows
            for page in range(max(first, 0) // self.bs, -(-n // self.bs) if n > 0 else 0):
                lo, hi = max(first, 0, page * self.bs), min(n, (page + 1) * self.bs)
                at = table[b][page] if page < len(table[b]) else -1
                if hi <= lo or not 0 <= at < self.n:
                    continue
                old_n, m = lo - page * self.bs, hi - page * self.bs
                for h, (name, x) in itertools.product(range(self.hkv), (("k", k), ("v", v))):
                    new = x[offsets[b] + lo - first:offsets[b] + hi - first, h]
                    old = self.scale[name][at, h] if old_n else np.float32(0)
                    s = max(old, plain_scale(new))
                    c = self.code[name][at, h]
                    bounds = [self.low[at, h], self.high[at, h]]
                    if old_n and s != old:
                        again = lambda x: np.rint(x.astype(np.float32) * (old / s)).astype(np.int64)  # noqa: E731
                        c[:old_n] = again(c[:old_n])
                        bounds = [again(x) for x in bounds]
                    c[old_n:m] = plain_codes(new, s)
                    self.scale[name][at, h] = s
                    if name == "k":
                        new = c[old_n:m].min(0), c[old_n:m].max(0)
                        self.low[at, h] = np.minimum(bounds[0], new[0]) if old_n else new[0]
                        self.high[at, h] = np.maximum(bounds[1], new[1]) if old_n else new[1]

    def values(self, name, at, h):
        return self.code[name][at, h].astype(np.float64) * np.float64(self.scale[name][at, h])


def places(lens, offsets):
    """(sequence, position) of every row."""
    return [(b, n - (offsets[b + 1] - offsets[b]) + i) for b, n in enumerate(lens)
            for i in range(offsets[b + 1] - offsets[b])]


def plain_attention(pc, table, lens, offsets, q, scale, blocks=None):
    """(out, lse, bound on the error without the output's rounding) in 64 bits."""
    T, H, D = q.shape
    G = H // pc.hkv
    out, lse, err = np.zeros((T, H, D)), np.full((T, H), -np.inf), np.zeros((T, H, D))
    for r, (b, pos) in enumerate(places(lens, offsets)):
        seen = min(pos + 1, lens[b], len(table[b]) * pc.bs)
        for h in range(pc.hkv):
            pages = range(-(-max(seen, 0) // pc.bs)) if blocks is None else [j for j in blocks[r, h]]
            ks, vs = [], []
            for j in pages:
                if not 0 <= j < len(table[b]) or not 0 <= table[b][j] < pc.n:
                    continue
                m = min(pc.bs, seen - j * pc.bs)
                if m > 0:
                    ks.append(pc.values("k", table[b][j], h)[:m])
                    vs.append(pc.values("v", table[b][j], h)[:m])
            if not ks:
                continue
            k, v = np.concatenate(ks), np.concatenate(vs)
            for g in range(h * G, (h + 1) * G):
                x = scale * (k @ q[r, g])
                top = x.max()
                p = np.exp(x - top)
                lse[r, g] = top + math.log(p.sum())
                p /= p.sum()
                out[r, g] = p @ v
                S = abs(scale) * (np.abs(k) @ np.abs(q[r, g])).max()
                err[r, g] = ((2.0 ** -11 + 2 * (D + 8) * 2.0 ** -23 * S + 2.0 ** -19) * (p @ np.abs(v))
                             + len(k) * 2.0 ** -39 * np.abs(v).max() + 2.0 ** -24)
    return out, lse, err


def plain_select(pc, table, lens, offsets, q, select, first, last):
    T, H, D = q.shape
    G = H // pc.hkv
    out = np.full((T, pc.hkv, select), -1, np.int64)
    for r, (b, pos) in enumerate(places(lens, offsets)):
        seen = min(pos + 1, lens[b], len(table[b]) * pc.bs)
        nb = -(-max(seen, 0) // pc.bs)
        for h in range(pc.hkv):
            score = np.full(nb, -np.inf, np.float32)
            for j in range(nb):
                at = table[b][j]
                if not 0 <= at < pc.n:
                    continue
                best = -np.inf
                for g in range(h * G, (h + 1) * G):
                    s = plain_scale(q[r, g])
                    c = plain_codes(q[r, g], s)
                    dot = np.maximum(c * pc.low[at, h], c * pc.high[at, h]).sum()
                    best = max(best, np.float32(dot) * s)
                score[j] = np.float32(best) * pc.scale["k"][at, h]
            score[:first] = np.inf
            score[max(nb - last, 0):] = np.inf
            best = sorted(range(nb), key=lambda j: (-score[j], j))[:select]
            out[r, h, :len(best)] = sorted(best)
    return out


# ------------------------------------------------------------------ the two sides together
class World:
    """A cache on the GPU and its plain twin, filled by appends."""

    def __init__(self, lens, rows, hkv, dim, bs, dtype, seed=0, holes=(), spread=1.0, steps=1, pool_extra=2):
        import torch
        from dance_b200 import kvcache
        self.rng = np.random.default_rng(seed)
        self.dtype = getattr(torch, dtype)
        self.lens, self.rows, self.hkv, self.dim, self.bs = list(lens), list(rows), hkv, dim, bs
        need = [-(-max(n, 0) // bs) for n in lens]
        self.width = max(1, max(need))
        pool = sum(need) + pool_extra
        ids = self.rng.permutation(pool)
        self.table = np.full((len(lens), self.width), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
        for b, j in holes:
            self.table[b, j] = -1 if (b + j) % 2 else pool + 7
        self.plain = PlainCache(pool, hkv, bs, dim)
        pooled = torch.full((pool, 2, hkv, bs, dim), 255, dtype=torch.uint8, device="cuda")  # keys and values side by side
        self.cache = kvcache.KVCache(pooled[:, 0], pooled[:, 1],
                                     torch.full((pool, hkv), float("nan"), device="cuda"),
                                     torch.full((pool, hkv), float("nan"), device="cuda"),
                                     torch.full((pool, hkv, 2, dim), 77, dtype=torch.uint8, device="cuda"))
        for part in range(steps):
            upto = [n * (part + 1) // steps for n in lens]
            since = [n * part // steps for n in lens]
            size = (0.2 + part) * spread
            self.append(upto, [max(0, u - s) for u, s in zip(upto, since)], size)

    def device(self, a):
        import torch
        return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")

    def batch(self, lens=None, rows=None):
        from dance_b200 import kvcache
        lens, rows = list(self.lens if lens is None else lens), list(self.rows if rows is None else rows)
        off = np.concatenate([[0], np.cumsum(rows)])
        return kvcache.KVBatch(self.device(self.table), self.device(lens), self.device(off), max(rows),
                               max(0, max(lens))), lens, off

    def tensor(self, x):
        """A tensor of the dtype, and the values that it holds."""
        import torch
        t = torch.tensor(np.asarray(x, np.float32), device="cuda").to(self.dtype)
        return t, t.float().cpu().numpy()

    def append(self, lens, rows, size=1.0, make=None):
        from dance_b200 import kvcache
        if max(rows) == 0:
            return
        batch, lens, off = self.batch(lens, rows)
        T = int(off[-1])
        make = make or (lambda: self.rng.normal(size=(T, self.hkv, self.dim)) * size
                        * np.exp(self.rng.normal(size=(1, self.hkv, 1))))
        (k, kn), (v, vn) = self.tensor(make()), self.tensor(make())
        kvcache.append(self.cache, batch, k, v)
        self.plain.append(self.table, lens, off, kn, vn)

    def check_cache(self, exact_bounds=True):
        """Codes, scales and bounds of every block that holds tokens; the bounds
        are those of the codes unless rows were written again."""
        c, p = self.cache, self.plain
        code = {"k": c.k.cpu().numpy().astype(np.int64) - 128, "v": c.v.cpu().numpy().astype(np.int64) - 128}
        scale = {"k": c.k_scale.cpu().numpy(), "v": c.v_scale.cpu().numpy()}
        bounds = c.bounds.cpu().numpy().astype(np.int64) - 128
        for b, n in enumerate(self.lens):
            for j in range(-(-max(n, 0) // self.bs)):
                at = self.table[b, j]
                if not 0 <= at < p.n:
                    continue
                m = min(self.bs, n - j * self.bs)
                for name in "kv":
                    assert np.array_equal(scale[name][at], p.scale[name][at])
                    assert np.array_equal(code[name][at, :, :m], p.code[name][at, :, :m])
                assert np.array_equal(bounds[at, :, 0], p.low[at]) and np.array_equal(bounds[at, :, 1], p.high[at])
                if exact_bounds:
                    assert np.array_equal(bounds[at, :, 0], code["k"][at, :, :m].min(1))
                    assert np.array_equal(bounds[at, :, 1], code["k"][at, :, :m].max(1))

    def q(self, heads, size=1.0):
        return self.tensor(self.rng.normal(size=(sum(self.rows), heads, self.dim)) * size)


def check_out(got, want, err, dtype):
    u = 2.0 ** -11 if dtype == "float16" else 2.0 ** -8
    got = got.float().cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all()
    excess = np.abs(got - want) - (u * np.abs(want) + err)
    assert excess.max() <= 0, f"off by {np.abs(got - want).max()} where {err.flat[excess.argmax()]} is allowed"


def check_lse(got, want, err_s):
    got = got.cpu().numpy().astype(np.float64)
    none = np.isinf(want)
    assert np.array_equal(np.isneginf(got), none)
    assert np.abs(got[~none] - want[~none]).max(initial=0.0) <= err_s


# ------------------------------------------------------------------ append and read
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,bs", [(64, 16), (96, 32), (128, 64), (64, 128), (128, 16), (96, 128)])
def test_append_equals_the_definition(dance_lib, dim, bs, dtype):
    lens = [1, bs, bs + 1, 3 * bs - 1, 0, 2 * bs + 5]
    w = World(lens, [0] * 6, 3, dim, bs, dtype, seed=dim + bs, steps=3)  # later parts are larger: scales grow
    w.check_cache()


@pytest.mark.gpu
def test_append_token_by_token(dance_lib):
    """Single tokens of growing and shrinking size: every step either keeps the scale or rounds again."""
    w = World([5, 37], [0, 0], 2, 96, 16, "bfloat16", seed=5)
    for step in range(20):
        w.lens = [n + 1 for n in w.lens]
        if max(w.lens) > w.width * w.bs:
            break
        w.append(w.lens, [1, 1], size=[0.1, 3.0, 0.5, 9.0][step % 4])
        w.check_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_odd_values(dance_lib, dtype):
    """Zeros, values without a finite reciprocal scale, infinities and NaN."""
    w = World([40], [0], 2, 64, 32, dtype, seed=1)
    kinds = [lambda x: x * 0, lambda x: x * 1e-40, lambda x: np.where(x > 1, np.inf, x),
             lambda x: np.where(x < -1, -np.inf, np.where(x > 1, np.nan, x)), lambda x: x * np.nan]
    for kind in kinds:
        w = World([33], [0], 2, 64, 32, dtype, seed=3)
        w.plain = PlainCache(w.plain.n, 2, 32, 64)
        w.append([33], [33], make=lambda: kind(w.rng.normal(size=(33, 2, 64))))
        w.check_cache()
        w.lens = [50]
        w.append([50], [17], size=2.0)
        w.check_cache()


@pytest.mark.gpu
def test_append_outside_the_table_and_before_the_start(dance_lib):
    """Tokens without a block, or of negative position, are dropped; sequences without new rows stay."""
    w = World([70, 20, 64], [0, 0, 0], 2, 128, 32, "float16", seed=2, holes=[(0, 1), (1, 0)])
    w.check_cache()
    before = w.cache.k.clone()
    w.append([70, 20, 64], [0, 0, 0])
    assert (w.cache.k == before).all()
    w.append([3, 20, 64], [9, 0, 1])  # six of the nine rows lie before the start
    w.lens = [3, 20, 64]
    w.check_cache(exact_bounds=False)


@pytest.mark.gpu
def test_append_strided_and_unaligned(dance_lib):
    import torch
    from dance_b200 import kvcache
    w = World([50, 9], [0, 0], 2, 96, 16, "float16", seed=8)
    batch, lens, off = w.batch([50, 9], [50, 9])
    big = torch.randn((59, 4, 2 * 97 + 6), device="cuda").half()
    for k, v in ((big[:, 0:2, :96], big[:, 2:4, :96]),          # rows and heads strided
                 (big[:, 0:2, 1:97], big[:, 2:4, 97:193]),      # not on 16 bytes
                 (big.transpose(0, 1)[0:2, :, 3:99].transpose(0, 1), big[:, ::2, 8:104])):
        kvcache.append(w.cache, batch, k, v)
        w.plain = PlainCache(w.plain.n, 2, 16, 96)
        w.plain.append(w.table, lens, off, k.float().cpu().numpy(), v.float().cpu().numpy())
        w.check_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("out", ("float16", "bfloat16", "float32"))
def test_read_gives_the_values(dance_lib, out):
    import torch
    from dance_b200 import kvcache
    w = World([70, 3, 100], [5, 4, 100], 3, 96, 32, "bfloat16", seed=4, holes=[(2, 1)])
    batch, lens, off = w.batch()
    k, v = kvcache.read(w.cache, batch, int(off[-1]), getattr(torch, out))
    for r, (b, pos) in enumerate(places(lens, off)):
        at = w.table[b, pos // 32] if pos >= 0 else -1
        for name, t in (("k", k), ("v", v)):
            if 0 <= at < w.plain.n:
                x = (w.plain.code[name][at, :, pos % 32].astype(np.float32) * w.plain.scale[name][at][:, None])
            else:
                x = np.zeros((3, 96), np.float32)
            assert torch.equal(t[r].cpu(), torch.tensor(x).to(getattr(torch, out)))


@pytest.mark.gpu
def test_append_keeps_values_within_half_a_step(dance_lib):
    """In 64 bits: a fresh token's value is within half a scale of the input."""
    import torch
    from dance_b200 import kvcache
    w = World([130], [130], 2, 128, 64, "float16", seed=6)
    batch, _, _ = w.batch()
    x = torch.randn((130, 2, 128), device="cuda").half()
    kvcache.append(w.cache, batch, x, -x)
    k, v = kvcache.read(w.cache, batch, 130, torch.float32)
    step = w.cache.k_scale[torch.tensor(w.table[0], device="cuda").long()].repeat_interleave(64, 0)[:130, :, None]
    for got, want in ((k, x), (v, -x)):
        assert ((got.double() - want.double()).abs() <= step.double() * (0.5 + 2.0 ** -15)).all()


# ------------------------------------------------------------------ attention
SHAPES = [  # lens, new rows, kv heads, group, dim, block
    ([1], [1], 1, 1, 64, 16),
    ([333], [1], 2, 4, 128, 16),
    ([700, 1, 64, 65, 0, 129], [1, 1, 1, 1, 0, 1], 2, 8, 128, 64),
    ([95, 31, 33], [1, 1, 1], 3, 5, 96, 32),
    ([257, 140], [1, 1], 1, 16, 96, 128),
    ([300, 40], [1, 1], 1, 24, 64, 16),       # more query heads than one tile
    ([100, 65, 7], [5, 3, 7], 2, 3, 64, 32),  # drafted tokens
    ([90, 200], [40, 129], 2, 4, 128, 64),    # prompt chunks
    ([77], [77], 1, 1, 96, 16),               # a prompt from nothing
    ([130, 20], [64, 9], 1, 2, 64, 128),
    ([5, 40], [9, 3], 2, 2, 128, 32),         # four rows lie before the start and see nothing
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_against_64_bits(dance_lib, shape, dtype):
    from dance_b200 import kvcache
    lens, rows, hkv, G, dim, bs = shape
    w = World(lens, rows, hkv, dim, bs, dtype, seed=len(lens) + dim, steps=2)
    batch, lens, off = w.batch()
    q, qn = w.q(hkv * G)
    out, lse = kvcache.attention(w.cache, batch, q, return_lse=True)
    want, want_lse, err = plain_attention(w.plain, w.table, lens, off, qn.astype(np.float64), dim ** -0.5)
    check_out(out, want, err, dtype)
    check_lse(lse, want_lse, 2.0 ** -11)
    none = np.isinf(want_lse)
    assert (out.float().cpu().numpy()[none] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,rows,G", [(128, 1, 8), (96, 1, 3), (64, 6, 4), (128, 150, 2)])
def test_attention_long_in_many_splits(dance_lib, dim, rows, G):
    """One sequence, cut over the whole GPU, and a short one next to it; peaked and flat rows."""
    from dance_b200 import kvcache
    w = World([4001, 90], [rows, 1], 1, dim, 32, "float16", seed=rows, steps=1)
    batch, lens, off = w.batch()
    for size in (0.05, 1.0, 12.0):
        q, qn = w.q(G, size)
        out, lse = kvcache.attention(w.cache, batch, q, 0.3, return_lse=True)
        want, want_lse, err = plain_attention(w.plain, w.table, lens, off, qn.astype(np.float64), 0.3)
        check_out(out, want, err, "float16")
        S = 0.3 * np.abs(qn).max() * 4 * dim
        check_lse(lse, want_lse, 2.0 ** -11 + 2 * (dim + 8) * 2.0 ** -23 * S)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", (1, 70))
def test_attention_with_missing_blocks(dance_lib, rows):
    """Blocks outside the pool hold nothing, at the start, inside and at the end."""
    from dance_b200 import kvcache
    w = World([200, 200, 128], [rows, rows, rows], 2, 64, 16, "bfloat16", seed=9,
              holes=[(0, 0), (0, 5), (1, 12), (1, 3)] + [(2, j) for j in range(8)])
    batch, lens, off = w.batch()
    q, qn = w.q(4)
    out, lse = kvcache.attention(w.cache, batch, q, return_lse=True)
    want, want_lse, err = plain_attention(w.plain, w.table, lens, off, qn.astype(np.float64), 64 ** -0.5)
    check_out(out, want, err, "bfloat16")
    assert np.isneginf(lse.cpu().numpy()).any() and np.array_equal(np.isneginf(lse.cpu().numpy()), np.isinf(want_lse))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", (1, 40))
def test_attention_extreme_queries(dance_lib, rows):
    """Very large, very small, zero and mixed-size queries; a row that is not a number stays in its row."""
    import torch
    from dance_b200 import kvcache
    w = World([150], [rows], 1, 128, 64, "bfloat16", seed=11)
    batch, lens, off = w.batch()
    sizes = np.resize([1e30, 1e-30, 0.0, 1.0, 1e-3, 40.0, 1e-38, 5.0], rows * 8).reshape(rows, 8, 1)
    q, qn = w.tensor(w.rng.normal(size=(rows, 8, 128)) * sizes)
    scale = 0.1
    out, lse = kvcache.attention(w.cache, batch, q, scale, return_lse=True)
    want, want_lse, err = plain_attention(w.plain, w.table, lens, off, qn.astype(np.float64), scale)
    keep = (sizes[:, :, 0] < 100)
    check_out(out[torch.tensor(keep)], want[keep], err[keep], "bfloat16")
    # the logits of the first are so far apart that one token takes it all
    assert torch.isfinite(out).all()
    qb = q.clone()
    qb[0, 3, 7] = float("nan")
    out2 = kvcache.attention(w.cache, batch, qb, scale)
    assert torch.isnan(out2[0, 3]).all()
    same = torch.ones((rows, 8), dtype=torch.bool)
    same[0, 3] = False
    assert torch.equal(out2[same], out[same])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", (1, 33))
def test_attention_strided_unaligned_queries(dance_lib, rows):
    import torch
    from dance_b200 import kvcache
    w = World([90, 300], [rows, rows], 2, 96, 32, "float16", seed=12)
    batch, _, _ = w.batch()
    big = torch.randn((2 * rows, 7, 211), device="cuda").half()
    for q in (big[:, :6, 8:104], big[:, 1:, 5:101], big.transpose(0, 1).contiguous().transpose(0, 1)[:, :6, 16:112]):
        assert torch.equal(kvcache.attention(w.cache, batch, q), kvcache.attention(w.cache, batch, q.contiguous()))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", (1, 40))
def test_attention_repeats_bit_for_bit(dance_lib, rows):
    """Splits are joined in their order: the same call gives the same bits, whatever the workspace held before."""
    import torch
    from dance_b200 import kvcache
    w = World([5000, 900, 77], [rows, rows, rows], 2, 128, 64, "bfloat16", seed=13)
    batch, _, _ = w.batch()
    q, _ = w.q(8)
    ws = kvcache.KVWorkspace()
    first = kvcache.attention(w.cache, batch, q, workspace=ws)
    small, _ = w.q(2)
    for _ in range(5):
        kvcache.attention(w.cache, batch, small, workspace=ws)
        kvcache.select_blocks(w.cache, batch, q, 5, workspace=ws)
        assert torch.equal(kvcache.attention(w.cache, batch, q, workspace=ws), first)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(dance_lib):
    """Blocks 2.2 GB apart: addresses of blocks, codes and outputs do not wrap."""
    import torch
    from dance_b200 import kvcache
    w = World([180], [2], 2, 64, 64, "float16", seed=14)
    batch, lens, off = w.batch()
    n, block = w.cache.num_blocks, 2 * 64 * 64
    stride = 2_200_000_000 // 16 * 16
    raw = torch.empty((n - 1) * stride + 2 * block, dtype=torch.uint8, device="cuda")
    k = raw.as_strided((n, 2, 64, 64), (stride, 64 * 64, 64, 1))
    v = raw.as_strided((n, 2, 64, 64), (stride, 64 * 64, 64, 1), block)
    k.copy_(w.cache.k)
    v.copy_(w.cache.v)
    far = kvcache.KVCache(k, v, w.cache.k_scale.clone(), w.cache.v_scale.clone(), w.cache.bounds.clone())
    q, _ = w.q(4)
    assert torch.equal(kvcache.attention(far, batch, q), kvcache.attention(w.cache, batch, q))
    x = torch.randn((2, 2, 64), device="cuda").half()
    kvcache.append(far, batch, x, x)
    kvcache.append(w.cache, batch, x, x)
    assert torch.equal(far.k, w.cache.k) and torch.equal(far.v, w.cache.v)
    a, b = kvcache.read(far, batch, 2), kvcache.read(w.cache, batch, 2)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ------------------------------------------------------------------ selection
SELECTS = [  # lens, new rows, kv heads, group, dim, block, select, first, last
    ([1], [1], 1, 1, 64, 16, 1, 0, 1),
    ([700], [1], 2, 4, 128, 16, 9, 1, 1),
    ([800, 33, 0, 400], [1, 1, 0, 1], 2, 8, 96, 16, 12, 2, 3),
    ([999], [1], 1, 16, 64, 16, 20, 0, 0),
    ([640, 500], [1, 1], 3, 3, 128, 32, 30, 1, 1),   # more asked for than there is
    ([900, 300], [20, 7], 2, 3, 96, 16, 7, 1, 1),
    ([400], [90], 1, 5, 64, 16, 4, 1, 2),
    ([300], [300], 1, 2, 128, 32, 3, 1, 1),          # rows of the first blocks see fewer
    ([9, 200], [15, 2], 1, 24, 64, 16, 5, 1, 1),     # rows before the start choose nothing
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", SELECTS)
def test_selection_equals_the_definition(dance_lib, case, dtype):
    from dance_b200 import kvcache
    lens, rows, hkv, G, dim, bs, select, first, last = case
    w = World(lens, rows, hkv, dim, bs, dtype, seed=select + dim, steps=2)
    batch, lens, off = w.batch()
    q, qn = w.q(hkv * G)
    got = kvcache.select_blocks(w.cache, batch, q, select, first_blocks=first, last_blocks=last)
    want = plain_select(w.plain, w.table, lens, off, qn, select, first, last)
    assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", (1, 9))
def test_selection_ties_and_missing_blocks(dance_lib, rows):
    """All scores equal (q of zeros, and of not-a-number), negative scores, blocks without tokens last."""
    import torch
    from dance_b200 import kvcache
    w = World([640], [rows], 2, 64, 16, "float16", seed=21, holes=[(0, 3), (0, 4), (0, 17)])
    batch, lens, off = w.batch()
    q, qn = w.q(4)
    for x in (torch.zeros_like(q), torch.full_like(q, float("nan")), -q.abs(), q):
        got = kvcache.select_blocks(w.cache, batch, x, 11)
        want = plain_select(w.plain, w.table, lens, off, x.float().cpu().numpy(), 11, 1, 1)
        assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,G", [(1, 4), (12, 3)])
def test_selection_of_a_long_sequence(dance_lib, rows, G):
    """Thousands of blocks, more than one pass of any thread; odd strides of q."""
    import torch
    from dance_b200 import kvcache
    w = World([16 * 5003], [rows], 1, 64, 16, "float16", seed=22, spread=0.3)
    batch, lens, off = w.batch()
    big = torch.randn((rows, G + 1, 67), device="cuda").half()
    q = big[:, 1:, 1:65]
    for select in (1, 64, 1500, 4096):
        got = kvcache.select_blocks(w.cache, batch, q, select, first_blocks=0, last_blocks=min(select, 1))
        c = q.float().cpu().numpy()
        low, high = w.plain.low[w.table[0], 0], w.plain.high[w.table[0], 0]
        for r in range(rows):
            nb = (lens[0] - rows + r) // 16 + 1
            score = np.full(nb, -np.inf, np.float32)
            for g in range(G):
                s = plain_scale(c[r, g])
                x = plain_codes(c[r, g], s)
                dot = np.maximum(x * low[:nb], x * high[:nb]).sum(1)
                score = np.maximum(score, dot.astype(np.float32) * s)
            score = score * w.plain.scale["k"][w.table[0, :nb], 0]
            score[nb - 1] = np.inf
            best = np.sort(np.lexsort((np.arange(nb), -score))[:select])
            want = np.full(select, -1)
            want[:len(best)] = best
            assert np.array_equal(got[r, 0].cpu().numpy(), want)


# ------------------------------------------------------------------ block-sparse attention
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("select", (1, 4, 11))
def test_sparse_attention_against_64_bits(dance_lib, shape, dtype, select):
    import torch
    from dance_b200 import kvcache
    lens, rows, hkv, G, dim, bs = shape
    w = World(lens, rows, hkv, dim, bs, dtype, seed=len(lens) + dim, steps=2, holes=[(0, 0)] if lens[0] > bs else ())
    batch, lens, off = w.batch()
    q, qn = w.q(hkv * G)
    # any blocks, in any order: beyond the row's position, outside the table, none at all
    blocks = w.rng.integers(-2, w.width + 2, size=(len(qn), hkv, select))
    for r in range(len(qn)):
        for h in range(hkv):
            vals, at = np.unique(blocks[r, h], return_index=True)
            keep = np.zeros(select, bool)
            keep[at] = True
            blocks[r, h][~keep] = -1
    blocks[0, 0] = -1
    out, lse = kvcache.sparse_attention(w.cache, batch, q, torch.tensor(blocks, dtype=torch.int32, device="cuda"),
                                        return_lse=True)
    want, want_lse, err = plain_attention(w.plain, w.table, lens, off, qn.astype(np.float64), dim ** -0.5, blocks)
    check_out(out, want, err, dtype)
    check_lse(lse, want_lse, 2.0 ** -11)
    assert (out[0, :G].float() == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,bs,rows", [(128, 64, 1), (96, 16, 30), (64, 128, 3)])
def test_sparse_over_all_blocks_is_attention(dance_lib, dim, bs, rows):
    """Chosen halves joined by their log-sums, and all blocks at once, give the whole attention."""
    import torch
    from dance_b200 import kvcache
    w = World([1500], [rows], 2, dim, bs, "float16", seed=31)
    batch, lens, off = w.batch()
    q, qn = w.q(8)
    want, want_lse, err = plain_attention(w.plain, w.table, lens, off, qn.astype(np.float64), dim ** -0.5)
    nb = -(-1500 // bs)
    all_blocks = torch.arange(nb, dtype=torch.int32, device="cuda").expand(rows, 2, nb).contiguous()
    check_out(kvcache.sparse_attention(w.cache, batch, q, all_blocks), want, err, "float16")
    parts = [kvcache.sparse_attention(w.cache, batch, q, all_blocks[:, :, i::2].contiguous(), return_lse=True)
             for i in range(2)]
    lse = torch.stack([p[1].double() for p in parts])
    weight = torch.softmax(lse, 0)[..., None].nan_to_num()
    joined = (weight * torch.stack([p[0].double() for p in parts])).sum(0).cpu().numpy()
    # each part carries its own output rounding
    u = sum((weight[i] * parts[i][0].double().abs()).cpu().numpy() for i in range(2)) * 2.0 ** -11
    assert (np.abs(joined - want) <= u + 2 * err + 2.0 ** -10 * np.abs(want)).all()
    assert np.abs(torch.logsumexp(lse, 0).cpu().numpy() - want_lse).max() <= 2.0 ** -10


# ------------------------------------------------------------------ streams, graphs, empties
@pytest.mark.gpu
def test_other_stream_and_graph(dance_lib):
    import torch
    from dance_b200 import kvcache
    w = World([500, 64], [1, 1], 2, 128, 32, "float16", seed=41)
    batch, _, _ = w.batch()
    q, _ = w.q(8)
    want = kvcache.attention(w.cache, batch, q)
    blocks = kvcache.select_blocks(w.cache, batch, q, 4)
    sparse = kvcache.sparse_attention(w.cache, batch, q, blocks)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        got = kvcache.attention(w.cache, batch, q, stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    ws = kvcache.KVWorkspace()
    ws.reserve(w.cache, batch, 2, 8)
    ws.reserve(w.cache, batch, 2, 8, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = kvcache.attention(w.cache, batch, q, workspace=ws)
        c = kvcache.select_blocks(w.cache, batch, q, 4, workspace=ws)
        s = kvcache.sparse_attention(w.cache, batch, q, c, workspace=ws)
    for _ in range(3):
        a.zero_(), c.zero_(), s.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(c, blocks) and torch.equal(s, sparse)


@pytest.mark.gpu
def test_no_rows_and_lengths_changed_in_place(dance_lib):
    import torch
    from dance_b200 import kvcache
    w = World([200], [1], 1, 64, 16, "float16", seed=42)
    batch, _, _ = w.batch()
    q, _ = w.q(2)
    none = kvcache.KVBatch(batch.block_table, batch.seq_lens, torch.zeros(2, dtype=torch.int32, device="cuda"), 0, 200)
    assert kvcache.attention(w.cache, none, q[:0]).shape == (0, 2, 64)
    assert kvcache.select_blocks(w.cache, none, q[:0], 3).shape == (0, 1, 3)
    assert kvcache.read(w.cache, none, 0)[0].shape == (0, 1, 64)
    long = kvcache.attention(w.cache, batch, q)
    batch.seq_lens.fill_(80)
    short, _ = w.batch([80], [1])[0], None
    assert torch.equal(kvcache.attention(w.cache, batch, q), kvcache.attention(w.cache, short, q))
    batch.seq_lens.fill_(10 ** 9)  # longer than the table and max_len: clipped, nothing beyond is read
    assert torch.isfinite(kvcache.attention(w.cache, batch, q)).all()
    batch.seq_lens.fill_(200)
    assert torch.equal(kvcache.attention(w.cache, batch, q), long)


# ------------------------------------------------------------------ refusals
def _structs(**over):
    from dance_b200 import DanceKvBatch, DanceKvCache, DanceKvRows
    c = dict(d_k=256, d_v=256, d_k_scale=256, d_v_scale=256, d_k_bounds=256, k_block_stride=2 * 64 * 128,
             v_block_stride=2 * 64 * 128, num_blocks=4, kv_heads=2, block_tokens=64, head_dim=128)
    b = dict(d_block_table=256, d_seq_lens=256, d_row_offsets=256, table_width=4, batch=1, max_rows=1, max_len=200)
    q = dict(d_data=256, row_stride=1024, head_stride=128, rows=1, dtype=1)
    for k, v in over.items():
        for d in (c, b, q):
            if k in d:
                d[k] = v
    return DanceKvCache(**c), DanceKvBatch(**b), DanceKvRows(**q)


@pytest.mark.parametrize("over", [
    dict(head_dim=80), dict(head_dim=256), dict(block_tokens=48), dict(kv_heads=0), dict(num_blocks=0),
    dict(d_k=0), dict(d_k_scale=0), dict(d_k=264), dict(k_block_stride=2 * 64 * 128 - 16),
    dict(v_block_stride=2 * 64 * 128 + 8), dict(d_seq_lens=0), dict(d_block_table=0), dict(batch=0),
    dict(batch=65536), dict(dtype=2), dict(dtype=0), dict(d_data=0), dict(d_data=257), dict(kv_heads=3)])
def test_c_calls_refuse_before_any_device_work(dance_lib, over):
    """The pointers are never followed: this runs without a GPU."""
    c, b, q = _structs(**over)
    a = [ctypes.addressof(x) for x in (c, b, q)]
    assert dance_lib.dance_kv_attention(*a, 8, 0.1, 256, None, 256, 1 << 40, None) == -1
    assert dance_lib.dance_kv_sparse_attention(*a, 8, 256, 4, 0.1, 256, None, 256, 1 << 40, None) == -1
    assert dance_lib.dance_kv_select_blocks(*a, 8, 4, 1, 1, 256, 256, 1 << 40, None) == -1
    if "kv_heads" not in over or over["kv_heads"] == 0:
        assert dance_lib.dance_kv_append(*a, a[2], None) == -1
    assert dance_lib.dance_last_error()


def test_c_calls_refuse_outputs_workspaces_and_counts(dance_lib):
    c, b, q = _structs()
    a = [ctypes.addressof(x) for x in (c, b, q)]
    big = 1 << 40
    att, spa, sel = (dance_lib.dance_kv_attention, dance_lib.dance_kv_sparse_attention,
                     dance_lib.dance_kv_select_blocks)
    assert att(*a, 7, 0.1, 256, None, 256, big, None) == -1           # heads are no multiple
    assert att(*a, 8, 0.1, None, None, 256, big, None) == -1          # no output
    assert att(*a, 8, 0.1, 264, None, 256, big, None) == -1           # misaligned output
    assert att(*a, 8, 0.1, 256, None, None, 0, None) == -1            # no workspace
    need = dance_lib.dance_kv_workspace_bytes(a[0], a[1], 1, 8, 0)
    assert need > 0 and att(*a, 8, 0.1, 256, None, 256, need - 1, None) == -1
    assert "are needed" in dance_lib.dance_last_error().decode()
    assert spa(*a, 8, None, 4, 0.1, 256, None, 256, big, None) == -1  # no selection
    assert spa(*a, 8, 256, 0, 0.1, 256, None, 256, big, None) == -1
    assert spa(*a, 8, 256, 4097, 0.1, 256, None, 256, big, None) == -1
    assert sel(*a, 8, 3, 2, 2, 256, 256, big, None) == -1             # first and last do not fit
    assert sel(*a, 8, 4, 1, 1, None, 256, big, None) == -1
    assert dance_lib.dance_kv_read(a[0], a[1], 1, 0, 256, 256, None) == -1
    assert dance_lib.dance_kv_read(a[0], a[1], 1, 1, 264, 256, None) == -1
    assert dance_lib.dance_kv_workspace_bytes(a[0], a[1], 1, 7, 0) == 0
    # nothing to do is no error, and touches nothing
    q.rows = 0
    assert att(*a, 8, 0.1, None, None, None, 0, None) == 0


def test_python_calls_refuse_host_tensors(dance_lib):
    import torch
    from dance_b200 import kvcache
    t = torch.zeros((2, 1, 16, 64), dtype=torch.uint8)
    s, b = torch.zeros((2, 1)), torch.zeros((2, 1, 2, 64), dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        kvcache.KVCache(t, t, s, s, b)
    with pytest.raises(ValueError, match="four dimensions"):
        kvcache.KVCache(t[0], t, s, s, b)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        kvcache.KVBatch(i[None], i[:1], i, 1, 1)


@pytest.mark.gpu
def test_python_calls_refuse_wrong_tensors(dance_lib):
    import torch
    from dance_b200 import kvcache
    w = World([40], [2], 2, 64, 16, "float16", seed=51)
    batch, _, _ = w.batch()
    q, _ = w.q(4)
    c = w.cache
    for bad, error in [(q.float(), TypeError), (q[0], ValueError), (q[:, :3], ValueError), (q[:, :, ::2], ValueError),
                       (q.cpu(), ValueError), (q.transpose(0, 2), ValueError)]:
        with pytest.raises(error):
            kvcache.attention(c, batch, bad)
        with pytest.raises(error):
            kvcache.select_blocks(c, batch, bad, 2)
    blocks = torch.zeros((2, 2, 3), dtype=torch.int32, device="cuda")
    for bad, error in [(blocks.long(), TypeError), (blocks[:1], ValueError), (blocks[:, :1], ValueError),
                       (blocks[:, :, :0], ValueError), (None, ValueError)]:
        with pytest.raises(error):
            kvcache.sparse_attention(c, batch, q, bad)
    for select, first, last in [(0, 0, 0), (4097, 1, 1), (3, 2, 2), (3, -1, 1)]:
        with pytest.raises(ValueError):
            kvcache.select_blocks(c, batch, q, select, first_blocks=first, last_blocks=last)
    with pytest.raises(ValueError):
        kvcache.attention(c, batch, q, out=torch.empty((2, 4, 65), dtype=q.dtype, device="cuda"))
    with pytest.raises(ValueError):
        kvcache.append(c, batch, q[:, :2], q[:1, :2])
    with pytest.raises(ValueError):
        kvcache.KVCache(c.k.transpose(1, 2), c.v, c.k_scale, c.v_scale, c.bounds)
    with pytest.raises(TypeError):
        kvcache.KVCache(c.k, c.v, c.k_scale.double(), c.v_scale, c.bounds)
    with pytest.raises(ValueError):
        kvcache.KVCache(torch.zeros((2, 1, 16, 80), dtype=torch.uint8, device="cuda"), c.v, c.k_scale, c.v_scale,
                        c.bounds)
    with pytest.raises(TypeError):
        kvcache.KVBatch(batch.block_table.long(), batch.seq_lens, batch.row_offsets, 1, 1)
