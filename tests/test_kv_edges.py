"""The key/value cache operators where they can go wrong: codes at ties,
factors of any sign, value scales far apart, rows that see nothing of a large
value, workspaces that grow, lists that share blocks.

Expected values come from the formulas in 64 bits (or exact fractions), of the
codes and scales that the cache holds, written apart from the kernels."""
from fractions import Fraction
from pathlib import Path

import numpy as np
import pytest

import test_kvcache

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


@pytest.mark.gpu
def test_tokens_beyond_the_largest_length_are_not_visited(dance_lib):
    """Appended rows beyond max_len are dropped, read as 0; rows of no sequence keep what their place held."""
    import torch
    from dance_b200 import kvcache
    cache = kvcache.KVCache.create(6, 1, 64, 16)
    x = torch.randn((40, 1, 64), device="cuda").half() + 3
    batch = batch_of([[0, 1, 2, 3]], [50], [40], max_len=33)
    kvcache.append(cache, batch, x, x)
    k = cache.k[:, 0].cpu().numpy()
    assert (k[0, :10] == 128).all() and (k[0, 10:] != 128).any(1).all() and (k[1] != 128).any(1).all()
    assert (k[2, 0] != 128).any() and (k[2, 1:] == 128).all() and (k[3:] == 128).all()
    assert (cache.k_scale[3:] == 0).all()
    got, _ = kvcache.read(cache, batch, 40, torch.float32)
    assert (got[23:] == 0).all() and (got[:23] != 0).any(2).all()
    assert torch.allclose(got[:23], x[:23].float(), atol=0.05)
    # rows 1 and 2 of four are a sequence's
    some = kvcache.KVBatch(int32([[0, 1, 2, 3]]), int32([30]), int32([1, 3]), 2, 30)
    out = torch.full((4, 2, 64), 7.0, device="cuda").half()
    kvcache.attention(cache, some, torch.randn((4, 2, 64), device="cuda").half(), out=out)
    assert (out[0] == 7).all() and (out[3] == 7).all() and (out[1:3] != 7).all()


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


# ------------------------------------------------------------------ the twin on the host, by the step
class StepCache(test_kvcache.PlainCache):
    """The cache on the host with codes at the step: half of a block's largest magnitude, an exact 63.5, is 64."""

    def append(self, table, lens, offsets, k, v):
        quotient, codes = test_kvcache.plain_scale, test_kvcache.plain_codes
        for b, n in enumerate(lens):
            first = n - (offsets[b + 1] - offsets[b])
            for page in range(max(first, 0) // self.bs, -(-n // self.bs) if n > 0 else 0):
                lo, hi = max(first, 0, page * self.bs), min(n, (page + 1) * self.bs)
                at = table[b][page] if page < len(table[b]) else -1
                if hi <= lo or not 0 <= at < self.n:
                    continue
                begun, end = lo - page * self.bs, hi - page * self.bs
                for h in range(self.hkv):
                    for name, x in (("k", k), ("v", v)):
                        new = x[offsets[b] + lo - first:offsets[b] + hi - first, h]
                        old = self.scale[name][at, h] if begun else np.float32(0)
                        largest = quotient(new)
                        step = old if old > largest else step_of(new)
                        c, ends = self.code[name][at, h], np.stack((self.low[at, h], self.high[at, h]))
                        if begun and largest > old:
                            c[:begun] = np.rint(c[:begun].astype(np.float32) * (old / step))
                            ends = np.rint(ends.astype(np.float32) * (old / step)).astype(np.int64)
                        c[begun:end] = codes(new, step)
                        self.scale[name][at, h] = max(old, largest)
                        if name == "k":
                            low, high = c[begun:end].min(0), c[begun:end].max(0)
                            self.low[at, h] = np.minimum(ends[0], low) if begun else low
                            self.high[at, h] = np.maximum(ends[1], high) if begun else high


def step_of(x):
    """The step of a set of values: the largest finite |x| times the float nearest 1/127."""
    a = np.abs(x[np.isfinite(x)])
    s = np.float32(a.max() if a.size else 0.0) * STEP
    return np.float32(0.0) if s < np.float32(2.0 ** -126) else s


@pytest.fixture
def twin(monkeypatch):
    monkeypatch.setattr(test_kvcache, "PlainCache", StepCache)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,bs", [(64, 16), (96, 32), (128, 64), (64, 128), (128, 16), (96, 128)])
def test_append_equals_the_twin(dance_lib, twin, dim, bs, dtype):
    test_kvcache.test_append_equals_the_definition(dance_lib, dim, bs, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_of_odd_values_equals_the_twin(dance_lib, twin, dtype):
    test_kvcache.test_append_odd_values(dance_lib, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("check", [
    test_kvcache.test_append_strided_and_unaligned, test_kvcache.test_append_outside_the_table_and_before_the_start])
def test_append_beside_the_twin(dance_lib, twin, check):
    for _ in range(4):
        check(dance_lib)


@pytest.mark.gpu
def test_append_token_by_token_equals_the_twin(dance_lib, twin):
    test_kvcache.test_append_token_by_token(dance_lib)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", test_kvcache.SHAPES)
def test_attention_over_the_twin(dance_lib, twin, shape, dtype):
    test_kvcache.test_attention_against_64_bits(dance_lib, shape, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", test_kvcache.SHAPES)
@pytest.mark.parametrize("select", (4, 11))
def test_sparse_attention_over_the_twin(dance_lib, twin, shape, dtype, select):
    test_kvcache.test_sparse_attention_against_64_bits(dance_lib, shape, dtype, select)


class QuotientFirst(StepCache):
    """StepCache where the module's scale of a set of values is the step, as a query's is."""

    def append(self, *args):
        with pytest.MonkeyPatch.context() as m:
            m.setattr(test_kvcache, "plain_scale", PLAIN_SCALE)
            super().append(*args)


PLAIN_SCALE = test_kvcache.plain_scale


@pytest.fixture
def select_twin(monkeypatch):
    monkeypatch.setattr(test_kvcache, "PlainCache", QuotientFirst)
    monkeypatch.setattr(test_kvcache, "plain_scale", step_of)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", test_kvcache.SELECTS)
def test_selection_equals_the_twin(dance_lib, select_twin, case, dtype):
    test_kvcache.test_selection_equals_the_definition(dance_lib, case, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,G", [(1, 4), (12, 3)])
def test_selection_of_a_long_sequence_equals_the_twin(dance_lib, select_twin, rows, G):
    for _ in range(4):
        test_kvcache.test_selection_of_a_long_sequence(dance_lib, rows, G)


# ------------------------------------------------------------------ attention
class Held:
    """A cache of given codes and scales, with the attention over it in 64 bits."""

    def __init__(self, lens, rows, hkv, dim, bs, dtype, seed, k_scale=None, v_scale=None, table=None):
        import torch
        from dance_b200 import kvcache
        rng = self.rng = np.random.default_rng(seed)
        self.lens, self.rows, self.hkv, self.dim, self.bs, self.dtype = lens, rows, hkv, dim, bs, dtype
        need = [-(-n // bs) for n in lens]
        pool, width = sum(need) + 2, max(need)
        ids = rng.permutation(pool)
        self.table = np.full((len(lens), width), -1)
        for b, n in enumerate(need):
            self.table[b, :n] = ids[sum(need[:b]):sum(need[:b + 1])]
        self.k = rng.integers(-127, 128, (pool, hkv, bs, dim))
        self.v = rng.integers(-127, 128, (pool, hkv, bs, dim))
        self.ks = np.full((pool, hkv), 0.02, np.float32) if k_scale is None else k_scale(self, pool)
        self.vs = np.full((pool, hkv), 0.01, np.float32) if v_scale is None else v_scale(self, pool)
        dev = [torch.tensor(x + 128, dtype=torch.uint8, device="cuda") for x in (self.k, self.v)]
        bounds = torch.stack((dev[0].amin(2), dev[0].amax(2)), 2).contiguous()
        self.cache = kvcache.KVCache(dev[0], dev[1], torch.tensor(self.ks, device="cuda"),
                                     torch.tensor(self.vs, device="cuda"), bounds)
        self.batch = batch_of(self.table, lens, rows)

    def q(self, heads, size=1.0):
        import torch
        t = torch.tensor(self.rng.normal(size=(sum(self.rows), heads, self.dim)) * size, device="cuda")
        t = t.to(getattr(torch, self.dtype))
        return t, t.double().cpu().numpy()

    def attention(self, q, scale, blocks=None):
        """(out, lse, allowed error without the output's rounding, the lse's) in 64 bits.

        Allowed: the weights' rounding to halves (2^-11), the logits' (products of D terms in float, S the largest sum
        of magnitudes), 2^x and the sums in float (2^-19), each of sum_j p_j |v_j|; and what weights below a half's
        range lose, 2^-30 of the row's largest p_j times its block's largest value, for each token."""
        T, H, D = q.shape
        G, bs = H // self.hkv, self.bs
        out, lse, err = np.zeros((T, H, D)), np.full((T, H), -np.inf), np.zeros((T, H, D))
        lse_err, r0 = np.zeros((T, H)), 0
        for b, n in enumerate(self.lens):
            rows, pages = self.rows[b], -(-n // bs)
            at, place = self.table[b, :pages], np.arange(pages * bs)
            for h in range(self.hkv):
                times = np.ones((rows, pages)) if blocks is None else np.array(
                    [[np.sum(blocks[r, h] == j) for j in range(pages)] for r in range(r0, r0 + rows)])
                times = times.repeat(bs, 1) * (place <= n - rows + np.arange(rows)[:, None])  # how often a row sees a token
                k = (self.k[at, h] * self.ks[at, h].astype(np.float64)[:, None, None]).reshape(-1, D)
                v = (self.v[at, h] * self.vs[at, h].astype(np.float64)[:, None, None]).reshape(-1, D)
                top = np.repeat(127 * self.vs[at, h].astype(np.float64), bs)
                for g in range(h * G, (h + 1) * G):
                    mine = slice(r0, r0 + rows)
                    x = np.where(times > 0, scale * (q[mine, g] @ k.T), -np.inf)
                    S = abs(scale) * np.where(times > 0, np.abs(q[mine, g]) @ np.abs(k).T, 0).max(1)
                    most = x.max(1)
                    p = times * np.exp(x - np.where(np.isinf(most), 0, most)[:, None])
                    total = p.sum(1)
                    some = total > 0
                    lse[mine, g][some] = (most + np.log(np.where(some, total, 1)))[some]
                    p /= np.where(some, total, 1)[:, None]
                    out[mine, g] = p @ v
                    lse_err[mine, g] = 2.0 ** -11 + 2 * (D + 8) * 2.0 ** -23 * S
                    err[mine, g] = ((2.0 ** -11 + 2 * (D + 8) * 2.0 ** -23 * S + 2.0 ** -19)[:, None] * (p @ np.abs(v))
                                    + (times.sum(1) * 2.0 ** -30 * (p * top).max(1))[:, None])
            r0 += rows
        return out, lse, err, lse_err


def check_out(got, want, err, dtype):
    u = 2.0 ** -11 if dtype == "float16" else 2.0 ** -8
    # float16 has no numbers below 2^-24
    err = err + (2.0 ** -25 if dtype == "float16" else 0.0)
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    excess = np.abs(got - want) - (u * np.abs(want) + err)
    at = np.unravel_index(excess.argmax(), excess.shape)
    assert excess.max() <= 0, f"{at}: {got[at]} where {want[at]} +- {err[at]} is right"


def check_lse(got, want, err):
    got = got.double().cpu().numpy()
    none = np.isinf(want)
    assert np.array_equal(np.isneginf(got), none)
    assert (np.abs(got[~none] - want[~none]) <= err[~none]).all()


ROWS = (1, 5, 40, 300)  # of a sequence: few rows, drafts, one row tile, two


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("scale", (-0.1, 0.0, 0.1, -3.0))
def test_attention_factor_of_any_sign(dance_lib, rows, scale, dtype):
    from dance_b200 import kvcache
    w = Held([700, 333], [rows, 1], 1, 128, 64, dtype, seed=rows)
    q, qn = w.q(2)
    out, lse = kvcache.attention(w.cache, w.batch, q, scale, return_lse=True)
    want, want_lse, err, lse_err = w.attention(qn, scale)
    check_out(out, want, err, dtype)
    check_lse(lse, want_lse, lse_err)


def far_apart(power, where):
    """Value scales 0.01, and 2^power times that in the blocks of the first sequence that `where` names."""
    def make(w, pool):
        s = np.full((pool, w.hkv), 0.01, np.float32)
        s[w.table[0, where]] *= np.float32(2.0 ** power)
        return s
    return make


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dtype,power", [("float16", 15), ("float16", -16), ("bfloat16", 24), ("bfloat16", 34),
                                         ("bfloat16", 90), ("bfloat16", -24), ("bfloat16", -100)])
def test_attention_value_scales_far_apart(dance_lib, rows, dtype, power):
    """One block's values are larger or smaller than the others' by a power of two; rows weigh it much and little."""
    from dance_b200 import kvcache
    w = Held([700, 65], [rows, 1], 1, 128, 64, dtype, seed=3, v_scale=far_apart(power, 4))
    for size in (0.3, 2.0, 20.0):
        q, qn = w.q(2, size)
        out, lse = kvcache.attention(w.cache, w.batch, q, 0.1, return_lse=True)
        want, want_lse, err, lse_err = w.attention(qn, 0.1)
        check_out(out, want, err, dtype)
        check_lse(lse, want_lse, lse_err)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS[1:])
@pytest.mark.parametrize("dtype,power", [("float16", 15), ("bfloat16", 20), ("bfloat16", 34), ("bfloat16", 90)])
def test_rows_do_not_depend_on_values_they_may_not_see(dance_lib, rows, dtype, power):
    """The last block's values are far larger: rows before it give what they give where it is like the others."""
    import torch
    from dance_b200 import kvcache
    outs, bs, last = [], 16, 2
    lens = [19 * bs + last]
    for p in (0, power):
        w = Held(lens, [rows], 4, 96, bs, dtype, seed=5, v_scale=far_apart(p, -1))
        q, qn = w.q(8)
        outs.append(kvcache.attention(w.cache, w.batch, q, 0.1))
        check_out(outs[-1], *w.attention(qn, 0.1)[::2], dtype)
    assert torch.equal(outs[0][:rows - last], outs[1][:rows - last])
    # adjacent rows that choose apart: only some of them the large block
    blocks = np.full((rows, 4, 3), -1)
    blocks[:, :, 0] = np.arange(rows)[:, None] % 3
    blocks[1::2, :, 1] = 19
    out = kvcache.sparse_attention(w.cache, w.batch, q, int32(blocks), 0.1)
    check_out(out, *w.attention(qn, 0.1, blocks)[::2], dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", (1, 40))
def test_scales_without_an_inverse(dance_lib, rows):
    """Blocks whose scales have no finite inverse: new rows become 0, attention stays finite."""
    import torch
    from dance_b200 import kvcache
    w = Held([320], [rows], 1, 64, 32, "bfloat16", seed=2, k_scale=far_apart(-126, 3), v_scale=far_apart(-126, 3))
    assert 0 < w.ks.min() < 2.0 ** -126
    q, qn = w.q(2)
    out, lse = kvcache.attention(w.cache, w.batch, q, 0.1, return_lse=True)
    want, want_lse, err, lse_err = w.attention(qn, 0.1)
    check_out(out, want, err, "bfloat16")
    check_lse(lse, want_lse, lse_err)
    x = torch.zeros((8, 1, 64), dtype=torch.bfloat16, device="cuda")
    x[1::2] = 2.0 ** -130
    kvcache.append(w.cache, batch_of(w.table, [3 * 32 + 10], [8]), x, x)
    for t in (w.cache.k, w.cache.v):
        assert (t[int(w.table[0, 3]), 0, 2:10] == 128).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("size", (1e6, 1e7, 3e7, 1e8, 3e8, 1e12, 1e30))
def test_attention_far_logits(dance_lib, rows, size):
    """Logits of a million and more: one token takes all where it leads by more than the logits' error; its values are
    the output."""
    from dance_b200 import kvcache
    w = Held([700], [rows], 1, 128, 64, "bfloat16", seed=rows, v_scale=far_apart(20, 4))
    q, qn = w.q(2, size)
    out, lse = kvcache.attention(w.cache, w.batch, q, 0.1, return_lse=True)
    got, clear = out.double().cpu().numpy(), 0
    assert np.isfinite(got).all() and np.isfinite(lse.cpu().numpy()).all()
    at = w.table[0]
    k = (w.k[at, 0] * w.ks[at, 0].astype(np.float64)[:, None, None]).reshape(-1, 128)
    v = (w.v[at, 0] * w.vs[at, 0].astype(np.float64)[:, None, None]).reshape(-1, 128)
    for r in range(rows):
        n = 700 - rows + r + 1
        for g in range(2):
            x = 0.1 * (k[:n] @ qn[r, g])
            first, second = np.argsort(-x)[:2]
            error = 2 * (128 + 8) * 2.0 ** -23 * 0.1 * (np.abs(k[:n]) @ np.abs(qn[r, g])).max()
            if x[first] - x[second] > 2 * error + 60:
                clear += 1
                want = v[first]
                assert (np.abs(got[r, g] - want) <= (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -19) * np.abs(want)).all()
    assert clear > rows


# ------------------------------------------------------------------ rows that share their chosen blocks
def lists(kind, rows, heads, select, pages, rng):
    """Block lists of adjacent rows: alike, apart, out of order, with repeats, with places past the end."""
    out = np.full((rows, heads, select), -1)
    common = rng.permutation(pages)[:select]
    for r in range(rows):
        for h in range(heads):
            mine = rng.permutation(pages)[:select]
            take = common if kind == "same" else np.where(rng.random(len(mine)) < 0.5, common[:len(mine)], mine)
            got = np.unique(take)
            if kind == "short":
                got = got[:rng.integers(0, len(got) + 1)]
            if kind == "unsorted":
                got = rng.permutation(got)
            if kind == "twice":
                got = np.concatenate([got, got])[:select]
            if kind == "outside":
                got = np.concatenate([got[:select - 2], [pages + 3, 1 << 30]])
            out[r, h, :len(got)] = got
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ("same", "apart", "short", "unsorted", "twice", "outside"))
@pytest.mark.parametrize("G,dim,bs,select,rows", [
    (1, 64, 16, 7, 301), (2, 128, 64, 11, 299), (3, 96, 16, 5, 333), (4, 64, 32, 60, 301), (1, 128, 128, 32, 300)])
def test_sparse_attention_of_adjacent_rows(dance_lib, kind, G, dim, bs, select, rows):
    """Hundreds of rows over four heads: a thread block takes several tokens (8 / G, a last group of fewer)."""
    from dance_b200 import kvcache
    pages = max(select + 3, 9)
    w = Held([pages * bs - 3], [rows], 4, dim, bs, "float16", seed=G + select)
    table = w.table.copy()
    table[0, 1] = -1 if G % 2 else 10 ** 6  # a block that holds nothing
    w.batch = batch_of(table, w.lens, w.rows)
    blocks = lists(kind, rows, 4, select, pages, w.rng)
    q, qn = w.q(4 * G)
    out, lse = kvcache.sparse_attention(w.cache, w.batch, q, int32(blocks), 0.1, return_lse=True)
    blocks[blocks == 1] = -1
    want, want_lse, err, lse_err = w.attention(qn, 0.1, blocks)
    check_out(out, want, err, "float16")
    check_lse(lse, want_lse, lse_err)
    assert kind != "short" or np.isinf(want_lse).any()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,G,blocks", [(1, 2, 9729), (3, 1, 20001), (2, 3, 9728)])
def test_selection_of_more_blocks_than_shared_memory_holds(dance_lib, rows, G, blocks):
    """Scores read from memory in every cut; and the most that shared memory holds."""
    import torch
    from dance_b200 import kvcache
    rng = np.random.default_rng(blocks)
    low = rng.integers(-127, 20, (blocks, 64))
    high = low + rng.integers(0, 107, (blocks, 64))
    ks = rng.choice(np.array([0.01, 0.02, 0.03], np.float32), (blocks, 1))
    code = torch.full((blocks, 1, 16, 64), 128, dtype=torch.uint8, device="cuda")
    bounds = torch.tensor(np.stack((low, high), 1)[:, None] + 128, device="cuda").to(torch.uint8)
    scale = torch.tensor(ks, device="cuda")
    cache = kvcache.KVCache(code, code, scale, scale, bounds)
    q = torch.tensor(rng.normal(size=(rows, G, 64)), device="cuda").half()
    batch = batch_of([np.arange(blocks)], [16 * blocks], [rows])
    for select, first, last in ((1, 0, 0), (64, 1, 1), (4096, 3, 5)):
        got = kvcache.select_blocks(cache, batch, q, select, first_blocks=first, last_blocks=last).cpu().numpy()
        for r in range(rows):
            score = np.full(blocks, -np.inf, np.float32)
            for g in range(G):
                x = q[r, g].float().cpu().numpy()
                s = step_of(x)
                c = np.rint(x * (np.float32(1) / s)).astype(np.int64)
                score = np.maximum(score, np.maximum(c * low, c * high).sum(1).astype(np.float32) * s)
            score = score * ks[:, 0]
            score[:first] = np.inf
            score[blocks - last:] = np.inf
            assert np.array_equal(got[r, 0], np.sort(np.lexsort((np.arange(blocks), -score))[:select]))


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


# ------------------------------------------------------------------ several devices
FAKE_RUNTIME = r'''
#include "func_attr.cuh"
#include <cstdio>
static int device, fails, asked[2];
extern "C" cudaError_t cudaGetDevice(int *d) { *d = device; return cudaSuccess; }
extern "C" cudaError_t cudaFuncSetAttribute(const void *, cudaFuncAttribute, int bytes)
{
    ++asked[device];
    return fails && fails-- ? cudaErrorInvalidValue : bytes == 70000 ? cudaSuccess : cudaErrorUnknown;
}
int main()
{
    static dance::SmemAllowed a;
    fails = 1;
    const cudaError_t first = a.on_current(nullptr, 70000), second = a.on_current(nullptr, 70000);
    cudaError_t later = a.on_current(nullptr, 70000);
    device = 1;
    const cudaError_t other = a.on_current(nullptr, 70000);
    for (device = 0; device < 2; ++device)
        later = a.on_current(nullptr, 70000);
    printf("%d %d %d %d %d %d\n", first != cudaSuccess, second, other, later, asked[0], asked[1]);
}
'''


def test_shared_memory_is_asked_for_on_every_device(tmp_path):
    """Against a fake of the runtime with two devices: once on each, again after a failure."""
    import shutil
    import subprocess
    from dance_b200 import build
    nvcc = build.nvcc()
    root = Path(shutil.which(nvcc) or nvcc).resolve().parent.parent
    (tmp_path / "t.cpp").write_text("#include <cuda_runtime_api.h>\n" + FAKE_RUNTIME)
    exe = tmp_path / "t"
    subprocess.run(["g++", "-std=c++17", "-I", str(root / "include"), "-I", str(build.CSRC), str(tmp_path / "t.cpp"),
                    "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split() == list("100021")


def test_no_attribute_is_remembered_for_the_process():
    from dance_b200 import build
    for src in build.SOURCES:
        text = (build.CSRC / src).read_text()
        assert "static const cudaError_t" not in text, src


@pytest.mark.gpu
def test_attention_on_a_second_device(dance_lib):
    import torch
    from dance_b200 import kvcache
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    for rows in (1, 40):
        outs = []
        for dev in (0, 1):
            with torch.cuda.device(dev):
                w = Held([300], [rows], 1, 128, 64, "float16", seed=rows)
                q, _ = w.q(2)
                outs.append(kvcache.attention(w.cache, w.batch, q).cpu())
        assert torch.equal(*outs)


# ------------------------------------------------------------------ waits that run out
@pytest.mark.gpu
@pytest.mark.parametrize("tokens", (700, 30000))
def test_waits_that_run_out_are_told(dance_lib, monkeypatch, tokens):
    """With a limit of nothing the blocks give up and say so; the calls after it are whole again."""
    import torch
    from dance_b200 import DanceError, kvcache
    cache, _, _ = decode_step(tokens)
    batch = batch_of([list(range(cache.num_blocks))], [tokens], [300])
    q = torch.randn((300, 8, 64), device="cuda").half()
    ws = kvcache.KVWorkspace()
    want, lse = kvcache.attention(cache, batch, q, return_lse=True, workspace=ws)
    kvcache.status()
    assert torch.isfinite(want).all()
    monkeypatch.setenv("DANCE_KV_WAIT_CLOCKS", "0")
    out = kvcache.attention(cache, batch, q, workspace=ws)
    with pytest.raises(DanceError, match="gave up waiting"):
        kvcache.status()
    assert torch.isnan(out).any()
    kvcache.status()  # told once
    monkeypatch.delenv("DANCE_KV_WAIT_CLOCKS")
    again, lse_again = kvcache.attention(cache, batch, q, return_lse=True, workspace=ws)
    kvcache.status()
    assert torch.equal(again, want) and torch.equal(lse_again, lse)
