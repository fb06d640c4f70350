"""Cases of the key/value cache operators: append and read, attention, block selection, block-sparse attention.

The cache holds 8-bit codes c in 1..255 standing for (c - 128) * scale, with one float32 scale for each block of
`block` tokens and key/value head, keys and values apart; a sequence's blocks are named by its row of a block table.
A batch names its sequences' lengths after the new rows and their new rows (row offsets); row i of a sequence with
r new rows and length n has position n - r + i and sees positions up to its own.

* append: the new rows' keys and values enter the cache.  A block's scale is max(its scale so far, the largest finite
  |x| of its new rows / 127); where it grows, the block's earlier codes are rounded again to the new scale.  With the
  keys, each block keeps the smallest and the largest code of every channel (its bounds).  The case reads the touched
  blocks' tokens back as the values that they stand for.
* attention: softmax(scale * q k) v over the sequence, heads / kv_heads query heads to one key/value head.
* select: each row and key/value head takes `select` blocks: the first and the last that it sees, the rest by the
  largest score, the largest over its query heads of sum_d max(c_d * low_d, c_d * high_d), where c is the head's query
  in 8 bits and low, high the block's bounds: an upper bound of the logits in the block.  The score's sum is an integer,
  so the order does not depend on how it is summed; ties go to the lowest block.  Blocks ascend; -1 fills.
* sparse: attention over the tokens of the selected blocks.
"""
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
TINY = 2.0 ** -126


def _case(name, op, dtype, batch, heads, kv_heads, dim, block, rows, length, ragged, select=0):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "block": block, "rows": rows, "length": length, "ragged": ragged, "select": select}


def listed():
    return [
        # one new token of each of 64 conversations: the write of every decode step
        _case("append_step", "append", "bf16", 64, 8, 8, 128, 64, 1, 8000, True),
        # three documents enter the cache whole, their lengths not multiples of the block
        _case("append_prompt", "append", "f16", 3, 8, 8, 96, 32, 9001, 9001, True),
        # the smallest call: one short conversation on few heads, where latency counts
        _case("attend_short", "attention", "bf16", 1, 8, 2, 128, 16, 1, 333, False),
        # an ordinary decode step of a busy server
        _case("attend_step", "attention", "bf16", 96, 32, 8, 128, 64, 1, 8192, True),
        # one reader of a very long document: the cache's offsets pass 31 bits
        _case("attend_long", "attention", "f16", 1, 64, 8, 128, 64, 1, 2200003, False),
        # a few drafted tokens of each conversation are checked at once; three query heads to one
        _case("attend_draft", "attention", "f16", 24, 12, 4, 64, 32, 5, 6000, True),
        # prompt chunks that follow what the cache holds
        _case("attend_prompt", "attention", "bf16", 2, 32, 8, 128, 64, 2048, 16000, True),
        # decode over long memories: which blocks each conversation's token reads
        _case("select_step", "select", "bf16", 32, 32, 8, 128, 64, 1, 120000, True, 64),
        # a question's tokens choose the blocks of one long document
        _case("select_prompt", "select", "f16", 1, 24, 8, 96, 32, 700, 65537, False, 48),
        # and the attention over what was chosen, for single tokens
        _case("sparse_step", "sparse", "bf16", 32, 32, 8, 128, 64, 1, 120000, True, 64),
        # and for a prompt's
        _case("sparse_prompt", "sparse", "f16", 1, 24, 8, 96, 32, 700, 65537, False, 48),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    op = rng.choice(("append", "attention", "select", "sparse"))
    dim, block = rng.choice((64, 96, 128)), rng.choice((16, 32, 64))
    kv_heads, group = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 3, 4, 5, 8, 16))
    dtype, ragged = rng.choice(("bf16", "f16")), rng.random() < 0.7
    if op == "append":
        rows = 1 if rng.random() < 0.5 else spread(2, 8000)
        batch = spread(1, max(1, min(128, 32000 // rows)))
        length = max(rows, spread(1, 16000))
        return _case("", op, dtype, batch, kv_heads, kv_heads, dim, block, rows, length, ragged) | {"name": "drawn"}
    if rng.random() < 0.55:
        rows, length = 1, spread(100, 150000)
        batch = spread(1, max(1, min(100, 600000 // length)))
    else:
        length = spread(1500, 40000)
        most = 700 if op != "attention" else 1000000000 // (length * kv_heads * group)
        rows = spread(2, min(1500, most))
        batch = 1 if op != "attention" else spread(1, max(1, min(8, most // rows)))
    select = spread(2, 64) if op in ("sparse", "select") else 0
    return _case("drawn", op, dtype, batch, kv_heads * group, kv_heads, dim, block, rows, length, ragged, select)


def _lengths(case):
    """(lengths, new rows) of the sequences: of the case alone."""
    n, r, b = case["length"], case["rows"], case["batch"]
    if not case["ragged"]:
        return [n] * b, [r] * b
    rng = random.Random(n * 1000003 + r * 10007 + b * 101 + case["dim"])
    rows = [r] + [1 + int(rng.random() * r) for _ in range(b - 1)]
    lens = [n] + [max(rows[i + 1], int(n * (0.1 + 0.9 * rng.random()))) for i in range(b - 1)]
    return lens, [min(x, y) for x, y in zip(rows, lens)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed) + 7)
    op, block, dim, hkv, heads = case["op"], case["block"], case["dim"], case["kv_heads"], case["heads"]
    dtype, dev = TYPES[case["dtype"]], "cuda"
    lens, rows = _lengths(case)
    B, T = len(lens), sum(rows)
    need = [-(-n // block) for n in lens]
    width, pool = max(need), sum(need) + 3
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32, device=dev)
    at = 0
    for b in range(B):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]

    def codes():
        # channels of a block share a direction, as neighbouring tokens do
        x = torch.empty((pool, hkv, block, dim), dtype=torch.uint8, device=dev)
        for i in range(0, pool, 2048):
            m = min(2048, pool - i)
            y = torch.randn((m, hkv, block, dim), generator=g, device=dev).mul_(26)
            y += torch.randn((m, hkv, 1, dim), generator=g, device=dev).mul_(15)
            x[i:i + m] = y.round_().clamp_(-127, 127).add_(128).to(torch.uint8)
        return x

    def scales(mean):
        return torch.randn((pool, hkv), generator=g, device=dev).mul_(0.3).exp_().mul_(mean)

    k = codes()
    v = k if op == "select" else codes()
    k_scale, v_scale = scales(0.04), scales(0.02)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device=dev)
    offsets = torch.tensor([0] + [sum(rows[:i + 1]) for i in range(B)], dtype=torch.int32, device=dev)
    # the bounds of a block are those of its tokens within the sequence
    held = torch.full((pool,), block, dtype=torch.int32, device=dev)
    before = [n - r for n, r in zip(lens, rows)] if op == "append" else lens
    for b in range(B):
        if before[b] % block:
            held[table[b, before[b] // block].long()] = before[b] % block
    bounds = torch.empty((pool, hkv, 2, dim), dtype=torch.uint8, device=dev)
    out_of = torch.arange(block, device=dev)[None, :] >= held[:, None]
    for i in range(0, pool, 4096):
        m = out_of[i:i + 4096, None, :, None]
        bounds[i:i + 4096, :, 0] = k[i:i + 4096].masked_fill(m, 255).amin(2)
        bounds[i:i + 4096, :, 1] = k[i:i + 4096].masked_fill(m, 0).amax(2)
    s = {"case": case, "k": k, "v": v, "k_scale": k_scale, "v_scale": v_scale, "bounds": bounds, "table": table,
         "lens": seq_lens, "offsets": offsets, "rows": T, "max_rows": max(rows), "max_len": max(lens),
         "scale": dim ** -0.5}
    if op == "append":
        s["k_new"] = torch.randn((T, hkv, dim), generator=g, device=dev).mul_(1.2).to(dtype)
        s["v_new"] = torch.randn((T, hkv, dim), generator=g, device=dev).mul_(0.7).to(dtype)
        back = [r + (n - r) % block for n, r in zip(lens, rows)]
        s["back_offsets"] = torch.tensor([0] + [sum(back[:i + 1]) for i in range(B)], dtype=torch.int32, device=dev)
        s["back_rows"], s["back_max"] = sum(back), max(back)
    else:
        s["q"] = torch.randn((T, heads, dim), generator=g, device=dev).mul_(1.5).to(dtype)
    if op == "sparse":
        s["blocks"] = _blocks(s, g)
    if own:
        from dance_b200 import kvcache
        s["cache"] = kvcache.KVCache(k, v, k_scale, v_scale, bounds)
        s["batch"] = kvcache.KVBatch(table, seq_lens, offsets, s["max_rows"], s["max_len"])
        if op == "append":
            s["back"] = kvcache.KVBatch(table, seq_lens, s["back_offsets"], s["back_max"], s["max_len"])
        s["workspace"] = kvcache.KVWorkspace()
    return s


def _blocks(s, g):
    """Chosen blocks as neighbouring rows choose them: much alike, the last always among them; some rows come up short."""
    case = s["case"]
    seq, pos = _row_places(s)
    seen = pos.div(case["block"], rounding_mode="floor") + 1
    B, W, hkv, n = s["table"].shape[0], s["table"].shape[1], case["kv_heads"], case["select"]
    score = torch.rand((B, hkv, W), generator=g, device="cuda")[seq]
    score += 0.3 * torch.rand(score.shape, generator=g, device="cuda")
    at = torch.arange(W, device="cuda")
    score = score.masked_fill(at == seen[:, None, None] - 1, 9.0).masked_fill(at >= seen[:, None, None], -9.0)
    got = score.topk(min(n, W), dim=2)
    keep = got.indices.masked_fill(got.values < 0, W).sort(dim=2).values
    blocks = torch.full((s["rows"], hkv, n), -1, dtype=torch.int32, device="cuda")
    blocks[:, :, :keep.shape[2]] = keep.masked_fill(keep == W, -1).to(torch.int32)
    return blocks


def run(s):
    return _run_own(s) if own else _PLAIN[s["case"]["op"]](s)


def _run_own(s):
    from dance_b200 import kvcache
    op, case = s["case"]["op"], s["case"]
    if op == "append":
        kvcache.append(s["cache"], s["batch"], s["k_new"], s["v_new"])
        k, v = kvcache.read(s["cache"], s["back"], s["back_rows"], s["k_new"].dtype)
        return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"], "bounds": s["bounds"]}
    if op == "attention":
        return kvcache.attention(s["cache"], s["batch"], s["q"], s["scale"], workspace=s["workspace"])
    if op == "select":
        return kvcache.select_blocks(s["cache"], s["batch"], s["q"], case["select"], workspace=s["workspace"])
    return kvcache.sparse_attention(s["cache"], s["batch"], s["q"], s["blocks"], s["scale"], workspace=s["workspace"])


# ------------------------------------------------------------------ plain forms
def _row_places(s, offsets=None, rows=None):
    """The sequence and the position of every row."""
    off = (s["offsets"] if offsets is None else offsets).long()
    rows = s["rows"] if rows is None else rows
    i = torch.arange(rows, device=off.device)
    seq = torch.searchsorted(off, i, right=True) - 1
    return seq, s["lens"].long()[seq] - off[seq + 1] + i


def _values(codes, scale):
    return (codes.float() - 128.0) * scale


def _quantised(x, scale):
    """Codes - 128 of x at a scale."""
    inv = torch.where(scale > 0, 1.0 / scale, 0.0)
    return (x * inv).nan_to_num(nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127, 127)


def _append(s):
    case = s["case"]
    bs, hkv, dim = case["block"], case["kv_heads"], case["dim"]
    off, lens, table = s["offsets"].long(), s["lens"].long(), s["table"].long()
    B = lens.shape[0]
    first = lens - (off[1:] - off[:-1])  # position of the first new row
    J = (s["max_rows"] + bs - 2) // bs + 1
    j = first[:, None] // bs + torch.arange(J, device=off.device)
    used = j * bs < lens[:, None]
    blk = table.gather(1, j.clamp(max=table.shape[1] - 1))
    pos = j[:, :, None] * bs + torch.arange(bs, device=off.device)
    fresh = (pos >= first[:, None, None]) & (pos < lens[:, None, None])
    older = pos < first[:, None, None]
    src = (off[:-1, None, None] + pos - first[:, None, None]).clamp(0, s["rows"] - 1)
    blk_ids = blk[used]
    for name in ("k", "v"):
        x = s[name + "_new"].float()[src]  # B, J, bs, hkv, dim
        x = torch.where(fresh[..., None, None], x, 0.0).permute(0, 1, 3, 2, 4)[used]
        f, o = fresh[used][:, None, :, None], older[used][:, None, :, None]
        size = torch.where(x.isfinite(), x.abs(), 0.0).amax((2, 3))
        new = size / 127.0
        new = torch.where(new < TINY, 0.0, new)
        old = torch.where(o.any(2)[:, :, 0], s[name + "_scale"][blk_ids], 0.0)
        scale = torch.maximum(old, new)
        codes = s[name][blk_ids].float() - 128.0
        shrink = torch.where(scale > 0, old / scale, 0.0)[:, :, None, None]
        codes = torch.where(o, (codes * shrink).round(), codes)
        codes = torch.where(f, _quantised(x, scale[:, :, None, None]), codes) + 128.0
        s[name][blk_ids] = codes.to(torch.uint8)
        s[name + "_scale"][blk_ids] = scale
        if name == "k":
            live = f | o
            low = torch.where(live, codes, 255.0).amin(2)
            high = torch.where(live, codes, 0.0).amax(2)
            s["bounds"][blk_ids] = torch.stack((low, high), 2).to(torch.uint8)
    seq, pos = _row_places(s, s["back_offsets"], s["back_rows"])
    at, slot = table[seq, pos // bs], pos % bs
    dtype = s["k_new"].dtype
    return {"k": _values(s["k"][at, :, slot], s["k_scale"][at][:, :, None]).to(dtype),
            "v": _values(s["v"][at, :, slot], s["v_scale"][at][:, :, None]).to(dtype),
            "k_scale": s["k_scale"], "v_scale": s["v_scale"], "bounds": s["bounds"]}


def _softmax_parts(score):
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top == float("-inf"), 0.0, top)).exp()
    return p, p.sum(-1, keepdim=True)


def _attention(s):
    case = s["case"]
    hkv, dim, bs = case["kv_heads"], case["dim"], case["block"]
    G, R = case["heads"] // hkv, s["max_rows"]
    off, lens, q = s["offsets"].long(), s["lens"].long(), s["q"]
    B = lens.shape[0]
    i = torch.arange(R, device=q.device)
    n = off[1:] - off[:-1]
    at = (off[:-1, None] + i).clamp(max=s["rows"] - 1)
    table = s["table"].clamp(min=0).long()

    def gather(codes, scale):
        x = _values(codes[table], scale[table][..., None, None])  # B, W, hkv, bs, dim
        return x.transpose(1, 2).reshape(B, hkv, -1, dim)

    x = q.float()[at].view(B, R, hkv, G, dim).permute(0, 2, 1, 3, 4).reshape(B, hkv, R * G, dim)
    score = (x @ gather(s["k"], s["k_scale"]).transpose(2, 3)).mul_(s["scale"]).view(B, hkv, R, G, -1)
    pos = lens[:, None] - n[:, None] + i
    seen = torch.arange(score.shape[-1], device=q.device) <= pos[:, :, None]
    score = score.masked_fill_(~seen[:, None, :, None, :], float("-inf")).view(B, hkv, R * G, -1)
    p, total = _softmax_parts(score)
    y = (p @ gather(s["v"], s["v_scale"])) / torch.where(total == 0, 1.0, total)
    y = y.view(B, hkv, R, G, dim).transpose(1, 2).reshape(B, R, hkv * G, dim).to(q.dtype)
    return y[i < n[:, None]]


def _select(s):
    case = s["case"]
    hkv, dim, bs, k = case["kv_heads"], case["dim"], case["block"], case["select"]
    G, R, q = case["heads"] // hkv, s["max_rows"], s["q"].float()
    off = s["offsets"].long()
    B, W = s["table"].shape
    size = torch.where(q.isfinite(), q.abs(), 0.0).amax(-1, keepdim=True) / 127.0
    size = torch.where(size < TINY, 0.0, size)
    c = _quantised(q, size).view(-1, hkv, G, dim)
    table = s["table"].clamp(min=0).long()
    bounds = s["bounds"][table].float() - 128.0  # B, W, hkv, 2, dim
    low, high = bounds[:, :, :, 0].permute(0, 2, 3, 1), bounds[:, :, :, 1].permute(0, 2, 3, 1)  # B, hkv, dim, W
    i = torch.arange(R, device=q.device)
    at = (off[:-1, None] + i).clamp(max=s["rows"] - 1)
    x = c[at].permute(0, 2, 1, 3, 4).reshape(B, hkv, R * G, dim)
    total = x.clamp(min=0) @ high + x.clamp(max=0) @ low  # whole numbers under 2^24
    total = total.view(B, hkv, R, G, W) * size.view(-1, hkv, G)[at].permute(0, 2, 1, 3)[..., None]
    score = total.amax(3) * s["k_scale"][table].transpose(1, 2)[:, :, None]
    score = score.transpose(1, 2)[i < (off[1:] - off[:-1])[:, None]]  # rows, hkv, W
    seq, pos = _row_places(s)
    seen = (pos // bs + 1)[:, None, None]
    j = torch.arange(W, device=q.device)
    score = torch.where((j == 0) | (j == seen - 1), float("inf"), score)
    score = torch.where(j >= seen, float("-inf"), score)
    got = score.sort(dim=-1, descending=True, stable=True).indices[:, :, :k]
    got = torch.where(got < seen, got, W).sort(dim=-1).values
    out = torch.full((got.shape[0], hkv, k), -1, dtype=torch.int32, device=q.device)
    out[:, :, :got.shape[2]] = torch.where(got == W, -1, got)
    return out


def _sparse(s):
    case = s["case"]
    hkv, dim, bs, n = case["kv_heads"], case["dim"], case["block"], case["select"]
    G, q, blocks = case["heads"] // hkv, s["q"], s["blocks"].long()
    seq, pos = _row_places(s)
    T = q.shape[0]
    at = s["table"].long()[seq[:, None, None], blocks.clamp(min=0)].clamp(min=0)  # T, hkv, n
    h = torch.arange(hkv, device=q.device)[None, :, None]
    k = _values(s["k"][at, h], s["k_scale"][at, h][..., None, None]).view(T, hkv, n * bs, dim)
    score = (q.float().view(T, hkv, G, dim) @ k.transpose(2, 3)).mul_(s["scale"])
    del k
    place = blocks[..., None] * bs + torch.arange(bs, device=q.device)
    seen = (blocks >= 0)[..., None] & (place <= pos[:, None, None, None])
    score = score.masked_fill_(~seen.view(T, hkv, 1, n * bs), float("-inf"))
    p, total = _softmax_parts(score)
    v = _values(s["v"][at, h], s["v_scale"][at, h][..., None, None]).view(T, hkv, n * bs, dim)
    return ((p @ v) / torch.where(total == 0, 1.0, total)).reshape(T, hkv * G, dim).to(q.dtype)


_PLAIN = {"append": _append, "attention": _attention, "select": _select, "sparse": _sparse}


# ------------------------------------------------------------------ work
def work(case):
    lens, rows = _lengths(case)
    bs, hkv, dim, heads = case["block"], case["kv_heads"], case["dim"], case["heads"]
    T, op = sum(rows), case["op"]
    if op == "append":
        part = sum((n - r) % bs for n, r in zip(lens, rows))  # tokens of blocks that were begun before
        touched = sum(-(-n // bs) - (n - r) // bs for n, r in zip(lens, rows))
        by = 2 * hkv * dim * (2 * T + T + part + 3 * (T + part)) + hkv * touched * (2 * dim + 16)
        return {"bytes": by, "flops": 4 * 2 * hkv * dim * T}
    rows_by = 2 * T * heads * dim
    if op == "attention":
        pairs = sum(r * (n - r) + r * (r + 1) // 2 for n, r in zip(lens, rows))
        return {"bytes": sum(lens) * hkv * 2 * dim + sum(-(-n // bs) for n in lens) * (8 * hkv + 4) + 2 * rows_by,
                "flops": 4 * pairs * heads * dim}
    blocks = sum(-(-n // bs) for n in lens)
    if op == "select":
        seen = sum((n - r + i) // bs + 1 for n, r in zip(lens, rows) for i in range(r))
        return {"bytes": blocks * (hkv * (2 * dim + 4) + 4) + rows_by + 4 * T * hkv * case["select"],
                "flops": 2 * seen * heads * dim}
    taken = [min(case["select"], (n - r + i) // bs + 1) for n, r in zip(lens, rows) for i in range(r)]
    per = [min(case["select"] * r, -(-n // bs)) for n, r in zip(lens, rows)]  # a sequence's rows may choose alike
    return {"bytes": sum(per) * hkv * (2 * dim * bs + 8) + 2 * rows_by + 4 * T * hkv * case["select"],
            "flops": 4 * sum(taken) * bs * heads * dim}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "select": _exact_select,
            "sparse": _exact_attention}[case["op"]](s)


def _exact_append(s):
    """Sequence by sequence and block by block, the whole heads of a block at once."""
    case = s["case"]
    bs = case["block"]
    lens, off = s["lens"].tolist(), s["offsets"].tolist()
    pool = {n: s[n].double() - 128 for n in ("k", "v")}
    scales = {n: s[n + "_scale"].double() for n in ("k", "v")}
    back = {"k": [], "v": []}
    for b, n in enumerate(lens):
        first = n - (off[b + 1] - off[b])
        for j in range(first // bs, -(-n // bs)):
            lo, hi = max(first, j * bs), min(n, (j + 1) * bs)
            at = int(s["table"][b, j])
            for name in ("k", "v"):
                x = s[name + "_new"][off[b] + lo - first:off[b] + hi - first].double().transpose(0, 1)
                old = scales[name][at] if lo > j * bs else torch.zeros_like(scales[name][at])
                scale = torch.maximum(old, x.abs().amax((1, 2)) / 127)
                pool[name][at, :, :lo - j * bs] = (pool[name][at, :, :lo - j * bs] * (old / scale)[:, None, None]).round()
                pool[name][at, :, lo - j * bs:hi - j * bs] = (x / scale[:, None, None]).round()
                scales[name][at] = scale
                back[name].append((pool[name][at, :, :hi - j * bs] * scale[:, None, None]).transpose(0, 1))
    return {"k": torch.cat(back["k"]), "v": torch.cat(back["v"]), "k_scale": scales["k"], "v_scale": scales["v"],
            "bounds": None}


def _exact_attention(s):
    """One sequence and one key/value head at a time; chosen blocks as a mask over the whole sequence."""
    case = s["case"]
    bs, hkv, G = case["block"], case["kv_heads"], case["heads"] // case["kv_heads"]
    lens, off = s["lens"].tolist(), s["offsets"].tolist()
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        a, e = off[b], off[b + 1]
        at = s["table"][b, :-(-n // bs)].long()
        pos = torch.arange(n - (e - a), n, device="cuda")
        for h in range(hkv):
            k = ((s["k"][at, h].double() - 128) * s["k_scale"][at, h].double()[:, None, None]).flatten(0, 1)
            v = ((s["v"][at, h].double() - 128) * s["v_scale"][at, h].double()[:, None, None]).flatten(0, 1)
            seen = torch.arange(k.shape[0], device="cuda")[None] <= pos[:, None]
            if case["op"] == "sparse":
                chosen = torch.zeros((e - a, at.shape[0] + 1), dtype=torch.bool, device="cuda")
                mine = s["blocks"][a:e, h].long()
                chosen.scatter_(1, torch.where(mine < 0, at.shape[0], mine), True)
                seen &= chosen[:, :-1].repeat_interleave(bs, dim=1)
            for i in range(0, e - a, 256):
                q = s["q"][a + i:min(e, a + i + 256), h * G:(h + 1) * G].double()
                logit = (q @ k.T * s["scale"]).masked_fill(~seen[i:i + 256, None], float("-inf"))
                out[a + i:a + i + q.shape[0], h * G:(h + 1) * G] = torch.softmax(logit, -1) @ v
    return out


def _exact_select(s):
    """The definition with its products and their maximum per channel written out, one block range at a time."""
    case = s["case"]
    bs, hkv, G, k = case["block"], case["kv_heads"], case["heads"] // case["kv_heads"], case["select"]
    lens, off = s["lens"].tolist(), s["offsets"].tolist()
    q = s["q"].float()
    size = q.abs().amax(-1, keepdim=True) / 127
    c = (q * (1 / size)).round()
    out = torch.full((q.shape[0], hkv, k), -1, dtype=torch.int32, device="cuda")
    for b, n in enumerate(lens):
        a, e = off[b], off[b + 1]
        at = s["table"][b, :-(-n // bs)].long()
        seen = torch.arange(n - (e - a), n, device="cuda")[:, None] // bs + 1
        j = torch.arange(at.shape[0], device="cuda")[None]
        for h in range(hkv):
            low, high = (s["bounds"][at, h, i].double() - 128 for i in (0, 1))
            score = torch.full((e - a, at.shape[0]), float("-inf"), dtype=torch.float64, device="cuda")
            for g in range(h * G, (h + 1) * G):
                x = c[a:e, g].double()
                total = torch.cat([torch.maximum(y[:, None] * low, y[:, None] * high).sum(-1)
                                   for y in x.split(max(1, 100_000_000 // low.numel()))])
                score = torch.maximum(score, total * size[a:e, g].double())
            score = score * s["k_scale"][at, h].double()
            score = torch.where((j == 0) | (j == seen - 1), float("inf"), score)
            score = score.masked_fill(j >= seen, float("-inf"))
            best = score.sort(dim=-1, descending=True, stable=True).indices[:, :k]
            best = torch.where(best < seen, best, at.shape[0]).sort(-1).values
            out[a:e, h, :best.shape[1]] = torch.where(best == at.shape[0], -1, best).to(torch.int32)
    return out
