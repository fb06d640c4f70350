"""Long-context memory end to end: an 8-bit key/value cache, the attention over
all of it, and the attention over the blocks that a cheap score or a proximity
graph over the keys picked.

    python -m dance_b200.memory --tokens 65536 --select 32

writes a synthetic context into a cache (whole, then token by token), takes
decode steps from its end and prints, for each way of choosing blocks, the time
of a step, the share of the softmax's mass that the chosen blocks hold and how
far the output is from attention over every token.

The graph is the package's Vamana graph over one head's keys, read back from
the cache.  Attention ranks keys by inner product, the graph by distance; with
one more channel sqrt(max |k|^2 - |k|^2) on every key and 0 on the queries the
two orders agree: |q' - k'|^2 = |q|^2 + max |k|^2 - 2 q.k.
"""
from __future__ import annotations

import argparse
import json
import sys

from . import kvcache, vamana

MOST_FOUND = 256  # the search's list


class KeyIndex:
    """Vamana graph over the keys of one sequence and key/value head, those of its building: tokens appended later are
    chosen with the last block only, which blocks_of_tokens always takes."""

    def __init__(self, keys, R: int = 32, L: int = 64, C: int = 64, steps: int = 32):
        """keys: CUDA tensor (tokens, head_dim), as kvcache.read gives them."""
        import torch
        if keys.dim() != 2 or not keys.is_cuda or keys.shape[0] < 2:
            raise ValueError("keys must be a CUDA tensor (tokens, head_dim) of at least two tokens")
        n, dim = keys.shape
        x = keys.float()
        norms = (x * x).sum(1)
        lifted = torch.zeros((n, dim + 2), dtype=torch.float16, device=keys.device)  # the store wants an even dimension
        lifted[:, :dim] = x
        lifted[:, dim] = (norms.max() - norms).clamp(min=0).sqrt()
        self.dim, self.tokens, self.R = dim, n, R
        self.store, self.stride = vamana.padded_store(lifted)
        self.graph, _, _, self.start = vamana.build_resident(self.store, dim + 2, self.stride, R, L, C, steps)

    def search(self, q, K: int, L: int | None = None):
        """The K (at most 256) keys of largest inner product with each row of q (rows, head_dim), approximately: int32
        (rows, K).  L: length of the search's list, K to 256, more is better (None: 2 K)."""
        import torch
        L = min(2 * K, MOST_FOUND) if L is None else L
        if not 1 <= K <= L <= MOST_FOUND:
            raise ValueError(f"K {K} and L {L}: 1 <= K <= L <= {MOST_FOUND} is needed")
        lifted = torch.zeros((q.shape[0], self.dim + 2), dtype=torch.float16, device=q.device)
        lifted[:, :self.dim] = q
        ids, _ = vamana.search_queries(self.store, self.dim + 2, self.stride, self.graph, self.R, self.start, lifted,
                                       L, K)
        return ids


def blocks_of_tokens(tokens, seen, block_tokens: int, select: int):
    """Block lists for sparse attention from found tokens.

    tokens: integer (rows, kv_heads, found), positions, others than [0, seen)
    ignored; seen: (rows,), tokens that each row sees.  The first and the last
    block that a row sees are taken, then those with the most found tokens
    (lower blocks first among equals), ``select`` in all: int32 (rows,
    kv_heads, select), ascending, -1 filled.
    """
    import torch
    if select < 2:
        raise ValueError("select must hold the first and the last block")
    rows, heads, _ = tokens.shape
    last = (seen.long() - 1).clamp(min=0) // block_tokens
    n = int(last.max()) + 1
    hit = (tokens >= 0) & (tokens < seen[:, None, None])
    at = torch.where(hit, tokens.long() // block_tokens, n)
    count = torch.zeros((rows, heads, n + 1), dtype=torch.int32, device=tokens.device)
    count.scatter_add_(2, at, torch.ones_like(at, dtype=torch.int32))
    count = count[:, :, :n]
    most = tokens.shape[2] + 1
    count[:, :, 0] = most
    count.scatter_(2, last[:, None, None].expand(rows, heads, 1), most)
    best = count.sort(dim=2, descending=True, stable=True)
    idx = torch.where(best.values > 0, best.indices, n)[:, :, :select].sort(dim=2).values
    out = torch.full((rows, heads, select), -1, dtype=torch.int32, device=tokens.device)
    out[:, :, :idx.shape[2]] = torch.where(idx == n, -1, idx)
    out[seen <= 0] = -1
    return out


def synthetic_context(tokens: int, kv_heads: int, dim: int, seed: int, topics: int = 64, device="cuda"):
    """Keys and values (tokens, kv_heads, dim) float16 of a context that moves from topic to topic, and the topics'
    directions (topics, kv_heads, dim)."""
    import torch
    g = torch.Generator(device=device).manual_seed(seed)
    centre = torch.randn((topics, kv_heads, dim), generator=g, device=device)
    run = (torch.arange(tokens, device=device) // 96 * 7919 + seed) % topics
    k = centre[run] + 0.7 * torch.randn((tokens, kv_heads, dim), generator=g, device=device)
    v = torch.randn((tokens, kv_heads, dim), generator=g, device=device)
    return k.half(), v.half(), centre


def demonstrate(tokens: int = 65536, steps: int = 8, kv_heads: int = 4, group: int = 4, dim: int = 128,
                block_tokens: int = 64, select: int = 32, seed: int = 0, graph: bool = True) -> dict:
    """What the command prints, as a dict."""
    import torch
    dev = torch.device("cuda", torch.cuda.current_device())
    total = tokens + steps
    width = -(-total // block_tokens)
    k, v, centre = synthetic_context(total, kv_heads, dim, seed, topics=max(16, tokens // 1024))
    cache = kvcache.KVCache.create(width, kv_heads, dim, block_tokens, dev)
    table = torch.randperm(width, device=dev).to(torch.int32)[None]
    ws = kvcache.KVWorkspace()

    def batch(length, rows):
        return kvcache.KVBatch(table, torch.tensor([length], dtype=torch.int32, device=dev),
                               torch.tensor([0, rows], dtype=torch.int32, device=dev), rows, length)

    kvcache.append(cache, batch(tokens, tokens), k[:tokens], v[:tokens])  # the prompt
    index = None
    if graph:
        keys, _ = kvcache.read(cache, batch(tokens, tokens), tokens, torch.float16)
        index = [KeyIndex(keys[:, h]) for h in range(kv_heads)]
    gen = torch.Generator(device=dev).manual_seed(seed + 1)
    ways = ["all", "bounds"] + (["graph"] if graph else [])
    report = {w: {"seconds": 0.0, "mass": 0.0, "error": 0.0} for w in ways}
    for step in range(steps):
        n = tokens + step + 1
        b = batch(n, 1)
        kvcache.append(cache, b, k[n - 1:n], v[n - 1:n])
        # each query head asks for one topic
        topic = torch.randint(0, centre.shape[0], (kv_heads * group,), generator=gen, device=dev)
        q = centre[topic, torch.arange(kv_heads * group, device=dev) // group] * 0.9
        q = (q + 0.3 * torch.randn(q.shape, generator=gen, device=dev)).half()[None]
        full = None
        for way in ways:
            for timed in (False, True):  # once to warm up
                ev = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
                ev[0].record()
                if way == "all":
                    out, lse = kvcache.attention(cache, b, q, return_lse=True, workspace=ws)
                else:
                    if way == "bounds":
                        blocks = kvcache.select_blocks(cache, b, q, select, workspace=ws)
                    else:
                        found = torch.stack([index[h].search(q[0, h * group:(h + 1) * group],
                                                             min(2 * select, MOST_FOUND)).flatten()
                                             for h in range(kv_heads)])
                        blocks = blocks_of_tokens(found[None], b.seq_lens, block_tokens, select)
                    out, lse = kvcache.sparse_attention(cache, b, q, blocks, return_lse=True, workspace=ws)
                ev[1].record()
                torch.cuda.synchronize()
            if way == "all":
                full = out.float(), lse
            r = report[way]
            r["seconds"] += ev[0].elapsed_time(ev[1]) * 1e-3 / steps
            r["mass"] += float((lse - full[1]).exp().mean()) / steps
            r["error"] += float((out.float() - full[0]).norm() / full[0].norm()) / steps
    return {"tokens": tokens, "blocks": width, "select": select, "kv_heads": kv_heads, "heads": kv_heads * group,
            "head_dim": dim, "block_tokens": block_tokens, "ways": report}


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--tokens", type=int, default=65536)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--kv_heads", type=int, default=4)
    ap.add_argument("--group", type=int, default=4, help="query heads of a key/value head")
    ap.add_argument("--head_dim", type=int, default=128, choices=kvcache.HEAD_DIMS)
    ap.add_argument("--block_tokens", type=int, default=64, choices=kvcache.BLOCK_TOKENS)
    ap.add_argument("--select", type=int, default=32, help="blocks that a row reads per key/value head")
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--no_graph", action="store_true", help="skip the graph over the keys")
    ap.add_argument("--json", action="store_true", help="print one JSON line instead of the table")
    a = ap.parse_args(argv)
    r = demonstrate(a.tokens, a.steps, a.kv_heads, a.group, a.head_dim, a.block_tokens, a.select, a.seed,
                    not a.no_graph)
    if a.json:
        print(json.dumps(r))
        return 0
    print(f"{r['tokens']} tokens in {r['blocks']} blocks, {r['heads']} query heads on {r['kv_heads']}; "
          f"{r['select']} blocks chosen per row and head")
    print(f"{'blocks':>8} {'us per step':>12} {'mass held':>10} {'output off':>11}")
    for way, x in r["ways"].items():
        print(f"{way:>8} {x['seconds'] * 1e6:>12.1f} {x['mass']:>10.4f} {x['error']:>11.4f}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
