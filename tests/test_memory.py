"""The long-context command: cache, block choice by bounds and by a graph over
the keys, and the attention over what was chosen."""
import json

import numpy as np
import pytest


def test_blocks_of_tokens_by_hand():
    import torch
    from dance_b200.memory import blocks_of_tokens
    tokens = torch.tensor([[[17, 18, 35, -1, 90], [3, 3, 3, 3, 3]],
                           [[1, 40, 41, 42, 63], [20, 21, 36, 37, 50]],
                           [[1, 2, 3, 4, 5], [1, 2, 3, 4, 5]]], dtype=torch.int32)
    seen = torch.tensor([80, 64, 0], dtype=torch.int32)
    got = blocks_of_tokens(tokens, seen, 16, 4).numpy()
    want = np.array([[[0, 1, 2, 4], [0, 4, -1, -1]],      # first and last block, then the found; 90 lies beyond
                     [[0, 2, 3, -1], [0, 1, 2, 3]],
                     [[-1] * 4, [-1] * 4]])               # a row that sees nothing
    assert np.array_equal(got, want)
    assert np.array_equal(blocks_of_tokens(tokens, seen, 16, 3).numpy()[1, 1], [0, 1, 3])  # equals: the lower block
    with pytest.raises(ValueError):
        blocks_of_tokens(tokens, seen, 16, 1)


def test_index_refuses_host_keys():
    import torch
    from dance_b200.memory import KeyIndex
    with pytest.raises(ValueError, match="CUDA"):
        KeyIndex(torch.zeros((10, 64)))


@pytest.mark.gpu
def test_graph_finds_the_largest_products(dance_lib):
    import torch
    from dance_b200 import memory
    k, _, centre = memory.synthetic_context(6000, 1, 64, seed=3)
    index = memory.KeyIndex(k[:, 0])
    q = (centre[:40, 0] * 0.9).half()
    found = index.search(q, 20, L=120).cpu().numpy()
    product = (q.double() @ k[:, 0].double().T).cpu().numpy()
    best = np.argsort(-product, axis=1)[:, :20]
    hits = np.mean([len(set(f) & set(b)) / 20 for f, b in zip(found.tolist(), best.tolist())])
    assert hits > 0.8, hits


@pytest.mark.gpu
@pytest.mark.parametrize("dim,block", [(128, 64), (64, 16)])
def test_ways_hold_the_mass(dance_lib, dim, block):
    from dance_b200 import memory
    r = memory.demonstrate(tokens=8192, steps=2, kv_heads=2, group=4, dim=dim, block_tokens=block,
                           select=2048 // block, seed=1)
    ways = r["ways"]
    assert abs(ways["all"]["mass"] - 1) < 1e-6 and ways["all"]["error"] == 0
    for way in ("bounds", "graph"):
        assert 0.5 < ways[way]["mass"] <= 1 + 1e-3 and ways[way]["error"] < 0.5, (way, ways[way])
    # all blocks chosen: the same attention
    r = memory.demonstrate(tokens=1000, steps=1, kv_heads=2, group=2, dim=dim, block_tokens=block,
                           select=-(-1001 // block), seed=2, graph=False)
    assert abs(r["ways"]["bounds"]["mass"] - 1) < 1e-4 and r["ways"]["bounds"]["error"] < 2e-3


@pytest.mark.gpu
def test_command_prints(dance_lib, capsys):
    from dance_b200 import memory
    assert memory.main(["--tokens", "2000", "--steps", "1", "--select", "8", "--head_dim", "96", "--json"]) == 0
    r = json.loads(capsys.readouterr().out)
    assert set(r["ways"]) == {"all", "bounds", "graph"}
    assert memory.main(["--tokens", "2000", "--steps", "1", "--select", "8", "--no_graph"]) == 0
    assert "mass held" in capsys.readouterr().out
