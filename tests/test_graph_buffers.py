"""Graphs captured between eager steps that replace the cache's buffers by larger ones.

The same steps run eagerly and with two of them by graph replay; the bound on their
logits is test_graphs_gpu.py's for graph and eager steps (GEMMs of padded M)."""

import numpy as np
import pytest
import torch

from pagedkv import BlockManager, PagedKVCache
from pagedkv.graphs import StepGraphs
from pagedkv.model import PagedQwen2Model, SequenceForwardInfo, random_weights
from test_int8_cache import CFG

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model():
    return PagedQwen2Model(CFG, random_weights(CFG, seed=3, final_norm_scale=4.0), device="cuda", dtype=torch.float16)


def steps(model, dtype, graphs):
    """Logits of the two small steps (by graph replay, if graphs)."""
    mgr = BlockManager(200, 16, CFG.num_hidden_layers, CFG.num_key_value_heads, CFG.head_dim, device="cuda", dtype=dtype)
    kv = PagedKVCache(mgr)
    for s in range(18):
        kv.add_sequence(s, [mgr.allocate() for _ in range(8)], 0)

    def step(new, by=model):
        infos, at, ids = [], 0, []
        for s, n in new:
            p = kv.seq_len(s)
            infos.append(SequenceForwardInfo(s, at, n, np.arange(p, p + n)))
            ids += [(s * 131 + t * 7 + p * 3) % CFG.vocab_size for t in range(n)]
            at += n
        ids = torch.tensor(ids, device="cuda")
        return (by.forward(ids, infos, kv) if by is model else by.forward(ids, infos)).float().clone()

    runner = StepGraphs(model, kv, 4, max_tokens=64, max_blocks_per_seq=8) if graphs else model
    # eager steps larger than what the graphs were sized for, then a capture, then larger ones again
    step([(s, 30) for s in range(6)])
    step([(s, 1) for s in range(6)])
    small = [[(0, 1), (1, 1), (2, 1), (6, 20)], [(0, 1), (1, 1), (2, 1), (3, 1), (17, 20)]]
    out = [step(small[0], runner)]
    used = kv.step_buffers()
    step([(s, 1) for s in range(6)] + [(s, 40) for s in range(7, 17)])
    step([(s, 1) for s in range(17)])
    junk = []
    if graphs:
        (held,) = runner.held.values()
        assert all(any(b is h for h in held) for b in used if b is not None)
        replaced = [b for b, now in zip(used, kv.step_buffers()) if b is not None and b is not now]
        assert replaced
        sizes = [b.numel() * b.element_size() for b in replaced]
        del held, used, replaced
        junk = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(4)]
    out.append(step(small[1], runner))
    assert all(bool((j == 255).all()) for j in junk)
    assert not graphs or runner.replays == 2
    mgr.check_errors()
    return out


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn, torch.float16])
def test_a_graph_keeps_the_buffers_it_was_captured_with(model, dtype):
    eager, graph = steps(model, dtype, False), steps(model, dtype, True)
    for a, b in zip(eager, graph):
        assert float((a - b).abs().max()) <= 16 * float(a.abs().max()) * 2.0 ** -10
