"""int8 pools, packed scoring and device-side tables through the cache, the model and the engine.

Attention is compared with 64-bit arithmetic over the values the pools hold
(test_int8_pools.check_rows); results that go the same way twice must be the same
bits.  Logits of two batchings of the same tokens differ by GEMM rounding only;
their bound is the one test_graphs_gpu.py uses for graph and eager steps."""

import math

import numpy as np
import pytest
import torch

from pagedkv import BlockManager, DeviceStepTables, OutOfBlocks, PagedKVCache, ops
from pagedkv.engine import Engine, Seq
from pagedkv.graphs import DecodeStepGraph, StepGraphs
from pagedkv.migration import PeerPools
from pagedkv.model import PagedQwen2Model, Qwen2Config, Rope, SequenceForwardInfo, random_weights
from test_int8_pools import check_rows, oracle_append, u

CFG = Qwen2Config(vocab_size=512, hidden_size=256, intermediate_size=320, num_hidden_layers=3, num_attention_heads=6,
                  num_key_value_heads=2)


def test_bookkeeping_without_a_gpu():
    m = BlockManager(4, 16, 2, 2, 64, device=None, dtype=torch.int8)
    assert m.int8 and m.block_bytes == 16 * 2 * 64
    for kw in (dict(head_dim=80), dict(block_size=8)):
        with pytest.raises(ValueError, match="int8"):
            BlockManager(**{**dict(num_blocks=4, block_size=16, num_layers=1, num_kv_heads=2, head_dim=64, device=None, dtype=torch.int8), **kw})
    with pytest.raises(ValueError, match="migrate"):
        PeerPools(m)
    with pytest.raises(RuntimeError):
        DeviceStepTables(m, 2, 4, 3)


def values(mgr, layer, table, n):
    ids = table[:-(-n // mgr.block_size)]
    return [(p[layer][ids].cpu().double() * s[layer][ids].cpu().double()[:, None, :, None]).flatten(0, 1)[:n]
            for p, s in ((mgr.k_pool, mgr.k_scale), (mgr.v_pool, mgr.v_scale))]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_append_and_fetch_and_copy_on_write(dtype):
    mgr = BlockManager(12, 16, 2, 2, 64, device="cuda", dtype=torch.int8)
    kv = PagedKVCache(mgr)
    table = [mgr.allocate() for _ in range(4)]
    kv.add_sequence(7, table, 0)
    g = torch.Generator().manual_seed(1)
    pools = [[torch.zeros(12, 16, 2, 64).double(), torch.zeros(12, 2).double()] for _ in range(4)]
    total = 0
    for n in (5, 1, 30, 0, 3):
        if n == 3:  # the tail block is shared now: it is copied first, scales too
            shared = table[2]
            mgr.incref(shared)
            kv.ensure_writable_tail(7)
            assert table[2] != shared
            for p, s in pools:
                p[table[2]], s[table[2]] = p[shared], s[shared]
        for layer in range(2):
            x = (torch.randn(n, 4, 64, generator=g) * 2.0 ** total).to(dtype) if n else torch.zeros(0, 4, 64, dtype=dtype)
            k, v, prior = kv.append_and_fetch(layer, 7, x[:, :2].cuda(), x[:, 2:].cuda())
            assert prior == total
            for j, (got, y) in enumerate(((k, x[:, :2]), (v, x[:, 2:]))):
                p, s = pools[2 * layer + j]
                oracle_append(p, s, y, [table], [total + n], [0, n], 16)
                ids = table[:-(-(total + n) // 16)]
                want = (p[ids] * s[ids][:, None, :, None]).flatten(0, 1)[:total + n].to(dtype)
                assert torch.equal(got.cpu(), want)
        total += n
        assert kv.seq_len(7) == total
    mgr.check_errors()


def mixed_step(mgr, seed, layer_inputs):
    """Sequences of 40, 16 and 0 cached tokens; a step of two decodes and two chunks on each layer."""
    kv = PagedKVCache(mgr)
    lens = {1: 40, 2: 16, 3: 21, 4: 0}
    for s, n in lens.items():
        kv.add_sequence(s, [mgr.allocate() for _ in range(6)], 0)
    g = torch.Generator().manual_seed(seed)
    steps = [[(s, n) for s, n in lens.items() if n], [(1, 1), (2, 1), (3, 30), (4, 9)]]
    outs = []
    for seqs in steps:
        meta = kv.prepare_step(seqs)
        for layer in range(mgr.num_layers):
            x = torch.randn(meta.n_tokens, 14 + 4, 64, generator=g).half().cuda()
            outs.append((layer, meta, x, layer_inputs(kv, layer, x, meta)))
    return kv, outs


@pytest.mark.gpu
def test_forward_layer_over_int8_pools():
    mgr = BlockManager(40, 16, 2, 2, 64, device="cuda", dtype=torch.int8)

    def run(kv, layer, x, meta):
        out = kv.forward_layer(layer, x[:, :14], x[:, 14:16], x[:, 16:], meta, 0.125)
        # checked at once: the next layer's step rewrites nothing of this layer
        o = 0
        for s, p, n in zip(meta.seq_ids, meta.num_prior, meta.num_new):
            k, v = values(mgr, layer, kv.block_tables[s], p + n)
            check_rows(out[o:o + n].cpu(), torch.float16, x[o:o + n, :14].cpu(), k, v, p, 0.125, u_p=u(torch.float16) + 2.0 ** -13)
            o += n
        return out

    kv, outs = mixed_step(mgr, 3, run)
    assert [kv.seq_len(s) for s in (1, 2, 3, 4)] == [41, 17, 51, 9]
    mgr.check_errors()
    # the whole-run call over int8 pools goes layer by layer: the same bits
    other = BlockManager(40, 16, 2, 2, 64, device="cuda", dtype=torch.int8)

    def again(kv, layer, x, meta):
        if layer:
            return None
        xs = torch.stack([o[2] for o in outs if o[1].n_tokens == meta.n_tokens])
        return kv.forward_layers(0, xs[:, :, :14], xs[:, :, 14:16], xs[:, :, 16:], meta, 0.125)

    _, outs2 = mixed_step(other, 3, again)
    for a, b in ((outs[0], outs2[0][3][0]), (outs[1], outs2[0][3][1]), (outs[2], outs2[2][3][0]), (outs[3], outs2[2][3][1])):
        assert torch.equal(a[3], b)
    with pytest.raises(ValueError):
        kv.forward_layers(0, outs[0][2][None, :1, :14], outs[0][2][None, :1, 14:16], outs[0][2][None, :1, 16:],
                          outs[2][1], 0.125, defer_first=True)


@pytest.mark.gpu
def test_fused_projection_rows_over_int8_pools():
    """forward_layer_qkv: the bits of rotating with torch and calling forward_layer."""
    rope = Rope(64, 1e6, torch.device("cuda"), torch.float16)
    cos, sin = rope.tables(128)
    mgrs = [BlockManager(40, 16, 2, 2, 64, device="cuda", dtype=torch.int8) for _ in range(2)]

    def positions(meta):
        return torch.cat([torch.arange(p, p + n) for p, n in zip(meta.num_prior, meta.num_new)]).cuda()

    def fused(kv, layer, x, meta):
        return kv.forward_layer_qkv(layer, x.flatten(1), positions(meta), cos, sin, meta, 0.125)

    def plain(kv, layer, x, meta):
        pos = positions(meta)
        c, s = cos[pos].unsqueeze(1), sin[pos].unsqueeze(1)
        return kv.forward_layer(layer, Rope.rotate(x[:, :14], c, s), Rope.rotate(x[:, 14:16], c, s), x[:, 16:], meta, 0.125)

    a, b = mixed_step(mgrs[0], 5, fused)[1], mixed_step(mgrs[1], 5, plain)[1]
    for (_, _, _, x), (_, _, _, y) in zip(a, b):
        assert torch.equal(x, y)
    for name in ("k_cache", "v_cache", "k_scale_cache", "v_scale_cache"):
        assert torch.equal(getattr(mgrs[0], name), getattr(mgrs[1], name))


@pytest.fixture(scope="module")
def model():
    return PagedQwen2Model(CFG, random_weights(CFG, seed=3, final_norm_scale=4.0), device="cuda", dtype=torch.float16)


def generate(model, dtype, graphs, n_new=12):
    mgr = BlockManager(120, 16, CFG.num_hidden_layers, CFG.num_key_value_heads, CFG.head_dim, device="cuda", dtype=dtype)
    eng = Engine(model, mgr, max_seqs=6, token_budget=64, cuda_graphs=graphs, graph_max_blocks=8)
    rng = np.random.default_rng(0)
    seqs = [eng.submit(Seq(i, rng.integers(0, 512, n).tolist(), limit=n_new)) for i, n in enumerate((5, 40, 17, 100, 1, 33, 64))]
    eng.run()
    mgr.check_errors()
    return [s.generated for s in seqs], eng


@pytest.mark.gpu
def test_engine_over_int8_pools(model):
    """Generation over int8 pools runs eagerly and in graphs, and mostly agrees with 16-bit pools."""
    exact, _ = generate(model, torch.float16, False)
    eager, _ = generate(model, torch.int8, False)
    graph, eng = generate(model, torch.int8, True)
    assert eng.graphs is not None and eng.graphs.replays > 0
    for a in (eager, graph):
        assert [len(x) for x in a] == [len(x) for x in exact]
        # the first token of a prompt of one chunk comes from its own values alone; later ones may
        # part where two logits are near
        same = np.mean([x[0] == y[0] for x, y in zip(a, exact)])
        assert same >= 0.5


@pytest.mark.gpu
def test_graph_step_over_int8_pools_equals_the_eager_step(model):
    lens = [30, 17, 64, 5]
    outs = []
    for graphs in (False, True):
        mgr = BlockManager(60, 16, CFG.num_hidden_layers, CFG.num_key_value_heads, CFG.head_dim, device="cuda", dtype=torch.int8)
        kv = PagedKVCache(mgr)
        g = torch.Generator(device="cuda").manual_seed(1)
        for t in (mgr.k_cache, mgr.v_cache):
            t.copy_(torch.randint(-127, 128, t.shape, generator=g, device="cuda"))
        mgr.k_scale_cache.fill_(2.0 ** -6), mgr.v_scale_cache.fill_(2.0 ** -6)
        for s, n in enumerate(lens):
            kv.add_sequence(s, [mgr.allocate() for _ in range(8)], n)
        kv.add_sequence(9, [mgr.allocate() for _ in range(8)], 0)
        infos = [SequenceForwardInfo(s, s, 1, np.array([n])) for s, n in enumerate(lens)]
        infos.append(SequenceForwardInfo(9, 4, 25, np.arange(25)))
        ids = torch.arange(29, device="cuda") * 7 % 512
        if graphs:
            sg = StepGraphs(model, kv, 6, max_tokens=64, max_blocks_per_seq=8)
            assert sg.supports(infos)
            logits = sg.forward(ids, infos).clone()
        else:
            logits = model.forward(ids, infos, kv)
        mgr.check_errors()
        outs.append(logits.float())
        assert [kv.seq_len(s) for s in (0, 1, 2, 3, 9)] == [31, 18, 65, 6, 25]
    # 3 layers of fp16 GEMMs whose padded M may pick another algorithm: a few ulps of the largest logit
    assert float((outs[0] - outs[1]).abs().max()) <= 16 * float(outs[0].abs().max()) * 2.0 ** -10


@pytest.mark.gpu
def test_decode_step_graph_refuses_int8_pools():
    mgr = BlockManager(8, 16, 2, 2, 64, device="cuda", dtype=torch.int8)
    z = torch.zeros(2, 2, 18, 64, dtype=torch.float16).pin_memory()
    with pytest.raises((ValueError, RuntimeError)):
        DecodeStepGraph(PagedKVCache(mgr), z, z[:, :, :14], 0.125)


@pytest.mark.gpu
def test_scoring_prompts_without_a_cache(model):
    """forward_all_logits: the last token's logits are forward()'s, every token's those of its prompt scored alone."""
    lengths = [7, 0, 64, 1, 33]
    ids = torch.randint(0, 512, (sum(lengths),), generator=torch.Generator().manual_seed(2)).cuda()
    logits = model.forward_all_logits(ids, lengths).float()
    assert logits.shape == (sum(lengths), 512)
    mgr = BlockManager(60, 16, CFG.num_hidden_layers, CFG.num_key_value_heads, CFG.head_dim, device="cuda", dtype=torch.float16)
    kv = PagedKVCache(mgr)
    tol = 16 * float(logits.abs().max()) * 2.0 ** -10
    o = 0
    for s, n in enumerate(lengths):
        if n == 0:
            continue
        kv.add_sequence(s, [mgr.allocate() for _ in range(8)], 0)
        last = model.forward(ids[o:o + n], [SequenceForwardInfo(s, 0, n, np.arange(n))], kv).float()
        assert float((last[0] - logits[o + n - 1]).abs().max()) <= tol
        alone = model.forward_all_logits(ids[o:o + n], [n]).float()
        assert float((alone - logits[o:o + n]).abs().max()) <= tol
        o += n
    with pytest.raises(ValueError):
        model.forward_all_logits(ids, [1, 2])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.int8])
def test_device_tables_drive_the_cache(dtype):
    """The same steps through host tables and through DeviceStepTables: the same outputs, bit for bit."""
    steps = [[1, 20, 33], [1, 1, 1], [1, 1, 1], [1, 16, 0], [1, 1, 1]]
    outs, mgrs = [], []
    for device_side in (False, True):
        mgr = BlockManager(30, 16, 2, 2, 64, device="cuda", dtype=dtype)
        kv = PagedKVCache(mgr)
        mgr.allocate()  # not the pool's first block
        dst = DeviceStepTables(mgr, 3, 8, 20) if device_side else None
        if not device_side:
            for s in range(3):
                kv.add_sequence(s, [], 0)
        g = torch.Generator().manual_seed(4)
        got = []
        for new in steps:
            if device_side:
                meta = dst.step(new)
                assert dst.positions.tolist() == [t for p, n in zip(meta.num_prior, new) for t in range(p, p + n)]
            else:
                for s, n in enumerate(new):
                    t = kv.block_tables[s]
                    t.extend(mgr.allocate() for _ in range(-(-(kv.seq_len(s) + n) // 16) - len(t)))
                live = [(s, n) for s, n in enumerate(new) if n]
                meta = kv.prepare_step(live)
            x = torch.randn(2, sum(new), 18, 64, generator=g).half().cuda()
            for layer in range(2):
                got.append(kv.forward_layer(layer, x[layer, :, :14], x[layer, :, 14:16], x[layer, :, 16:], meta, 0.125,
                                            advance=not device_side))
        outs.append(got)
        mgrs.append(mgr)
        mgr.check_errors()
        if device_side:
            free = mgr.num_free
            with pytest.raises(OutOfBlocks):
                dst.step([120, 80, 80])  # within the tables, past the free list
            with pytest.raises(ValueError):
                dst.step([200, 0, 0])
            with pytest.raises(ValueError):
                dst.step([1, 1])
            dst.release()
            assert mgr.num_free == free + 20
            with pytest.raises(RuntimeError):
                dst.step([1, 1, 1])
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert torch.equal(mgrs[0].k_cache, mgrs[1].k_cache)
    with pytest.raises(OutOfBlocks):
        DeviceStepTables(mgrs[0], 2, 4, 1000)


@pytest.mark.gpu
def test_cache_of_a_whole_prompt_against_no_cache():
    """A prompt through int8 pools stays near the same prompt without a cache: within the quantisation of K and V."""
    g = torch.Generator().manual_seed(8)
    x = torch.randn(200, 18, 64, generator=g).half()
    mgr = BlockManager(20, 16, 1, 2, 64, device="cuda", dtype=torch.int8)
    kv = PagedKVCache(mgr)
    kv.add_sequence(0, [mgr.allocate() for _ in range(13)], 0)
    xd = x.cuda()
    a = kv.forward_layer(0, xd[:, :14], xd[:, 14:16], xd[:, 16:], kv.prepare_step([(0, 200)]), 0.125).float()
    b = ops.packed_prompt_attention(xd[:, :14], xd[:, 14:16], xd[:, 16:], torch.tensor([0, 200], dtype=torch.int32, device="cuda"), 0.125).float()
    # a value is off by at most absmax / 127 (half a step of a scale up to 2 absmax / 127); a score by
    # scale sum|q| absmax / 127 at most, so p by a factor e^(2 dx)
    top = float(x.abs().max())
    dx = 0.125 * float(x[:, :14].abs().sum(-1).max()) * top / 127
    assert math.isfinite(dx)
    bound = top / 127 + top * (math.exp(2 * dx) - 1) + 2 * u(torch.float16) * top
    assert float((a - b).abs().max()) <= bound
