"""Calls of the step tables, the int8 pools and the packed attention that their
documentation allows and that are easy to get wrong: rows before the first
sequence, many sequences and heads, capture and replay with other lengths, two
streams at once, rows of non-finite queries, in-place outputs.

Tolerances are those of test_int8_pools.py and test_packed_prompts.py."""

import math

import pytest
import torch

from pagedkv import _lib, ops
from test_int8_pools import DT, check_rows, ints, layout, random_pool, starts_of, u, values
from test_packed_prompts import check


def chunk_call(ctx, bs, hq, hkv, d, dt, rows, seed=3):
    """Pools and a query for sequences of ctx tokens; rows: of q."""
    tables, nb = layout(ctx, bs, 11)
    (kp, ks), (vp, vs) = random_pool(nb, bs, hkv, d, 1), random_pool(nb, bs, hkv, d, 2)
    q = torch.randn(rows, hq, d, generator=torch.Generator().manual_seed(seed)).to(dt)
    return tables, (kp, vp, ks, vs), q


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hq,hkv,d", [("f16", 14, 2, 64), ("bf16", 16, 2, 128)])
def test_split_chunks_in_a_graph_follow_their_lengths(dtype, hq, hkv, d):
    """Replays after the lengths changed (the split changes with them, its counters
    start anew), each equal to an eager call; the same bits every time."""
    bs, dt = 16, DT[dtype]
    new, cases = [40, 3, 90], [[5000, 0, 2500], [10, 6000, 0], [0, 0, 5900], [5000, 0, 2500]]
    ctx = [max(p[i] for p in cases) + new[i] for i in range(3)]
    tables, pools, q = chunk_call(ctx, bs, hq, hkv, d, dt, sum(new))
    dev = [t.cuda() for t in pools]
    qd, tab, start, prior = q.cuda(), ints(tables), ints(starts_of(new)), ints(cases[0])
    out, other = torch.empty_like(qd), torch.empty_like(qd)
    need = ops.prefill_int8_scratch_bytes(3, sum(new), tab.shape[1], hq, hkv, d, bs, dt)
    scratch, scratch2 = (torch.full((need,), 255, dtype=torch.uint8, device="cuda") for _ in range(2))

    def call(o, s):
        return ops.paged_prefill_attention_int8(qd, *dev, tab, start, prior, max(new), d ** -0.5, out=o, scratch=s)

    call(out, scratch)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(out, scratch)
    seen = []
    for p in cases:
        prior.copy_(ints(p))
        out.fill_(7)
        g.replay()
        call(other, scratch2)
        assert torch.equal(out, other)
        seen.append(out.cpu())
        at = starts_of(new)
        for i in range(3):
            c = p[i] + new[i]
            check_rows(seen[-1][at[i]:at[i + 1]], dt, q[at[i]:at[i + 1]], values(pools[0], pools[2], tables[i], c, bs),
                       values(pools[1], pools[3], tables[i], c, bs), p[i], d ** -0.5, u_p=u(dt) + 2.0 ** -13)
    assert torch.equal(seen[0], seen[3])


@pytest.mark.gpu
def test_non_finite_queries_stay_in_their_rows():
    """In split items too: NaN and infinite query rows give NaN there and nowhere else."""
    bs, hq, hkv, d, prior, n = 16, 14, 2, 64, 5000, 40
    tables, pools, q = chunk_call([prior + n], bs, hq, hkv, d, torch.float16, n)
    dev = [t.cuda() for t in pools]
    args = (ints(tables), ints([0, n]), ints([prior]), n, 0.125)
    plain = ops.paged_prefill_attention_int8(q.cuda(), *dev, *args).cpu()
    bad = q.clone()
    bad[3, 2] = math.nan
    bad[17, 9, 5] = math.inf
    got = ops.paged_prefill_attention_int8(bad.cuda(), *dev, *args).cpu()
    spoilt = torch.zeros(n, hq, dtype=torch.bool)
    spoilt[3, 2] = spoilt[17, 9] = True
    assert bool(got[spoilt].isnan().all()) and torch.equal(got[~spoilt], plain[~spoilt])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_two_streams_at_once(dtype):
    """Decode and chunks on two streams, a workspace each, against the same calls alone."""
    bs, hq, hkv, d, dt = 16, 14, 2, 64, DT[dtype]
    ctx = [3000, 17, 0, 900]
    tables, pools, q = chunk_call(ctx, bs, hq, hkv, d, dt, 64)
    dev, qd, tab = [t.cuda() for t in pools], q.cuda(), ints(tables)
    new = [20, 17, 0, 27]
    start, prior, lens = ints(starts_of(new)), ints([c - n for c, n in zip(ctx, new)]), ints(ctx)
    calls = [lambda: ops.paged_decode_attention_int8(qd[:4], *dev, tab, lens, 0.125),
             lambda: ops.paged_prefill_attention_int8(qd, *dev, tab, start, prior, 27, 0.125)]
    alone = [f() for f in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[j].append(calls[j]())
    torch.cuda.synchronize()
    assert all(torch.equal(x, alone[j]) for j in range(2) for x in got[j])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hq,hkv,n", [("f16", 14, 2, 500), ("bf16", 2, 1, 390), ("f16", 80, 1, 6), ("f32", 80, 1, 6)])
def test_packed_many_sequences_and_many_heads_a_group(dtype, hq, hkv, n):
    d, dt = 64, DT[dtype]
    starts = starts_of([(i * 29) % 60 for i in range(n)])
    x = torch.randn(starts[-1], hq + 2 * hkv, d, generator=torch.Generator().manual_seed(n)).to(dt)
    xd = x.cuda()
    out = ops.packed_prompt_attention(xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:], ints(starts), 0.125).cpu()
    check(out, dt, x, hq, hkv, starts, 0.125)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_rows_before_the_first_sequence(dtype):
    """query_start_loc[0] > 0 (the tail of a larger batch): packed, append, chunks."""
    hq, hkv, d, bs, dt = 14, 2, 64, 16, DT[dtype]
    new, skip = [20, 0, 45], 7
    starts = [skip + s for s in starts_of(new)]
    x = torch.randn(starts[-1] + 2, hq + 2 * hkv, d, generator=torch.Generator().manual_seed(8)).to(dt)
    x[:skip] = math.nan
    xd = x.cuda()
    q, k, v = xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:]
    out = torch.full((x.shape[0], hq, d), 7.0, dtype=dt, device="cuda")
    err = ops.new_error_flags("cuda")
    ops.packed_prompt_attention(q, k, v, ints(starts), 0.125, out=out, err=err)
    got = out.cpu()
    assert int(err) == 0 and bool((got[:skip] == 7).all()) and bool((got[starts[-1]:] == 7).all())
    check(got, dt, x, hq, hkv, starts, 0.125)

    tables, nb = layout(new, bs, 11)
    pools = [torch.zeros(nb, bs, hkv, d, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(nb, hkv, device="cuda") for _ in range(2)]
    ops.reshape_and_cache_int8(k, v, *pools, *scales, ints(tables), ints(new), ints(starts), err)
    out.fill_(7)
    ops.paged_prefill_attention_int8(q, *pools, *scales, ints(tables), ints(starts), ints([0, 0, 0]), 45, 0.125, out=out, err=err)
    got = out.cpu()
    assert int(err) == 0 and bool((got[:skip] == 7).all()) and bool((got[starts[-1]:] == 7).all())
    kp, vp, ks, vs = (t.cpu() for t in (*pools, *scales))
    for i, n in enumerate(new):
        if n:
            held = values(kp, ks, tables[i], n, bs)
            rows = slice(starts[i], starts[i + 1])
            assert bool(((held - x[rows, hq:hq + hkv].double()).abs() <= ks[tables[i][:-(-n // bs)]].max() / 2).all())
            check_rows(got[rows], dt, x[rows, :hq], held, values(vp, vs, tables[i], n, bs), 0, 0.125, u_p=u(dt) + 2.0 ** -13)


@pytest.mark.gpu
def test_step_tables_largest_batch_and_odd_outputs():
    """16,384 requests, outputs that are not 16-byte aligned, and the entries behind them left alone."""
    B, bs, width = 16384, 16, 3
    prior = torch.arange(B, dtype=torch.int32) * 7 % 30
    new = (torch.arange(B, dtype=torch.int32) % 5 == 0).int() * 2
    need = (prior + new + bs - 1) // bs - (prior + bs - 1) // bs
    T, F = int(new.sum()), int(need.sum())
    tables = torch.arange(B * width, dtype=torch.int32).view(B, width)
    free = torch.arange(F, dtype=torch.int32) + B * width
    plain, first = tables.clone(), F
    for i in torch.nonzero(need)[:, 0].tolist():
        for j in range(int(need[i])):
            first -= 1
            plain[i, int(prior[i] + bs - 1) // bs + j] = free[first]
    dev = tables.cuda()
    room = torch.full((2, T + 3), -9, dtype=torch.int64, device="cuda")
    small = torch.full((2 * B + 3,), -9, dtype=torch.int32, device="cuda")
    out = ops.StepTables(small[:B], small[B:2 * B + 1], room[0, 1:T + 1], room[1, 1:T + 1], small[2 * B + 1:2 * B + 2])
    err = ops.new_error_flags("cuda")
    ops.build_step_tables(dev, free.cuda(), ints([F]), prior.cuda(), new.cuda(), bs, T, out=out, err=err)
    seq = torch.repeat_interleave(torch.arange(B), new.long())
    start = torch.cat([torch.zeros(1, dtype=torch.long), new.long().cumsum(0)])
    pos = prior.long()[seq] + torch.arange(T) - start[seq]
    slot = plain[seq, pos // bs].long() * bs + pos % bs
    assert int(err) == 0 and torch.equal(dev.cpu(), plain) and int(out.n_free) == 0
    assert torch.equal(out.positions.cpu(), pos) and torch.equal(out.slot_mapping.cpu(), slot)
    assert torch.equal(out.context_lens.cpu(), prior + new) and torch.equal(out.query_start_loc.cpu().long(), start)
    assert bool((room[:, 0] == -9).all()) and bool((room[:, T + 1:] == -9).all()) and int(small[-1]) == -9


@pytest.mark.gpu
def test_a_request_without_blocks_leaves_the_others_as_they_are():
    """A batch whose free list runs short, through append and decode: the requests
    that were served get what a batch of them alone gets, the others zero rows."""
    bs, hq, hkv, d = 16, 14, 2, 64
    prior, new = [16, 5, 32, 0], [1, 1, 1, 1]
    tables = torch.tensor([[0, 0, 0], [1, 0, 0], [2, 3, 0], [0, 0, 0]], dtype=torch.int32).cuda()
    x = torch.randn(4, hq + 2 * hkv, d, generator=torch.Generator().manual_seed(2)).half().cuda()
    (kp, ks), (vp, vs) = random_pool(8, bs, hkv, d, 1), random_pool(8, bs, hkv, d, 2)

    def run(n, tab):
        pools = [t.cuda() for t in (kp, vp, ks, vs)]
        err = ops.new_error_flags("cuda")
        st = ops.build_step_tables(tab, ints([7, 6, 5, 4]), ints([1]), ints(prior[:n]), ints(new[:n]), bs, n, err=err)
        ops.reshape_and_cache_int8(x[:n, hq:hq + hkv], x[:n, hq + hkv:], *pools, tab, st.context_lens, st.query_start_loc, err)
        return ops.paged_decode_attention_int8(x[:n, :hq], *pools, tab, st.context_lens, 0.125, err=err), int(err), pools

    a, flags, pools_a = run(4, tables.clone())
    b, none, pools_b = run(2, tables.clone()[:2])
    assert flags == _lib.FLAG_OUT_OF_BLOCKS and none == 0
    assert torch.equal(a[:2], b) and bool((a[2:] == 0).all())
    assert all(torch.equal(s, t) for s, t in zip(pools_a, pools_b))


@pytest.mark.gpu
def test_in_place_outputs_are_refused():
    x = torch.randn(20, 18, 64, device="cuda").half()
    q, k, v = x[:, :14], x[:, 14:16], x[:, 16:]
    with pytest.raises(_lib.PagedKVError):
        ops.packed_prompt_attention(q, k, v, ints([0, 20]), 0.125, out=q)
    tables, pools, _ = chunk_call([20], 16, 14, 2, 64, torch.float16, 1)
    with pytest.raises(_lib.PagedKVError):
        ops.paged_prefill_attention_int8(q, *[t.cuda() for t in pools], ints(tables), ints([0, 20]), ints([0]), 20, 0.125, out=q)


@pytest.mark.gpu
def test_split_chunks_flag_bad_layouts():
    """Starts that go back or pass the rows, lengths past the tables: flagged, and a good call after them is right."""
    bs, hq, hkv, d = 16, 14, 2, 64
    tables, pools, q = chunk_call([5030, 20, 5030], bs, hq, hkv, d, torch.float16, 50)
    dev, qd, tab = [t.cuda() for t in pools], q.cuda(), ints(tables)
    need = ops.prefill_int8_scratch_bytes(3, 50, tab.shape[1], hq, hkv, d, bs, torch.float16)
    scratch = torch.zeros(need, dtype=torch.uint8, device="cuda")
    err = ops.new_error_flags("cuda")

    def call(starts, prior):
        err.zero_()
        out = ops.paged_prefill_attention_int8(qd, *dev, tab, ints(starts), ints(prior), 50, 0.125, err=err, scratch=scratch)
        return out, int(err)

    good, flags = call([0, 20, 20, 50], [5000, 0, 5000])
    assert flags == 0
    assert call([0, 30, 20, 50], [5000, 0, 5000])[1] & _lib.FLAG_BAD_QUERY_LAYOUT
    assert call([0, 20, 20, 70], [5000, 0, 5000])[1] & _lib.FLAG_BAD_QUERY_LAYOUT
    assert call([0, 20, 20, 50], [2 ** 30, 0, 5000])[1] & _lib.FLAG_CONTEXT_EXCEEDS_TABLE
    again, flags = call([0, 20, 20, 50], [5000, 0, 5000])
    assert flags == 0 and torch.equal(again, good)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [("f16", 64), ("bf16", 128), ("f32", 64)])
def test_non_finite_values_of_a_rows_own(dtype, d):
    """NaN in a key makes NaN of every later row of its sequence and heads; an infinity or
    NaN in a value of its column there; no other row or column changes."""
    hq, hkv, dt, starts = 6, 2, DT[dtype], [0, 90, 200]
    x = torch.randn(200, hq + 2 * hkv, d, generator=torch.Generator().manual_seed(5)).to(dt)

    def run(y):
        y = y.cuda()
        return ops.packed_prompt_attention(y[:, :hq], y[:, hq:hq + hkv], y[:, hq + hkv:], ints(starts), 0.125).cpu()

    plain, bad = run(x), x.clone()
    bad[40, hq, 3] = math.nan           # a key of KV head 0 in the first sequence
    bad[130, hq + hkv + 1, 7] = math.inf  # a value of KV head 1 in the second
    bad[150, hq + hkv + 1, 9] = math.nan
    got, want = run(bad), plain.clone()
    want[40:90, :3] = math.nan
    want[130:200, 3:, 7] = math.inf
    want[150:200, 3:, 9] = math.nan
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan) and torch.equal(got.isinf(), want.isinf())
    # bit for bit where no key tile holds a bad value of a key that the row must not see;
    # rows of the second sequence are computed again on their own, within the bounds of any result
    assert torch.equal(got[:90][~nan[:90]], plain[:90][~nan[:90]])
    check(torch.where(nan | want.isinf(), plain, got), dt, x, hq, hkv, starts, 0.125)
