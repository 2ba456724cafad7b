"""Packed attention beside rows that a row must not see (later tokens, the next prompt, rows
behind the last one) and beside values that are not finite."""

import math

import pytest
import torch

from pagedkv import ops
from test_int8_pools import DT, ints
from test_packed_prompts import check


def run(x, hq, hkv, starts, scale=0.125):
    err = ops.new_error_flags("cuda")
    x = x.cuda()
    out = torch.zeros(x.shape[0], hq, x.shape[2], dtype=x.dtype, device="cuda")
    ops.packed_prompt_attention(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], ints(starts), scale, out=out, err=err)
    assert int(err) == 0
    return out.cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("f16", 64), ("f32", 64)])
def test_largest_finite_values_stay_hidden(dtype, d):
    """A value of the type's largest magnitude at each position of a key tile in turn, in the
    next prompt and behind the last one: rows that must not see it have the bits they have without it."""
    hq, hkv, dt, starts = 6, 2, DT[dtype], [0, 200, 330]
    x = torch.randn(340, hq + 2 * hkv, d, generator=torch.Generator().manual_seed(2)).to(dt)
    plain, top = run(x, hq, hkv, starts), torch.finfo(dt).max
    for at in range(60, 60 + 128):
        y = x.clone()
        y[at, hq + hkv:] = top
        got = run(y, hq, hkv, starts)
        assert torch.equal(got[:at], plain[:at]) and torch.equal(got[200:330], plain[200:330]), at
    y = x.clone()
    y[200:, hq + hkv:] = top
    assert torch.equal(run(y, hq, hkv, starts)[:200], plain[:200])
    y = x.clone()
    y[330:, hq + hkv:] = -top
    assert torch.equal(run(y, hq, hkv, starts)[:330], plain[:330])


@pytest.mark.gpu
def test_largest_finite_values_stay_hidden_in_paged_chunks():
    """The same behind a block table (bf16): later tokens of the chunk, and what the last block holds behind the sequence."""
    hq, hkv, d, bs, n = 14, 2, 64, 16, 200
    g = torch.Generator().manual_seed(2)
    q = torch.randn(n, hq, d, generator=g).bfloat16().cuda()
    pools = [torch.randn(14, bs, hkv, d, generator=g).bfloat16().cuda() for _ in range(2)]
    table = torch.randperm(14, generator=g).int().cuda()[None]

    def chunk(v):
        return ops.paged_prefill_attention(q, pools[0], v, table[:, :13].contiguous(), ints([0, n]), ints([0]), n, 0.125)

    plain = chunk(pools[1])
    for at in list(range(60, 190, 3)) + [n]:
        v = pools[1].clone()
        v.view(-1, hkv, d)[int(table[0, at // bs]) * bs + at % bs] = torch.finfo(torch.bfloat16).max
        assert torch.equal(chunk(v)[:at], plain[:at]), at


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_a_value_that_is_not_finite_costs_little(dtype):
    """A NaN in the first value of a long prompt makes a column of its later rows NaN and
    nothing else, in a small multiple of the time without it (every row computed again, key by
    key, takes a hundred times as long)."""
    hq, hkv, d, n = 14, 2, 64, 8191 if dtype == "f16" else 2000
    x = torch.randn(n, hq + 2 * hkv, d, generator=torch.Generator().manual_seed(2)).to(DT[dtype])
    bad = x.clone()
    bad[0, hq + hkv, 5] = math.nan
    plain, got = run(x, hq, hkv, [0, n]), run(bad, hq, hkv, [0, n])
    assert bool(got[:, :7, 5].isnan().all())
    got[:, :7, 5] = plain[:, :7, 5]
    assert torch.equal(got, plain)

    def best(t):
        t, start = t.cuda(), ints([0, n])
        times = []
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            ops.packed_prompt_attention(t[:, :hq], t[:, hq:hq + hkv], t[:, hq + hkv:], start, 0.125)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    assert best(bad) < 4 * best(x)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [("bf16", 64), ("bf16", 128), ("f32", 64)])
def test_largest_finite_values_of_a_rows_own(dtype, d):
    """Values near the type's end in keys that a row sees: sums that pass fp32 on the way give a finite row all the same."""
    hq, hkv, starts = 6, 2, [0, 150, 300]
    x = torch.randn(300, hq + 2 * hkv, d, generator=torch.Generator().manual_seed(4)).to(DT[dtype])
    x[40, hq + hkv] = 3e38
    x[200, hq + hkv + 1, ::2] = -3e38
    out = run(x, hq, hkv, starts)
    assert bool(out.isfinite().all())
    check(out, DT[dtype], x, hq, hkv, starts, 0.125)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_a_score_of_minus_infinity_counts_for_nothing(dtype):
    """The first key's scores are -infinity: the row that sees nothing else is NaN, the others are as without that key."""
    hq, hkv, d, n = 6, 2, 64, 200
    x = torch.randn(n, hq + 2 * hkv, d, generator=torch.Generator().manual_seed(4)).to(DT[dtype])
    x[:, :hq, 3] = 1
    x[0, hq:hq + hkv, 3] = -math.inf
    out = run(x, hq, hkv, [0, n])
    assert bool(out[0].isnan().all())
    check(out[1:], DT[dtype], x[1:], hq, hkv, [0, n - 1], 0.125)
