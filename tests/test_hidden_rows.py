"""Packed attention beside rows that a row must not see (later tokens, the next prompt, rows
behind the last one)."""

import pytest
import torch

from pagedkv import ops
from test_int8_pools import DT, ints


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
