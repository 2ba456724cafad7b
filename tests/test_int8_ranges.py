"""Decode over int8 pools where the range of scores is wide.

Tolerances are those of test_int8_pools.py."""

import pytest
import torch

from pagedkv import ops
from test_int8_pools import DT, check_rows, ints, layout, random_pool, values


def decode(q, kp, vp, ks, vs, tables, ctx, scale):
    err = ops.new_error_flags("cuda")
    out = ops.paged_decode_attention_int8(q.cuda(), kp.cuda(), vp.cuda(), ks.cuda(), vs.cuda(), ints(tables), ints(ctx), scale, err=err).cpu()
    assert int(err) == 0
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hq,hkv,d", [("f16", 14, 2, 64), ("bf16", 8, 2, 128), ("f32", 14, 2, 64), ("f16", 16, 1, 64),
                                            ("f32", 12, 1, 128)])
def test_scores_far_below_zero(dtype, hq, hkv, d):
    """Every score some hundreds below zero: in one tile, in tiles that the warps of a CTA
    share, in ranges that several CTAs share (few and many of them)."""
    bs, dt, ctx = 16, DT[dtype], [5, 16, 40, 400, 3000, 20000]
    tables, nb = layout(ctx, bs, 7)
    (kp, ks), (vp, vs) = random_pool(nb, bs, hkv, d, 1), random_pool(nb, bs, hkv, d, 2)
    kp[..., : d // 2] = -100  # half of each key is far from q, the other half random
    ks = torch.full_like(ks, 2.0 ** -5)
    q = torch.randn(len(ctx), hq, d, generator=torch.Generator().manual_seed(4)) * 0.5
    q[..., : d // 2] = 16.0 if d == 64 else 8.0
    q = q.to(dt)
    out = decode(q, kp, vp, ks, vs, tables, ctx, 0.125)
    for i, c in enumerate(ctx):
        k, v = values(kp, ks, tables[i], c, bs), values(vp, vs, tables[i], c, bs)
        top = torch.einsum("hd,khd->hk", q[i].double(), k.repeat_interleave(hq // hkv, 1)).amax() * 0.125
        assert float(top) < -130  # -90 is where 2^(-score) leaves fp32
        check_rows(out[i:i + 1], dt, q[i:i + 1], k, v, c - 1, 0.125)
