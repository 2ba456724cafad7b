"""Decode over int8 pools where the range of scores or of V's scales is wide.

Tolerances are those of test_int8_pools.py, with the absolute term stated by weight (see
weighted_tolerance)."""

import pytest
import torch

from pagedkv import ops
from test_int8_pools import DT, attend, check_rows, ints, layout, random_pool, values


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


def weighted_tolerance(dt, q, k, v, vscale, scale):
    """The bound for one row: P has 2^-11 of its value (fp32: 2^-22) or, in the subnormals of fp16, an
    error of 2^-25 where the largest weight of a key, p_j s_j (s: the scale of V's block), is at least
    2^6: n 127 2^-31 max_j(p_j s_j).  The rest as in test_int8_pools.tolerance, whose absolute term
    counts the loudest block whatever its weight."""
    n, hq, d = q.shape
    grp = hq // k.shape[1]
    o, A, S, S_max = attend(q.double(), k, v, k.shape[0] - 1, scale)
    x = torch.einsum("nhd,khd->hk", q.double(), k.repeat_interleave(grp, 1)) * scale
    w = (torch.softmax(x, -1) * vscale.repeat_interleave(grp, 1).T).amax(-1)[None, :, None]
    dx = (16 + d / 2 + 2) * 2.0 ** -23 * S + (2.0 ** -22 * S_max if dt == torch.float32 else 0)
    keys = k.shape[0]
    part = 2.0 ** -22 if dt == torch.float32 else 2.0 ** -11
    return o, (torch.finfo(dt).eps / 2 * o.abs() + A * (part * 1.01 + 2 * dx + (keys / 16 + 64) * 2.0 ** -23) +
               keys * 127 * 2.0 ** -31 * w)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["loud first", "loud last", "loud between"])
@pytest.mark.parametrize("dtype,hq,hkv,d,ratio", [
    ("f16", 14, 2, 64, 20), ("bf16", 14, 2, 64, 20), ("bf16", 8, 2, 128, 40), ("f32", 14, 2, 64, 20), ("f32", 6, 3, 128, 40),
    ("f32", 16, 1, 64, 60), ("bf16", 16, 1, 128, 20)])
def test_loud_blocks_of_no_weight(dtype, hq, hkv, d, ratio, order):
    """A block whose V scale is 2^ratio above the others' and whose keys have next to no weight
    (their scores are far below): the quiet blocks keep their precision."""
    bs, dt, ctx = 16, DT[dtype], [40, 1024, 9000]
    tables, nb = layout(ctx, bs, 3)
    (kp, ks), (vp, vs) = random_pool(nb, bs, hkv, d, 1), random_pool(nb, bs, hkv, d, 2)
    ks, vs = torch.full_like(ks, 2.0 ** -6), torch.full_like(vs, 2.0 ** -14)
    q = torch.randn(len(ctx), hq, d, generator=torch.Generator().manual_seed(4))
    q[..., :8] = 16.0
    kp[..., :8] = 0
    for t, c in zip(tables, ctx):
        last = (c - 1) // bs
        loud = t[{"loud first": 0, "loud last": last, "loud between": last // 2}[order]]
        kp[loud, ..., :8] = -120  # 8 x 16 x 120 / 64 / 8: 30 nats below; more for the larger ratios
        ks[loud] *= max(1, ratio // 20) ** 2
        vs[loud] = 2.0 ** (ratio - 14)
    q = q.to(dt)
    out = decode(q, kp, vp, ks, vs, tables, ctx, 0.125)
    for i, c in enumerate(ctx):
        k, v = values(kp, ks, tables[i], c, bs), values(vp, vs, tables[i], c, bs)
        vscale = vs[tables[i][:-(-c // bs)]].double().repeat_interleave(bs, 0)[:c]
        o, tol = weighted_tolerance(dt, q[i:i + 1], k, v, vscale, 0.125)
        off = (out[i:i + 1].double() - o).abs()
        assert bool((off <= tol).all()), f"context {c} off by up to {float((off / tol).max()):.2f} of the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["first", "last", "all"])
@pytest.mark.parametrize("dtype,hq,hkv,d", [("f16", 14, 2, 64), ("bf16", 16, 1, 128), ("f32", 14, 2, 64)])
def test_blocks_of_zeros(dtype, hq, hkv, d, where):
    """Blocks whose rows are all zeros have the least scale, 2^-120: as any other block."""
    bs, dt, ctx = 16, DT[dtype], [7, 40, 1500, 9000]
    tables, nb = layout(ctx, bs, 3)
    (kp, ks), (vp, vs) = random_pool(nb, bs, hkv, d, 1), random_pool(nb, bs, hkv, d, 2)
    for t, c in zip(tables, ctx):
        n = -(-c // bs)
        zero = t[:n] if where == "all" else t[:(n + 2) // 3] if where == "first" else t[n // 2:n]
        kp[zero], vp[zero], ks[zero], vs[zero] = 0, 0, 2.0 ** -120, 2.0 ** -120
    q = torch.randn(len(ctx), hq, d, generator=torch.Generator().manual_seed(4)).to(dt)
    out = decode(q, kp, vp, ks, vs, tables, ctx, 0.125)
    for i, c in enumerate(ctx):
        k, v = values(kp, ks, tables[i], c, bs), values(vp, vs, tables[i], c, bs)
        vscale = vs[tables[i][:-(-c // bs)]].double().repeat_interleave(bs, 0)[:c]
        o, tol = weighted_tolerance(dt, q[i:i + 1], k, v, vscale, 0.125)
        assert bool(((out[i:i + 1].double() - o).abs() <= tol).all())
