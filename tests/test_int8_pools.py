"""int8 pools with a power-of-two scale per (block, KV head): the append and the
fetch exactly, the attention over them against 64-bit arithmetic, refusals.

Tolerances of the attention, per element, from the arithmetic (A = sum_j p_j |v_j|
over the normalised p, all in 64 bits; u(t) = finfo(t).eps / 2):
  output rounding          u(dtype) |o|
  rounding of P            u(fp16) A for 16-bit q, 2^-22 A for fp32 (two fp16 parts)
  P below fp16's range     n 2^-25 max|v|  (an absolute error of 2^-25 per key, against a sum >= 1)
  scores                   2 A dx, dx = error of a score: (16 + D / 2) sums of 2^-23 of S = scale sum|q||k|,
                           the scale products 2^-22 |x| with |x| <= S, fp32 q in two parts 2^-22 S_max,
                           S_max = scale max|q| sum|k|
  sums over n keys         (n / 16 + 64) 2^-23 A (fp32, one tile of 16 at a time, then joined partials)
"""

import ctypes
import math

import pytest
import torch

from pagedkv import _lib, ops

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
FAKE = ctypes.c_void_p(0x1000)


def u(dt):
    return torch.finfo(dt).eps / 2


def block_scale(amax):
    """The smallest 2^e, e >= -120, with amax <= 127 * 2^e."""
    if amax == 0:
        return 2.0 ** -120
    m, e = math.frexp(amax)
    return 2.0 ** max(-120, e - 7 if m * 128 <= 127 else e - 6)


def rne(x):
    return torch.round(x)  # half to even


def oracle_append(pool, scale, x, tables, ctx, starts, bs):
    """pool [NB, bs, H, D] and scale [NB, H] as float64 CPU tensors, changed in place."""
    for i, c in enumerate(ctx):
        n = starts[i + 1] - starts[i]
        if c == 0 or n == 0:
            continue
        rows, p = x[starts[i]:starts[i + 1]].double(), c - n
        for jb in range(p // bs, -(-c // bs)):
            b = tables[i][jb]
            lo, hi = max(p, jb * bs), min(c, (jb + 1) * bs)
            part = rows[lo - p:hi - p]
            held = lo - jb * bs
            for h in range(pool.shape[2]):
                y = part[:, h]
                fin = y[torch.isfinite(y)]
                s = block_scale(float(fin.abs().max()) if fin.numel() else 0.0)
                if held:
                    old = float(scale[b, h])
                    s = max(s, old)
                    pool[b, :held, h] = rne(pool[b, :held, h] * (old / s))
                q = torch.nan_to_num(y / s, nan=0.0, posinf=127.0, neginf=-127.0)
                pool[b, held:held + hi - lo, h] = rne(q).clamp(-127, 127)
                scale[b, h] = s


def layout(ctx, bs, seed, extra_cols=0, spare=3):
    """Scattered disjoint tables for the contexts: (rows of ids, number of blocks)."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-c // bs) for c in ctx]
    nb = sum(need) + spare
    ids = torch.randperm(nb, generator=g).tolist()
    width = max(1, max(need, default=1)) + extra_cols
    tables, o = [], 0
    for k in need:
        tables.append(ids[o:o + k] + [-5] * (width - k))  # entries past a sequence's blocks are never read
        o += k
    return tables, nb


def starts_of(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def ints(v, dt=torch.int32):
    return torch.tensor(v, dtype=dt, device="cuda")


def random_pool(nb, bs, hkv, d, seed):
    g = torch.Generator().manual_seed(seed)
    pool = torch.randint(-127, 128, (nb, bs, hkv, d), generator=g).to(torch.int8)
    scale = 2.0 ** torch.randint(-9, -3, (nb, hkv), generator=g).float()
    return pool, scale


# contexts before the call and new tokens of it, by name
APPENDS = {
    "one token": ([0], [1]),
    "tokens": ([0, 1, 15, 16, 31, 200, 7], [1] * 7),
    "prompts": ([0, 0, 0], [1, 16, 75]),
    "chunks": ([5, 16, 40, 63, 0], [11, 33, 1, 70, 0]),
    "padding": ([3, -1, 8, -1], [2, 1, 0, 1]),  # -1: a padding row, context length 0
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(APPENDS))
@pytest.mark.parametrize("dtype,hkv,d,bs", [("f16", 2, 64, 16), ("bf16", 8, 128, 16), ("f32", 1, 64, 32), ("f16", 3, 128, 48)])
def test_append_and_fetch_are_exact(name, dtype, hkv, d, bs):
    prior, new = APPENDS[name]
    ctx = [p + n if p >= 0 else 0 for p, n in zip(prior, new)]
    starts = starts_of(new)
    T = starts[-1]
    tables, nb = layout(ctx, bs, 3)
    g = torch.Generator().manual_seed(7)
    # rows of very different loudness: scales grow at some tokens, and not at others
    x = torch.randn(T + 2, 2 * hkv, d, generator=g) * torch.exp2(torch.randint(-3, 4, (T + 2, 2 * hkv, 1), generator=g).float())
    x = x.to(DT[dtype])
    (kp, ks), (vp, vs) = random_pool(nb, bs, hkv, d, 1), random_pool(nb, bs, hkv, d, 2)
    dev = [t.cuda() for t in (kp, vp, ks, vs)]
    err = ops.new_error_flags("cuda")
    xd = x.cuda()
    ops.reshape_and_cache_int8(xd[:, :hkv], xd[:, hkv:], *dev, ints(tables), ints(ctx), ints(starts), err=err)
    want = []
    for pool, scale, y in ((kp, ks, x[:, :hkv]), (vp, vs, x[:, hkv:])):
        pool, scale = pool.double(), scale.double()
        oracle_append(pool, scale, y, tables, ctx, starts, bs)
        want.append((pool, scale))
    assert int(err) == 0
    for got, (pool, scale), s in ((dev[0], want[0], dev[2]), (dev[1], want[1], dev[3])):
        assert torch.equal(got.cpu().double(), pool) and torch.equal(s.cpu().double(), scale)
    # the whole contexts back as values
    fs = starts_of(ctx)
    k, v = ops.fetch_int8(*dev, ints(tables), ints(ctx), ints(fs), fs[-1], DT[dtype], err=err)
    for got, (pool, scale) in ((k, want[0]), (v, want[1])):
        for i, c in enumerate(ctx):
            ids = tables[i][:-(-c // bs)]
            rows = (pool[ids] * scale[ids][:, None, :, None]).flatten(0, 1)[:c]
            assert torch.equal(got[fs[i]:fs[i + 1]].cpu(), rows.to(DT[dtype]))
    assert int(err) == 0


@pytest.mark.gpu
def test_append_boundaries_and_non_finite_rows():
    """absmax at 127 steps and just above it, zeros, subnormals, the largest values, infinities and NaN."""
    d, bs = 64, 16
    tops = [127.0, 127.25, 127 * 2.0 ** -5, 128.0, 0.0, 2.0 ** -24, 65504.0, 1e-45, 3.0e38, 2.0 ** -119, 1.0]
    x = torch.zeros(len(tops), 1, d)
    for i, t in enumerate(tops):
        x[i, 0, 0], x[i, 0, 1], x[i, 0, 2] = t, -t / 3, t / 2
    x[10, 0, 5], x[10, 0, 6], x[10, 0, 7] = math.inf, -math.inf, math.nan
    for dtype in ("f32", "f16", "bf16"):
        y = x.clone()
        if dtype != "f32":
            y[7:10] = 0.5
        y = y.to(DT[dtype])
        n = len(tops)
        tables = [[i] for i in range(n)]
        pool, scale = torch.zeros(n, bs, 1, d), torch.zeros(n, 1)
        dev = [pool.to(torch.int8).cuda(), pool.to(torch.int8).cuda(), scale.cuda(), scale.cuda()]
        ops.reshape_and_cache_int8(y.cuda(), y.cuda(), *dev, ints(tables), ints([1] * n), ints(list(range(n + 1))))
        p, s = pool.double(), scale.double()
        oracle_append(p, s, y, tables, [1] * n, list(range(n + 1)), bs)
        assert torch.equal(dev[0].cpu().double(), p) and torch.equal(dev[3].cpu().double(), s)


@pytest.mark.gpu
def test_a_growing_block_is_off_by_less_than_a_step():
    """Sixteen tokens one by one, each louder than the last: within one step of the block's final scale."""
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(16, 1, 64, generator=g) * torch.exp2(torch.arange(16.0) / 2)[:, None, None]).half()
    dev = [torch.zeros(1, 16, 1, 64, dtype=torch.int8, device="cuda") for _ in range(2)] + \
          [torch.zeros(1, 1, device="cuda") for _ in range(2)]
    for t in range(16):
        ops.reshape_and_cache_int8(x[t:t + 1].cuda(), x[t:t + 1].cuda(), *dev, ints([[0]]), ints([t + 1]), ints([0, 1]))
    k, _ = ops.fetch_int8(*dev, ints([[0]]), ints([16]), ints([0, 16]), 16, torch.float32)
    assert (k.cpu().double() - x.double()).abs().max() < float(dev[2])  # 1/2 + 1/4 + ... of a step


# ---- attention

def attend(q, k, v, prior, scale):
    """Rows q [n, Hq, D] over k, v [keys, Hkv, D] (float64), row r sees keys 0 .. prior + r: (o, A, S, S_max)."""
    n, hq, d = q.shape
    grp = hq // k.shape[1]
    k, v = k.repeat_interleave(grp, 1), v.repeat_interleave(grp, 1)
    hidden = torch.arange(k.shape[0])[None, :] > prior + torch.arange(n)[:, None]
    s = torch.einsum("nhd,khd->hnk", q, k) * scale
    p = torch.softmax(s.masked_fill(hidden, -math.inf), dim=-1)
    mag = (torch.einsum("nhd,khd->hnk", q.abs(), k.abs()) * scale).masked_fill(hidden, 0).amax(-1)      # [H, n]
    top = q.abs().amax(-1).T * k.abs().sum(-1).amax(0)[:, None] * scale                                   # [H, n]
    return (torch.einsum("hnk,khd->nhd", p, v), torch.einsum("hnk,khd->nhd", p, v.abs()), mag.T[..., None], top.T[..., None])


def tolerance(dt, o, A, S, S_max, n, vmax, d, u_p=None):
    part = 2.0 ** -22 if dt == torch.float32 else u(torch.float16) if u_p is None else u_p
    dx = (16 + d / 2 + 2) * 2.0 ** -23 * S + (2.0 ** -22 * S_max if dt == torch.float32 else 0)
    return u(dt) * o.abs() + A * (part * 1.01 + 2 * dx + (n / 16 + 64) * 2.0 ** -23) + n * 2.0 ** -25 * vmax


def check_rows(got, dt, q, k, v, prior, scale, u_p=None):
    o, A, S, S_max = attend(q.double(), k, v, prior, scale)
    tol = tolerance(dt, o, A, S, S_max, k.shape[0], float(v.abs().max()), q.shape[2], u_p)
    off = (got.double() - o).abs()
    assert bool((off <= tol).all()), f"off by up to {float((off / tol).max()):.2f} of the bound"


def values(pool, scale, table, c, bs):
    ids = table[:-(-c // bs)]
    return (pool[ids].double() * scale[ids].double()[:, None, :, None]).flatten(0, 1)[:c]


CONTEXTS = {
    "one key": [1],
    "edges": [1, 15, 16, 17, 31, 32, 33, 0, 47, 48, 49, 0],
    "long": [5000],
    "mixed": [0, 3, 700, 16, 2049, 1, 0, 90, 1000, 5],
    "many": [(i * 37) % 130 for i in range(300)],
}


@pytest.mark.gpu
@pytest.mark.parametrize("ctxs", list(CONTEXTS))
@pytest.mark.parametrize("dtype,hq,hkv,d,bs", [
    ("f16", 14, 2, 64, 16), ("bf16", 14, 2, 64, 16), ("f32", 14, 2, 64, 16), ("f16", 12, 1, 64, 32), ("bf16", 32, 8, 128, 32),
    ("f32", 6, 3, 128, 16), ("f16", 40, 2, 128, 16), ("f32", 16, 1, 128, 16), ("bf16", 20, 20, 64, 48), ("f32", 9, 1, 64, 16)])
def test_decode(ctxs, dtype, hq, hkv, d, bs):
    ctx, dt = CONTEXTS[ctxs], DT[dtype]
    tables, nb = layout(ctx, bs, 11, extra_cols=2)
    (kp, ks), (vp, vs) = random_pool(nb, bs, hkv, d, 1), random_pool(nb, bs, hkv, d, 2)
    g = torch.Generator().manual_seed(4)
    q = (torch.randn(len(ctx), hq, d, generator=g) * 2).to(dt)
    scale = d ** -0.5
    err = ops.new_error_flags("cuda")
    out = ops.paged_decode_attention_int8(q.cuda(), kp.cuda(), vp.cuda(), ks.cuda(), vs.cuda(), ints(tables), ints(ctx), scale, err=err).cpu()
    assert int(err) == 0
    pick = range(len(ctx)) if len(ctx) < 50 else range(0, len(ctx), 7)
    for i in pick:
        if ctx[i] == 0:
            assert bool((out[i] == 0).all())
            continue
        check_rows(out[i:i + 1], dt, q[i:i + 1], values(kp, ks, tables[i], ctx[i], bs), values(vp, vs, tables[i], ctx[i], bs),
                   ctx[i] - 1, scale)


@pytest.mark.gpu
def test_decode_in_parts_of_the_batch():
    """More sequences than one launch takes, strided q and out rows, rows past the batch left as they are."""
    ctx = [(i * 7) % 23 for i in range(1100)]
    bs, hq, hkv, d = 16, 14, 2, 64
    tables, nb = layout(ctx, bs, 5)
    (kp, ks), (vp, vs) = random_pool(nb, bs, hkv, d, 1), random_pool(nb, bs, hkv, d, 2)
    q = torch.randn(len(ctx), hq + 3, d, generator=torch.Generator().manual_seed(1)).half()
    qd = q.cuda()[:, :hq]
    out = torch.full((len(ctx) + 5, hq + 1, d), 7.0, dtype=torch.float16, device="cuda")
    ops.paged_decode_attention_int8(qd, kp.cuda(), vp.cuda(), ks.cuda(), vs.cuda(), ints(tables), ints(ctx), 0.125,
                                    out=out[:len(ctx), :hq])
    out = out.cpu()
    assert bool((out[len(ctx):] == 7).all()) and bool((out[:, hq:] == 7).all())
    for i in list(range(0, 1100, 53)) + [1023, 1024, 1099]:
        if ctx[i]:
            check_rows(out[i:i + 1, :hq], torch.float16, q[i:i + 1, :hq], values(kp, ks, tables[i], ctx[i], bs),
                       values(vp, vs, tables[i], ctx[i], bs), ctx[i] - 1, 0.125)
        else:
            assert bool((out[i, :hq] == 0).all())


@pytest.mark.gpu
def test_decode_scales_far_apart():
    """Blocks whose scales differ by 2^30, quiet ones first and loud ones first; scores that jump by hundreds."""
    bs, hq, hkv, d, ctx = 16, 14, 2, 64, [400, 400, 330]
    tables, nb = layout(ctx, bs, 2)
    (kp, ks), (vp, vs) = random_pool(nb, bs, hkv, d, 1), random_pool(nb, bs, hkv, d, 2)
    for j in range(25):
        vs[tables[0][j]] = 2.0 ** (-20 + j)
        vs[tables[1][j]] = 2.0 ** (10 - j)
    for j in range(21):
        ks[tables[2][j]] = 2.0 ** (-2 if j % 5 == 4 else -8)
    q = torch.randn(3, hq, d, generator=torch.Generator().manual_seed(9)).half()
    out = ops.paged_decode_attention_int8(q.cuda(), kp.cuda(), vp.cuda(), ks.cuda(), vs.cuda(), ints(tables), ints(ctx), 0.125).cpu().float()
    # 16-bit results near fp16's largest value saturate; these stay below it
    for i in range(3):
        check_rows(out[i:i + 1].half(), torch.float16, q[i:i + 1], values(kp, ks, tables[i], ctx[i], bs),
                   values(vp, vs, tables[i], ctx[i], bs), ctx[i] - 1, 0.125)


@pytest.mark.gpu
def test_decode_bf16_rows_past_fp16_range():
    bs, hq, hkv, d, ctx = 16, 6, 2, 64, [50, 200]
    tables, nb = layout(ctx, bs, 2)
    (kp, ks), (vp, vs) = random_pool(nb, bs, hkv, d, 1), random_pool(nb, bs, hkv, d, 2)
    ks = ks * 2.0 ** -20
    for dt in (torch.bfloat16, torch.float32):
        q = (torch.randn(2, hq, d, generator=torch.Generator().manual_seed(9)) * 2.0 ** 20).to(dt)
        out = ops.paged_decode_attention_int8(q.cuda(), kp.cuda(), vp.cuda(), ks.cuda(), vs.cuda(), ints(tables), ints(ctx), 0.125).cpu()
        for i in range(2):
            check_rows(out[i:i + 1], dt, q[i:i + 1], values(kp, ks, tables[i], ctx[i], bs), values(vp, vs, tables[i], ctx[i], bs),
                       ctx[i] - 1, 0.125)


@pytest.mark.gpu
def test_decode_same_bits_and_bad_ids():
    """Two calls give the same bits; a bad id is flagged; a context past its table is cut to the table."""
    ctx, bs, hq, hkv, d = CONTEXTS["mixed"], 16, 14, 2, 64
    tables, nb = layout(ctx, bs, 2)
    (kp, ks), (vp, vs) = random_pool(nb, bs, hkv, d, 1), random_pool(nb, bs, hkv, d, 2)
    q = torch.randn(len(ctx), hq, d, generator=torch.Generator().manual_seed(9)).half().cuda()
    dev = [t.cuda() for t in (kp, vp, ks, vs)]
    a = ops.paged_decode_attention_int8(q, *dev, ints(tables), ints(ctx), 0.125)
    b = ops.paged_decode_attention_int8(q, *dev, ints(tables), ints(ctx), 0.125)
    assert torch.equal(a, b)
    err = ops.new_error_flags("cuda")
    bad = [list(r) for r in tables]
    bad[2][3] = nb
    ops.paged_decode_attention_int8(q, *dev, ints(bad), ints(ctx), 0.125, err=err)
    assert int(err) == _lib.FLAG_BLOCK_OUT_OF_RANGE
    err.zero_()
    long = list(ctx)
    long[4] = len(tables[0]) * bs + 9
    c = ops.paged_decode_attention_int8(q, *dev, ints(tables), ints(long), 0.125, err=err)
    assert int(err) == _lib.FLAG_CONTEXT_EXCEEDS_TABLE and torch.equal(c[5:], a[5:])


CHUNKS = {
    "one": ([0], [1]),
    "small": ([0, 7, 70, 33], [5, 1, 45, 0]),
    "tiles": ([128, 0, 1, 255], [128, 129, 300, 17]),
    "behind": ([1500, 3], [200, 257]),
    "far behind": ([6000, 0, 2500], [3, 40, 90]),  # few rows behind many keys: split over the keys
    "far alone": ([9001], [2]),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(CHUNKS))
@pytest.mark.parametrize("dtype,hq,hkv,d,bs", [("f16", 14, 2, 64, 16), ("bf16", 14, 2, 64, 32), ("f32", 6, 3, 64, 16),
                                               ("bf16", 16, 2, 128, 16), ("f16", 20, 1, 128, 48), ("f32", 4, 4, 128, 32)])
def test_chunks(name, dtype, hq, hkv, d, bs):
    prior, new = CHUNKS[name]
    ctx, dt = [p + n for p, n in zip(prior, new)], DT[dtype]
    starts = starts_of(new)
    tables, nb = layout(ctx, bs, 11, extra_cols=1)
    (kp, ks), (vp, vs) = random_pool(nb, bs, hkv, d, 1), random_pool(nb, bs, hkv, d, 2)
    g = torch.Generator().manual_seed(4)
    q = torch.randn(starts[-1] + 3, hq, d, generator=g).to(dt)
    out = torch.full(q.shape, 7.0, dtype=dt, device="cuda")
    err = ops.new_error_flags("cuda")
    ops.paged_prefill_attention_int8(q.cuda(), kp.cuda(), vp.cuda(), ks.cuda(), vs.cuda(), ints(tables), ints(starts), ints(prior),
                                     max(new), d ** -0.5, out=out, err=err)
    assert int(err) == 0
    out = out.cpu()
    assert bool((out[starts[-1]:] == 7).all())  # rows behind the last sequence stay as they were
    for i in range(len(ctx)):
        if new[i]:
            check_rows(out[starts[i]:starts[i + 1]], dt, q[starts[i]:starts[i + 1]], values(kp, ks, tables[i], ctx[i], bs),
                       values(vp, vs, tables[i], ctx[i], bs), prior[i], d ** -0.5,
                       # P in q's type, its exponentials to 7.5e-5
                       u_p=u(dt) + 2.0 ** -13)


@pytest.mark.gpu
def test_a_decode_loop_of_the_operators_together():
    """Tables from lengths, append, attention, step by step on the GPU: equal to a loop that fetches and attends in 64 bits."""
    bs, hq, hkv, d, dt = 16, 14, 2, 64, torch.float16
    g = torch.Generator().manual_seed(3)
    lens = [0, 5, 30, 16]
    B, width, nb = len(lens), 6, 30
    tables = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(nb, generator=g).int().cuda()
    n_free = ints([nb])
    dev = [torch.zeros(nb, bs, hkv, d, dtype=torch.int8, device="cuda") for _ in range(2)] + \
          [torch.zeros(nb, hkv, device="cuda") for _ in range(2)]
    err = ops.new_error_flags("cuda")
    prior = ints([0] * B)
    for step, new in enumerate([[3, 5, 30, 16], [1] * 4, [1] * 4, [20, 1, 0, 33]]):
        T = sum(new)
        x = torch.randn(T, hq + 2 * hkv, d, generator=g).to(dt)
        xd = x.cuda()
        st = ops.build_step_tables(tables, free, n_free, prior, ints(new), bs, T, err=err)
        ops.reshape_and_cache_int8(xd[:, hq:hq + hkv], xd[:, hq + hkv:], *dev, tables, st.context_lens, st.query_start_loc, err=err)
        q = xd[:, :hq]
        if new == [1] * 4:
            out = ops.paged_decode_attention_int8(q, *dev, tables, st.context_lens, 0.125, err=err)
        else:
            out = ops.paged_prefill_attention_int8(q, *dev, tables, st.query_start_loc, prior, max(new), 0.125, err=err)
        ctx = st.context_lens.tolist()
        fs = starts_of(ctx)
        k, v = ops.fetch_int8(*dev, tables, st.context_lens, ints(fs), fs[-1], torch.float32, err=err)
        starts = starts_of(new)
        for i in range(B):
            if new[i]:
                check_rows(out[starts[i]:starts[i + 1]].cpu(), dt, x[starts[i]:starts[i + 1], :hq], k[fs[i]:fs[i + 1]].cpu().double(),
                           v[fs[i]:fs[i + 1]].cpu().double(), ctx[i] - new[i], 0.125, u_p=u(dt) + 2.0 ** -13)
        prior, n_free = st.context_lens, st.n_free
    assert int(err) == 0


@pytest.mark.gpu
def test_captured_decode_follows_its_inputs():
    """Append and decode captured once and replayed with other lengths, rows and tables."""
    bs, hq, hkv, d = 16, 14, 2, 64
    ctx = [40, 17, 300, 1]
    tables, nb = layout([320] * 4, bs, 2)
    (kp, ks), (vp, vs) = random_pool(nb, bs, hkv, d, 1), random_pool(nb, bs, hkv, d, 2)
    dev = [t.cuda() for t in (kp, vp, ks, vs)]
    t, c = ints(tables), ints(ctx)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, hq + 2 * hkv, d, generator=g).half().cuda()
    one = ints([0, 1, 2, 3, 4])
    ws = torch.empty(ops.decode_int8_workspace_bytes(hq, d), dtype=torch.uint8, device="cuda")
    out = torch.empty(4, hq, d, dtype=torch.float16, device="cuda")

    def step():
        ops.reshape_and_cache_int8(x[:, hq:hq + hkv], x[:, hq + hkv:], *dev, t, c, one)
        ops.paged_decode_attention_int8(x[:, :hq], *dev, t, c, 0.125, workspace=ws, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for lens in ([41, 18, 301, 2], [0, 320, 5, 16]):
        c.copy_(ints(lens))
        x.copy_(torch.randn(4, hq + 2 * hkv, d, generator=g).half())
        graph.replay()
        got = out.clone()
        step()
        assert torch.equal(got, out)
        fs = starts_of(lens)
        k, v = ops.fetch_int8(*dev, t, c, ints(fs), fs[-1], torch.float32)
        for i, n in enumerate(lens):
            if n:
                check_rows(got[i:i + 1].cpu(), torch.float16, x[i:i + 1, :hq].cpu(), k[fs[i]:fs[i + 1]].cpu().double(),
                           v[fs[i]:fs[i + 1]].cpu().double(), n - 1, 0.125)
            else:
                assert bool((got[i] == 0).all())


# ---- refusals

def test_c_refusals():
    L = _lib.load()
    names = dict(k=FAKE, v=FAKE, ks=128, vs=128, kp=FAKE, vp=FAKE, ksc=FAKE, vsc=FAKE, nb=64, tables=FAKE, bts=8, width=8,
                 ctx=FAKE, qsl=FAKE, n=2, T=5, hkv=2, d=64, bs=16, dt=1, err=None, stream=None)
    for f in (L.pkv_reshape_and_cache_int8, L.pkv_fetch_int8):
        def call(**kw):
            return f(*{**names, **kw}.values())

        assert call(n=0) == call(T=0) == _lib.OK
        for name in ("k", "v", "kp", "vp", "ksc", "vsc", "tables", "ctx", "qsl"):
            assert call(**{name: None}) == _lib.ERR_NULL_POINTER, name
        assert call(n=-1) == call(T=-1) == call(ks=127) == call(vs=1) == call(bts=7) == call(nb=0) == call(hkv=0) == _lib.ERR_BAD_SHAPE
        assert call(dt=3) == _lib.ERR_BAD_DTYPE
        assert call(d=80, ks=160, vs=160) == call(bs=8) == _lib.ERR_UNSUPPORTED
        assert call(kp=ctypes.c_void_p(0x1008)) == call(k=ctypes.c_void_p(0x1001)) == _lib.ERR_MISALIGNED
    dec = dict(out=FAKE, os=896, q=FAKE, qs=896, kp=FAKE, vp=FAKE, ksc=FAKE, vsc=FAKE, nb=64, tables=FAKE, bts=8, width=8, ctx=FAKE,
               n=2, hq=14, hkv=2, d=64, bs=16, scale=0.125, dt=1, ws=FAKE, wsb=1 << 30, err=None, stream=None)

    def call(**kw):
        return L.pkv_paged_decode_attention_int8(*{**dec, **kw}.values())

    assert call(n=0) == _lib.OK
    for name in ("out", "q", "kp", "vp", "ksc", "vsc", "tables", "ctx", "ws"):
        assert call(**{name: None}) == _lib.ERR_NULL_POINTER, name
    assert call(n=-1) == call(hq=13) == call(qs=895) == call(os=10) == call(bts=7) == _lib.ERR_BAD_SHAPE
    assert call(n=1024, width=1 << 22, bts=1 << 22) == _lib.ERR_BAD_SHAPE  # tiles past 32 bits
    assert call(dt=-1) == _lib.ERR_BAD_DTYPE
    assert call(wsb=L.pkv_decode_int8_workspace_bytes(14, 64) - 1) == _lib.ERR_WORKSPACE_TOO_SMALL
    assert call(ws=ctypes.c_void_p(0x1004)) == _lib.ERR_MISALIGNED
    assert call(d=32, qs=896) == call(bs=24) == _lib.ERR_UNSUPPORTED
    assert L.pkv_decode_int8_workspace_bytes(0, 64) == 0 and L.pkv_prefill_int8_scratch_bytes(1, 5, 0, 14, 2, 64, 16, 1) == 0
    # K and V rows of two sequences, 9 blocks of 16 rounded up to 256 rows; no splitting of fp32 rows
    assert L.pkv_prefill_int8_scratch_bytes(2, 9, 9, 14, 2, 64, 16, 0) == 2 * 2 * 256 * 2 * 64 * 4
    assert L.pkv_prefill_int8_scratch_bytes(2, 9, 9, 14, 2, 64, 16, 1) == 2 * 2 * 256 * 2 * 64 * 2
    # long ones in 16-bit types also get room for the parts of a split
    assert L.pkv_prefill_int8_scratch_bytes(2, 9, 512, 14, 2, 64, 16, 0) == 2 * 2 * 8192 * 2 * 64 * 4
    assert L.pkv_prefill_int8_scratch_bytes(2, 9, 512, 14, 2, 64, 16, 1) > 2 * 2 * 8192 * 2 * 64 * 2
    pre = dict(out=FAKE, os=896, q=FAKE, qs=896, kp=FAKE, vp=FAKE, ksc=FAKE, vsc=FAKE, nb=64, tables=FAKE, bts=8, width=8, qsl=FAKE,
               prior=FAKE, n=2, T=5, hq=14, hkv=2, d=64, bs=16, scale=0.125, dt=1, sc=FAKE, scb=1 << 30, err=None, stream=None)

    def call(**kw):
        return L.pkv_paged_prefill_attention_int8(*{**pre, **kw}.values())

    assert call(n=0) == call(T=0) == _lib.OK
    for name in ("out", "q", "kp", "ksc", "tables", "qsl", "prior", "sc"):
        assert call(**{name: None}) == _lib.ERR_NULL_POINTER, name
    assert call(scale=0.0) == call(scale=float("nan")) == call(T=-1) == call(n=70000) == _lib.ERR_BAD_SHAPE
    assert call(scb=10) == _lib.ERR_WORKSPACE_TOO_SMALL and call(sc=ctypes.c_void_p(0x1010)) == _lib.ERR_MISALIGNED


def test_wrappers_refuse_cpu_tensors():
    p, s = torch.zeros(2, 16, 2, 64, dtype=torch.int8), torch.zeros(2, 2)
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(1, 2, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.reshape_and_cache_int8(x, x, p, p, s, s, i[:, None], i[:1], i)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_decode_attention_int8(x, p, p, s, s, i[:, None], i, 1.0)


@pytest.mark.gpu
def test_wrapper_refusals():
    z = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    p, s = z(4, 16, 2, 64, dt=torch.int8), z(4, 2, dt=torch.float32)
    t, c, qsl, x, q = ints([[0], [1]]), ints([1, 1]), ints([0, 1, 2]), z(2, 2, 64), z(2, 14, 64)
    app = dict(k=x, v=x, k_pool=p, v_pool=p.clone(), k_scale=s, v_scale=s.clone(), block_tables=t, context_lens=c, query_start_loc=qsl)
    ops.reshape_and_cache_int8(**app)
    for kw, exc in [(dict(k_pool=z(4, 16, 2, 64)), TypeError), (dict(k_scale=z(4, 2)), TypeError), (dict(k_scale=z(4, 16, 2, dt=torch.float32)), ValueError),
                    (dict(k=z(2, 2, 64, dt=torch.float32)), TypeError), (dict(k=z(2, 1, 64)), ValueError), (dict(context_lens=ints([1])), ValueError),
                    (dict(query_start_loc=ints([0, 1, 2], torch.int64)), TypeError), (dict(block_tables=ints([[0]])), ValueError),
                    (dict(k=x.double(), v=x.double()), TypeError), (dict(k=z(2, 64, 2).transpose(1, 2)), ValueError)]:
        with pytest.raises(exc):
            ops.reshape_and_cache_int8(**{**app, **kw})
    dec = dict(q=q, k_pool=p, v_pool=p, k_scale=s, v_scale=s, block_tables=t, context_lens=c, scale=0.125)
    ops.paged_decode_attention_int8(**dec)
    for kw, exc in [(dict(q=z(2, 13, 64)), ValueError), (dict(q=z(2, 14, 128)), ValueError), (dict(context_lens=ints([1])), ValueError),
                    (dict(out=z(2, 14, 64, dt=torch.float32)), ValueError), (dict(workspace=z(16, dt=torch.uint8)), _lib.PagedKVError),
                    (dict(err=z(1)), TypeError), (dict(k_pool=z(4, 8, 2, 64, dt=torch.int8), v_pool=z(4, 8, 2, 64, dt=torch.int8)), _lib.PagedKVError)]:
        with pytest.raises(exc):
            ops.paged_decode_attention_int8(**{**dec, **kw})
