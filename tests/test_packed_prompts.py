"""Packed-prompt attention against 64-bit arithmetic, and its refusals.

Tolerances as in test_int8_pools.py, with P rounded to the input type (its
exponentials to 2^-13 relative in 16 bits, 2^-21 in fp32)."""

import ctypes
import math

import pytest
import torch

from pagedkv import _lib, ops
from test_int8_pools import DT, attend, ints, starts_of, tolerance, u

FAKE = ctypes.c_void_p(0x1000)


def check(out, dt, x, hq, hkv, starts, scale):
    q, k, v = x[:, :hq].double(), x[:, hq:hq + hkv].double(), x[:, hq + hkv:hq + 2 * hkv].double()
    for a, b in zip(starts, starts[1:]):
        if a == b:
            continue
        o, A, S, S_max = attend(q[a:b], k[a:b], v[a:b], 0, scale)
        u_p = u(dt) + 2.0 ** -13 if dt != torch.float32 else 2.0 ** -21
        tol = tolerance(dt, o, A, S, S_max, b - a, float(v[a:b].abs().max()), q.shape[2], u_p)
        off = (out[a:b].double() - o).abs()
        assert bool((off <= tol).all()), f"rows {a}:{b} off by up to {float((off / tol).max()):.2f} of the bound"


LENGTHS = {
    "one": [1],
    "short": [1, 0, 2, 17, 18, 19, 0, 35, 36, 37, 5],
    "tiles": [63, 64, 65, 127, 128, 129, 255, 256, 257],
    "long": [1500],
    "many": [(i * 29) % 60 for i in range(70)],
    "skewed": [3, 900, 1, 0, 40, 300, 0],
}
HEADS = [("f16", 14, 2, 64), ("bf16", 14, 2, 64), ("f32", 14, 2, 64), ("f16", 8, 8, 64), ("bf16", 32, 8, 128), ("f32", 6, 3, 128),
         ("f16", 12, 1, 128), ("bf16", 40, 1, 64), ("f16", 3, 1, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(LENGTHS))
@pytest.mark.parametrize("dtype,hq,hkv,d", HEADS)
def test_against_64_bits(name, dtype, hq, hkv, d):
    dt, starts = DT[dtype], starts_of(LENGTHS[name])
    T = starts[-1]
    x = (torch.randn(T + 5, hq + 2 * hkv, d, generator=torch.Generator().manual_seed(T)) * 1.5).to(dt)
    x[T:] = math.nan  # rows behind the last sequence
    xd = x.cuda()
    out = torch.full((T + 5, hq, d), 7.0, dtype=dt, device="cuda")
    err = ops.new_error_flags("cuda")
    ops.packed_prompt_attention(xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:], ints(starts), d ** -0.5, out=out, err=err)
    out = out.cpu()
    assert int(err) == 0 and bool((out[T:] == 7).all())
    check(out, dt, x, hq, hkv, starts, d ** -0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [("f16", 64), ("bf16", 128), ("f32", 64)])
def test_what_a_row_must_not_see_never_enters_it(dtype, d):
    """Infinities and NaN in a later row's and the next prompt's K and V: earlier rows are as without them."""
    dt, hq, hkv, starts = DT[dtype], 14, 2, [0, 40, 170, 300]
    x = torch.randn(300, hq + 2 * hkv, d, generator=torch.Generator().manual_seed(2)).to(dt)
    y = x.clone()
    y[30, hq:] = math.nan          # K and V of row 30 of the first prompt
    y[160, hq + hkv:] = math.inf   # V near the end of the second
    y[171, hq:hq + hkv] = -math.inf
    run = lambda t: ops.packed_prompt_attention(t[:, :hq], t[:, hq:hq + hkv], t[:, hq + hkv:], ints(starts), d ** -0.5).cpu()  # noqa: E731
    a, b = run(x.cuda()), run(y.cuda())
    clean = torch.cat([a[:30], a[40:160], a[170:171]])
    got = torch.cat([b[:30], b[40:160], b[170:171]])
    assert bool(torch.isfinite(got).all())
    check(torch.cat([b[:30], a[30:40], b[40:160], a[160:170], b[170:171], a[171:]]), dt, x, hq, hkv, starts, d ** -0.5)
    assert float((clean.double() - got.double()).abs().max()) < 0.05
    assert not bool(torch.isfinite(b[30:40]).any()) and not bool(torch.isfinite(b[160:170]).any())


@pytest.mark.gpu
def test_large_scores_and_equal_scores():
    """Scores of several hundred (one key takes all) and all-equal scores (the mean)."""
    hq, hkv, d, starts = 14, 2, 64, [0, 300]
    x = torch.randn(300, hq + 2 * hkv, d, generator=torch.Generator().manual_seed(3)).half()
    x[:, :hq] *= 8
    x[:, hq:hq + hkv] *= 8
    xd = x.cuda()
    out = ops.packed_prompt_attention(xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:], ints(starts), 0.125).cpu()
    check(out, torch.float16, x, hq, hkv, starts, 0.125)
    x[:, :hq] = 0
    xd = x.cuda()
    out = ops.packed_prompt_attention(xd[:, :hq], xd[:, hq:hq + hkv], xd[:, hq + hkv:], ints(starts), 0.125).cpu()
    check(out, torch.float16, x, hq, hkv, starts, 0.125)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_rows_at_any_stride_and_alignment(dtype):
    """Row strides and first elements that no wide load can take, and out rows inside a wider buffer."""
    dt, hq, hkv, d, starts = DT[dtype], 6, 2, 64, [0, 150, 151, 260]
    for pad, off in ((1, 0), (0, 1), (8, 8)):
        width = (hq + 2 * hkv) * d + pad
        flat = torch.randn(260 * width + off, generator=torch.Generator().manual_seed(3)).to(dt).cuda()
        rows = flat[off:].view(260, width)
        x = rows[:, :(hq + 2 * hkv) * d].unflatten(1, (hq + 2 * hkv, d))
        wide = torch.full((260, hq * d + pad), 7.0, dtype=dt, device="cuda")
        out = wide[:, :hq * d].unflatten(1, (hq, d))
        ops.packed_prompt_attention(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], ints(starts), 0.125, out=out)
        check(out.cpu(), dt, x.cpu(), hq, hkv, starts, 0.125)
        assert bool((wide[:, hq * d:] == 7).all())


@pytest.mark.gpu
def test_same_bits_graph_and_other_stream():
    hq, hkv, d, starts = 14, 2, 64, [0, 5, 400, 900]
    x = torch.randn(900, hq + 2 * hkv, d, generator=torch.Generator().manual_seed(3)).half().cuda()
    args = (x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], ints(starts), 0.125)
    a = ops.packed_prompt_attention(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b = ops.packed_prompt_attention(*args)
    side.synchronize()
    out = torch.zeros_like(a)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.packed_prompt_attention(*args, out=out)
    g.replay()
    assert torch.equal(a, b) and torch.equal(a, out)
    x.copy_(torch.randn(900, hq + 2 * hkv, d, generator=torch.Generator().manual_seed(4)).half())
    g.replay()
    assert torch.equal(out, ops.packed_prompt_attention(*args))


@pytest.mark.gpu
def test_bad_starts_are_flagged():
    hq, hkv, d = 14, 2, 64
    x = torch.randn(50, hq + 2 * hkv, d).half().cuda()
    for starts in ([0, 10, 70], [0, 30, 20, 50], [-3, 20]):
        err = ops.new_error_flags("cuda")
        ops.packed_prompt_attention(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], ints(starts), 0.125, err=err)
        assert int(err) == _lib.FLAG_BAD_QUERY_LAYOUT, starts


def test_c_refusals():
    f = _lib.load().pkv_packed_prompt_attention
    base = dict(out=FAKE, os=896, q=FAKE, qs=896, k=FAKE, ks=128, v=FAKE, vs=128, qsl=FAKE, n=2, T=5, hq=14, hkv=2, d=64, scale=0.125,
                dt=1, err=None, stream=None)

    def call(**kw):
        return f(*{**base, **kw}.values())

    assert call(n=0) == call(T=0) == _lib.OK
    for name in ("out", "q", "k", "v", "qsl"):
        assert call(**{name: None}) == _lib.ERR_NULL_POINTER, name
    assert call(n=-1) == call(T=-1) == call(hq=13) == call(ks=127) == call(os=1) == call(scale=0.0) == call(scale=-1.0) == _lib.ERR_BAD_SHAPE
    assert call(T=0x7fffffff) == _lib.ERR_BAD_SHAPE
    assert call(dt=7) == _lib.ERR_BAD_DTYPE and call(d=32) == _lib.ERR_UNSUPPORTED
    assert call(q=ctypes.c_void_p(0x1001)) == _lib.ERR_MISALIGNED


@pytest.mark.gpu
def test_wrapper_refusals():
    z = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    good = dict(q=z(4, 14, 64), k=z(4, 2, 64), v=z(4, 2, 64), query_start_loc=ints([0, 4]), scale=0.125)
    ops.packed_prompt_attention(**good)
    for kw, exc in [(dict(k=z(4, 2, 64, dt=torch.float32)), TypeError), (dict(k=z(3, 2, 64)), ValueError), (dict(k=z(4, 3, 64), v=z(4, 3, 64)), ValueError),
                    (dict(query_start_loc=ints([0, 4], torch.int64)), TypeError), (dict(scale=0.0), _lib.PagedKVError), (dict(out=z(4, 14, 32)), ValueError),
                    (dict(q=torch.zeros(4, 14, 64).half()), RuntimeError), (dict(q=z(4, 14, 32), k=z(4, 2, 32), v=z(4, 2, 32)), _lib.PagedKVError)]:
        with pytest.raises(exc):
            ops.packed_prompt_attention(**{**good, **kw})
