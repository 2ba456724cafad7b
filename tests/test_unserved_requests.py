"""Requests that build_step_tables does not serve (the free list is short): through append,
chunk attention and fetch over int8 pools they leave the others as they are and give zeros."""

import ctypes

import pytest
import torch

from pagedkv import _lib, ops
from test_int8_pools import DT, ints, random_pool, starts_of

FAKE = ctypes.c_void_p(0x1000)


def step(prior, new, n_free, dtype, hq, hkv, d, bs, served):
    """A step over `served` requests of the batch (all of them, or those that get blocks)."""
    n, dt = len(prior), DT[dtype]
    width = max(-(-(p + m) // bs) for p, m in zip(prior, new))
    have = [-(-p // bs) for p in prior]
    pool = sum(have) + n_free + 5
    # what a table holds behind a request's blocks: the first request's, another's, out of range
    tables, at = [], 0
    for i, h in enumerate(have):
        tables.append(list(range(at, at + h)) + [[0, max(0, at - 1), pool + 7][i % 3]] * (width - h))
        at += h
    (kp, ks), (vp, vs) = random_pool(pool, bs, hkv, d, 1), random_pool(pool, bs, hkv, d, 2)
    dev = [t.cuda() for t in (kp, vp, ks, vs)]
    T = sum(new)
    x = torch.randn(T, hq + 2 * hkv, d, generator=torch.Generator().manual_seed(5)).to(dt)
    prior, new = prior[:served], new[:served]
    T = sum(new)
    xd, tab, err = x[:T].cuda(), ints(tables[:served]), ops.new_error_flags("cuda")
    p = ints(prior)
    free = torch.arange(pool - 1, pool - 1 - n_free, -1, dtype=torch.int32, device="cuda")
    st = ops.build_step_tables(tab, free, ints([n_free]), p, ints(new), bs, T, err=err)
    built = int(err)
    err.zero_()
    ops.reshape_and_cache_int8(xd[:, hq:hq + hkv], xd[:, hq + hkv:], *dev, tab, st.context_lens, st.query_start_loc, err=err)
    out = torch.full((T + 2, hq, d), 7.0, dtype=dt, device="cuda")
    ops.paged_prefill_attention_int8(xd[:, :hq], *dev, tab, st.query_start_loc, p, max(new), 0.125, out=out[:T], err=err,
                                     context_lens=st.context_lens)
    k, v = ops.fetch_int8(*dev, tab, st.context_lens, st.query_start_loc, T, dt, err=err)
    assert int(err) == 0 and bool((out[T:] == 7).all())
    return out[:T].cpu(), k.cpu(), v.cpu(), [t.cpu() for t in dev], built, st.context_lens.tolist()


BATCHES = {
    # prior, new, requests whose blocks are there (the next one is a block short, if it needs any)
    "prompts": ([0, 20, 5, 0], [40, 30, 70, 9], 2),
    "behind long contexts": ([9000, 3, 5000, 100], [20, 16, 33, 1], 2),  # split over the keys in 16 bits
    "many": ([(i * 7) % 40 for i in range(500)], [(i * 5) % 7 for i in range(500)], 200),  # taken as they come
    "the first": ([0, 0], [40, 3], 0),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(BATCHES))
@pytest.mark.parametrize("dtype,hq,hkv,d,bs", [("f16", 14, 2, 64, 16), ("bf16", 8, 2, 128, 32), ("f32", 6, 3, 64, 16)])
def test_unserved_requests_give_zeros(name, dtype, hq, hkv, d, bs):
    prior, new, served = BATCHES[name]
    need = [-(-(p + m) // bs) - -(-p // bs) for p, m in zip(prior, new)]
    n_free = sum(need[:served]) + max(0, need[served] - 1)
    count = next(i for i in range(len(need)) if sum(need[:i + 1]) > n_free)
    out, k, v, pools, flags, ctx = step(prior, new, n_free, dtype, hq, hkv, d, bs, len(prior))
    assert flags == _lib.FLAG_OUT_OF_BLOCKS and ctx[count] == 0 and ctx[count:] == [0] * (len(prior) - count)
    rows = starts_of(new)[count]
    assert not bool(out[rows:].any()) and not bool(k[rows:].any()) and not bool(v[rows:].any())
    if not rows:
        return
    alone = step(prior, new, n_free, dtype, hq, hkv, d, bs, count)
    assert alone[4] == 0 and torch.equal(k[:rows], alone[1]) and torch.equal(v[:rows], alone[2])
    assert all(torch.equal(a, b) for a, b in zip(pools, alone[3]))
    # (a split over the keys goes by the batch: other partial sums)
    tol = {"f16": 2.0 ** -9, "bf16": 2.0 ** -6, "f32": 2.0 ** -18}[dtype]
    assert float((out[:rows].double() - alone[0].double()).abs().max()) <= tol * float(alone[0].abs().max())


def test_c_refusals():
    L = _lib.load()
    pre = dict(out=FAKE, os=896, q=FAKE, qs=896, kp=FAKE, vp=FAKE, ksc=FAKE, vsc=FAKE, nb=64, tables=FAKE, bts=8, width=8, qsl=FAKE,
               prior=FAKE, ctx=None, n=2, T=5, hq=14, hkv=2, d=64, bs=16, scale=0.125, dt=1, sc=FAKE, scb=1 << 30, err=None, stream=None)

    def call(**kw):
        return L.pkv_paged_prefill_attention_int8_served(*{**pre, **kw}.values())

    assert call(n=0) == call(T=0, ctx=FAKE) == _lib.OK
    for name in ("out", "q", "kp", "ksc", "tables", "qsl", "prior", "sc"):
        assert call(**{name: None}) == _lib.ERR_NULL_POINTER, name
    assert call(scale=0.0) == call(hq=13) == _lib.ERR_BAD_SHAPE
    assert call(scb=10) == _lib.ERR_WORKSPACE_TOO_SMALL


@pytest.mark.gpu
def test_wrapper_refusals():
    z = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    p, s = z(4, 16, 2, 64, dt=torch.int8), z(4, 2, dt=torch.float32)
    good = dict(q=z(4, 14, 64), k_pool=p, v_pool=p, k_scale=s, v_scale=s, block_tables=ints([[0], [1]]), query_start_loc=ints([0, 2, 4]),
                num_prior=ints([0, 0]), max_query_len=2, scale=0.125, context_lens=ints([2, 2]))
    ops.paged_prefill_attention_int8(**good)
    for kw, exc in [(dict(context_lens=ints([2])), ValueError), (dict(context_lens=ints([2, 2], torch.int64)), TypeError),
                    (dict(context_lens=torch.tensor([2, 2], dtype=torch.int32)), RuntimeError)]:
        with pytest.raises(exc):
            ops.paged_prefill_attention_int8(**{**good, **kw})
