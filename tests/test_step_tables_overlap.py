"""build_step_tables refuses outputs that lie over its inputs: every CTA reads the lengths,
the free list and its count while others write."""

import ctypes

import pytest
import torch

from pagedkv import _lib, ops
from test_int8_pools import ints

AT = {n: 0x10000 * (i + 1) for i, n in enumerate(("tables", "free", "n_free", "n_out", "prior", "new", "ctx", "qsl", "slots", "pos"))}


def c_call(**kw):
    """5 requests, 40 tokens, 30 free blocks at addresses of their own."""
    a = {**AT, **kw}
    p = {k: ctypes.c_void_p(v) for k, v in a.items()}
    return _lib.load().pkv_build_step_tables(p["tables"], 8, 8, p["free"], 30, p["n_free"], p["n_out"], p["prior"], p["new"], 5, 16,
                                             p["ctx"], p["qsl"], p["slots"], p["pos"], 40, None, None)


@pytest.mark.parametrize("out,size", [("n_out", 4), ("ctx", 20), ("qsl", 24), ("slots", 320), ("pos", 320)])
@pytest.mark.parametrize("into,room", [("n_free", 4), ("prior", 20), ("new", 20), ("free", 120)])
def test_overlaps_are_refused(out, size, into, room):
    for at in (AT[into], AT[into] + room - 4, AT[into] - size + 4):  # the whole, the last and the first word
        assert c_call(**{out: at}) == _lib.ERR_UNSUPPORTED


@pytest.mark.gpu
def test_lengths_that_advance_in_place_are_refused():
    t, prior, new = ints([[0, 0], [1, 0]]), ints([3, 16]), ints([1, 1])
    out = ops.new_step_tables(2, 2, "cuda")
    for bad in (out._replace(context_lens=prior), out._replace(query_start_loc=torch.cat([new, new])[:3], context_lens=new)):
        with pytest.raises(_lib.PagedKVError):
            ops.build_step_tables(t, ints([7, 6]), ints([2]), prior, new, 16, 2, out=bad)
    both = torch.arange(4, dtype=torch.int32, device="cuda")  # neighbours in one buffer do not overlap
    st = ops.build_step_tables(t, ints([7, 6]), ints([2]), both[:2], new, 16, 2, out=out._replace(context_lens=both[2:]))
    assert st.context_lens.tolist() == [1, 2] and both.tolist() == [0, 1, 1, 2]
