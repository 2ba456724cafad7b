"""build_step_tables against a plain Python statement of the same rules, exactly
(every output is a whole number), and its refusals."""

import ctypes
import random

import pytest
import torch

from pagedkv import _lib, ops

FAKE, FAKE2 = ctypes.c_void_p(0x1000), ctypes.c_void_p(0x2000)


def oracle(tables, free, n_free, prior, new, bs, width, n_tokens):
    """(tables, context_lens, query_start_loc, slots, positions, n_free, flags)."""
    tables = [list(r) for r in tables]
    ctx, starts, slots, pos, flags = [], [0], [], [], 0
    taken = wanted = 0
    for i, (p, n) in enumerate(zip(prior, new)):
        valid = p >= 0 and n >= 0 and p + n <= width * bs
        if not valid:
            flags |= _lib.FLAG_BAD_QUERY_LAYOUT if p < 0 or n < 0 else _lib.FLAG_CONTEXT_EXCEEDS_TABLE
            ctx.append(0)
            starts.append(starts[-1])
            continue
        have, need = -(-p // bs), -(-(p + n) // bs) - -(-p // bs)
        wanted += need
        starts.append(starts[-1] + n)
        served = wanted <= n_free and starts[-1] <= n_tokens
        if served:
            for j in range(need):
                tables[i][have + j] = free[n_free - 1 - (wanted - need) - j]
            taken = wanted
        else:
            flags |= _lib.FLAG_BAD_QUERY_LAYOUT if starts[-1] > n_tokens else _lib.FLAG_OUT_OF_BLOCKS
        ctx.append(p + n if served else 0)
        for t in range(p, p + n):
            pos.append(t)
            slots.append(tables[i][t // bs] * bs + t % bs if served else -1)
    slots = (slots + [-1] * n_tokens)[:n_tokens]
    pos = (pos + [0] * n_tokens)[:n_tokens]
    return tables, ctx, starts, slots, pos, n_free - taken, flags


def batch(seed, n, bs, p_hi, n_hi, n_lo=0):
    rng = random.Random(seed)
    prior = [rng.choice([0, bs, rng.randint(0, p_hi)]) for _ in range(n)]
    new = [rng.randint(n_lo, n_hi) for _ in range(n)]
    width = max(1, max(-(-(p + m) // bs) for p, m in zip(prior, new)) if n else 1)
    held = sum(-(-p // bs) for p in prior)
    wanted = sum(-(-(p + m) // bs) - -(-p // bs) for p, m in zip(prior, new))
    ids = list(range(held + wanted + 7))
    rng.shuffle(ids)
    tables, o = [], 0
    for p in prior:
        k = -(-p // bs)
        tables.append(ids[o:o + k] + [-9] * (width - k))
        o += k
    return prior, new, width, tables, ids[o:], wanted


def run(tables, free, n_free, prior, new, bs, n_tokens, row_pad=0, out=None):
    dev = "cuda"
    n, width = len(prior), len(tables[0]) if tables else 1
    full = torch.full((max(n, 1), width + row_pad), -9, dtype=torch.int32, device=dev)
    if n:
        full[:, :width] = torch.tensor(tables, dtype=torch.int32, device=dev)
    t = full[:, :width]
    err = ops.new_error_flags(dev)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    r = ops.build_step_tables(t, ints(free), ints([n_free]), ints(prior), ints(new), bs, n_tokens, out=out, err=err)
    return [t[:n].tolist(), r.context_lens[:n].tolist(), r.query_start_loc[:n + 1].tolist(),
            r.slot_mapping[:n_tokens].tolist(), r.positions[:n_tokens].tolist(), int(r.n_free), int(err)]


CASES = [
    # seed, requests, block size, longest prior, longest new, extra tokens
    (1, 1, 16, 0, 1, 0), (2, 1, 16, 40, 0, 3), (3, 256, 16, 4000, 1, 0), (4, 37, 8, 100, 33, 5),
    (5, 513, 16, 300, 40, 1), (6, 1025, 32, 64, 3, 0), (7, 5, 1, 9, 9, 2), (8, 3, 16, 17, 5000, 0),
    (9, 4000, 16, 50, 4, 11), (10, 60, 24, 700, 300, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("seed,n,bs,p_hi,n_hi,extra", CASES)
@pytest.mark.parametrize("short", [False, True])
def test_against_plain_rules(seed, n, bs, p_hi, n_hi, extra, short):
    prior, new, width, tables, free, wanted = batch(seed, n, bs, p_hi, n_hi)
    n_free = wanted // 2 if short else len(free)
    n_tokens = sum(new) + extra
    got = run(tables, free, n_free, prior, new, bs, n_tokens, row_pad=seed % 3)
    assert got == list(oracle(tables, free, n_free, prior, new, bs, width, n_tokens))


@pytest.mark.gpu
def test_no_requests_and_no_tokens():
    got = run([], [3, 4], 2, [], [], 16, 4)
    assert got == [[], [], [0], [-1] * 4, [0] * 4, 2, 0]
    got = run([[5, -9]], [3, 4], 2, [7], [0], 16, 0)
    assert got == [[[5, -9]], [7], [0, 0], [], [], 2, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("prior,new,n_free,n_tokens", [
    ([5, -1, 3], [4, 2, 30], 6, 40),                       # a negative length
    ([5, 20, 3], [4, 2 ** 31 - 1, 30], 6, 40),             # past its table, and past 2^31 in all
    ([5, 2 ** 31 - 1, 3], [4, 1, 30], 6, 40),              # their sum wraps 32 bits
    ([0, 0, 3], [20, 40, 10], 6, 25),                      # more tokens than rows
    ([0, 0, 3], [20, 40, 10], 99, 90),                     # a free count past the list
    ([0, 0, 3], [20, 40, 10], -4, 90),                     # a negative free count
])
def test_bad_lengths_are_flagged(prior, new, n_free, n_tokens):
    width, bs, free = 6, 16, [7, 8, 9, 10, 11, 12]
    tables = [[i + 1] + [-9] * 5 for i in range(3)]
    got = run(tables, free, n_free, prior, new, bs, n_tokens)
    fit = min(max(n_free, 0), len(free))
    want = list(oracle(tables, free, fit, prior, new, bs, width, n_tokens))
    if fit != n_free:
        want[-1] |= _lib.FLAG_BLOCK_OUT_OF_RANGE
    assert got == want and got[-1]


@pytest.mark.gpu
def test_steps_in_a_captured_graph_keep_the_state_on_the_gpu():
    """Ten replays of one captured step: lengths, tables and free count advance on the GPU."""
    n, bs, width, dev = 9, 16, 12, "cuda"
    prior = torch.tensor([i * 5 for i in range(n)], dtype=torch.int32, device=dev)
    new = torch.tensor([1, 2, 0, 16, 3, 1, 1, 7, 17], dtype=torch.int32, device=dev)
    host_prior = prior.tolist()
    ids = list(range(200))
    random.Random(0).shuffle(ids)
    tables, o = [], 0
    for p in host_prior:
        k = -(-p // bs)
        tables.append(ids[o:o + k] + [-9] * (width - k))
        o += k
    free = ids[o:]
    t = torch.tensor(tables, dtype=torch.int32, device=dev)
    f = torch.tensor(free, dtype=torch.int32, device=dev)
    left = torch.tensor([len(free)], dtype=torch.int32, device=dev)
    T = int(new.sum())
    out = ops.new_step_tables(n, T + 2, dev)
    err = ops.new_error_flags(dev)

    def step():
        ops.build_step_tables(t, f, left, prior, new, bs, T + 2, out=out, err=err)
        left.copy_(out.n_free)
        prior.copy_(out.context_lens)

    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # step 0, uncaptured
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(g):
        step()
    n_free, hn = len(free), new.tolist()
    for k in range(5):
        if k:
            g.replay()
        tables, ctx, starts, slots, pos, n_free, flags = oracle(tables, free, n_free, host_prior, hn, bs, width, T + 2)
        host_prior = ctx
        assert t.tolist() == tables and prior.tolist() == ctx and int(left) == n_free and int(err) == flags == 0
        assert out.slot_mapping.tolist() == slots and out.positions.tolist() == pos
        assert out.query_start_loc.tolist() == starts


def test_c_refusals():
    f = _lib.load().pkv_build_step_tables
    base = [FAKE, 8, 8, FAKE, 4, FAKE, FAKE2, FAKE, FAKE, 2, 16, FAKE, FAKE, FAKE, FAKE, 5, None, None]

    def call(**kw):
        names = ["tables", "stride", "width", "free", "n_list", "n_free", "n_out", "prior", "new", "n", "bs",
                 "ctx", "qsl", "slots", "pos", "tokens", "err", "stream"]
        a = dict(zip(names, base))
        a.update(kw)
        return f(*a.values())

    assert call(n=-1) == call(tokens=-1) == call(bs=0) == call(stride=7) == call(width=0) == _lib.ERR_BAD_SHAPE
    assert call(width=1 << 28, stride=1 << 28) == _lib.ERR_BAD_SHAPE  # 2^28 blocks of 16 pass 32 bits
    for name in ("tables", "free", "n_free", "n_out", "prior", "new", "ctx", "qsl", "slots", "pos"):
        assert call(**{name: None}) == _lib.ERR_NULL_POINTER, name
    assert call(n_out=FAKE) == _lib.ERR_UNSUPPORTED   # the count read and written in one word
    assert call(n=16385) == _lib.ERR_UNSUPPORTED


def test_wrapper_refuses_cpu_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.build_step_tables(torch.zeros(2, 4, dtype=torch.int32), i, i, i, i, 16, 4)


@pytest.mark.gpu
def test_wrapper_refusals():
    z = lambda *s, dt=torch.int32: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    t, i = z(2, 4), z(2)
    good = dict(block_tables=t, free_blocks=z(3), n_free=z(1), num_prior=i, num_new=i, block_size=16, n_tokens=4)
    ops.build_step_tables(**good)
    for kw, exc in [(dict(block_tables=z(2, 4, dt=torch.int64)), TypeError), (dict(num_prior=z(2, dt=torch.int64)), TypeError),
                    (dict(num_new=z(3)), ValueError), (dict(block_tables=z(1, 4)), ValueError), (dict(free_blocks=z(3, 1)), TypeError),
                    (dict(err=z(1, dt=torch.int64)), TypeError), (dict(num_prior=torch.zeros(2, dtype=torch.int32)), RuntimeError),
                    (dict(out=ops.new_step_tables(2, 3, "cuda")), ValueError)]:
        with pytest.raises(exc):
            ops.build_step_tables(**{**good, **kw})
    out = ops.new_step_tables(2, 4, "cuda")
    with pytest.raises(ValueError, match="tensor of its own"):
        ops.build_step_tables(**{**good, "n_free": out.n_free, "out": out})
