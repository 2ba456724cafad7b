"""Cases of the packed-prompt, 8-bit cache and step-table operators: inputs, plain forms, calls, work and exact values.

Four operators of a serving step:

* packed   causal attention with grouped heads over whole prompts packed one behind the other
           (scoring prompts without a cache).
* append   new K/V rows written into int8 pools with one power-of-two scale per (block, KV head),
           and the touched rows fetched back as values (the append-and-fetch contract of the cache).
* decode / chunk   attention over such pools: one query row per sequence, or a chunk of a prompt
           behind its cached tokens.
* tables   the step's block tables, slot map, positions and lengths from request lengths, with new
           blocks taken from a free list that lives on the GPU.

With `own` false, run() computes them with elementary torch operations in 32 bits; with `own` true it
makes the calls a user of pagedkv makes.  A scale is the smallest power of two 2^e (e >= -120) with
absmax <= 127 * 2^e over the block's rows of that head, so quantising, rescaling and dequantising are
exact but for the rounding to an integer.
"""

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MIN_EXP = -120  # smallest scale exponent of a block
LARGEST = 3_500_000_000  # scores of a drawn attention case in its plain form


def _ops():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm-inference-scheduler_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from pagedkv import ops

    return ops


# ---- lengths, decided by the case alone -----------------------------------------------------


def _spread(n, low, high, salt):
    """n lengths: `high` first, the others spread over the logarithm of low .. high; low = 0 gives some empty ones."""
    rng = random.Random(salt)
    out = [high]
    for _ in range(n - 1):
        if low == 0 and rng.random() < 0.08:
            out.append(0)
        else:
            out.append(min(high, max(low, round(math.exp(rng.uniform(math.log(max(1, low)), math.log(max(1, high))))))))
    return out


def _bell(n, median, high, salt):
    """n lengths around a median (lognormal, sigma 1/2), as context lengths of a running batch are."""
    rng = random.Random(salt)
    return [min(high, max(16, round(median * math.exp(0.5 * rng.gauss(0, 1))))) for _ in range(n)]


def _lengths(case):
    """(tokens before the call, tokens of the call) of each sequence."""
    n, salt = case["n"], case["salt"]
    op = case["op"]
    if op == "packed":
        return [0] * n, _spread(n, case["low"], case["longest"], salt)
    if op == "decode":
        ctx = _bell(n, case["median"], case["longest"], salt) if case["median"] else _spread(n, 0, case["longest"], salt)
        return [max(0, c - 1) for c in ctx], [1 if c else 0 for c in ctx]
    prior = _spread(n, 0, case["prior"], salt + 1) if case["prior"] else [0] * n
    return prior, _spread(n, case["low"], case["longest"], salt)


def listed():
    qwen = {"hq": 14, "hkv": 2, "d": 64}  # this repository's model
    wide = {"hq": 32, "hkv": 8, "d": 128}  # the usual larger head layout
    return [
        # scoring four documents of very different lengths in one call, the longest past 8,000 tokens
        {"name": "packed_documents", "op": "packed", "dtype": "f16", **qwen, "n": 4, "low": 30, "longest": 8191, "salt": 3},
        # a batch of ordinary prompts at 128-wide heads, as a larger model scores them
        {"name": "packed_prompts_wide", "op": "packed", "dtype": "bf16", **wide, "n": 12, "low": 200, "longest": 2048, "salt": 5},
        # a few short prompts in full precision: the latency of the smallest calls
        {"name": "packed_short_f32", "op": "packed", "dtype": "f32", **qwen, "n": 3, "low": 1, "longest": 250, "salt": 1},
        # the prompts of a large prefill step entering the cache: 64 prompts
        {"name": "append_prompts", "op": "append", "dtype": "bf16", **wide, "bs": 16, "n": 64, "prior": 0, "low": 200, "longest": 2000, "salt": 7},
        # one token for each of 256 running sequences: most blocks part full, some scales grow
        {"name": "append_tokens", "op": "append", "dtype": "f16", **qwen, "bs": 16, "n": 256, "prior": 4000, "low": 1, "longest": 1, "salt": 9},
        # the decode step of a full batch (256 sequences, contexts around 1,024)
        {"name": "decode_batch", "op": "decode", "dtype": "f16", **qwen, "bs": 16, "n": 256, "median": 1024, "longest": 8192, "salt": 3},
        # one long conversation alone on the GPU
        {"name": "decode_one_long", "op": "decode", "dtype": "f16", **qwen, "bs": 16, "n": 1, "median": 0, "longest": 131000, "salt": 2},
        # a batch with 128-wide heads and larger blocks
        {"name": "decode_wide", "op": "decode", "dtype": "bf16", **wide, "bs": 32, "n": 48, "median": 4096, "longest": 16384, "salt": 4},
        # chunked prefill: 16 chunks of up to 512 tokens behind up to 4,096 cached ones
        {"name": "chunk_batch", "op": "chunk", "dtype": "f16", **qwen, "bs": 16, "n": 16, "prior": 4096, "low": 500, "longest": 512, "salt": 6},
        # one odd chunk behind a short prefix
        {"name": "chunk_small", "op": "chunk", "dtype": "bf16", **qwen, "bs": 16, "n": 2, "prior": 70, "low": 3, "longest": 45, "salt": 8},
        # a decode step of 256 requests: latency
        {"name": "tables_tokens", "op": "tables", "bs": 16, "n": 256, "prior": 4000, "low": 1, "longest": 1, "short": False, "salt": 10},
        # many prompts and chunks at once, more tokens than blocks are left for
        {"name": "tables_prompts", "op": "tables", "bs": 16, "n": 1000, "prior": 2000, "low": 1, "longest": 2000, "short": True, "salt": 11},
    ]


def _log(rng, low, high):
    return round(math.exp(rng.uniform(math.log(low), math.log(high))))


def draw(rng):
    op = rng.choice(["packed", "packed", "append", "append", "decode", "decode", "decode", "chunk", "tables"])
    salt = rng.randrange(1 << 30)
    if op == "tables":
        n = _log(rng, 1, 4000)
        longest = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, min(8000, 600000 // n)))
        return {"op": op, "bs": rng.choice([8, 16, 16, 32]), "n": n, "prior": _log(rng, 1, 6000), "low": rng.choice([0, 1]),
                "longest": longest, "short": rng.random() < 0.3, "salt": salt}
    hq, hkv = rng.choice([(14, 2), (14, 2), (8, 8), (32, 8), (16, 2), (12, 1), (40, 8), (20, 4), (6, 3)])
    case = {"op": op, "dtype": rng.choice(["f16", "f16", "bf16", "bf16", "f32"]), "hq": hq, "hkv": hkv, "d": rng.choice([64, 64, 128])}
    if op == "packed":
        n = _log(rng, 1, 64)
        longest = _log(rng, 1, int(math.sqrt(LARGEST / (n * hq * (2 if case["d"] == 128 else 1)))) // (3 if case["dtype"] == "f32" else 1))
        return {**case, "n": n, "low": min(longest, rng.choice([0, 1, 1, 100])), "longest": longest, "salt": salt}
    case["bs"] = rng.choice([16, 16, 16, 32])
    if op == "append":
        n = _log(rng, 1, 512)
        longest = 1 if rng.random() < 0.4 else _log(rng, 1, min(4000, 40000 // n + 1))
        return {**case, "n": n, "prior": _log(rng, 1, 200000 // n), "low": min(longest, rng.choice([0, 1])), "longest": longest, "salt": salt}
    if op == "decode":
        n = _log(rng, 1, 512)
        if rng.random() < 0.5 and n >= 8:
            median = _log(rng, 16, 130000 // n)
            return {**case, "n": n, "median": median, "longest": 8 * median, "salt": salt}
        return {**case, "n": n, "median": 0, "longest": _log(rng, 1, min(131000, 400000 // n)), "salt": salt}
    n = _log(rng, 1, 32)
    return {**case, "n": n, "prior": _log(rng, 1, 8000 // n + 500), "low": 1, "longest": _log(rng, 2, 6000 // n + 100), "salt": salt}


# ---- inputs -----------------------------------------------------------------------------


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype).cuda()


def _starts(counts):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return out


def _two_to(e):
    """2^e in 32 bits for whole e in -126 .. 127, exactly (torch.ldexp goes by pow, which rounds)."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    op = case["op"]
    prior, new = _lengths(case)
    n = case["n"]
    ctx = [p + c for p, c in zip(prior, new)]
    tokens = sum(new)
    state = {"case": case, "ctx": ctx, "new": new, "tokens": tokens, "err": torch.zeros(1, dtype=torch.int32, device="cuda"),
             "query_start_loc": _ints(_starts(new)), "context_lens": _ints(ctx), "num_prior": _ints(prior), "num_new": _ints(new)}
    if op == "packed":
        # q, k and v are the rows of one fused projection, as the model has them
        dt, hq, hkv, d = DTYPES[case["dtype"]], case["hq"], case["hkv"], case["d"]
        rows = randn(tokens, hq + 2 * hkv, d).to(dt)
        state.update(q=rows[:, :hq], k=rows[:, hq:hq + hkv], v=rows[:, hq + hkv:], scale=d ** -0.5)
        return state

    bs = case["bs"]
    blocks = [-(-c // bs) for c in ctx]
    width = max(1, max(blocks))
    have = blocks if op != "tables" else [-(-p // bs) for p in prior]
    total = sum(blocks)
    pool = total + 5
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(n, width, dtype=torch.int32, device="cuda")
    counts = _ints(have, torch.int64)
    first = _ints(_starts(have)[:-1], torch.int64)
    column = torch.arange(width, device="cuda")
    at = (first[:, None] + column[None, :]).clamp(max=pool - 1)
    table = torch.where(column[None, :] < counts[:, None], order[at], table)
    state.update(block_tables=table, num_blocks=pool)
    if op == "tables":
        spare = order[sum(have):].contiguous()
        wanted = total - sum(have)
        state.update(free_blocks=spare, n_free=_ints([wanted * 2 // 3 if case["short"] else spare.numel()]))
        return state

    dt, hq, hkv, d = DTYPES[case["dtype"]], case["hq"], case["hkv"], case["d"]

    def bytes_of_pool():
        x = torch.empty(pool, bs, hkv, d, dtype=torch.int8, device="cuda")
        for i in range(0, pool, 4096):  # in parts: the normal values take four times the pool's bytes
            part = x[i:i + 4096]
            part.copy_((randn(*part.shape) * 36).round_().clamp_(-127, 127))
        return x

    def scales():
        return _two_to(torch.randint(-7, -4, (pool, hkv), generator=g, device="cuda"))

    state.update(k_pool=bytes_of_pool(), v_pool=bytes_of_pool(), k_scale=scales(), v_scale=scales())
    if op == "append":
        # token rows of different loudness, so that some blocks' scales have to grow
        rows = randn(tokens, 2 * hkv, d) * torch.exp(0.6 * randn(tokens, 2 * hkv, 1))
        rows = rows.to(dt)
        # what changes: every row of the touched blocks
        back = [c - p // bs * bs if m else 0 for c, p, m in zip(ctx, prior, new)]
        state.update(k=rows[:, :hkv], v=rows[:, hkv:], fetch_start_loc=_ints(_starts(back)), fetch_tokens=sum(back))
        return state
    state.update(q=randn(tokens if op == "chunk" else n, hq, d).to(dt), scale=d ** -0.5)
    if op == "decode":
        # the split-K scratch that a serving program keeps
        state["workspace"] = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    return state


# ---- plain forms -------------------------------------------------------------------------


def _owners(start_loc, total):
    """The sequence of each of `total` packed rows, and the row's index in it."""
    t = torch.arange(total, device="cuda")
    seq = torch.searchsorted(start_loc[1:].contiguous(), t, right=True)
    return seq, t - start_loc[seq].long()


def _padded(rows, start_loc, longest):
    """[B, longest, ...] of packed rows (rows behind a sequence's end are some other row's)."""
    at = start_loc[:-1].long()[:, None] + torch.arange(longest, device="cuda")[None, :]
    return rows[at.clamp(max=rows.shape[0] - 1)].float()


def _attend(q, k, v, seen, scale):
    """softmax(scale q k^T) v for padded q [B, Lq, Hq, D], k / v [B, Lk, Hkv, D]; seen [B, Lq, Lk]."""
    b, lq, hq, d = q.shape
    hkv = k.shape[2]
    q = q.view(b, lq, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4)
    s = torch.matmul(q, k.permute(0, 2, 3, 1).unsqueeze(2))
    s.mul_(scale).masked_fill_(~seen[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s, v.permute(0, 2, 1, 3).unsqueeze(2)) / total
    return o.permute(0, 3, 1, 2, 4).reshape(b, lq, hq, d)


def _plain_packed(st):
    longest = max(st["new"])
    start = st["query_start_loc"]
    q, k, v = (_padded(st[x], start, longest) for x in "qkv")
    at = torch.arange(longest, device="cuda")
    seen = (at[None, :] <= at[:, None])[None].expand(q.shape[0], -1, -1)
    o = _attend(q, k, v, seen, st["scale"])
    seq, i = _owners(start, st["tokens"])
    return o[seq, i].to(st["q"].dtype)


def _need(amax):
    """The block scale that holds absmax."""
    m, e = torch.frexp(amax)
    e = torch.where(m * 128 <= 127, e - 7, e - 6)
    e = torch.where(amax > 0, e, torch.full_like(e, MIN_EXP)).clamp(min=MIN_EXP)
    return _two_to(e)


def _plain_append_one(x, pool, scale, block, offset, tail, partial):
    """Write rows x [T, Hkv, D] at (block, offset); tail / partial: each sequence's first block and whether it held rows."""
    x = x.float()
    amax = torch.where(x.isfinite(), x.abs(), torch.zeros((), device="cuda")).amax(-1)
    most = torch.zeros_like(scale).index_reduce_(0, block, amax, "amax")
    held = torch.zeros(scale.shape[0], dtype=torch.bool, device="cuda")
    held[tail[partial]] = True
    touched = torch.zeros_like(held)
    touched[block] = True
    wanted = _need(most)
    new = torch.where(touched[:, None], torch.where(held[:, None], torch.maximum(scale, wanted), wanted), scale)
    old_rows = tail[partial]
    pool[old_rows] = (pool[old_rows].float() * (scale[old_rows] / new[old_rows])[:, None, :, None]).round().to(torch.int8)
    y = x / new[block][:, :, None]
    y = torch.nan_to_num(y, nan=0.0, posinf=127.0, neginf=-127.0)
    pool[block, offset] = y.round().to(torch.int8)
    scale.copy_(new)


def _rows_of(start_loc, total, ctx, table, bs):
    """(block, offset) of the last start_loc[i + 1] - start_loc[i] tokens of each context."""
    seq, i = _owners(start_loc, total)
    counts = (start_loc[1:] - start_loc[:-1]).long()
    pos = ctx.long()[seq] - counts[seq] + i
    return table[seq, pos // bs].long(), pos % bs


def _plain_append(st):
    bs, table, ctx = st["case"]["bs"], st["block_tables"], st["context_lens"]
    block, offset = _rows_of(st["query_start_loc"], st["tokens"], ctx, table, bs)
    prior = st["num_prior"].long()
    partial = (prior % bs != 0) & (st["num_new"] > 0)
    tail = table.gather(1, (prior // bs).clamp(max=table.shape[1] - 1)[:, None])[:, 0].long()
    out = {}
    for x in "kv":
        pool, scale = st[x + "_pool"], st[x + "_scale"]
        _plain_append_one(st[x], pool, scale, block, offset, tail, partial)
        b, o = _rows_of(st["fetch_start_loc"], st["fetch_tokens"], ctx, table, bs)
        out[x] = (pool[b, o].float() * scale[b][:, :, None]).to(st[x].dtype)
        out[x + "_scale"] = scale
    return out


def _plain_decode(st):
    bs, table, q = st["case"]["bs"], st["block_tables"], st["q"]
    n, hq, d = q.shape
    total = sum(st["ctx"])
    ctx = st["context_lens"].long()
    seq = torch.repeat_interleave(torch.arange(n, device="cuda"), ctx, output_size=total)
    pos = torch.arange(total, device="cuda") - (ctx.cumsum(0) - ctx)[seq]
    block, offset = table[seq, pos // bs].long(), pos % bs
    k = st["k_pool"][block, offset].float() * st["k_scale"][block][:, :, None]
    g = hq // k.shape[1]
    s = (q.float()[seq].view(total, -1, g, d) * k[:, :, None]).sum(-1).view(total, hq) * st["scale"]
    most = torch.full((n, hq), -math.inf, device="cuda").index_reduce_(0, seq, s, "amax")
    p = torch.exp(s - most[seq])
    bottom = torch.zeros(n, hq, device="cuda").index_add_(0, seq, p)
    v = st["v_pool"][block, offset].float() * st["v_scale"][block][:, :, None]
    o = torch.zeros(n, hq, d, device="cuda").index_add_(0, seq, (p.view(total, -1, g, 1) * v[:, :, None]).view(total, hq, d))
    return torch.where(bottom[..., None] > 0, o / bottom[..., None], torch.zeros((), device="cuda")).to(q.dtype)


def _plain_chunk(st):
    bs, table = st["case"]["bs"], st["block_tables"]
    longest, most = max(st["new"]), max(st["ctx"])
    pos = torch.arange(most, device="cuda")
    block, offset = table[:, pos // bs].long(), (pos % bs).expand(table.shape[0], -1)
    k, v = (st[x + "_pool"][block, offset].float() * st[x + "_scale"][block][..., None] for x in "kv")
    q = _padded(st["q"], st["query_start_loc"], longest)
    at = torch.arange(longest, device="cuda")
    seen = pos[None, None, :] <= st["num_prior"][:, None, None] + at[None, :, None]
    o = _attend(q, k, v, seen, st["scale"])
    seq, i = _owners(st["query_start_loc"], st["tokens"])
    return o[seq, i].to(st["q"].dtype)


def _plain_tables(st):
    bs, table, free = st["case"]["bs"], st["block_tables"], st["free_blocks"]
    prior, new, total = st["num_prior"].long(), st["num_new"].long(), st["tokens"]
    have = (prior + bs - 1) // bs
    need = (prior + new + bs - 1) // bs - have
    upto = need.cumsum(0)
    served = upto <= st["n_free"]
    start = torch.zeros(new.numel() + 1, dtype=torch.int32, device="cuda")
    start[1:] = new.cumsum(0)
    seq, i = _owners(start, total)
    pos = prior[seq] + i
    column = pos // bs
    fresh = column >= have[seq]
    index = st["n_free"].long() - 1 - (upto - need)[seq] - (column - have[seq])
    block = torch.where(fresh, free[index.clamp(0, free.numel() - 1)], table[seq, column])
    ok = served[seq]
    slot = torch.where(ok, block.long() * bs + pos % bs, -1)
    # a new block begins with a token of this step; the other tokens write what is there
    table[seq, column] = torch.where(ok & fresh, block, table[seq, column])
    left = st["n_free"] - torch.where(served, upto, 0).amax().to(torch.int32)
    return {"block_tables": table, "context_lens": torch.where(served, prior + new, 0).to(torch.int32), "query_start_loc": start,
            "slot_mapping": slot, "positions": pos, "n_free": left}


# ---- the framework's calls --------------------------------------------------------------------


def _own(st):
    ops, op, err = _ops(), st["case"]["op"], st["err"]
    if op == "packed":
        return ops.packed_prompt_attention(st["q"], st["k"], st["v"], st["query_start_loc"], st["scale"], err=err)
    if op == "tables":
        t = ops.build_step_tables(st["block_tables"], st["free_blocks"], st["n_free"], st["num_prior"], st["num_new"], st["case"]["bs"],
                                  n_tokens=st["tokens"], err=err)
        return {"block_tables": st["block_tables"], "context_lens": t.context_lens, "query_start_loc": t.query_start_loc,
                "slot_mapping": t.slot_mapping, "positions": t.positions, "n_free": t.n_free}
    pools = (st["k_pool"], st["v_pool"], st["k_scale"], st["v_scale"])
    if op == "append":
        ops.reshape_and_cache_int8(st["k"], st["v"], *pools, st["block_tables"], st["context_lens"], st["query_start_loc"], err=err)
        k, v = ops.fetch_int8(*pools, st["block_tables"], st["context_lens"], st["fetch_start_loc"], st["fetch_tokens"], st["k"].dtype, err=err)
        return {"k": k, "v": v, "k_scale": st["k_scale"], "v_scale": st["v_scale"]}
    if op == "decode":
        return ops.paged_decode_attention_int8(st["q"], *pools, st["block_tables"], st["context_lens"], st["scale"],
                                               workspace=st["workspace"], err=err)
    return ops.paged_prefill_attention_int8(st["q"], *pools, st["block_tables"], st["query_start_loc"], st["num_prior"],
                                            max(st["new"]), st["scale"], err=err)


def run(state):
    if own:
        return _own(state)
    return {"packed": _plain_packed, "append": _plain_append, "decode": _plain_decode, "chunk": _plain_chunk,
            "tables": _plain_tables}[state["case"]["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------


def work(case):
    prior, new = _lengths(case)
    ctx = [p + c for p, c in zip(prior, new)]
    tokens, op = sum(new), case["op"]
    if op == "tables":
        bs = case["bs"]
        fresh = sum(-(-c // bs) - -(-p // bs) for c, p in zip(ctx, prior))
        # lengths read; lengths, starts, slots and positions written; a block id read and written for each
        # new block, and read for each sequence that goes on in a part-full one
        return {"bytes": 8 * case["n"] + 8 * case["n"] + 16 * tokens + 8 * fresh + 4 * case["n"], "flops": 0}
    size, hq, hkv, d = {"f32": 4}.get(case["dtype"], 2), case["hq"], case["hkv"], case["d"]
    if op == "packed":
        return {"bytes": tokens * (2 * hq + 2 * hkv) * d * size, "flops": 4 * d * hq * sum(c * (c + 1) // 2 for c in new)}
    bs = case["bs"]
    blocks = sum(-(-c // bs) for c in ctx)
    if op == "append":
        back = sum(c - p // bs * bs if m else 0 for c, p, m in zip(ctx, prior, new))
        touched = sum(-(-c // bs) - p // bs for c, p, m in zip(ctx, prior, new) if m)
        # rows read, their bytes written, the touched rows given back as values, two scales a block and head
        return {"bytes": 2 * hkv * (d * (tokens * (size + 1) + back * size) + 4 * touched) + 4 * touched, "flops": 0}
    rows = case["n"] if op == "decode" else tokens
    seen = sum(ctx) if op == "decode" else sum(c * p + c * (c + 1) // 2 for c, p in zip(new, prior))
    return {"bytes": 2 * sum(ctx) * hkv * d + 8 * blocks * hkv + 4 * blocks + 2 * rows * hq * d * size, "flops": 4 * d * hq * seen}


# ---- exact values ------------------------------------------------------------------------


def _exact_rows(st, x, i, upto):
    """The dequantised rows 0 .. upto - 1 of sequence i, in 64 bits."""
    bs = st["case"]["bs"]
    ids = st["block_tables"][i, : -(-upto // bs)].long()
    rows = st[x + "_pool"][ids].double() * st[x + "_scale"][ids].double()[:, None, :, None]
    return rows.flatten(0, 1)[:upto]


def _exact_attention(q, k, v, prior, scale):
    """One sequence, head group by head group: row r sees keys 0 .. prior + r."""
    out = torch.empty_like(q, dtype=torch.float64)
    group = q.shape[1] // k.shape[1]
    rows, keys = q.shape[0], k.shape[0]
    hidden = torch.arange(keys, device="cuda")[None, :] > prior + torch.arange(rows, device="cuda")[:, None]
    for h in range(q.shape[1]):
        s = (q[:, h].double() @ k[:, h // group].double().T) * scale
        s[hidden] = -math.inf
        out[:, h] = torch.softmax(s, dim=1) @ v[:, h // group].double()
    return out


def _exact_append(st, x):
    bs, table = st["case"]["bs"], st["block_tables"].cpu()
    pool, scale = st[x + "_pool"].double(), st[x + "_scale"].double()
    rows, parts, first = st[x].double(), [], 0
    powers = torch.tensor([2.0 ** e for e in range(MIN_EXP, 130)], dtype=torch.float64, device="cuda")
    for i, (c, m) in enumerate(zip(st["ctx"], st["new"])):
        if not m:
            continue
        p = c - m
        begin = p // bs * bs
        ids = table[i, begin // bs: -(-c // bs)].long().cuda()
        held = pool[ids].flatten(0, 1)
        content = torch.zeros(ids.numel() * bs, *rows.shape[1:], dtype=torch.float64, device="cuda")
        content[p - begin: c - begin] = rows[first: first + m]
        top = content.view(ids.numel(), bs, *rows.shape[1:]).abs().amax(dim=(1, 3))
        # the first of the powers 2^-120, 2^-119, ... that holds the largest value
        step = powers[torch.searchsorted(127 * powers, top.contiguous())]
        if p > begin:
            step[0] = torch.maximum(step[0], scale[ids[0]])
            kept = (held[: p - begin] * scale[ids[0]][None, :, None] / step[0][None, :, None]).round()
        each = step.repeat_interleave(bs, dim=0)[: c - begin, :, None]
        ints = (content[: c - begin] / each).round()
        if p > begin:
            ints[: p - begin] = kept
        parts.append(ints * each)
        scale[ids] = step
        first += m
    return torch.cat(parts) if parts else rows[:0], scale


def exact(case, seed):
    op = case["op"]
    if op == "tables":
        return None
    st = prepare(case, seed)
    if op == "append":
        out = {}
        for x in "kv":
            out[x], out[x + "_scale"] = _exact_append(st, x)
        return out
    start, parts = _starts(st["new"] if op != "decode" else [1] * case["n"]), []
    for i, (c, m) in enumerate(zip(st["ctx"], st["new"])):
        q = st["q"][start[i]: start[i + 1]]
        if c == 0:
            parts.append(torch.zeros_like(q, dtype=torch.float64))
        elif op == "packed":
            parts.append(_exact_attention(q, st["k"][start[i]: start[i + 1]], st["v"][start[i]: start[i + 1]], 0, st["scale"]))
        else:
            parts.append(_exact_attention(q, _exact_rows(st, "k", i, c), _exact_rows(st, "v", i, c), c - m, st["scale"]))
    return torch.cat(parts)
