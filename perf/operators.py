"""Measured cases of the ragged-chunk operators of the paged KV cache.

A step of an env loop feeds every row of the batch its own number of new
tokens: one for a row that goes on, a whole window for a row that is rebuilt,
none for a row that sits out. The new tokens of all rows lie one after the
other in a packed stream. Two operators serve such a step:

* ``slots``: from the rows' new-token counts and cached lengths, the packed
  stream's offsets, every token's position and cache slot, the new lengths,
  and the block table with the pages that the step opens.
* ``attention``: the packed queries over the rows' paged K/V cache. The token
  at position p of row b sees the cached slots 0..p of its row.

Lengths are spread evenly over a case's range (the same multiset for every
seed, so that the work is known); the seed decides the order of the rows, the
pages they lie on and all values.
"""

import math
import random

import torch

own = False  # set by whoever measures: False computes the plain forms, True calls the framework


# ------------------------------------------------------------------- cases
def listed():
    qwen = dict(q_heads=16, kv_heads=8, head_dim=128, page=128)  # the 16/8-head backbone, 128-token pages
    llama = dict(q_heads=32, kv_heads=8, head_dim=64, page=64)  # the 32/8-head backbone, 64-token pages
    return [
        # An env batch's plain step: every row appends one token.
        dict(name="slots_step_256", op="slots", rows=256, ctx_lo=64, ctx_hi=4096, log=False, new_lo=1, new_hi=1,
             windows=0, window=0, page=128),
        # The same batch while six rows are rebuilt from 1024-token windows.
        dict(name="slots_rebuild_256", op="slots", rows=256, ctx_lo=64, ctx_hi=4096, log=False, new_lo=1, new_hi=1,
             windows=6, window=1024, page=128),
        # A large env shard, transitions of 0 to 4 tokens a row.
        dict(name="slots_envs_4096", op="slots", rows=4096, ctx_lo=128, ctx_hi=16384, log=True, new_lo=0, new_hi=4,
             windows=0, window=0, page=64),
        # Root contexts prefilled from empty: a few hundred thousand tokens.
        dict(name="slots_prefill_64", op="slots", rows=64, ctx_lo=0, ctx_hi=0, log=False, new_lo=1024, new_hi=8192,
             windows=0, window=0, page=128),
        # One env, one token, a short context: latency.
        dict(name="attn_one_token", op="attention", rows=1, ctx_lo=300, ctx_hi=300, log=False, new_lo=1, new_hi=1,
             windows=0, window=0, **qwen),
        # The plain step of 256 envs.
        dict(name="attn_step_256", op="attention", rows=256, ctx_lo=64, ctx_hi=4096, log=False, new_lo=1, new_hi=1,
             windows=0, window=0, **qwen),
        # Transitions of 0 to 4 tokens (observation, action, reward, done) over log-uniform contexts.
        dict(name="attn_transitions_128", op="attention", rows=128, ctx_lo=128, ctx_hi=16380, log=True, new_lo=0,
             new_hi=4, windows=0, window=0, **llama),
        # Four rows rebuilt from their windows while the others step.
        dict(name="attn_rebuild_48", op="attention", rows=48, ctx_lo=64, ctx_hi=2047, log=False, new_lo=1, new_hi=1,
             windows=4, window=1024, **qwen),
        # Branches of forked rollouts: 256 new tokens each over a long prefix.
        dict(name="attn_branches_48", op="attention", rows=48, ctx_lo=1024, ctx_hi=8192, log=False, new_lo=256,
             new_hi=256, windows=0, window=0, **qwen),
        # Ragged windows prefilled from an empty cache.
        dict(name="attn_windows_64", op="attention", rows=64, ctx_lo=0, ctx_hi=0, log=False, new_lo=500, new_hi=1024,
             windows=0, window=0, **llama),
        # One long row taking a chunk of 700 tokens: few query tiles, a long key axis.
        dict(name="attn_long_chunk", op="attention", rows=1, ctx_lo=60001, ctx_hi=60001, log=False, new_lo=700,
             new_hi=700, windows=0, window=0, **qwen),
        # Three very long rows, a handful of tokens.
        dict(name="attn_long_rows_3", op="attention", rows=3, ctx_lo=90000, ctx_hi=131000, log=False, new_lo=1,
             new_hi=5, windows=0, window=0, **llama),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], uniform in its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.3:
        rows = _spread(rng, 1, 4096)
        page = rng.choice([64, 128, 192, 256])
        hi = _spread(rng, 64, 16384)
        lo = rng.randrange(0, 3)
        most = max(lo + 1, min(8192, 300000 // rows))
        case = dict(op="slots", rows=rows, ctx_lo=rng.randrange(1, 64), ctx_hi=hi, log=rng.random() < 0.5, new_lo=lo,
                    new_hi=_spread(rng, lo + 1, most), windows=0, window=0, page=page)
        if rows >= 8 and rng.random() < 0.5:
            case.update(windows=rng.randrange(1, 5), window=rng.randrange(65, 1025))
        return case
    q_heads, kv_heads = rng.choice([(16, 8), (32, 8), (8, 8), (4, 2), (12, 4), (14, 2), (16, 1)])
    head_dim, page = rng.choice([(128, 128), (64, 64), (128, 64), (64, 128), (128, 192)])
    ctx_hi = _spread(rng, 64, 65536)
    new_hi = _spread(rng, 1, 1024)
    rows = _spread(rng, 1, 256)
    case = dict(op="attention", rows=rows, ctx_lo=rng.randrange(0, 64), ctx_hi=ctx_hi, log=rng.random() < 0.5,
                new_lo=rng.randrange(0, min(new_hi, 9) + 1), new_hi=new_hi, windows=0, window=0, q_heads=q_heads,
                kv_heads=kv_heads, head_dim=head_dim, page=page)
    if rows >= 8 and new_hi <= 8 and rng.random() < 0.5:
        case.update(windows=rng.randrange(1, 4), window=rng.randrange(65, 1025))
    # No drawn case takes more than the largest listed ones: neither as work nor as the plain form's padded batch.
    while True:
        s = max(new_hi, case["window"])
        kv = ctx_hi + new_hi
        w = work(case)
        if (4 * case["rows"] * q_heads * s * kv <= 6 << 30 and 4 * case["rows"] * kv * kv_heads * head_dim <= 4 << 30
                and w["bytes"] <= 2e9 and w["flops"] <= 4e11) or case["rows"] == 1:
            return case
        case["rows"] = max(1, case["rows"] * 3 // 4)
        if case["rows"] < 8:
            case.update(windows=0, window=0)


def _lengths(case):
    """(cached, new) tokens of every row, in an order of no meaning."""
    rows, windows = case["rows"], case["windows"]
    n = rows - windows
    got = [(0, case["window"])] * windows
    step = next(s for s in (7919, 104729, 1) if math.gcd(s, n) == 1)
    for i in range(n):
        u = (i + 0.5) / n
        lo, hi = case["ctx_lo"], case["ctx_hi"]
        c = math.exp(math.log(lo + 1) + u * (math.log(hi + 1) - math.log(lo + 1))) - 1 if case["log"] else lo + u * (hi - lo)
        v = ((i * step) % n + 0.5) / n
        got.append((int(round(c)), min(case["new_hi"], case["new_lo"] + int(v * (case["new_hi"] - case["new_lo"] + 1)))))
    return got


def _pages(tokens, page):
    return -(-tokens // page)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator("cuda").manual_seed(seed)
    page, rows = case["page"], case["rows"]
    order = _lengths(case)
    rng.shuffle(order)
    held = [_pages(c, page) for c, _ in order]
    opened = [_pages(c + n, page) - h for (c, n), h in zip(order, held)]
    width = max(1, max(h + o for h, o in zip(held, opened)))
    total = sum(held) + sum(opened)
    pool = total + max(64, total // 16)
    ids = torch.randperm(pool, generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
    column = torch.arange(width, device="cuda")[None, :]
    cached, new = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in zip(*order))
    held_t = torch.tensor(held, device="cuda")
    table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    table[column < held_t[:, None]] = ids[: sum(held)]
    state = dict(op=case["op"], page=page, tokens=sum(n for _, n in order), block_table=table)
    if case["op"] == "slots":
        state.update(lengths=new, kv_len=cached, free_pages=ids[sum(held):total].contiguous())
        return state
    full = torch.tensor([h + o for h, o in zip(held, opened)], device="cuda")
    table[(column < full[:, None]) & (column >= held_t[:, None])] = ids[sum(held):total]
    hd, hq, hkv = case["head_dim"], case["q_heads"], case["kv_heads"]
    shape = (pool, hkv, page, hd)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.bfloat16)

    state.update(q=normal(max(state["tokens"], 1), hq, hd)[: state["tokens"]], k_pool=normal(*shape), v_pool=normal(*shape),
                 cu_q=torch.cat([new.new_zeros(1), new.cumsum(0, dtype=torch.int32)]), kv_len=cached + new, scale=hd ** -0.5,
                 most_new=max(n for _, n in order), most_kv=max(c + n for c, n in order))
    return state


# -------------------------------------------------------------------- runs
def _slots_plain(s):
    page = s["page"]
    n, old = s["lengths"].long(), s["kv_len"].long()
    free, table = s["free_pages"], s["block_table"]
    rows = torch.arange(n.numel(), device=n.device)
    cu_q = torch.nn.functional.pad(n.cumsum(0), (1, 0))
    held = (old + page - 1) // page
    opened = (old + n + page - 1) // page - held
    cu_pages = torch.nn.functional.pad(opened.cumsum(0), (1, 0))
    k = torch.arange(free.numel(), device=n.device)
    row = torch.repeat_interleave(rows, opened, output_size=free.numel())
    table[row, held[row] + k - cu_pages[row]] = free
    t = torch.arange(s["tokens"], device=n.device)
    row = torch.repeat_interleave(rows, n, output_size=s["tokens"])
    pos = old[row] + t - cu_q[row]
    slot = table[row, pos // page].long() * page + pos % page
    return dict(cu_q=cu_q.int(), q_pos=pos.int(), slot=slot.int(), kv_len=(old + n).int(), cu_pages=cu_pages.int(),
                block_table=table)


def _attention_plain(s):
    """The batch padded to its longest chunk and its longest cache, in 32 bits."""
    q, cu, lens = s["q"], s["cu_q"].long(), s["kv_len"].long()
    tokens, hq, hd = q.shape
    batch, hkv, page = lens.numel(), s["k_pool"].shape[1], s["page"]
    most_new, width = max(s["most_new"], 1), max(1, _pages(s["most_kv"], page))
    n = cu[1:] - cu[:-1]
    row = torch.repeat_interleave(torch.arange(batch, device=q.device), n, output_size=tokens)
    col = torch.arange(tokens, device=q.device) - cu[row]
    padded = torch.zeros(batch, most_new, hq, hd, device=q.device)
    padded[row, col] = q.float()
    padded = padded.view(batch, most_new, hkv, hq // hkv, hd).permute(0, 2, 3, 1, 4).reshape(batch, hkv, -1, hd)
    pages = s["block_table"][:, :width].clamp(min=0).long()
    key = torch.arange(width * page, device=q.device)
    inside = (key < lens[:, None])[:, None, :, None]

    def cached(pool):
        x = pool[pages].transpose(1, 2).reshape(batch, hkv, width * page, hd).float()
        return x.masked_fill_(~inside, 0.0)

    scores = torch.matmul(padded, cached(s["k_pool"]).transpose(2, 3)).mul_(s["scale"])
    scores = scores.view(batch, hkv, hq // hkv, most_new, width * page)
    pos = (lens - n)[:, None] + torch.arange(most_new, device=q.device)
    scores.masked_fill_((key > pos[:, :, None])[:, None, None], float("-inf"))
    scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-3e38)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(batch, hkv, -1, width * page), cached(s["v_pool"]))
    out = out.view(batch, hkv, hq // hkv, most_new, hd) / total.clamp(min=1e-30)
    return out.permute(0, 3, 1, 2, 4).reshape(batch, most_new, hq, hd)[row, col].to(torch.bfloat16)


def run(state):
    if own:
        from mouse_core_b200 import kernels

        if state["op"] == "slots":
            cu_q, q_pos, slot, kv_len, cu_pages = kernels.chunk_meta(
                state["lengths"], state["kv_len"], state["block_table"], state["free_pages"], state["page"], state["tokens"])
            return dict(cu_q=cu_q, q_pos=q_pos, slot=slot, kv_len=kv_len, cu_pages=cu_pages,
                        block_table=state["block_table"])
        return kernels.chunk_attention(state["q"], state["k_pool"], state["v_pool"], state["block_table"], state["cu_q"],
                                       state["kv_len"], state["scale"])
    return _slots_plain(state) if state["op"] == "slots" else _attention_plain(state)


# ------------------------------------------------------------------- work
def work(case):
    order, page = _lengths(case), case["page"]
    tokens = sum(n for _, n in order)
    if case["op"] == "slots":
        opened = sum(_pages(c + n, page) - _pages(c, page) for c, n in order)
        # counts and lengths in; offsets, lengths, page offsets out; a started page's id in; opened ids in and out
        started = sum(1 for c, n in order if n and c % page)
        return {"bytes": 4.0 * (5 * len(order) + started + 2 * opened + 2 * tokens), "flops": 4.0 * tokens}
    hd, hq, hkv = case["head_dim"], case["q_heads"], case["kv_heads"]
    keys = sum(c + n for c, n in order if n)
    pairs = sum(n * c + n * (n + 1) // 2 for c, n in order)
    return {"bytes": 4.0 * keys * hkv * hd + 4.0 * tokens * hq * hd, "flops": 4.0 * pairs * hq * hd}


# ------------------------------------------------------------- definitions
def exact(case, seed):
    s = prepare(case, seed)
    page, table = s["page"], s["block_table"]
    if s["op"] == "slots":
        n, old, free, table = (s[k].tolist() for k in ("lengths", "kv_len", "free_pages", "block_table"))
        cu_q, cu_pages, q_pos, slot, took = [0], [0], [], [], 0
        for b in range(len(n)):
            need = max(0, -(-(old[b] + n[b]) // page) - -(-old[b] // page))
            for k in range(need):
                table[b][-(-old[b] // page) + k] = free[took + k]
            took += need
            q_pos += range(old[b], old[b] + n[b])
            slot += [table[b][p // page] * page + p % page for p in range(old[b], old[b] + n[b])]
            cu_q.append(cu_q[-1] + n[b])
            cu_pages.append(took)
        return {k: torch.tensor(v, dtype=torch.int32) for k, v in dict(
            cu_q=cu_q, q_pos=q_pos, slot=slot, kv_len=[a + b for a, b in zip(old, n)], cu_pages=cu_pages,
            block_table=table).items()}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    cu, lens = s["cu_q"].tolist(), s["kv_len"].tolist()
    group = case["q_heads"] // case["kv_heads"]
    for b, length in enumerate(lens):
        if cu[b] == cu[b + 1]:
            continue
        ids = table[b, : _pages(length, page)].long()
        k, v = (s[name][ids].double().transpose(0, 1).flatten(1, 2)[:, :length] for name in ("k_pool", "v_pool"))
        first = length - (cu[b + 1] - cu[b])
        for lo in range(cu[b], cu[b + 1], 128):
            hi = min(lo + 128, cu[b + 1])
            see = first + hi - cu[b]
            a = torch.einsum("thgd,hkd->htgk", s["q"][lo:hi].double().unflatten(1, (-1, group)), k[:, :see]) * s["scale"]
            late = torch.arange(see, device="cuda")[None, :] > torch.arange(first + lo - cu[b], see, device="cuda")[:, None]
            a = torch.softmax(a.masked_fill_(late[None, :, None], -math.inf), -1)
            out[lo:hi] = torch.einsum("htgk,hkd->thgd", a, v[:, :see]).flatten(1, 2)
    return out
