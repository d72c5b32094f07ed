"""GPU parity of the ragged step: K14 (slot maps and block tables) against a
loop over the rows, exactly, and K15 (attention of packed chunks over the paged
cache) against its formula in 64 bits.

Tolerance of K15, element by element. With p the softmax weights, o = sum p v
and A = sum p |v| over the visible keys (64 bits): the kernel rounds the weights
to bf16 before the second product (at most 2^-8 of each term: 2^-8 A), and the
output to bf16 (2^-8 |o|); scores, exponentials, sums and the merge of split
keys are held in fp32 (relative 2^-20 of a term or better). A quarter of a
2^-8 of both is left for those: |out - o| <= (2^-8 + 2^-10) (A + |o|), plus
the smallest bf16 step near zero."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = 2.0 ** -8 + 2.0 ** -10


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from mouse_core_b200 import build

    build.build()
    return torch.device("cuda")


def _status():
    from mouse_core_b200 import _lib

    return _lib.device_status()


# ------------------------------------------------------------------ K14
def _meta_reference(n, c, table, free, page, tokens):
    """Loop over rows and tokens; a step that does not fit keeps what does."""
    table = table.copy()
    cu_q, cu_pages, pos, slot = [0], [0], np.zeros(tokens, np.int64), np.full(tokens, -1, np.int64)
    t = taken = 0
    for b in range(len(n)):
        held, total = -(-c[b] // page), -(-(c[b] + n[b]) // page)
        for col in range(held, total):
            if taken < len(free) and col < table.shape[1]:
                table[b, col] = free[taken]
            taken += 1
        for i in range(n[b]):
            p = c[b] + i
            if t < tokens:
                pos[t] = p
                col = p // page
                fits = col < table.shape[1] and (col < held or cu_pages[-1] + col - held < len(free))
                if fits and table[b, col] >= 0:
                    slot[t] = table[b, col] * page + p % page
            t += 1
        cu_q.append(t)
        cu_pages.append(taken)
    return np.array(cu_q), pos, slot, np.array(n) + np.array(c), np.array(cu_pages), table


def _meta_case(n, c, page, seed, extra_width=1, spare=3):
    rng = np.random.default_rng(seed)
    held = [-(-x // page) for x in c]
    total = [-(-(x + y) // page) for x, y in zip(c, n)]
    need = sum(t - h for t, h in zip(total, held))
    width = max(total + [1]) + extra_width
    ids = rng.permutation(sum(held) + need + spare).astype(np.int32)
    table = np.full((len(n), width), -1, np.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = ids[at:at + h]
        at += h
    return table, ids[at:at + need + spare]


def _check_meta(n, c, page, table, free, tokens, status=0):
    dev = _dev()
    from mouse_core_b200 import kernels as K

    t = torch.from_numpy(table.copy()).to(dev)
    got = K.chunk_meta(torch.tensor(n, dtype=torch.int32, device=dev), torch.tensor(c, dtype=torch.int32, device=dev), t,
                       torch.from_numpy(free.copy()).to(dev), page, tokens)
    assert _status() == status
    ref = _meta_reference(n, c, table, free, page, tokens)
    for name, g, r in zip(("cu_q", "q_pos", "slot", "new_len", "cu_pages", "block_table"), (*got, t), ref):
        assert np.array_equal(g.cpu().numpy(), r), name


@pytest.mark.parametrize("page", [1, 64, 128, 192])
@pytest.mark.parametrize("rows,most,seed", [(1, 1, 0), (1, 700, 1), (5, 3, 2), (33, 200, 3), (1023, 4, 4), (1024, 4, 5),
                                            (1025, 9, 6), (4100, 2, 7)])
def test_chunk_meta_matches_the_row_loop(page, rows, most, seed):
    rng = np.random.default_rng(seed)
    n = rng.integers(0, most + 1, rows).tolist()
    c = rng.integers(0, 5 * page, rows).tolist()
    n[rng.integers(rows)] = most
    c[0] = 0
    if rows > 3:
        c[1], n[2], c[3] = page, 0, 2 * page - 1  # a full page, a row that sits out, one slot left
        n[0] = n[3] = 1
    table, free = _meta_case(n, c, page, seed)
    _check_meta(n, c, page, table, free, sum(n) + (seed % 3) * 7)


def test_chunk_meta_edges():
    _check_meta([], [], 64, np.zeros((0, 3), np.int32), np.zeros(0, np.int32), 0)
    _check_meta([], [], 64, np.zeros((0, 3), np.int32), np.zeros(0, np.int32), 5)
    _check_meta([0, 0], [0, 70], 64, *_meta_case([0, 0], [0, 70], 64, 1), 0)
    n, c = [100000, 0, 1, 3], [17, 5, 64, 200000]
    _check_meta(n, c, 64, *_meta_case(n, c, 64, 2), sum(n))


def test_chunk_meta_reports_a_step_that_does_not_fit():
    n, c = [70, 1, 130], [60, 64, 0]
    table, free = _meta_case(n, c, 64, 3, spare=0)
    _check_meta(n, c, 64, table, free[:3], sum(n), status=3)  # out of free pages
    _check_meta(n, c, 64, np.ascontiguousarray(table[:, :2]), free, sum(n), status=3)  # out of table columns
    _check_meta(n, c, 64, table, free, 150, status=7)  # out of tokens
    _check_meta(n, c, 64, table, free, 0, status=7)


def test_chunk_meta_reports_every_token_without_a_page():
    """Also where the step itself opens none: a cached length past the table,
    a table entry without a page, and a page whose slots pass 32 bits."""
    free = np.array([7, 8], np.int32)
    table = np.array([[5, 6], [3, -1], [1 << 26, 4]], np.int32)
    _check_meta([1, 0, 0], [190, 10, 1], 64, table, free, 1, status=3)
    _check_meta([0, 1, 1], [300, 100, 0], 64, table, free, 2, status=3)
    _check_meta([1, 0, 0], [10, 0, 300], 64, table, free, 1)  # idle rows are nobody's tokens
    dev = _dev()
    from mouse_core_b200 import kernels as K

    args = [torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 0, 2], [0, 0, 1], table, free)]
    got = K.chunk_meta(*args, 64, 2)
    assert _status() == 3 and got[2].tolist() == [-1, -1] and got[1].tolist() == [1, 2]


def test_chunk_meta_refuses_bad_arguments():
    dev = _dev()
    from mouse_core_b200 import kernels as K

    i = torch.zeros(2, dtype=torch.int32, device=dev)
    table = torch.zeros(2, 4, dtype=torch.int32, device=dev)
    for bad in ((i.long(), i, table, i, 64, 5), (i, i[:1], table, i, 64, 5), (i, i, table[:1], i, 64, 5),
                (i, i, table.t(), i, 64, 5), (i, i, table, i, 64, -1), (i, i, table, i, 0, 5)):
        with pytest.raises((TypeError, ValueError)):
            K.chunk_meta(*bad)


# ------------------------------------------------------------------ K15
def _paged(rows, Hq, Hkv, hd, page, seed, poison=float("nan"), spread=1.0):
    """Packed queries and a shuffled page pool for ``rows`` of (cached, new)
    tokens. Every slot without a token holds ``poison`` and every table entry
    without a page an id far outside the pool."""
    g = torch.Generator("cuda").manual_seed(seed)
    lens = [c + n for c, n in rows]
    pages = [-(-x // page) for x in lens]
    P = sum(pages) + 3
    perm = torch.randperm(P, generator=g, device="cuda").tolist()
    table = torch.full((len(rows), max(pages + [1]) + 1), 1 << 30, dtype=torch.int32)
    kp = torch.full((P, Hkv, page, hd), poison, dtype=torch.bfloat16, device="cuda")
    vp = kp.clone()
    at = 0
    for b, x in enumerate(lens):
        for i in range(pages[b]):
            table[b, i] = perm[at]
            m = min(page, x - i * page)
            kp[perm[at], :, :m] = (torch.randn(Hkv, m, hd, generator=g, device="cuda") * spread).bfloat16()
            vp[perm[at], :, :m] = torch.randn(Hkv, m, hd, generator=g, device="cuda").bfloat16()
            at += 1
    T = sum(n for _, n in rows)
    q = (torch.randn(T, Hq, hd, generator=g, device="cuda") * spread).bfloat16()
    cu = torch.tensor(np.concatenate([[0], np.cumsum([n for _, n in rows])]), dtype=torch.int32, device="cuda")
    return q, kp, vp, table.cuda(), cu, torch.tensor(lens, dtype=torch.int32, device="cuda")


def _attention_reference(q, kp, vp, table, cu, kv_len, scale):
    """(o, A) of the module's docstring in 64 bits, row by row."""
    T, Hq, hd = q.shape
    Hkv, page = kp.shape[1:3]
    o = torch.zeros(T, Hq, hd, dtype=torch.float64, device=q.device)
    A = torch.zeros_like(o)
    cu = cu.tolist()
    for b, length in enumerate(kv_len.tolist()):
        n = cu[b + 1] - cu[b]
        if n == 0 or length <= 0:
            continue
        ids = table[b, : -(-length // page)].long()
        k = kp[ids].transpose(0, 1).flatten(1, 2)[:, :length].double()
        v = vp[ids].transpose(0, 1).flatten(1, 2)[:, :length].double()
        for lo in range(cu[b], cu[b + 1], 64):
            hi = min(lo + 64, cu[b + 1])
            s = torch.einsum("thgd,hkd->thgk", q[lo:hi].double().unflatten(1, (Hkv, -1)), k) * scale
            pos = torch.arange(lo, hi, device=q.device) - cu[b] + length - n
            seen = torch.arange(length, device=q.device) <= pos[:, None]
            s.masked_fill_(~seen[:, None, None], -torch.inf)
            w = torch.softmax(s, -1).nan_to_num(0.0)  # a token that sees nothing
            o[lo:hi] = torch.einsum("thgk,hkd->thgd", w, v).flatten(1, 2)
            A[lo:hi] = torch.einsum("thgk,hkd->thgd", w, v.abs()).flatten(1, 2)
    return o, A


def _check(out, ref, what=""):
    o, A = ref
    err = (out.double() - o).abs()
    assert bool(torch.isfinite(out.float()).all()), f"{what}: not finite"
    over = (err / (TOL * (A + o.abs()) + 1e-30)).max().item() if out.numel() else 0.0
    assert over <= 1.0, f"{what}: error {over:.2f} times the bound"


CASES = {
    # name: (rows of (cached, new), Hq, Hkv, hd, page)
    "one_token": ([(0, 1)], 16, 8, 128, 128),
    "one_token_cached": ([(300, 1)], 16, 8, 128, 128),
    "step_with_idle_rows": ([(64, 1), (0, 0), (127, 1), (128, 1), (700, 0), (2049, 1), (5, 1)], 16, 8, 128, 128),
    "transitions_hd64": ([(9000, 4), (63, 3), (64, 0), (1, 2), (4095, 1), (130, 4)], 32, 8, 64, 64),
    "at_most_16_query_rows": ([(500, 8), (31, 7), (128, 5)], 4, 2, 128, 64),
    "just_over_16_query_rows": ([(500, 9), (31, 17), (128, 1)], 4, 2, 128, 64),
    "windows_from_empty": ([(0, 1024), (0, 1), (0, 129), (0, 64), (0, 65), (0, 257)], 16, 8, 128, 128),
    "windows_hd64": ([(0, 500), (0, 33), (0, 1000), (0, 31), (0, 32)], 32, 8, 64, 64),
    "mixed": ([(1500, 1), (0, 300), (10, 0), (777, 1), (200, 130), (4000, 1), (3, 2)], 16, 8, 128, 128),
    "chunk_over_prefix": ([(1023, 256), (1024, 256), (2500, 255), (40, 256)], 16, 8, 128, 128),
    "no_gqa": ([(100, 300), (513, 1), (0, 256), (5, 257)], 4, 4, 128, 128),
    "group_of_3": ([(100, 50), (1000, 1), (0, 43), (64, 84), (63, 85), (7, 6)], 12, 4, 128, 64),
    "group_of_7": ([(100, 50), (1000, 1), (0, 18), (64, 36), (63, 37), (7, 2), (700, 3)], 14, 2, 64, 128),
    "group_of_16": ([(100, 50), (1000, 1), (0, 8), (64, 16), (63, 17), (7, 2)], 16, 1, 128, 192),
    "group_of_32": ([(100, 9), (1000, 1), (0, 4), (64, 8)], 32, 1, 64, 64),
    "one_sub_tile_even_and_odd_key_tiles": ([(100, 20), (220, 40), (500, 64), (700, 33), (2500, 9), (0, 50), (128, 64)],
                                            16, 8, 128, 64),
    "one_sub_tile_hd64": ([(100, 5), (240, 16), (500, 32), (9000, 20), (380, 7), (0, 31)], 32, 8, 64, 64),
    "one_sub_tile_split": ([(30000, 40), (17, 3)], 16, 8, 128, 128),
    "one_head": ([(0, 5), (600, 1), (128, 128), (127, 257)], 1, 1, 64, 64),
    "long_axis_few_rows": ([(40000, 1), (30001, 3)], 16, 8, 128, 128),
    "long_axis_chunk": ([(20011, 200)], 16, 8, 128, 128),
    "long_axis_hd64": ([(33333, 5), (65000, 1)], 32, 8, 64, 64),
    "many_rows": ([(17 * i % 900, (i * 7) % 3) for i in range(1500)], 4, 2, 64, 64),
    "large_pages": ([(1000, 3), (0, 700), (319, 2)], 8, 2, 128, 320),
}


@pytest.mark.parametrize("name", list(CASES))
def test_chunk_attention_matches_the_formula(name):
    _dev()
    from mouse_core_b200 import kernels as K

    rows, Hq, Hkv, hd, page = CASES[name]
    args = _paged(rows, Hq, Hkv, hd, page, seed=len(name))
    out = K.chunk_attention(*args, hd ** -0.5)
    assert _status() == 0
    _check(out, _attention_reference(*args, hd ** -0.5), name)
    again = K.chunk_attention(*args, hd ** -0.5)
    assert torch.equal(out, again), "the same call twice gives other bits"


@pytest.mark.parametrize("poison", [float("inf"), float("-inf"), torch.finfo(torch.bfloat16).min])
def test_slots_without_a_token_are_not_read(poison):
    _dev()
    from mouse_core_b200 import kernels as K

    rows = [(1, 1), (63, 1), (64, 2), (100, 40), (0, 129), (191, 1)]
    args = _paged(rows, 16, 8, 128, 64, seed=5, poison=poison)
    out = K.chunk_attention(*args, 128 ** -0.5)
    assert _status() == 0
    _check(out, _attention_reference(*args, 128 ** -0.5))


def test_large_scores():
    """Scores in the hundreds: one key carries nearly all the weight."""
    _dev()
    from mouse_core_b200 import kernels as K

    rows = [(900, 1), (300, 200), (0, 70), (2300, 3)]
    for hd in (64, 128):
        args = _paged(rows, 8, 4, hd, 64, seed=9, spread=4.0)
        out = K.chunk_attention(*args, hd ** -0.5)
        assert _status() == 0
        _check(out, _attention_reference(*args, hd ** -0.5))


def test_tokens_before_the_cache_get_zero():
    """kv_len below the row's token count: the first tokens sit at negative positions."""
    _dev()
    from mouse_core_b200 import kernels as K

    q, kp, vp, table, cu, kv_len = _paged([(0, 5), (0, 200), (0, 1), (0, 40)], 16, 8, 128, 128, seed=3)
    kv_len = torch.tensor([3, 70, 0, 0], dtype=torch.int32, device="cuda")
    out = K.chunk_attention(q, kp, vp, table, cu, kv_len, 0.1)
    assert _status() == 0
    assert bool((out[:2] == 0).all()) and bool((out[5:135] == 0).all()) and bool((out[205:] == 0).all())
    _check(out, _attention_reference(q, kp, vp, table, cu, kv_len, 0.1))


def test_strided_queries_and_rows_behind_the_last_sequence():
    _dev()
    from mouse_core_b200 import kernels as K

    rows, Hq, Hkv, hd = [(100, 1), (30, 70), (260, 2)], 16, 8, 128
    q, kp, vp, table, cu, kv_len = _paged(rows, Hq, Hkv, hd, 64, seed=11)
    ref = _attention_reference(q, kp, vp, table, cu, kv_len, 0.1)
    T, extra = q.shape[0], 37
    fused = torch.full((T + extra, (Hq + 2 * Hkv) * hd), float("nan"), dtype=torch.bfloat16, device="cuda")
    view = fused[:, : Hq * hd].unflatten(1, (Hq, hd))
    view[:T] = q
    out = torch.full((T + extra, Hq, hd), 7.0, dtype=torch.bfloat16, device="cuda")
    got = K.chunk_attention(view, kp, vp, table, cu, kv_len, 0.1, out=out)
    assert got is out and _status() == 0
    _check(out[:T], ref)
    assert bool((out[T:] == 7.0).all())


def test_empty_calls():
    _dev()
    from mouse_core_b200 import kernels as K

    q, kp, vp, table, cu, kv_len = _paged([(10, 0), (0, 0)], 4, 2, 64, 64, seed=1)
    assert K.chunk_attention(q, kp, vp, table, cu, kv_len, 0.1).shape == (0, 4, 64)
    out = torch.full((3, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    K.chunk_attention(torch.zeros_like(out), kp, vp, table, cu, kv_len, 0.1, out=out)  # no row has a token
    assert _status() == 0 and bool((out == 7.0).all())
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    K.chunk_attention(torch.zeros_like(out), kp, vp, table[:0], cu[:1], none, 0.1, out=out)
    assert _status() == 0 and bool((out == 7.0).all())


def test_a_page_outside_the_pool_reads_as_zero_and_is_reported():
    _dev()
    from mouse_core_b200 import kernels as K

    for rows in ([(500, 1), (40, 1)], [(400, 100), (40, 1)]):
        q, kp, vp, table, cu, kv_len = _paged(rows, 16, 8, 128, 128, seed=2)
        bad = table.clone()
        bad[0, 1] = -1
        kz, vz = kp.clone(), vp.clone()
        kz[table[0, 1]] = vz[table[0, 1]] = 0
        out = K.chunk_attention(q, kp, vp, bad, cu, kv_len, 0.1)
        assert _status() == 3
        _check(out, _attention_reference(q, kz, vz, table, cu, kv_len, 0.1))


def test_a_pool_beyond_32_bit_offsets():
    dev = _dev()
    from mouse_core_b200 import kernels as K

    Hkv, page, hd = 8, 128, 128
    P = (1 << 31) // (Hkv * page * hd) + 40  # the last pages' elements lie past 2^31
    kp, vp = (torch.zeros(P, Hkv, page, hd, dtype=torch.bfloat16, device=dev) for _ in range(2))
    g = torch.Generator("cuda").manual_seed(4)
    rows = [(500, 1), (300, 140), (2600, 3)]
    ids = torch.arange(P - 30, P, device=dev)
    kp[ids] = torch.randn(30, Hkv, page, hd, generator=g, device=dev).bfloat16()
    vp[ids] = torch.randn(30, Hkv, page, hd, generator=g, device=dev).bfloat16()
    table = torch.full((3, 21), -1, dtype=torch.int32, device=dev)
    table[0, :4], table[1, :4], table[2, :21] = ids[:4].int(), ids[4:8].int(), ids[9:].int()
    q = torch.randn(144, 16, hd, generator=g, device=dev).bfloat16()
    cu = torch.tensor([0, 1, 141, 144], dtype=torch.int32, device=dev)
    kv_len = torch.tensor([c + n for c, n in rows], dtype=torch.int32, device=dev)
    out = K.chunk_attention(q, kp, vp, table, cu, kv_len, 0.1)
    assert _status() == 0
    _check(out, _attention_reference(q, kp, vp, table, cu, kv_len, 0.1))


def test_refusals_of_the_attention_wrapper():
    _dev()
    from mouse_core_b200 import kernels as K

    q, kp, vp, table, cu, kv_len = _paged([(10, 3), (5, 1)], 4, 2, 64, 64, seed=1)
    good = dict(q=q, k_pool=kp, v_pool=vp, block_table=table, cu_q=cu, kv_len=kv_len, scale=0.1)
    bad = [dict(q=q.float()), dict(q=q[0]), dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)),
           dict(k_pool=kp.transpose(1, 2)), dict(v_pool=vp[:, :1].contiguous()), dict(q=q[:, :, :32].contiguous()),
           dict(cu_q=cu[:2]), dict(cu_q=cu.long()), dict(kv_len=kv_len[:1]), dict(block_table=table[:1]),
           dict(out=torch.empty(2, 4, 64, dtype=torch.bfloat16, device="cuda")), dict(out=torch.empty_like(q).float()),
           dict(q=q[:, :3].contiguous()), dict(block_table=table.cpu())]
    for b in bad:
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            K.chunk_attention(**{**good, **b})
    assert _status() == 0


def test_other_streams_and_captured_graphs():
    """Calls in flight together on two streams, and a captured call replayed
    after its inputs changed, each on its own workspace."""
    _dev()
    from mouse_core_b200 import kernels as K

    a = _paged([(3000, 1), (0, 200), (77, 3), (9000, 2)], 16, 8, 128, 128, seed=21)
    b = _paged([(50, 130), (6000, 1), (1, 1)], 32, 8, 64, 64, seed=22)
    ref_a, ref_b = _attention_reference(*a, 0.1), _attention_reference(*b, 0.1)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            outs.append((K.chunk_attention(*a, 0.1), ref_a))
        with torch.cuda.stream(s2):
            outs.append((K.chunk_attention(*b, 0.1), ref_b))
    torch.cuda.synchronize()
    assert _status() == 0
    for out, ref in outs:
        _check(out, ref)

    q, kp, vp, table, cu, kv_len = (t.clone() for t in a)
    K.chunk_attention(q, kp, vp, table, cu, kv_len, 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = K.chunk_attention(q, kp, vp, table, cu, kv_len, 0.1)
    graph.replay()
    torch.cuda.synchronize()
    _check(out, ref_a)
    # The same buffers with other lengths and another split of the tokens over the rows.
    cu.copy_(torch.tensor([0, 150, 151, 151, 206], dtype=torch.int32))
    kv_len.copy_(torch.tensor([2000, 199, 80, 9002], dtype=torch.int32))
    q.copy_(q.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert _status() == 0
    _check(out, _attention_reference(q, kp, vp, table, cu, kv_len, 0.1))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tiles", [1, 2, 3, 4, 5, 9])
def test_tables_no_wider_than_their_rows(hd, tiles):
    """Few rows whose longest tile is split or not, by a table of just the
    columns that the longest row needs."""
    _dev()
    from mouse_core_b200 import kernels as K

    keys = 128 * tiles
    for i, rows in enumerate(([(0, keys)], [(keys - 64, 64), (3, 1)], [(keys - 1, 1)], [(keys - 100, 90), (0, 20)],
                              [(0, keys - 84 + 1), (0, 1), (1, 19)])):
        q, kp, vp, table, cu, kv_len = _paged(rows, 4, 2, hd, 128, seed=tiles + 10 * i)
        args = q, kp, vp, table[:, :tiles].contiguous(), cu, kv_len, hd ** -0.5
        out = K.chunk_attention(*args)
        assert _status() == 0
        _check(out, _attention_reference(*args), (rows, tiles))


@pytest.mark.parametrize("hd", [64, 128])
def test_random_steps(hd):
    """Rows, lengths, groups and pages drawn at random, rows of every kind in
    one step."""
    _dev()
    from mouse_core_b200 import kernels as K

    rng = np.random.default_rng(hd)
    for i in range(40):
        Hkv = int(rng.choice([1, 2, 3, 8]))
        G = int(rng.choice([1, 2, 3, 4, 5, 8, 16]))
        page = int(rng.choice([64, 128, 192]))
        B = int(rng.choice([1, 2, 3, 8, 30]))
        most_c, most_n = int(rng.choice([1, 200, 5000])), int(rng.choice([1, 4, 40, 300]))
        rows = [(int(rng.integers(0, most_c + 1)), int(rng.integers(0, most_n + 1))) for _ in range(B)]
        rows[0] = (rows[0][0], most_n)
        args = (*_paged(rows, Hkv * G, Hkv, hd, page, seed=i), hd ** -0.5)
        out = K.chunk_attention(*args)
        assert _status() == 0
        _check(out, _attention_reference(*args), (i, Hkv, G, page, rows))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_a_token_sees_decides_whether_its_output_is_a_number(hd, bad):
    """A NaN (or an infinity whose scores are NaN or +inf) in one cached key
    makes NaN of the tokens that see it and leaves the others as they are, in
    every kind of tile; so does one in a token's query."""
    _dev()
    from mouse_core_b200 import kernels as K

    # (cached, new, position of the bad key): single tokens, one sub-tile, two, split rows.
    rows = [(700, 1, 90), (300, 40, 320), (100, 300, 250), (20000, 1, 3), (15000, 100, 15030), (64, 2, None)]
    q, kp, vp, table, cu, kv_len = _paged([r[:2] for r in rows], 8, 4, hd, 64, seed=hd)
    q[:, :, 0] = 1.0  # so that +inf in a key's first element is a score of +inf
    clean = kp.clone()
    for b, (_, _, at) in enumerate(rows):
        if at is not None:
            kp[table[b, at // 64], :, at % 64, 0] = bad
    q[-1, 3] = float("nan")
    out = K.chunk_attention(q, kp, vp, table, cu, kv_len, 0.1)
    assert _status() == 0
    zeroed = q.clone()
    zeroed[-1, 3] = 0.0
    o, A = _attention_reference(zeroed, clean, vp, table, cu, kv_len, 0.1)
    sees = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    for b, (c, n, at) in enumerate(rows):
        if at is not None:
            t = torch.arange(c, c + n, device="cuda")
            sees[cu[b]:cu[b + 1]] = (t >= at)[:, None]
    sees[-1, 3] = True
    assert bool(torch.isnan(out[sees].float()).all())
    _check(out[~sees], (o[~sees], A[~sees]))


@pytest.mark.parametrize("group,T,full", [(2, 2000, 40), (1, 300, 700), (128, 524288, 8192)])
def test_overlapping_rows_that_ask_for_more_tiles_than_the_stream_holds(group, T, full):
    """Offsets 0, T, 0, T, ...: every second row asks for the whole stream. The
    last case asks for 2^31 tiles, which no 32-bit count holds. The step is
    reported, no entry is written past the workspace, and (the sizes at which
    queries are worth making) the output stays as it was."""
    dev = _dev()
    from mouse_core_b200 import kernels as K

    B = 2 * full - 1
    cu = torch.tensor([0, T] * full, dtype=torch.int32, device=dev)
    kv_len = torch.full((B,), 100, dtype=torch.int32, device=dev)
    need = K.chunk_workspace_bytes(B, T, group, 1, 64)
    buf = torch.full((need + (1 << 22),), 0xA5, dtype=torch.uint8, device=dev)
    ws = buf[1 << 21: (1 << 21) + need]
    K.chunk_plan(cu, kv_len, T, group, 1, 64, 64, 2, ws)
    torch.cuda.synchronize()
    assert _status() == 7
    assert bool((buf[: 1 << 21] == 0xA5).all()) and bool((buf[(1 << 21) + need:] == 0xA5).all())
    if T > 4096:
        return
    pool = torch.zeros(2, 1, 64, 64, dtype=torch.bfloat16, device=dev)
    table = torch.zeros(B, 2, dtype=torch.int32, device=dev)
    out = torch.full((T, group, 64), 7.0, dtype=torch.bfloat16, device=dev)
    K.chunk_attention(torch.zeros_like(out), pool, pool, table, cu, kv_len, 0.1, out=out)
    assert _status() == 7 and bool((out == 7.0).all())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 4])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_which_tokens_a_bad_value_reaches(hd, group, bad):
    """One NaN or infinity in a cached value: the tokens that see it have no
    finite output in its element, earlier tokens of a tile that reads as far
    may have none, and every other token is as exact as without it. (A tile is
    128 / group tokens of the chunk and reads up to the end of the 128 slots of
    its last token.)"""
    _dev()
    from mouse_core_b200 import kernels as K

    # (cached, new, slot of the bad value): inside the prefix, among the new tokens of small, single and
    # paired tiles that straddle a multiple of 128, of split rows, and in nobody's tile but its own.
    rows = [(700, 1, 90), (124, 3, 126), (126, 3, 128), (100, 40, 135), (100, 128, 200), (50, 300, 320),
            (0, 500, 100), (0, 500, 127), (20000, 2, 20001), (15000, 100, 15090), (300, 60, None), (1000, 1, None)]
    q, kp, vp, table, cu, kv_len = _paged([r[:2] for r in rows], 2 * group, 2, hd, 64, seed=hd + group)
    clean = vp.clone()
    sees = torch.zeros(q.shape[0], dtype=torch.bool, device="cuda")
    may = sees.clone()
    ts = 128 // group
    for b, (c, n, at) in enumerate(rows):
        if at is None:
            continue
        vp[table[b, at // 64], :, at % 64, 1] = bad
        for i in range(n):
            last = c + min(n, (i // ts + 1) * ts) - 1
            sees[int(cu[b]) + i] = c + i >= at
            may[int(cu[b]) + i] = last >= at // 128 * 128
    assert bool((may | ~sees).all()) and bool((may & ~sees).any()) and bool((~may).any())
    out = K.chunk_attention(q, kp, vp, table, cu, kv_len, 0.1)
    assert _status() == 0
    assert not bool(torch.isfinite(out[sees][:, :, 1].float()).any())
    o, A = _attention_reference(q, kp, clean, table, cu, kv_len, 0.1)
    _check(out[~may], (o[~may], A[~may]))
    others = [e for e in range(hd) if e != 1]
    _check(out[:, :, others], (o[:, :, others], A[:, :, others]))


@pytest.mark.parametrize("hd", [64, 128])
def test_scores_in_the_hundreds(hd):
    """Scores of several hundred, where what fp32 holds of them counts.

    Tolerance. With S the largest sum |scale q_d k_d| over a token's visible keys
    (64 bits): the fp32 sum of hd exact products is off by at most hd 2^-23 S
    (each of its additions may truncate); scale, log2(e) and their product are
    rounded to fp32, as are the scaled score, the maximum and their difference:
    6 x 2^-24 S. So a weight is off by a factor of at most exp(d), d =
    (2 hd + 6) 2^-24 S, and a quotient of sums of weights by exp(2 d): 2.2 d (A +
    |o|) on top of the module's bound, as long as d is below 0.05."""
    _dev()
    from mouse_core_b200 import kernels as K

    scale = hd ** -0.5
    rows = [(900, 1), (300, 200), (0, 70), (2300, 3), (30000, 1), (9000, 100)]
    q, kp, vp, table, cu, kv_len = _paged(rows, 8, 4, hd, 64, seed=31, spread=10.0)
    S = torch.zeros(*q.shape[:2], 1, dtype=torch.float64, device="cuda")
    most = 0.0
    for b, (c, n) in enumerate(rows):
        ids = table[b, : -(-(c + n) // 64)].long()
        k = kp[ids].transpose(0, 1).flatten(1, 2)[:, : c + n].double()
        at = slice(int(cu[b]), int(cu[b]) + n)
        qb = q[at].double().unflatten(1, (4, 2))
        seen = torch.arange(c + n, device="cuda") <= torch.arange(c, c + n, device="cuda")[:, None]
        s = torch.einsum("thgd,hkd->thgk", qb, k).masked_fill_(~seen[:, None, None], 0.0)
        most = max(most, s.abs().max().item() * scale)
        s = torch.einsum("thgd,hkd->thgk", qb.abs(), k.abs()).masked_fill_(~seen[:, None, None], 0.0)
        S[at] = (s.amax(-1) * scale).flatten(1)[:, :, None]
    assert 300 < most < 1000
    d = (2 * hd + 6) * 2.0 ** -24 * S
    assert d.max().item() < 0.05
    out = K.chunk_attention(q, kp, vp, table, cu, kv_len, scale)
    assert _status() == 0
    o, A = _attention_reference(q, kp, vp, table, cu, kv_len, scale)
    assert bool(torch.isfinite(out.float()).all())
    assert bool(((out.double() - o).abs() <= (TOL + 2.2 * d) * (A + o.abs()) + 1e-30).all())


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("room", [0, 1, 3, 20, 100, 200, 333])
def test_rows_that_reach_past_the_stream_get_what_fits(hd, room):
    """The stream ends inside a row, or before it: the tokens that fit are those
    of the whole step, at their own positions, and the step is reported."""
    dev = _dev()
    from mouse_core_b200 import kernels as K

    rows = [(50, 3), (300, 330), (0, 40), (700, 1)]
    args = q, kp, vp, table, cu, kv_len = _paged(rows, 8, 4, hd, 64, seed=room)
    o, A = _attention_reference(*args, 0.1)
    T = 3 + room
    out = torch.full((T + 2, 8, hd), 7.0, dtype=torch.bfloat16, device=dev)
    K.chunk_attention(q[:T].contiguous(), kp, vp, table, cu, kv_len, 0.1, out=out[:T])
    assert _status() == 7
    _check(out[:T], (o[:T], A[:T]))
    assert bool((out[T:] == 7.0).all())
    # Fewer cached keys than tokens left out: those that fit see nothing.
    short = kv_len.clone()
    short[1] = 5
    K.chunk_attention(q[:T].contiguous(), kp, vp, table, cu, short, 0.1, out=out[:T])
    assert _status() == 7
    _check(out[:3], (o[:3], A[:3]))
    if room < 325:
        assert bool((out[3:3 + min(room, 325)] == 0).all())


@pytest.mark.parametrize("hd", [64, 128])
def test_keys_past_the_table_are_left_out_and_reported(hd):
    _dev()
    from mouse_core_b200 import kernels as K

    for rows in ([(500, 1), (40, 1)], [(500, 7), (40, 1)], [(400, 200), (70, 30)], [(20, 700), (1, 1)]):
        q, kp, vp, table, cu, kv_len = _paged(rows, 8, 4, hd, 64, seed=hd)
        narrow = table[:, :5].contiguous()  # 320 slots
        out = K.chunk_attention(q, kp, vp, narrow, cu, kv_len, 0.1)
        assert _status() == 3
        o, A = _attention_reference(q, kp, vp, table, cu, kv_len, 0.1)
        # Row 0 again, every token over the table's slots alone.
        n = rows[0][1]
        for i in range(n):
            if rows[0][0] + i >= 320:
                one = [t.to(q.device) for t in (torch.tensor([0, 1], dtype=torch.int32), torch.tensor([320], dtype=torch.int32))]
                o[i:i + 1], A[i:i + 1] = _attention_reference(q[i:i + 1], kp, vp, table[:1], *one, 0.1)
        _check(out, (o, A), rows)
