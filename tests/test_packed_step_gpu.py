"""Packed decode calls end to end on the GPU: K14 (slots and table entries),
K2 (append), K15 (attention) and the layer stack as ``forward_packed`` and
``GrowRebuildDecoder(packed=True)`` run them together, against the float64
oracle session on the same bf16-rounded weights and embeddings.

Tolerance: as for the other whole-decoder checks, 2e-2 x max(1, the token's
largest magnitude): the hidden states carry bf16 rounding (2^-8 relative) of
every GEMM input, q, k, v and the output over two layers, and the attention
probabilities' rounding to bf16, a few steps of 2^-8 = 0.0039 in all.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import attention as oatt
from oracle import decoder as odec
from tests.golden_io import grow_rebuild_schedule
from tests.test_failure_gpu import _timed_out_launches

pytestmark = pytest.mark.gpu

ATOL = 2e-2


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from mouse_core_b200 import build

    build.build()
    return torch.device("cuda")


def _model(dev, head_dim, q_heads, kv_heads, hidden=256, seed=7):
    from mouse_core_b200.backbone import Qwen3Backbone

    torch.manual_seed(seed)
    bb = Qwen3Backbone(hidden_dim=hidden, num_layers=2, num_heads=q_heads, num_key_value_heads=kv_heads,
                       head_dim=head_dim)
    with torch.no_grad():
        for name, p in bb.model.named_parameters():
            if "norm" in name:
                p.copy_(1 + 0.2 * torch.randn_like(p))
            else:
                p.mul_(3.0)  # make attention non-trivial
        for p in bb.model.parameters():
            p.copy_(p.bfloat16().float())
    sd = {k: v.detach().numpy() for k, v in bb.model.state_dict().items() if "rotary" not in k}
    dec = odec.DecoderOracle(sd, odec.config_from_hf(bb.model.config, bb.model.rotary_emb.inv_freq.numpy()))
    return bb.to(device=dev, dtype=torch.bfloat16).eval(), dec


def _close(got, ref, where):
    assert got.shape == ref.shape, where
    assert np.isfinite(got).all(), where
    bound = ATOL * np.maximum(1.0, np.abs(ref).max(axis=-1, keepdims=True))
    assert (np.abs(got - ref) <= bound).all(), (where, float(np.abs(got - ref).max()))


class _Rows:
    """The oracle session with ``reset_rows`` and ``fork``."""

    def __init__(self, dec, B):
        self.s = odec.DecodeSessionOracle(dec, B)

    def step(self, parts):
        """``parts[b] [n_b, D]`` float64; the packed hidden states and every layer's."""
        n = np.array([p.shape[0] for p in parts])
        S = max(int(n.max()), 1)
        x = np.zeros((len(parts), S, parts[0].shape[1]))
        for b, p in enumerate(parts):
            x[b, S - n[b]:] = p
        h, layers = self.s.forward(x, n, output_hidden_states=True)
        pack = lambda t: np.concatenate([t[b, S - n[b]:] for b in range(len(parts))])
        return pack(h), [pack(t) for t in layers]

    def reset(self, rows):
        for b in rows:
            self.fork(b, b, 0)

    def fork(self, src, dst, n):
        for li in range(len(self.s.k)):
            self.s.k[li][dst], self.s.v[li][dst] = self.s.k[li][src][:n].copy(), self.s.v[li][src][:n].copy()
        self.s.lengths[dst] = n


@pytest.mark.parametrize("head_dim,q_heads,kv_heads,page,residual_fp32,fused_qkv", [
    (128, 4, 2, 128, True, False),
    (128, 4, 2, 64, False, False),
    (64, 6, 2, 64, True, False),
    (64, 8, 1, 128, True, True),
])
def test_packed_calls_mixed_with_everything_else_match_the_oracle(head_dim, q_heads, kv_heads, page, residual_fp32,
                                                                  fused_qkv):
    """A random schedule of packed calls (long chunks beside single tokens and
    rows that sit out), padded calls, one-token steps replayed from a graph,
    emptied rows and branches; the pool starts too small and the block table
    too narrow, so both grow inside packed calls."""
    dev = _dev()
    bb, dec = _model(dev, head_dim, q_heads, kv_heads)
    rng = np.random.default_rng(head_dim + q_heads)
    gen = torch.Generator().manual_seed(11)
    B, D = 5, 256
    sess = bb.decode_session(batch_size=B, capacity=64, page_size=page, num_pages=2)
    sess.residual_fp32, sess.fused_qkv = residual_fp32, fused_qkv
    oracle = _Rows(dec, B)
    ops = ["packed", "one", "one", "one", "reset", "packed", "one", "padded", "packed", "fork", "packed", "reset",
           "one", "one", "packed", "packed", "fork", "one", "packed"]
    for ci, op in enumerate(ops):
        if op == "reset":
            rows = rng.choice(B, size=2, replace=False)
            sess.reset_rows(rows)
            oracle.reset(rows)
            continue
        if op == "fork":
            n = int(oracle.s.lengths[0]) - int(rng.integers(0, 40))
            n = max(n, 0)
            sess.fork([0], [3], [n])
            oracle.fork(0, 3, n)
            continue
        hi = {"packed": 90, "padded": 9, "one": 2}[op]
        n = rng.integers(0, hi, size=B)
        if op == "packed":
            n[rng.integers(0, B)] = 1
            n[rng.integers(0, B)] = 0
            if ci == 0:
                n[0] = 300
        parts = [torch.randn(int(k), D, generator=gen).bfloat16() for k in n]
        ref, ref_layers = oracle.step([p.double().numpy() for p in parts])
        if op == "packed":
            h, layers = sess.forward_packed(embeds=torch.cat(parts).to(dev), lengths=n.tolist(),
                                            output_hidden_states=True)
            assert h.dtype == torch.bfloat16 and len(layers) == 2
            for li, (a, r) in enumerate(zip(layers, ref_layers)):
                _close(a.float().cpu().numpy(), r, (ci, op, li))
            got = h.float().cpu().numpy()
        else:
            S = max(int(n.max()), 1)
            x = torch.zeros(B, S, D, dtype=torch.bfloat16)
            for b, p in enumerate(parts):
                x[b, S - len(p):] = p
            h = sess.forward(embeds=x.to(dev), lengths=n.tolist()).float().cpu().numpy()
            got = np.concatenate([h[b, S - n[b]:] for b in range(B)])
        _close(got, ref, (ci, op))
        assert sess.lengths.cpu().tolist() == oracle.s.lengths.tolist()
    # The device's table is the host's, entry for entry of the pages in use.
    table = sess.block_table.cpu().numpy()
    for b in range(B):
        k = int(sess.pages.npages[b])
        assert (table[b, :k] == sess.pages.table[b, :k]).all(), b
    from mouse_core_b200 import _lib

    assert _lib.device_status() == 0


def test_packed_call_leaves_clones_streams_and_graphs_alone():
    """A clone stepped on another stream beside its source, and a captured
    one-token graph replayed after packed calls that grew their workspace:
    each sequence is what it is alone."""
    dev = _dev()
    bb, dec = _model(dev, 128, 4, 2)
    gen = torch.Generator().manual_seed(3)
    B, D = 3, 256
    sess = bb.decode_session(batch_size=B, capacity=1024)
    oracle = _Rows(dec, B)
    mk = lambda n: [torch.randn(k, D, generator=gen).bfloat16() for k in n]

    def run(s, o, n, packed=True):
        parts = mk(n)
        ref, _ = o.step([p.double().numpy() for p in parts])
        x = torch.cat(parts).to(dev)
        if packed:
            return s.forward_packed(embeds=x, lengths=n), ref
        return s.forward(embeds=x.view(B, 1, D), lengths=n)[:, 0], ref

    for n, packed in (([5, 0, 70], True), ([1, 1, 1], False), ([1, 1, 1], False), ([1, 1, 1], False),
                      ([200, 1, 130], True), ([1, 1, 1], False), ([1, 1, 1], False)):
        got, ref = run(sess, oracle, n, packed)
        _close(got.float().cpu().numpy(), ref, (n, packed))
    import copy

    other, o2 = sess.clone(), _Rows(dec, B)
    o2.s.lengths, o2.s.k, o2.s.v = oracle.s.lengths.copy(), copy.deepcopy(oracle.s.k), copy.deepcopy(oracle.s.v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    results = []
    for n, m in (([1, 65, 3], [40, 1, 0]), ([0, 0, 250], [1, 1, 1]), ([2, 1, 1], [129, 0, 7])):
        results.append(run(sess, oracle, n))
        with torch.cuda.stream(side):
            results.append(run(other, o2, m))
    torch.cuda.synchronize()
    for i, (got, ref) in enumerate(results):
        _close(got.float().cpu().numpy(), ref, i)


def test_packed_call_without_tokens_and_refusals():
    dev = _dev()
    bb, _ = _model(dev, 64, 2, 1, hidden=128)
    sess = bb.decode_session(batch_size=2, capacity=64)
    x = torch.randn(3, 128, device=dev).bfloat16()
    h = sess.forward_packed(embeds=x[:0], lengths=[0, 0])
    assert h.shape == (0, 128) and sess.lengths.tolist() == [0, 0]
    a = sess.forward_packed(embeds=x, lengths=[1, 2])
    with pytest.raises(ValueError, match="lengths"):
        sess.forward_packed(embeds=x, lengths=[1, 1])
    graph = torch.cuda.CUDAGraph()
    y = torch.zeros(1, device=dev)
    with torch.cuda.graph(graph):
        y += 1
        with pytest.raises(RuntimeError, match="captured"):
            sess.forward_packed(embeds=x, lengths=[1, 2])
    assert sess.lengths.tolist() == [1, 2]
    sess.reset_rows([0, 1])
    # Strided embeddings of another type are taken as forward takes them.
    b = sess.forward_packed(embeds=x.float().repeat(1, 2)[:, :128], lengths=[1, 2])
    assert torch.equal(a, b)


@pytest.mark.parametrize("per_row", [False, True])
@pytest.mark.parametrize("with_head,with_hidden", [(False, False), (True, False), (False, True)])
def test_grow_rebuild_packed_matches_the_reference_loop(per_row, with_head, with_hidden):
    """The grow-then-rebuild loop with packed calls: rebuilt windows beside
    single appended tokens, one-token calls from a graph, emptied rows."""
    dev = _dev()
    from mouse_core_b200.grow_rebuild import GrowRebuildDecoder

    bb, dec = _model(dev, 128, 4, 2, seed=17)
    B, calls, vocab = 5, 30, 97
    table16 = torch.randn(vocab, 256, generator=torch.Generator().manual_seed(6)).bfloat16()
    table = table16.to(dev)
    oracle = odec.GrowRebuildOracle(dec, B, table16.float().numpy(), 72, 30, per_row=per_row)
    ours = GrowRebuildDecoder(bb, B, lambda ids: table[ids], max_cache=72, start_cache=30, per_row=per_row,
                              page_size=64, packed=True)
    head = (lambda h: 2.0 * h.float()) if with_head else None
    for ci, (hist, ends, ctx, ended) in enumerate(grow_rebuild_schedule(29, B, calls, vocab, max_append=5)):
        if ci % 4 == 3:
            ended[:] = ended & per_row
        rb = ended if per_row else bool(ended.any())
        out, fed, *layers = ours.step(hist, ends, ctx, rebuild=rb, head=head, output_hidden_states=with_hidden)
        if with_hidden:
            assert len(layers[0]) == 2 and all(t.shape == out.shape for t in layers[0])
            _close(layers[0][1].float().cpu().numpy(), out.double().cpu().numpy(), ci)  # (no final norm: the identity)
        ref, ref_fed = oracle.step(hist, ends, ctx, rebuild=rb)
        assert fed.tolist() == np.asarray(ref_fed).tolist(), ci
        S = ref.shape[1]
        got = out.float().cpu().numpy()
        if with_head:
            live = np.flatnonzero(fed)
            assert got.shape == (B, 256)
            _close(got[live] / 2.0, ref[live, -1], ci)
        else:
            _close(got, np.concatenate([ref[b, S - fed[b]:] for b in range(B)]), ci)
    assert ours.rebuild_calls >= 3


@pytest.mark.parametrize("head_dim,lens,news", [
    (128, [3000, 129, 700, 4100], [1, 129, 200, 1]),   # single-token tiles, tcgen05 tiles, joins
    (64, [2500, 300, 65], [300, 300, 1]),
])
def test_chunk_attention_wait_timeout_is_reported_and_recovers(head_dim, lens, news):
    """K15 with a wait limit of 0: every launch finishes and reports a
    timeout; with the default limit back the same call is exact again."""
    dev = _dev()
    from mouse_core_b200 import _lib
    from mouse_core_b200 import kernels as K

    Hq, Hkv, page = 4, 2, 64
    g = torch.Generator().manual_seed(head_dim)
    need = [-(-n // page) for n in lens]
    P = sum(need)
    kp = torch.randn(P, Hkv, page, head_dim, generator=g).bfloat16()
    vp = torch.randn(P, Hkv, page, head_dim, generator=g).bfloat16()
    q = torch.randn(sum(news), Hq, head_dim, generator=g).bfloat16()
    order = torch.randperm(P, generator=g).int().tolist()
    bt = torch.full((len(lens), max(need)), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        bt[b, :n] = torch.tensor(order[sum(need[:b]):sum(need[:b + 1])], dtype=torch.int32)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32)
    args = [t.to(dev) for t in (q, kp, vp, bt, cu, torch.tensor(lens, dtype=torch.int32))] + [head_dim ** -0.5]
    _timed_out_launches(lambda: K.chunk_attention(*args))
    out = K.chunk_attention(*args)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    got = out.float().cpu().numpy()
    for b, (n, m) in enumerate(zip(lens, news)):
        rows = [t[bt[b, :need[b]].long()].permute(1, 0, 2, 3).reshape(Hkv, -1, head_dim)[:, :n].permute(1, 0, 2)
                .float().numpy() for t in (kp, vp)]
        at = int(cu[b])
        pos = np.arange(n - m, n)[None, :]
        ref = oatt.cached_decode_attention(q[at:at + m].float().numpy()[None], [rows[0]], [rows[1]], pos,
                                           head_dim ** -0.5)[0]
        assert np.abs(got[at:at + m] - ref).max() < ATOL, b


def test_one_plan_serves_every_layer_and_no_other_sizes():
    """The work list of a step used for several layers' pools and queries; a
    workspace without one, or with one for other sizes, is reported and leaves
    the output as it was."""
    dev = _dev()
    from mouse_core_b200 import _lib
    from mouse_core_b200 import kernels as K
    from tests.test_chunk_gpu import _attention_reference, _check, _paged

    rows = [(6000, 1), (0, 200), (77, 30), (20000, 2)]
    layers = [_paged(rows, 16, 8, 128, 64, seed=i) for i in range(3)]
    table, cu, kv_len = layers[0][3:]
    T = layers[0][0].shape[0]
    ws = torch.zeros(K.chunk_workspace_bytes(len(rows), T, 16, 8, 128), dtype=torch.uint8, device=dev)
    out = torch.full((T, 16, 128), 7.0, dtype=torch.bfloat16, device=dev)
    q, kp, vp = layers[0][:3]
    K.chunk_attention(q, kp, vp, table, cu, kv_len, 0.1, out=out, workspace=ws, plan_ready=True)
    assert _lib.device_status() == 7 and bool((out == 7.0).all())
    K.chunk_plan(cu, kv_len, T, 16, 8, 128, 64, table.shape[1], ws)
    for q, kp, vp, t, c, n in layers:
        got = K.chunk_attention(q, kp, vp, t, c, n, 0.1, workspace=ws, plan_ready=True)
        _check(got, _attention_reference(q, kp, vp, t, c, n, 0.1))
    assert _lib.device_status() == 0
    narrow = t[:, :-1].contiguous()  # (the last layer's own table from here on)
    K.chunk_attention(q, kp, vp, narrow, cu, kv_len, 0.1, out=out, workspace=ws, plan_ready=True)
    assert _lib.device_status() == 7 and bool((out == 7.0).all())
    got = K.chunk_attention(q, kp, vp, t, cu, kv_len, 0.1, workspace=ws, plan_ready=True)
    _check(got, _attention_reference(q, kp, vp, t, cu, kv_len, 0.1))  # the plan is still there
    assert _lib.device_status() == 0


def test_growth_on_a_side_stream_beside_allocations_on_the_session_s_own():
    """A session made on one stream and stepped on another outgrows its pool
    and its table there, while the first stream allocates and fills memory of
    the sizes just given up."""
    dev = _dev()
    bb, dec = _model(dev, 128, 4, 2)
    gen = torch.Generator().manual_seed(8)
    B, D = 3, 256
    sess = bb.decode_session(batch_size=B, capacity=64, page_size=64, num_pages=3)
    oracle = _Rows(dec, B)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    # Work in front of the session's own, so that its copies are still to come
    # when the other stream allocates.
    busy = torch.randn(4096, 4096, device=dev)
    results = []
    for n in ([40, 3, 60], [500, 1, 1], [1, 900, 40], [1, 1, 1200], [2, 1, 1]):
        parts = [torch.randn(k, D, generator=gen).bfloat16() for k in n]
        ref, _ = oracle.step([p.double().numpy() for p in parts])
        x = torch.cat(parts).to(dev)
        side.wait_stream(torch.cuda.current_stream())
        sizes = [sess.k_pool.numel() * 2, sess.v_pool.numel() * 2, sess.block_table.numel() * 4]
        with torch.cuda.stream(side):
            for _ in range(4):
                busy @ busy
            results.append((sess.forward_packed(embeds=x, lengths=n), ref, n, x))  # (x is the default stream's)
        fill = [torch.full((k,), 0xFF, dtype=torch.uint8, device=dev) for k in sizes for _ in range(2)]
        del fill
    torch.cuda.synchronize()
    for got, ref, n, _ in results:
        _close(got.float().cpu().numpy(), ref, n)


def test_a_packed_call_that_raised_can_be_made_again(monkeypatch):
    """Out of memory before the metadata launch, and in a layer behind the
    first one's append: the rows keep their lengths, and the same call, another
    one and a one-token step come out as if nothing had happened."""
    dev = _dev()
    from mouse_core_b200 import decode

    bb, dec = _model(dev, 64, 6, 2)
    gen = torch.Generator().manual_seed(4)
    B, D = 3, 256
    sess = bb.decode_session(batch_size=B, capacity=64, page_size=64, num_pages=4)
    oracle = _Rows(dec, B)

    def run(n, fails_in=None):
        parts = [torch.randn(k, D, generator=gen).bfloat16() for k in n]
        x = torch.cat(parts).to(dev)
        if fails_in:
            def fail(*a, **k):
                raise torch.OutOfMemoryError(fails_in)

            before = sess.lengths.tolist()
            with monkeypatch.context() as m:
                m.setattr(decode.K, fails_in, fail)
                with pytest.raises(torch.OutOfMemoryError):
                    sess.forward_packed(embeds=x, lengths=n)
            assert sess.lengths.tolist() == before
            if fails_in == "chunk_meta":  # another call comes first
                run([1, 0, 2])
        ref, _ = oracle.step([p.double().numpy() for p in parts])
        _close(sess.forward_packed(embeds=x, lengths=n).float().cpu().numpy(), ref, (n, fails_in))
        assert sess.lengths.tolist() == oracle.s.lengths.tolist()

    run([3, 64, 1])
    run([200, 1, 70], "chunk_meta")
    run([1, 130, 2], "chunk_attention")
    run([1, 1, 300], "chunk_plan")
    run([5, 0, 1])
    run([1, 2, 1])
    lengths, x = sess.lengths.tolist(), torch.randn(3, D, device=dev).bfloat16()
    with monkeypatch.context() as m:
        m.setattr(sess, "_final", lambda h: 1 / 0)
        with pytest.raises(ZeroDivisionError):
            sess.forward_packed(embeds=x, lengths=[1, 0, 2])
    assert sess.lengths.tolist() == lengths
    run([1, 0, 2])
    from mouse_core_b200 import _lib

    assert _lib.device_status() == 0


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("limit", [0, 2000, 20000])
def test_after_a_timeout_an_output_is_the_result_or_as_it_was(head_dim, limit):
    """Waits of a few cycles run out somewhere in a step of single tokens,
    chunks of one and two sub-tiles and split rows. Nothing half done is
    written, and the same call is exact afterwards."""
    _dev()
    from mouse_core_b200 import _lib
    from mouse_core_b200 import kernels as K
    from tests.test_chunk_gpu import TOL, _attention_reference, _check, _paged

    rows = [(3000, 1), (900, 300), (0, 129), (40, 20), (12000, 2), (700, 1), (9000, 100)] * 3
    args = (*_paged(rows, 8, 4, head_dim, 64, seed=head_dim), 0.1)
    o, A = ref = _attention_reference(*args)
    assert _lib.device_status() == 0
    try:
        _lib.set_wait_limit(limit)
        for _ in range(3):
            out = torch.full_like(args[0], 7.0)
            K.chunk_attention(*args, out=out)
            torch.cuda.synchronize()
            assert _lib.device_status() in (0, 1, 2, 6)
            right = (out.double() - o).abs() <= TOL * (A + o.abs())
            assert bool((right | (out == 7.0)).all())
    finally:
        _lib.set_wait_limit(None)
    out = K.chunk_attention(*args)
    assert _lib.device_status() == 0
    _check(out, ref)


@pytest.mark.parametrize("head_dim", [64, 128])
def test_a_plan_serves_the_call_behind_one_that_timed_out(head_dim):
    """Split rows are joined again by the next call on the same work list."""
    dev = _dev()
    from mouse_core_b200 import _lib
    from mouse_core_b200 import kernels as K
    from tests.test_chunk_gpu import _attention_reference, _check, _paged

    rows = [(20000, 1), (300, 90), (9000, 100), (50, 1)]
    args = (*_paged(rows, 8, 4, head_dim, 64, seed=3), 0.1)
    q, _, _, table, cu, kv_len, _ = args
    ref = _attention_reference(*args)
    ws = torch.zeros(K.chunk_workspace_bytes(len(rows), q.shape[0], 8, 4, head_dim), dtype=torch.uint8, device=dev)
    K.chunk_plan(cu, kv_len, q.shape[0], 8, 4, head_dim, 64, table.shape[1], ws)
    run = lambda: K.chunk_attention(*args, out=torch.full_like(q, 7.0), workspace=ws, plan_ready=True)
    _check(run(), ref)
    _timed_out_launches(run)
    for _ in range(2):
        out = run()
        assert _lib.device_status() == 0
        _check(out, ref)
