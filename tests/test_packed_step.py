"""Host side of the packed decode call (no GPU): the page allocator's
``open_chunks``, which pages a call opens and in which order, and every
refusal of ``forward_packed`` before anything reaches the device."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from mouse_core_b200.decode import PagedDecodeSession
from mouse_core_b200.pages import PageTable


@pytest.mark.parametrize("add", [[0, 0, 0], [1, 0, 2], [0, 5, 1]])
def test_open_chunks_is_allocate_without_the_dirty_mark(add):
    a, b = PageTable(3, 8, 64, 6), PageTable(3, 8, 64, 6)
    a.dirty = b.dirty = False
    ids = a.open_chunks(np.array(add))
    b.allocate(np.array(add))
    assert (a.table == b.table).all() and (a.npages == b.npages).all() and (a.refcount == b.refcount).all()
    assert a.free_pages == b.free_pages
    assert not a.dirty and b.dirty == (sum(add) > 0)
    # Handed out row by row, as the device writes them into its table.
    assert ids.tolist() == [int(i) for r in range(3) for i in a.table[r, :add[r]]]


def test_open_chunks_marks_a_widened_table_and_refuses_an_empty_pool():
    t = PageTable(2, 6, 64, 1)
    t.dirty = False
    t.open_chunks(np.array([3, 0]))
    assert t.dirty and t.max_pages >= 3
    with pytest.raises(RuntimeError, match="exhausted"):
        t.open_chunks(np.array([0, 4]))
    assert t.free_pages == 3 and t.npages.tolist() == [3, 0]


def _stub():
    s = object.__new__(PagedDecodeSession)
    s.B, s.page_size, s.n_layers = 3, 64, 1
    s.device, s.dtype = torch.device("cpu"), torch.bfloat16
    s.model = SimpleNamespace(config=SimpleNamespace(hidden_size=16))
    s.pages = PageTable(3, 8, 64, 2)
    s._len = np.array([0, 5, 64])
    return s


@pytest.mark.parametrize("embeds", [torch.zeros(3, 1, 16), torch.zeros(16), torch.zeros(4, 8)])
def test_forward_packed_refuses_other_layouts(embeds):
    with pytest.raises(ValueError, match="hidden_size"):
        _stub().forward_packed(embeds=embeds, lengths=[1, 2, 1])


@pytest.mark.parametrize("lengths", [[1, 3], [1, 3, 0, 0], [5, -1, 0], [1, 1, 1], [4, 1, 0]])
def test_prepare_packed_refuses_lengths_that_do_not_fit(lengths):
    s = _stub()
    with pytest.raises(ValueError, match="lengths"):
        s.prepare_packed(lengths, 4)
    # Nothing was allocated or advanced by a refused call.
    assert s.pages.free_pages == 8 and s._len.tolist() == [0, 5, 64] and s.pages.npages.tolist() == [0, 0, 0]


@pytest.fixture
def recorded(monkeypatch):
    """Which tensors were put under which stream, and a stream to stand on."""
    seen = []
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: seen.append((t.data_ptr(), t.numel(), s)),
                        raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: "side")
    return seen


def test_pools_outgrown_on_another_stream_stay_until_that_stream_is_done(recorded):
    s = _stub()
    s.n_kv_heads, s.head_dim = 2, 64
    s.k_pool = torch.randn(1, 8, 2, 64, 64).bfloat16()
    s.v_pool = torch.randn(1, 8, 2, 64, 64).bfloat16()
    old = s.k_pool, s.v_pool
    s._grow_pool(12)
    assert s.pages.num_pages >= 12 and s.k_pool.shape[1] == s.v_pool.shape[1] == s.pages.num_pages
    assert torch.equal(s.k_pool[:, :8], old[0]) and torch.equal(s.v_pool[:, :8], old[1])
    for t in old:
        assert (t.data_ptr(), t.numel(), "side") in recorded


def test_a_pool_that_finds_no_memory_to_grow_stays_whole(recorded, monkeypatch):
    """The second of the two pools cannot be allocated: both keep their pages,
    layer by layer contiguous, and growing them again works."""
    s = _stub()
    s.n_layers, s.n_kv_heads, s.head_dim = 2, 2, 64
    k, v = (torch.randn(2, 8, 2, 64, 64).bfloat16() for _ in range(2))
    s.k_pool, s.v_pool = k.clone(), v.clone()
    real, left = torch.zeros, [1]

    def zeros(*a, **kw):
        left[0] -= 1
        if left[0] < 0:
            raise torch.OutOfMemoryError("zeros")
        return real(*a, **kw)

    with monkeypatch.context() as m:
        m.setattr(torch, "zeros", zeros)
        with pytest.raises(torch.OutOfMemoryError):
            s._grow_pool(12)
    assert s.pages.num_pages == s.pages.free_pages == 8
    assert torch.equal(s.k_pool, k) and torch.equal(s.v_pool, v)
    assert all(p[li].is_contiguous() for p in (s.k_pool, s.v_pool) for li in range(2))
    s._grow_pool(12)
    assert s.k_pool.shape == s.v_pool.shape and s.k_pool.shape[1] == s.pages.num_pages >= 12
    assert torch.equal(s.k_pool[:, :8], k) and torch.equal(s.v_pool[:, :8], v)


def test_metadata_outgrown_on_another_stream_stays_until_that_stream_is_done(recorded, monkeypatch):
    """A padded call that widens the block table and enlarges the metadata buffer."""
    s = _stub()
    s._pending_reset = np.zeros(3, dtype=bool)
    s._staging_ev = [SimpleNamespace(record=lambda: None)] * 2
    s._stage = lambda n: (torch.empty(n, dtype=torch.int32), 0)
    s._meta_dev, s._bt_dev = torch.zeros(2, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32)
    s.pages = PageTable(3, 20, 64, 2)
    s._len = np.zeros(3, dtype=np.int64)
    old = s._meta_dev, s._bt_dev
    s.prepare([200, 3, 0], 200)
    assert s._bt_dev.shape[1] > 2 and s._meta_dev.numel() > 2
    for t in old:
        assert (t.data_ptr(), t.numel(), "side") in recorded


def _device_table(table, n, c, free, page):
    """What K14 does to the device's block table, and the slots it makes."""
    slots, taken = [], 0
    for b in range(len(n)):
        held, total = -(-int(c[b]) // page), -(-int(c[b] + n[b]) // page)
        for col in range(held, total):
            if taken < len(free):
                table[b, col] = free[taken]
            taken += 1
        slots += [int(table[b, p // page]) * page + p % page for p in range(int(c[b]), int(c[b] + n[b]))]
    assert taken <= len(free), "K14 was given too few pages"
    return slots


@pytest.mark.parametrize("fails_in", ["stage", "upload", "K14"])
@pytest.mark.parametrize("retry", [[70, 1, 1], [3, 130, 0], [0, 0, 70]])
def test_a_packed_call_that_failed_leaves_the_next_one_right(recorded, monkeypatch, fails_in, retry):
    """Out of memory between the pages' opening and the K14 launch: the call
    made again, or another one, gives every token the slot of the host's table,
    and so does the padded call behind it."""
    from mouse_core_b200 import decode

    P = 64
    s = _stub()
    s._pending_reset = np.zeros(3, dtype=bool)
    s._staging_ev = [SimpleNamespace(record=lambda: None)] * 2
    s._meta_dev = torch.zeros(0, dtype=torch.int32)
    s._bt_dev = torch.full((3, 4), -1, dtype=torch.int32)
    s.pages = PageTable(3, 30, P, 4)
    s._len = np.zeros(3, dtype=np.int64)
    fail = {"stage": False, "upload": False, "K14": False}

    class Upload(torch.Tensor):
        def to(self, *a, **k):
            if fail["upload"]:
                raise torch.OutOfMemoryError("upload")
            return super().to(*a, **k).as_subclass(torch.Tensor)

    def stage(n):
        if fail["stage"]:
            raise torch.OutOfMemoryError("stage")
        return torch.empty(n, dtype=torch.int32).as_subclass(Upload), 0

    def chunk_meta(n, c, table, free, page, tokens):
        if fail["K14"]:
            raise torch.OutOfMemoryError("K14")
        assert n.sum() == tokens
        slots = _device_table(table.numpy(), n.numpy(), c.numpy(), free.tolist(), page)
        return None, None, torch.tensor(slots), n + c, None

    s._stage = stage
    monkeypatch.setattr(decode.K, "chunk_meta", chunk_meta)

    def check(lengths):
        before = s._len.copy()
        _, _, slots, _ = s.prepare_packed(lengths, sum(lengths))
        rows = np.repeat(np.arange(3), lengths)
        pos = np.concatenate([np.arange(c, c + n) for c, n in zip(before, lengths)]).astype(np.int64)
        assert slots.tolist() == s.pages.slots(rows, pos).tolist()
        for b in range(3):
            held = -(-int(s._len[b]) // P)
            assert s._bt_dev[b, :held].tolist() == s.pages.table[b, :held].tolist()

    check([5, 64, 1])
    fail[fails_in] = True
    with pytest.raises(torch.OutOfMemoryError):
        s.prepare_packed([70, 1, 1], 72)
    fail[fails_in] = False
    assert s._len.tolist() == [5, 64, 1]
    check(retry)
    check([1, 1, 80])
    # A padded call behind a failed one: its rows' pages reach the device, too.
    fail[fails_in] = True
    with pytest.raises(torch.OutOfMemoryError):
        s.prepare_packed([130, 60, 0], 190)
    fail[fails_in] = False
    s.prepare([2, 60, 0], 60)
    for b in range(3):
        held = int(s.pages.npages[b])
        assert s._bt_dev[b, :held].tolist() == s.pages.table[b, :held].tolist()
    ids = np.concatenate([s.pages.table[b, :int(s.pages.npages[b])] for b in range(3)])
    assert len(set(ids.tolist())) == ids.size == 30 - s.pages.free_pages


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("per_row", [True, False])
def test_a_rebuild_that_failed_is_fed_again(per_row, packed):
    """The session's call raises after the rows were emptied: the same step made
    again feeds them their whole windows, and the others what they missed."""
    from mouse_core_b200.grow_rebuild import GrowRebuildDecoder

    class Session:
        def __init__(self):
            self.rows, self.fail = [[], [], []], False

        def reset_rows(self, rows):
            for b in rows:
                self.rows[b] = []

        def _feed(self, parts):
            if self.fail:
                raise torch.OutOfMemoryError("layers")
            for row, part in zip(self.rows, parts):
                row += part

        def forward_packed(self, *, embeds, lengths, output_hidden_states):
            at = np.cumsum(lengths)
            self._feed([embeds[a - n:a, 0].tolist() for a, n in zip(at, lengths)])
            return embeds

        def forward(self, *, embeds, lengths, output_hidden_states=False):
            S = embeds.shape[1]
            self._feed([embeds[b, S - n:, 0].tolist() for b, n in enumerate(lengths)])
            return embeds

    d = object.__new__(GrowRebuildDecoder)
    d.B, d.max_cache, d.start_cache, d.per_row, d.packed = 3, 20, 8, per_row, packed
    d.session, d.embed = Session(), lambda ids: ids[..., None].float()
    d.cached_starts, d.cached_ends = np.zeros(3, dtype=np.int64), np.zeros(3, dtype=np.int64)
    d.rebuild_calls = d.rows_rebuilt = 0
    d._stage_ids = lambda ids: torch.from_numpy(ids.copy())
    hist = np.arange(3 * 40).reshape(3, 40)
    d.step(hist, [5, 6, 7])
    for ends in ([18, 9, 9], [25, 11, 10], [27, 31, 11]):  # row 0, then row 1 outgrow the cache
        d.session.fail = True
        with pytest.raises(torch.OutOfMemoryError):
            d.step(hist, ends)
        d.session.fail = False
        d.step(hist, ends)
        for b in range(3):
            assert d.session.rows[b] == hist[b, d.cached_starts[b]:ends[b]].tolist(), (b, ends)
    assert d.rebuild_calls >= 2
