"""Refusals of the ragged-step entry points (K14 metadata, K15 attention):
every one returns or raises before any CUDA call, so they run without a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from mouse_core_b200 import _lib, build


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


# Any non-NULL, 16-byte-aligned address: the refusals below are decided before it is read.
P = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 8)


def _meta(lib, lengths=P, kv_len=P, batch=2, table=P, max_pages=4, page=64, free=P, n_free=3, tokens=5, cu_q=P,
          cu_pages=P, new_len=ctypes.c_void_p(2 << 20), q_pos=P, slot=P):
    return lib.mb_chunk_meta(lengths, kv_len, batch, table, max_pages, page, free, n_free, tokens, cu_q, cu_pages,
                             new_len, q_pos, slot, None)


@pytest.mark.parametrize("bad", [
    dict(batch=-1), dict(max_pages=-1), dict(n_free=-1), dict(tokens=-1), dict(page=0), dict(page=-64),
    dict(lengths=None), dict(kv_len=None), dict(table=None), dict(free=None), dict(cu_q=None), dict(cu_pages=None),
    dict(new_len=None), dict(q_pos=None), dict(slot=None),
    dict(new_len=P),  # kv_len's own memory: another block may still read it
])
def test_chunk_meta_refusals(lib, bad):
    assert _meta(lib, **bad) == 1
    assert lib.mb_last_error()


def _attention(lib, q=P, q_stride=16 * 128, k=P, v=P, num_pages=8, table=P, max_pages=4, cu_q=P, kv_len=P, batch=2,
               tokens=5, q_heads=16, kv_heads=8, head_dim=128, page=128, scale=0.1, out=P, ws=P, ws_bytes=1 << 30):
    return lib.mb_chunk_attention(q, q_stride, k, v, num_pages, table, max_pages, cu_q, kv_len, batch, tokens, q_heads,
                                  kv_heads, head_dim, page, scale, 0, out, ws, ws_bytes, None)


@pytest.mark.parametrize("bad,code", [
    (dict(batch=-1), 1), (dict(tokens=-1), 1), (dict(q_heads=0), 1), (dict(kv_heads=0), 1), (dict(q_heads=12), 1),
    (dict(head_dim=96), 2), (dict(page=0), 2), (dict(page=96), 2), (dict(num_pages=0), 1), (dict(max_pages=0), 1),
    (dict(q=None), 1), (dict(k=None), 1), (dict(v=None), 1), (dict(table=None), 1), (dict(cu_q=None), 1),
    (dict(kv_len=None), 1), (dict(out=None), 1), (dict(q=ODD), 1), (dict(k=ODD), 1), (dict(v=ODD), 1),
    (dict(out=ODD), 1), (dict(q_stride=16 * 128 - 8), 1), (dict(q_stride=16 * 128 + 4), 1),
    (dict(num_pages=1 << 22), 2), (dict(max_pages=1 << 25), 2), (dict(q_heads=258, kv_heads=2, q_stride=1 << 16), 2),
    (dict(scale=0.0), 1), (dict(scale=-0.1), 1), (dict(scale=float("nan")), 1), (dict(scale=float("inf")), 1),
    (dict(ws=None), 3), (dict(ws=ODD), 3), (dict(ws_bytes=1000), 3),
])
def test_chunk_attention_refusals(lib, bad, code):
    assert _attention(lib, **bad) == code
    assert lib.mb_last_error()


def _plan(lib, cu_q=P, kv_len=P, batch=2, tokens=5, q_heads=16, kv_heads=8, head_dim=128, page=128, max_pages=4, ws=P,
          ws_bytes=1 << 30):
    return lib.mb_chunk_plan(cu_q, kv_len, batch, tokens, q_heads, kv_heads, head_dim, page, max_pages, ws, ws_bytes, None)


@pytest.mark.parametrize("bad,code", [
    (dict(batch=-1), 1), (dict(tokens=-1), 1), (dict(q_heads=12), 1), (dict(head_dim=80), 2), (dict(page=32), 2),
    (dict(cu_q=None), 1), (dict(kv_len=None), 1), (dict(max_pages=0), 1), (dict(max_pages=1 << 25), 2),
    (dict(ws=None), 3), (dict(ws=ODD), 3), (dict(ws_bytes=1000), 3), (dict(q_heads=258, kv_heads=2), 2),
])
def test_chunk_plan_refusals(lib, bad, code):
    assert _plan(lib, **bad) == code
    assert lib.mb_last_error()


def test_chunk_workspace_size_rules(lib):
    size = lib.mb_chunk_workspace_bytes
    assert 0 < size(1, 1, 16, 8, 128) < size(256, 256, 16, 8, 128) <= size(256, 6000, 16, 8, 128)
    for bad in ((0, 1, 16, 8, 128), (1, 0, 16, 8, 128), (1, 1, 12, 8, 128), (1, 1, 16, 8, 96), (1, 1, 129, 1, 64)):
        assert size(*bad) == 0


def test_empty_chunk_attention_is_a_noop(lib):
    assert _attention(lib, batch=0, q=None, k=None, v=None, table=None, cu_q=None, kv_len=None, out=None, ws=None) == 0
    assert _attention(lib, tokens=0, q=None, k=None, v=None, table=None, cu_q=None, kv_len=None, out=None, ws=None) == 0


def test_wrappers_refuse_host_tensors():
    from mouse_core_b200 import kernels as K

    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        K.chunk_meta(i, i, torch.zeros(2, 4, dtype=torch.int32), i, 64, 5)
    pool = torch.zeros(2, 1, 64, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        K.chunk_attention(torch.zeros(3, 1, 64, dtype=torch.bfloat16), pool, pool, i.view(2, 1),
                          torch.zeros(3, dtype=torch.int32), i, 1.0)
