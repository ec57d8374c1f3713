"""Paged 4-bit cache, without a GPU: sizes, refusals, and the documented layout against itself."""
import ctypes as C
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import _kv4  # noqa: E402


def descriptor(capi, lib, **over):
    """A descriptor whose pointers are numbers: every call below must be refused before it looks behind them."""
    v = dict(pages=1 << 20, table=1 << 20, lens=1 << 20, refs=1 << 20, work=1 << 20, work_bytes=1 << 40, n_pages=10, layers=2, kv_heads=8, q_heads=32,
             max_seqs=6, table_stride=4)
    v.update(over)
    return capi.Kv4(*(v[name] for name, _ in capi.Kv4._fields_))


def batch(capi, **over):
    v = dict(seqs=1 << 20, row0=1 << 20, pos0=1 << 20, n=2, rows=3, max_rows=2)
    v.update(over)
    return capi.Kv4Batch(*(v[name] for name, _ in capi.Kv4Batch._fields_))


def test_layout_covers_each_place_once():
    seen = []
    for which in (0, 1):
        byte, shift, s, m = _kv4.places(which)
        seen += sorted(zip(byte.flatten().tolist(), shift.flatten().tolist()))
        seen += [(b + o, 8) for at in (s, m) for b in sorted(set(at.flatten().tolist())) for o in (0, 1)]
    assert len(seen) == len(set(seen)) and {b for b, _ in seen} == set(range(_kv4.BLOCK))


def test_pack_and_unpack_are_inverses():
    g = torch.Generator().manual_seed(0)
    blocks = torch.zeros(3, _kv4.BLOCK, dtype=torch.uint8)
    want = {}
    for which in (0, 1):
        for i in range(16):
            want[which, i] = _kv4.quantise(torch.randn(3, 128, generator=g))
            _kv4.pack(blocks, which, i, *want[which, i])
    for which in (0, 1):
        c, s, m = _kv4.unpack(blocks, which)
        for i in range(16):
            for got, ref in zip((c, s, m), want[which, i]):
                assert torch.equal(got[:, i], ref.double())


def test_struct_layouts(capi):
    assert C.sizeof(capi.Kv4) == 72 and capi.Kv4.work_bytes.offset == 40 and capi.Kv4.n_pages.offset == 48 and capi.Kv4.table_stride.offset == 68
    assert C.sizeof(capi.Kv4Batch) == 40 and capi.Kv4Batch.n.offset == 24 and capi.Kv4Batch.max_rows.offset == 32


def test_sizes(mine, capi):
    assert mine.s2p_b200_kv4_page_bytes(36, 8) == 36 * 8 * 4 * 2560
    assert mine.s2p_b200_kv4_page_bytes(0, 8) == 0 and mine.s2p_b200_kv4_page_bytes(1, -1) == 0
    small, large = (mine.s2p_b200_kv4_work_bytes(C.byref(descriptor(capi, mine)), n) for n in (1, 100000))
    assert 0 < small < large
    for bad in (dict(q_heads=12), dict(q_heads=8 * 17), dict(kv_heads=0), dict(n_pages=0), dict(layers=0), dict(max_seqs=0), dict(table_stride=0),
                dict(table_stride=(1 << 24) + 1), dict(n_pages=(1 << 22) + 1)):
        assert mine.s2p_b200_kv4_work_bytes(C.byref(descriptor(capi, mine, **bad)), 1) == 0
    assert mine.s2p_b200_kv4_work_bytes(None, 1) == 0 and mine.s2p_b200_kv4_work_bytes(C.byref(descriptor(capi, mine)), -1) == 0


P = 1 << 20


def calls(mine, c, b, layer=0):
    """Every entry point that takes a cache, with otherwise fine arguments."""
    one, two, tok = ((C.c_int32 * 1)(v) for v in (0, 1, 5))
    yield lambda: mine.s2p_b200_kv4_reserve(c, b, None, None)
    yield lambda: mine.s2p_b200_kv4_append(c, b, layer, P, P, P, 1e-6, 1e6, P, None)
    yield lambda: mine.s2p_b200_kv4_attention(c, b, layer, P, P, None)
    yield lambda: mine.s2p_b200_kv4_read(c, b, layer, P, P, None)
    yield lambda: mine.s2p_b200_kv4_fork(c, one, two, tok, 1, None, None)
    yield lambda: mine.s2p_b200_kv4_release(c, one, 1, None)
    yield lambda: mine.s2p_b200_kv4_compact(c, None, None)
    yield lambda: mine.s2p_b200_kv4_status(c, None)


@pytest.mark.parametrize("bad", [dict(pages=None), dict(table=None), dict(lens=None), dict(refs=None), dict(work=None), dict(pages=P + 64), dict(work=P + 128),
                                 dict(table=P + 2), dict(refs=P + 1), dict(work_bytes=1000), dict(q_heads=30), dict(q_heads=136), dict(n_pages=-1),
                                 dict(table_stride=1 << 25)])
def test_every_call_refuses_a_bad_cache(mine, capi, bad):
    c, b = descriptor(capi, mine, **bad), batch(capi)
    for call in calls(mine, C.byref(c), C.byref(b)):
        assert call() == -1
    for call in calls(mine, None, C.byref(b)):
        assert call() == -1


@pytest.mark.parametrize("bad", [dict(n=-1), dict(rows=-1), dict(max_rows=-1), dict(n=1025), dict(seqs=None), dict(row0=None), dict(pos0=None), dict(row0=P + 2)])
def test_row_calls_refuse_a_bad_batch(mine, capi, bad):
    c, b = descriptor(capi, mine), batch(capi, **bad)
    for i, call in enumerate(calls(mine, C.byref(c), C.byref(b))):
        if i < 4:
            assert call() == -1
    for i, call in enumerate(calls(mine, C.byref(c), None)):
        if i < 4:
            assert call() == -1


def test_row_calls_refuse_layers_and_pointers(mine, capi):
    c, b = C.byref(descriptor(capi, mine)), C.byref(batch(capi))
    for layer in (-1, 2):
        for i, call in enumerate(calls(mine, c, b, layer)):
            if 1 <= i <= 3:
                assert call() == -1
    for qkv, qn, kn, q in ((None, P, P, P), (P, P, P, None), (P + 8, P, P, P), (P, P, P, P + 2), (P, P + 4, P, P), (P, P, P + 2, P)):
        assert mine.s2p_b200_kv4_append(c, b, 0, qkv, qn, kn, 1e-6, 1e6, q, None) == -1
    for eps, base in ((-1.0, 1e6), (float("nan"), 1e6), (1e-6, 0.0), (1e-6, -3.0), (1e-6, float("nan")), (1e-6, float("inf"))):
        assert mine.s2p_b200_kv4_append(c, b, 0, P, P, P, eps, base, P, None) == -1
    for x, y in ((None, P), (P, None), (P + 8, P), (P, P + 4)):
        assert mine.s2p_b200_kv4_attention(c, b, 0, x, y, None) == -1
        assert mine.s2p_b200_kv4_read(c, b, 0, x, y, None) == -1
    assert mine.s2p_b200_kv4_reserve(c, b, P + 2, None) == -1 and mine.s2p_b200_kv4_compact(c, P + 2, None) == -1


def test_attention_refuses_more_work_than_it_counts(mine, capi):
    c = C.byref(descriptor(capi, mine, table_stride=1 << 20))
    assert mine.s2p_b200_kv4_attention(c, C.byref(batch(capi, rows=65)), 0, P, P, None) == -1


def test_lists_are_checked(mine, capi):
    c = C.byref(descriptor(capi, mine))
    L = lambda *v: (C.c_int32 * len(v))(*v)  # noqa: E731
    fork = lambda p, k, t: mine.s2p_b200_kv4_fork(c, p, k, t, len(k), None, None)  # noqa: E731
    assert fork(L(0, 0), L(1, 1), L(3, 3)) == -1      # the same child twice
    assert fork(L(0, 1), L(1, 2), L(3, 3)) == -1      # a child that is a parent
    assert fork(L(3), L(3), L(1)) == -1
    assert fork(L(6), L(1), L(1)) == -1 and fork(L(-1), L(1), L(1)) == -1
    assert fork(L(0), L(6), L(1)) == -1 and fork(L(0), L(-1), L(1)) == -1
    assert fork(L(0), L(1), L(-2)) == -1
    assert mine.s2p_b200_kv4_fork(c, None, L(1), L(1), 1, None, None) == -1
    assert mine.s2p_b200_kv4_fork(c, L(0), L(1), None, 1, None, None) == -1
    assert mine.s2p_b200_kv4_fork(c, L(0), L(1), L(1), -1, None, None) == -1
    assert mine.s2p_b200_kv4_fork(c, L(0), L(1), L(1), 257, None, None) == -1
    assert mine.s2p_b200_kv4_release(c, L(1, 2, 1), 3, None) == -1
    assert mine.s2p_b200_kv4_release(c, L(6), 1, None) == -1 and mine.s2p_b200_kv4_release(c, None, 1, None) == -1
    assert mine.s2p_b200_kv4_release(c, L(1), 257, None) == -1 and mine.s2p_b200_kv4_release(c, L(1), -1, None) == -1


def test_calls_without_work_do_nothing(mine, capi):
    c = C.byref(descriptor(capi, mine))
    for b in (batch(capi, n=0, seqs=None, row0=None, pos0=None), batch(capi, rows=0)):
        assert mine.s2p_b200_kv4_append(c, C.byref(b), 0, None, None, None, 1e-6, 1e6, None, None) == 0
        assert mine.s2p_b200_kv4_attention(c, C.byref(b), 1, None, None, None) == 0
        assert mine.s2p_b200_kv4_read(c, C.byref(b), 0, None, None, None) == 0
    assert mine.s2p_b200_kv4_reserve(c, C.byref(batch(capi, n=0)), None, None) == 0
    assert mine.s2p_b200_kv4_fork(c, None, None, None, 0, None, None) == 0
    assert mine.s2p_b200_kv4_release(c, None, 0, None) == 0
