"""The C entry points of a drafted step refuse on the host what they cannot do, before any launch (runs without a GPU)."""

from __future__ import annotations

import ctypes

import pytest

from nanoserve_amd import _lib

BIG = 1 << 40  # aligned, never read: every call here returns before a launch
INVALID, UNSUPPORTED, WORKSPACE = _lib.NS_ERR_INVALID_ARG, _lib.NS_ERR_UNSUPPORTED, _lib.NS_ERR_WORKSPACE


def _attention(**over):
    a = dict(out=BIG, query=BIG, k=BIG, v=BIG, bt=BIG, bt_stride=64, bt_width=64, bt64=1, sl=BIG, sl64=1, qsl=BIG, qsl64=1,
             mask=BIG, S=2, T=16, maxq=8, maxs=1024, Hq=14, Hkv=2, D=64, bs=16, nb=128, scale=0.125,
             dtype=_lib.NS_DTYPE_F16, counters=BIG, ws=BIG, ws_bytes=1 << 40, stream=None)
    a.update(over)
    return _lib.load().ns_paged_attention_tree(*a.values())


@pytest.mark.parametrize("over,code", [
    (dict(Hq=15), INVALID), (dict(Hkv=0), INVALID), (dict(D=0), INVALID), (dict(bs=0), INVALID), (dict(nb=0), INVALID),
    (dict(S=-1), INVALID), (dict(T=-1), INVALID), (dict(maxq=-1), INVALID), (dict(maxs=-1), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID),
    (dict(out=None), INVALID), (dict(query=None), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID),
    (dict(bt=None), INVALID), (dict(sl=None), INVALID), (dict(mask=None), INVALID),
    (dict(qsl=None), INVALID), (dict(bt_width=0), INVALID), (dict(bt_stride=63), INVALID),
    (dict(out=BIG + 8), INVALID), (dict(query=BIG + 2), INVALID), (dict(k=BIG + 8), INVALID), (dict(v=BIG + 4), INVALID),
    (dict(bt=BIG + 4), INVALID), (dict(bt=BIG + 2, bt64=0), INVALID), (dict(sl=BIG + 4), INVALID),
    (dict(qsl=BIG + 4), INVALID), (dict(mask=BIG + 4), INVALID),
    (dict(dtype=7), UNSUPPORTED), (dict(D=320), UNSUPPORTED), (dict(maxq=65), UNSUPPORTED),
    (dict(maxs=(1 << 30) + 1, bt_width=1 << 28, bt_stride=1 << 28), UNSUPPORTED),
    (dict(T=1 << 30), UNSUPPORTED), (dict(S=1 << 28, T=1 << 28), UNSUPPORTED), (dict(Hq=1 << 17, Hkv=1 << 17), UNSUPPORTED),
    # More work than its line of 32 bits holds for one sequence.
    (dict(Hq=512, Hkv=64, maxq=64, maxs=1 << 30, bt_width=1 << 26, bt_stride=1 << 26), UNSUPPORTED),
    (dict(counters=None), WORKSPACE), (dict(counters=BIG + 2), WORKSPACE), (dict(ws=None), WORKSPACE),
    (dict(ws=BIG + 8), WORKSPACE), (dict(ws_bytes=1024), WORKSPACE),
])
def test_attention_refuses(over, code):
    assert _attention(**over) == code


def test_attention_of_nothing():
    assert _attention(S=0, T=0, out=None, query=None, qsl=None) == _lib.NS_OK
    assert _attention(T=0) == _lib.NS_OK


def test_attention_workspace_sizes():
    lib = _lib.load()
    size = lambda S, Hq, Hkv, D, bs, maxq, T, dt: lib.ns_paged_attention_tree_workspace_size(S, Hq, Hkv, D, bs, maxq, T, dt)  # noqa: E731
    f16, bf16, f32 = _lib.NS_DTYPE_F16, _lib.NS_DTYPE_BF16, _lib.NS_DTYPE_F32
    for dt in (f16, bf16):
        for D in (64, 128):
            n = size(2, 14, 2, D, 16, 8, 16, dt)
            assert n > 0 and n % 16 == 0
            assert _attention(D=D, dtype=dt, ws_bytes=n - 1) == WORKSPACE
    # Shapes of the plain kernel keep no partial results.
    for args in ((2, 14, 2, 64, 16, 8, 16, f32), (2, 14, 2, 80, 16, 8, 16, f16), (2, 14, 2, 64, 8, 8, 16, f16),
                 (0, 14, 2, 64, 16, 8, 16, f16), (2, 14, 2, 64, 16, 8, 0, f16), (2, 15, 2, 64, 16, 8, 16, f16)):
        assert size(*args) == 0
    assert lib.ns_paged_attention_tree_counters() > 0


def _inputs(**over):
    a = dict(tables=BIG, R=4, W=32, stride=32, t64=1, rows=BIG, computed=BIG, lens=BIG, new=BIG, start=BIG, held=BIG, N=3,
             parents=BIG, i64=1, S=2, T=16, bs=16, maxb=32, qsl=BIG, sl=BIG, pos=BIG, slots=BIG, packed=BIG, mask=BIG, stream=None)
    a.update(over)
    return _lib.load().ns_step_inputs(*a.values())


@pytest.mark.parametrize("over", [
    dict(R=-1), dict(W=-1), dict(stride=31), dict(N=-1), dict(S=-1), dict(T=-1), dict(bs=0), dict(maxb=-1),
    dict(rows=None), dict(computed=None), dict(lens=None), dict(new=None), dict(start=None), dict(held=None),
    dict(qsl=None), dict(sl=None), dict(pos=None), dict(slots=None), dict(packed=None), dict(mask=None), dict(tables=None),
    dict(rows=BIG + 4), dict(computed=BIG + 2, i64=0), dict(tables=BIG + 4), dict(tables=BIG + 2, t64=0), dict(qsl=BIG + 4),
    dict(packed=BIG + 4), dict(mask=BIG + 4),
])
def test_step_inputs_refuses(over):
    assert _inputs(**over) in (INVALID, UNSUPPORTED)


def _commit(caches=(BIG, BIG), **over):
    array = (ctypes.c_void_p * max(len(caches), 1))(*caches)
    a = dict(counts=BIG, tokens=BIG, chosen=BIG, ids=BIG, parents=BIG, i64=1, qsl=BIG, qsl64=1, slots=BIG, slots64=1, S=2, T=16,
             maxr=8, array=ctypes.addressof(array), n=len(caches), num_slots=512, row_bytes=256, stream=None)
    a.update(over)
    return _lib.load().ns_commit_drafts(*a.values())


@pytest.mark.parametrize("over", [
    dict(counts=None), dict(tokens=None), dict(chosen=None), dict(ids=None), dict(parents=None), dict(qsl=None),
    dict(slots=None), dict(S=-1), dict(T=-1), dict(maxr=-1), dict(maxr=65), dict(array=None), dict(n=-1),
    dict(num_slots=-1), dict(row_bytes=-1), dict(caches=(BIG, 0)), dict(counts=BIG + 4), dict(chosen=BIG + 4),
    dict(qsl=BIG + 4), dict(slots=BIG + 4), dict(chosen=BIG + 2, i64=0),
])
def test_commit_refuses(over):
    assert _commit(**over) in (INVALID, UNSUPPORTED)


def test_commit_of_nothing():
    assert _commit(S=0, T=0, caches=()) == _lib.NS_OK
