"""CPU checks of the C entry points for drafted trees and encoders over the
4-bit cache: arguments that are refused before any device is touched."""
from __future__ import annotations

import ctypes
import importlib

import pytest


@pytest.fixture(scope="module")
def kv4():
    pytest.importorskip("torch")
    return importlib.import_module("cis2-lab-archive_b200.kv4")


def message(kv4):
    return kv4._pkg.lib().cis2b_last_error().decode()


def cache(kv4, **more):
    c = kv4._Cache(0, 4, 16, 2, 64, 0, 256, None)
    for k, v in more.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("field,value,word", [("requests", 0, "requests"), ("rows", -1, "rows"), ("words", 0, "words"), ("words", 33, "words"),
                                              ("length", None, "NULL"), ("row_start", None, "NULL"), ("parent", None, "NULL"),
                                              ("mask", None, "NULL"), ("position", None, "NULL"), ("device", 64, "device"),
                                              ("device", -1, "device")])
def test_bad_trees_are_refused(kv4, field, value, word):
    t = kv4._Tree(0, 2, 4, 1, *([256] * 5), None)
    setattr(t, field, value)
    assert kv4._lib().cis2b_kv4_plan_tree(ctypes.byref(t), None) == 1 and word in message(kv4)
    assert kv4._lib().cis2b_kv4_plan_tree(None, None) == 1


@pytest.mark.parametrize("field,value,word", [("requests", 0, "requests"), ("rows", -1, "rows"), ("reserved", 1, "reserved"), ("device", 99, "device")] +
                         [(f, None, "NULL") for f in ("length", "row_start", "token", "parent", "target", "accepted", "path",
                                                      "next_token", "kept")])
def test_bad_drafts_are_refused(kv4, field, value, word):
    d = kv4._Draft(0, 2, 4, 0, *([256] * 9), None)
    setattr(d, field, value)
    assert kv4._lib().cis2b_kv4_accept(ctypes.byref(d), None) == 1 and word in message(kv4)
    assert kv4._lib().cis2b_kv4_accept(None, None) == 1


@pytest.mark.parametrize("field,value,word", [("requests", 0, "requests"), ("rows", -1, "rows"), ("reserved", 1, "reserved"), ("device", 1, "device"),
                                              ("row_start", None, "NULL"), ("accepted", None, "NULL"), ("path", None, "NULL"),
                                              ("slot", None, "NULL")])
def test_bad_moves_are_refused(kv4, field, value, word):
    k = kv4._Kept(0, 2, 4, 0, 256, 256, 256, 256)
    setattr(k, field, value)
    one = (kv4._Cache * 1)(cache(kv4))
    assert kv4._lib().cis2b_kv4_keep(one, 1, ctypes.byref(k), None) == 1 and word in message(kv4)
    assert kv4._lib().cis2b_kv4_keep(one, 1, None, None) == 1


@pytest.mark.parametrize("more", [dict(head_dim=128), dict(page_size=32), dict(kv_heads=1), dict(device=1), dict(pool=None), dict(pool=8)])
def test_caches_that_do_not_belong_together_are_refused(kv4, more):
    k = ctypes.byref(kv4._Kept(0, 2, 4, 0, 256, 256, 256, 256))
    two = (kv4._Cache * 2)(cache(kv4), cache(kv4, **more))
    assert kv4._lib().cis2b_kv4_keep(two, 2, k, None) == 1
    assert kv4._lib().cis2b_kv4_keep(two, 0, k, None) == 1
    assert kv4._lib().cis2b_kv4_keep(None, 1, k, None) == 1


def attention(kv4, **more):
    a = kv4._Attn(2, 8, 2, 12, 4, 6, 0, 0, 0.125, 0, 256, 256, 512, 64, 512, 64, 256, 256, 256, 256, 2 ** 40)
    for k, v in more.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("max_new", [1, 2, 6])
@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("field,value", [("dtype", 3), ("heads", 5), ("heads", 66), ("requests", 0), ("rows", -1), ("width", 0), ("width", 2 ** 28),
                                         ("max_new", 0), ("window", -1), ("sinks", -1), ("scale", float("inf")), ("flags", 2), ("q", None),
                                         ("out", None), ("table", None), ("length", None), ("row_start", None), ("work", None),
                                         ("work", 8), ("work_bytes", 4), ("requests", 2 ** 30)])
def test_bad_attention_calls_are_refused(kv4, field, value, dtype, max_new):
    L, c = kv4._lib(), cache(kv4)
    a = attention(kv4, dtype=dtype, max_new=max_new)
    setattr(a, field, value)
    assert L.cis2b_kv4_tree_attention(ctypes.byref(c), ctypes.byref(a), 256, 1, 256, None) == 1
    assert L.cis2b_kv4_cross_attention(ctypes.byref(c), ctypes.byref(a), None) == 1


def test_masks_positions_and_windows_are_checked(kv4):
    L, c = kv4._lib(), ctypes.byref(cache(kv4))
    for mask, words, position, window in [(None, 1, 256, 0), (256, 0, 256, 0), (256, 2 ** 26, 256, 0), (256, 1, None, 9)]:
        a = attention(kv4, window=window)
        assert L.cis2b_kv4_tree_attention(c, ctypes.byref(a), mask, words, position, None) == 1
    for more in (dict(window=5), dict(sinks=1)):
        assert L.cis2b_kv4_cross_attention(c, ctypes.byref(attention(kv4, **more)), None) == 1
    assert L.cis2b_kv4_tree_attention(c, None, 256, 1, 256, None) == 1 and L.cis2b_kv4_cross_attention(c, None, None) == 1
    n = ctypes.c_uint64()
    assert L.cis2b_kv4_tree_workspace(c, None, ctypes.byref(n)) == 1
    assert L.cis2b_kv4_tree_workspace(c, ctypes.byref(attention(kv4)), None) == 1
    for dtype in range(3):
        for new in (1, 2, 6, 100):
            assert L.cis2b_kv4_tree_workspace(c, ctypes.byref(attention(kv4, dtype=dtype, max_new=new)), ctypes.byref(n)) == 0
            assert n.value >= 266240

