"""CPU checks of the 4-bit cache's C entry points: sizes, and arguments that
are refused before any device is touched."""
from __future__ import annotations

import ctypes
import importlib

import pytest


@pytest.fixture(scope="module")
def kv4():
    pytest.importorskip("torch")
    return importlib.import_module("cis2-lab-archive_b200.kv4")


def test_pool_size(kv4):
    c = kv4._Cache(0, 10, 64, 8, 128, 0, None, None)
    n = ctypes.c_uint64()
    assert kv4._lib().cis2b_kv4_bytes(ctypes.byref(c), ctypes.byref(n)) == 0
    assert n.value == 10 * 64 * 8 * 136
    c = kv4._Cache(0, 2 ** 22, 256, 100, 128, 0, None, None)  # past 32 bits
    assert kv4._lib().cis2b_kv4_bytes(ctypes.byref(c), ctypes.byref(n)) == 0 and n.value == 2 ** 30 * 13600


def test_the_package_does_not_need_torch(pkg):
    """Only kv4.py imports torch; loading the library and the other modules stays free of it."""
    import subprocess
    import sys
    code = ("import sys, importlib; sys.path.insert(0, %r); importlib.import_module('cis2-lab-archive_b200').lib(); "
            "assert 'torch' not in sys.modules" % pkg.ROOT_DIR)
    subprocess.run([sys.executable, "-c", code], check=True, timeout=120)


@pytest.mark.parametrize("field,value,word", [("pages", 0, "pages"), ("page_size", 48, "page_size"),
                                              ("page_size", 512, "page_size"), ("kv_heads", 0, "kv_heads"),
                                              ("head_dim", 96, "head_dim"), ("pages", 2 ** 27, "pages"),
                                              ("reserved", 1, "reserved"), ("pool", None, "pool"), ("pool", 24, "pool")])
def test_bad_caches_are_refused(kv4, field, value, word):
    L = kv4._lib()
    c = kv4._Cache(0, 4, 16, 2, 64, 0, 256, None)
    setattr(c, field, value)
    assert L.cis2b_kv4_append(ctypes.byref(c), 0, 256, 256, 1, 1, 1, 1, 256, 1, None) == 1
    assert word in kv4._pkg.lib().cis2b_last_error().decode()
    assert L.cis2b_kv4_append(None, 0, 256, 256, 1, 1, 1, 1, 256, 1, None) == 1


def test_bad_rows_are_refused(kv4):
    L = kv4._lib()
    c = ctypes.byref(kv4._Cache(0, 4, 16, 2, 64, 0, 256, None))
    for dtype, k, v, slot, rows in [(3, 256, 256, 256, 1), (-1, 256, 256, 256, 1), (0, None, 256, 256, 1),
                                    (0, 256, None, 256, 1), (0, 256, 256, None, 1), (0, 256, 256, 256, -1)]:
        assert L.cis2b_kv4_append(c, dtype, k, v, 1, 1, 1, 1, slot, rows, None) == 1
        assert L.cis2b_kv4_gather(c, dtype, k, v, slot, rows, None) == 1


@pytest.mark.parametrize("field,value", [("requests", 0), ("requests", 16385), ("rows", -1), ("width", 0), ("page_size", 8),
                                         ("free_count", -1), ("cached", None), ("table", None), ("slot", None),
                                         ("counts", None), ("free_pages", None), ("device", 64), ("device", -1)])
def test_bad_steps_are_refused(kv4, field, value):
    s = kv4._Step(0, 2, 4, 2, 16, 1, *([256] * 10))
    setattr(s, field, value)
    assert kv4._lib().cis2b_kv4_plan(ctypes.byref(s), None) == 1


@pytest.mark.parametrize("field,value", [("dtype", 3), ("heads", 5), ("heads", 66), ("heads", 0), ("requests", 0), ("rows", -1),
                                         ("width", 0), ("width", 2 ** 28), ("max_new", 0), ("window", -1), ("sinks", -1),
                                         ("scale", float("inf")), ("flags", 2), ("q", None), ("out", None), ("table", None),
                                         ("length", None), ("row_start", None), ("work", None), ("work", 8), ("work_bytes", 4)])
def test_bad_attention_calls_are_refused(kv4, field, value):
    c = kv4._Cache(0, 4, 16, 2, 64, 0, 256, None)
    a = kv4._Attn(0, 4, 2, 3, 4, 1, 0, 0, 0.125, 0, 256, 256, 256, 64, 256, 64, 256, 256, 256, 256, 2 ** 40)
    setattr(a, field, value)
    assert kv4._lib().cis2b_kv4_attention(ctypes.byref(c), ctypes.byref(a), None) == 1
    n = ctypes.c_uint64()
    assert kv4._lib().cis2b_kv4_workspace(ctypes.byref(c), None, ctypes.byref(n)) == 1


def test_batches_live_on_the_gpu(kv4):
    with pytest.raises(ValueError):
        kv4.Batch(1, 1, 1, 16, device="cpu")


def test_sizes_past_32_bits_are_refused(kv4):
    """A field of 32 bits would take 2^32 + 4 for 4."""
    for args in [(2 ** 32 + 4, 16, 1, 64), (4, 2 ** 32 + 16, 1, 64), (4, 16, 2 ** 32 + 1, 64), (4, 16, 1, 2 ** 32 + 64)]:
        with pytest.raises(ValueError):
            kv4.Cache(*args, device="cuda:0")
