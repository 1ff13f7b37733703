"""CPU checks of what the forms of attention over the 4-bit cache ask for: the workspace's size shows which
kernel a call takes."""
from __future__ import annotations

import ctypes

import pytest

from test_kv4_tree_abi import attention, cache, kv4, message  # noqa: F401


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("new", [1, 2, 4, 5, 8, 16, 17, 32, 33, 64, 128, 129, 1000])
def test_a_whole_request_takes_the_same_kernel_in_any_batch(kv4, dtype, new):  # noqa: F811
    sizes = set()
    for requests in (1, 2, 40, 81, 160, 161, 1000):
        a = attention(kv4, dtype=dtype, max_new=new, requests=requests, rows=requests * new, flags=1)
        n = ctypes.c_uint64()
        assert kv4._lib().cis2b_kv4_tree_workspace(ctypes.byref(cache(kv4)), ctypes.byref(a), ctypes.byref(n)) == 0
        sizes.add(n.value)
    assert len(sizes) == 1


@pytest.mark.parametrize("window,sinks", [(-1, 0), (0, -1), (-2 ** 31, 3)])
def test_bad_windows_of_a_tree_are_refused(kv4, window, sinks):  # noqa: F811
    t = kv4._Tree(0, 2, 4, 1, *([256] * 5), None)
    assert kv4._lib().cis2b_kv4_plan_tree_window(ctypes.byref(t), window, sinks, None) == 1 and "window" in message(kv4)
    assert kv4._lib().cis2b_kv4_plan_tree_window(None, 0, 0, None) == 1
