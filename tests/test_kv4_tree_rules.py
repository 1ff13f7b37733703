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


@pytest.mark.parametrize("requests,width,window,few", [(20, 4, 0, True), (21, 4, 0, False), (50, 62, 0, False), (50, 63, 0, True),
                                                       (160, 2000, 0, True), (161, 2000, 0, False), (50, 2000, 900, False),
                                                       (50, 2000, 968, True), (1, 1, 1, True)])
def test_which_kernel_128_columns_take_goes_by_items_and_keys(kv4, requests, width, window, few):  # noqa: F811
    """2 KV heads: up to 40 items take the kernel of 64 columns, else a tenth of the keys that a row may see, up to
    320.  The window with 32 new tokens: 968 + 32 = 1,000 keys."""
    n = ctypes.c_uint64()
    c, sizes = cache(kv4, head_dim=128, page_size=16), []
    for flags in (0, 1):
        a = attention(kv4, dtype=2, max_new=32, requests=requests, rows=32 * requests, width=width, window=window, flags=flags)
        assert kv4._lib().cis2b_kv4_tree_workspace(ctypes.byref(c), ctypes.byref(a), ctypes.byref(n)) == 0
        sizes.append(n.value)
    columns = 266240 + 160 * 2 * 64 * 130 * 4  # two parts of 64 columns for each of 160 blocks
    assert (sizes[0] == columns) == few and sizes[1] != columns
