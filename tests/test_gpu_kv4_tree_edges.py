"""Drafted trees and encoders over the 4-bit cache at their edges: hand-offs between warps, the ends of the
number range, requests alone and in large batches, windows shorter than a path, what a batch allocates.

Tolerances are those of test_gpu_kv4_tree.py; where a test needs another one its comment derives it."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from test_gpu_kv4 import World
from test_gpu_kv4_tree import DTYPES, NEW, Trees, check, everyone, i32, write

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return importlib.import_module("torch")


@pytest.fixture(scope="module")
def kv4():
    return importlib.import_module("cis2-lab-archive_b200.kv4")


# ---------------------------------------------------------------- hand-offs between warps

@pytest.mark.parametrize("new", [5, 14])  # of 4 heads of one KV head: 20 and 56 query columns
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("whole", [False, True])
def test_short_items_hand_over(torch, kv4, head_dim, new, whole):
    """Many items of none to a few key tiles behind one another in each block, some with missing pages: what is
    there, the last tile of an item and the end of the work are known in time, call after call."""
    g = np.random.default_rng(5)
    lengths = [int(n) for n in g.choice([0, 1, 15, 127, 128, 129, 300, 700], 350)]
    w = World(torch, kv4, lengths, [new] * 350, 1, head_dim, 16, "bfloat16", seed=4)
    gone = [r for r in range(350) if lengths[r] > 200 and r % 3 == 0]
    for r in gone:
        w.table[r, 3] = -1
    q = w.queries(4, head_dim)

    def see(r, i):
        j = np.arange(lengths[r])
        return (j // 16 != 3) | (r not in gone)
    want = w.cache.cross_attention(q, w.batch, max_new=new, whole=whole)
    check(w, q, want, see)
    for _ in range(100):
        assert torch.equal(w.cache.cross_attention(q, w.batch, max_new=new, whole=whole), want)
    assert w.cache.errors() == kv4.BAD_PAGE


# ---------------------------------------------------------------- the ends of the number range

@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("size", [2.0 ** 125, 2.0 ** 126, 2.0 ** 127])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_few_keys_of_the_largest_values(torch, kv4, dtype, size, new):
    """One key, or a few, whose values are the largest that a cache holds: their mean is one that the type holds."""
    g = np.random.default_rng(3)
    w = World(torch, kv4, [1, 2, 40], [new] * 3, 1, 64, 16, dtype)
    for r, n in enumerate(w.lengths):
        write(torch, w, w.x[r], np.float32(size) * g.uniform(1, 1.8, (n, 1, 64)).astype(np.float32), r)
    q = w.queries(4, 64)
    check(w, q, w.cache.cross_attention(q, w.batch, max_new=new), everyone(w))


# ---------------------------------------------------------------- alone and in a batch

@pytest.mark.parametrize("heads,new", [(8, 17), (64, 8), (8, 65), (64, 9), (64, 16), (8, 129)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_request_alone_gives_the_bits_it_gives_in_a_large_batch(torch, kv4, dtype, heads, new):
    """17, 64, 65, 72, 128 and 129 query columns a KV head, 8 KV heads, alone and with 47 other requests."""
    n, g = 48, np.random.default_rng(9)
    t = Trees(torch, kv4, [int(x) for x in g.integers(new, 400, n)], [new] * n, 8, 64, 16, dtype, seed=81)
    w, q = t.w, t.w.queries(heads, 64)
    more = dict(max_new=new, whole=True)
    tree, cross = w.cache.tree_attention(q, w.batch, **t.args, **more), w.cache.cross_attention(q, w.batch, **more)
    for r in (0, 41):
        rows = slice(r * new, (r + 1) * new)
        one = kv4.Batch.of(w.table[r:r + 1], w.batch.length[r:r + 1].clone(), i32(torch, [0, new]), 16)
        assert torch.equal(w.cache.tree_attention(q[rows], one, mask=t.args["mask"][rows], **more), tree[rows])
        assert torch.equal(w.cache.cross_attention(q[rows], one, **more), cross[rows])
