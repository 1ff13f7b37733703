"""Drafted trees and encoders over the 4-bit cache at their edges: hand-offs between warps, the ends of the
number range, requests alone and in large batches, windows shorter than a path, what a batch allocates.

Tolerances are those of test_gpu_kv4_tree.py; where a test needs another one its comment derives it."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from test_gpu_kv4 import World, stands_for
from test_gpu_kv4_tree import DTYPES, NEW, Trees, bits, check, everyone, i32, plain_plan, plain_rows, random_parents, sees_tree, tolerance, write

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


@pytest.mark.parametrize("new", [5, 14, 30])  # of 4 heads: query columns that k_kv4_columns takes
@pytest.mark.parametrize("q_power,k_power,scale,elements", [(0, 125, 1.0, 1), (-3, 126, 0.125, 1), (-100, 126, 0.125, 64),
                                                            (-60, 120, 1.0, 64), (126, -100, 2.0, 64), (127, -110, 4.0, 64),
                                                            (127, -5, 1.0, 1), (-110, 126, 16.0, 64), (-125, 120, 1.0, 64)])
def test_scores_whose_factors_are_far_apart(torch, kv4, q_power, k_power, scale, elements, new):
    """Queries and keys of the largest and smallest sizes, whose scores fp32 holds: the first is far above the
    others, or all are near 0."""
    d, n = 64, 300
    g = np.random.default_rng(3)
    w = World(torch, kv4, [n], [new], 1, d, 16, "bfloat16")
    first = 77
    t = np.where(np.arange(n) == first, 1.0, g.uniform(-1, 0.4, n))
    write(torch, w, t[:, None, None] * g.uniform(1, 1.2, (n, 1, d)) * 2.0 ** k_power, w.y[0])
    q = torch.zeros((new, 4, d), device="cuda")
    q[:, :, :elements] = 2.0 ** q_power
    q = q.to(w.dtype)
    out = w.cache.cross_attention(q, w.batch, scale=scale, max_new=new)
    want = plain_rows(q.double().cpu().numpy(), w.k, w.v, w.new, scale, everyone(w))
    # Scores: a key's elements are rounded to 2^-11, and the largest score is 1.2 / (0.4 * 1.2) of the next: far apart,
    # or (-125 + 120 + 6 bits) below 2^2, where tolerance() holds.  Values and weights: 11 bits, the result 8.
    limit = 2 * (2.0 ** -11 * 4 + 2.0 ** -11) + 2.0 ** -11 + 2.0 ** -15 + 2.0 ** -8
    assert np.abs(out.double().cpu().numpy() - want).max() <= limit * np.abs(w.v[0]).max()


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("q_power,k_power", [(119, -100), (-100, 117), (0, 117), (119, 0)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_scores_within_every_kernels_range(torch, kv4, dtype, q_power, k_power, new):
    """Queries below 2^120 and keys below 2^118, all elements of one sign, in every kernel."""
    d, n = 128, 300
    g = np.random.default_rng(3)
    w = World(torch, kv4, [n], [new], 1, d, 16, dtype)
    t = np.where(np.arange(n) == 77, 1.0, g.uniform(0, 0.4, n))
    write(torch, w, t[:, None, None] * g.uniform(1, 1.2, (n, 1, d)) * 2.0 ** k_power, w.y[0])
    q = torch.full((new, 4, d), 2.0 ** q_power, device="cuda").to(w.dtype)
    out = w.cache.cross_attention(q, w.batch, max_new=new).double().cpu().numpy()
    # One key has all the weight: its value, in 22 or 11 bits, and the result's rounding.
    assert np.abs(out - w.v[0][77]).max() <= {"float32": 2.0 ** -20, "bfloat16": 2.0 ** -10 + 2.0 ** -8}[dtype] * np.abs(w.v[0][77]).max()


@pytest.mark.parametrize("new", [5, 14, 30])
def test_unseen_keys_of_the_largest_size_change_no_bit(torch, kv4, new):
    """Scores are formed in two ways, by the sizes of the keys beside them: with the same bits."""
    d, n = 64, 300
    w = World(torch, kv4, [n], [new], 1, d, 16, "bfloat16")
    q = w.queries(4, d)
    clean = w.cache.cross_attention(q, w.batch, max_new=new)
    check(w, q, clean, everyone(w))
    slot = i32(torch, [int(w.table[0, (n - 1) // 16]) * 16 + n % 16])  # behind the last key, in its tile and page
    huge = torch.full((1, 1, d), 3e38, device="cuda")
    huge[0, 0, ::2] = 1e30
    w.cache.append(huge, huge, slot)
    assert torch.equal(w.cache.cross_attention(q, w.batch, max_new=new), clean)


# ---------------------------------------------------------------- sums over many keys

@pytest.mark.parametrize("new", [1, 4, 12, 20, 70])  # 4 to 280 query columns
def test_fp32_sums_over_many_keys_are_rounded(torch, kv4, new):
    """Every token has the same value, so that is the result, whatever the weights; what is off is sums.  Of 32,768
    keys each of a block's eight warps adds up 256 records of 16.  Rounded to nearest, 256 adds are off by a standard
    deviation of 2^-23 sqrt(256 / 36) (the sum so far grows evenly), the denominators' in eight lanes by less, and
    eight warps' mean by 1 / sqrt(8) of that: 1.3e-7, eight of which are 1.1e-6.  Within a record two products of 16
    addends and a sum cut off up to 2^-24 of the largest each, at most 2 * 17 * 2^-24 = 2.0e-6 of the whole.  Chains of
    products over all records would cut off half of 2^-24 to 2^-23 of the sum so far, twice a record, always
    towards zero: about 1.1e-5."""
    n, d, page = 32768, 64, 64
    cache = kv4.Cache(n // page, page, 1, d)
    g = np.random.default_rng(0)
    x = g.standard_normal((n, 1, d)).astype(np.float32)
    y = np.where(np.arange(d) < d // 2, 1.0, -1.0).astype(np.float32)
    cache.append(torch.from_numpy(x).cuda(), torch.from_numpy(y).cuda().expand(n, 1, d).contiguous(), i32(torch, np.arange(n)))
    q = torch.from_numpy(g.standard_normal((new, 4, d)).astype(np.float32)).cuda()
    batch = kv4.Batch.of(i32(torch, np.arange(n // page)[None]), i32(torch, [n]), i32(torch, [0, new]), page)
    out = cache.cross_attention(q, batch, max_new=new, whole=True).double().cpu().numpy()
    assert np.abs(out - stands_for(y[None])[0]).max() <= 3.2e-6


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
    if new == 16:  # and beside many others, in parts or not, they are right
        check(w, q, tree, t.see())
        check(w, q, w.cache.tree_attention(q, w.batch, **t.args, max_new=new), t.see())
    for r in (0, 41):
        rows = slice(r * new, (r + 1) * new)
        one = kv4.Batch.of(w.table[r:r + 1], w.batch.length[r:r + 1].clone(), i32(torch, [0, new]), 16)
        assert torch.equal(w.cache.tree_attention(q[rows], one, mask=t.args["mask"][rows], **more), tree[rows])
        assert torch.equal(w.cache.cross_attention(q[rows], one, **more), cross[rows])


# ---------------------------------------------------------------- paths longer than the window

WINDOWS = [(1, 0), (7, 0), (16, 2), (5, 43), (30, 300), (33, 0), (1000, 4)]


def plain_window(parent, lengths, new, rows, words, window, sinks):
    """plan_tree's masks and positions, less the ancestors that the window hides."""
    mask, position = plain_plan(parent, lengths, new, rows, words)
    start = np.concatenate([[0], np.cumsum(new)])
    for r, n in enumerate(new):
        for i in range(min(n, 32 * words)):
            for b in range(i):
                at = position[start[r] + b]
                if at <= position[start[r] + i] - window and at >= sinks:
                    mask[start[r] + i, b // 32] &= ~np.uint32(1 << (b % 32))
    return mask, position


@pytest.mark.parametrize("window,sinks", WINDOWS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_chain_longer_than_the_window_is_causal_attention(torch, kv4, dtype, window, sinks):
    """Tokens that each continue the last see what a layer with a sliding window shows them: the same rows as
    attention()'s, within both kernels' tolerances."""
    lengths, new, d = [300, 41, 5], [40, 33, 5], 64
    w = World(torch, kv4, lengths, new, 2, d, 16, dtype, seed=9)
    batch = kv4.Batch.of(w.table, w.batch.length, w.batch.row_start, 16, rows=78, tree=40)
    batch.plan_tree(i32(torch, np.concatenate([np.arange(n) - 1 for n in new])), window, sinks)
    q = w.queries(8, d)
    more = dict(window=window, sinks=sinks, max_new=40)
    a, b = w.cache.attention(q, w.batch, **more), w.cache.tree_attention(q, batch, **more)
    top = max(np.abs(v).max() for v in w.v)
    assert (a.double() - b.double()).abs().max().item() <= 2 * tolerance(w, q, d ** -0.5) * top
    assert batch.tree_errors() == 0


@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_plan_tree_with_a_window_matches_the_loops(torch, kv4, window, sinks):
    g = np.random.default_rng(window)
    for new, pad in (([1], 0), ([0, 5, 70], 3), ([31, 32, 33, 64, 65], 0), ([300, 3], 7)):
        rows, tree, words = sum(new) + pad, max(new), (max(new) + 31) // 32
        lengths = np.array(new) + g.integers(0, 60, len(new))
        for parent in (random_parents(g, new, roots=True), random_parents(g, new, 1)):
            given = i32(torch, np.concatenate([parent, np.zeros(pad, np.int64)]))
            batch = kv4.Batch.of(i32(torch, np.zeros((len(new), 1))), i32(torch, lengths),
                                 i32(torch, np.concatenate([[0], np.cumsum(new)])), 16, rows=rows, tree=tree)
            own, other = plain_plan(parent, lengths, new, rows, words), torch.empty_like(batch.mask)
            mask, position = plain_window(parent, lengths, new, rows, words, window, sinks)
            batch.plan_tree(given)
            batch.plan_tree(given, window, sinks, mask=other)  # the batch's own stays as it is
            assert np.array_equal(other.cpu().numpy().view(np.uint32), mask)
            assert np.array_equal(batch.mask.cpu().numpy().view(np.uint32), own[0])
            assert np.array_equal(batch.position.cpu().numpy(), position)
            batch.plan_tree(given, window, sinks)
            assert torch.equal(batch.mask, other) and batch.tree_errors() == 0


@pytest.mark.parametrize("heads", [2, 8, 24])
@pytest.mark.parametrize("dtype", DTYPES)
def test_trees_deeper_than_their_window(torch, kv4, dtype, heads):
    lengths, new, window, sinks = [200, 44, 40], [40, 20, 40], 6, 3
    t = Trees(torch, kv4, lengths, new, 2, 64, 16, dtype, seed=17)
    w, q = t.w, t.w.queries(heads, 64)
    mask, position = plain_window(t.parent, lengths, new, w.rows, 2, window, sinks)
    assert not np.array_equal(mask, t.mask)
    out = w.cache.tree_attention(q, w.batch, mask=bits(torch, mask), position=i32(torch, position), window=window,
                                 sinks=sinks, max_new=40)
    check(w, q, out, sees_tree(mask, position, lengths, new, window, sinks))


def test_windows_of_plan_tree_are_checked(torch, kv4):
    batch = kv4.Batch.of(i32(torch, [[0]]), i32(torch, [4]), i32(torch, [0, 4]), 16, rows=4, tree=4)
    parent = i32(torch, [-1, 0, 1, 2])
    for more in (dict(window=-1), dict(sinks=-1), dict(window=2 ** 31), dict(mask=batch.mask[:3]), dict(mask=batch.mask.long()),
                 dict(mask=batch.mask.cpu())):
        with pytest.raises((ValueError, kv4.Cis2Error)):
            batch.plan_tree(parent, **more)


# ---------------------------------------------------------------- what a batch allocates

def test_a_batch_over_the_callers_tensors_allocates_nothing(torch, kv4):
    """Neither memory nor a kernel that would fill it: also inside a capture, where it would be a node."""
    given = i32(torch, [[0]]), i32(torch, [4]), i32(torch, [0, 4])
    slot = i32(torch, [0, 1, 2, 3])
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    kept = [kv4.Batch.of(*given, 16), kv4.Batch.of(*given, 16, slot=slot)]
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before
    assert [b.tree_errors() for b in kept] == [0, 0]
    kept[0].accept(slot, slot, slot)  # row 0 is not before itself
    assert kept[0].tree_errors() == kv4.TREE_PARENT and kept[0].tree_errors() == 0 and kept[1].tree_errors() == 0


def test_accepts_of_any_number_of_rows_share_their_outputs(torch, kv4):
    """What a captured call writes to stays the batch's, whatever calls come between."""
    batch = kv4.Batch.of(i32(torch, [[0]]), i32(torch, [4]), i32(torch, [0, 4]), 16)
    few, many = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (4, 900))
    chain = i32(torch, [-1, 0, 1, 2])
    batch.accept(few, chain, few)
    first, outputs = batch.path, (batch.accepted, batch.next_token, batch.kept)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batch.accept(few, chain, few)
    assert batch.path.data_ptr() == first.data_ptr()
    place = first.data_ptr()
    del first
    for rows in (900, 3, 0, 4, 700):
        batch.accept(many[:rows], many[:rows] - 1, many[:rows])
        assert all(a is b for a, b in zip(outputs, (batch.accepted, batch.next_token, batch.kept)))
        assert batch.path.shape == (rows,)
    others = [torch.full((n,), 77, dtype=torch.int32, device="cuda") for n in (1, 4, 900) for _ in range(20)]
    assert all(x.data_ptr() != place for x in others)
    graph.replay()
    assert all((x == 77).all() for x in others)
    assert batch.accepted.tolist() == [4] and batch.kept.tolist() == [4]
    batch.accept(few, chain, few)
    assert batch.path.tolist() == [0, 1, 2, 3]
