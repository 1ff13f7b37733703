"""Drafted trees and encoders over the 4-bit cache on the device, against plain
64-bit restatements.

Tolerances of attention, relative to the largest |value| that a row can see.
fp32 rows: those of test_gpu_kv4.py, 4e-5.  16-bit rows: with W the largest
sum of |q_d k_d| times the scale over rows and keys,
  a key's elements rounded to 11 bits (half a step is 2^-11 of each): 2^-11 W in
  an exponent, and weights rounded to 11 bits, both in the numerator and, the
  first, in the denominator: 2 (2^-11 W + 2^-11)
  values rounded to 11 bits, and sums in fp32: 2^-11 + 2^-15
  the result's own rounding: 2^-11 (fp16) or 2^-8 (bf16)
which also covers the kernel for up to 8 query columns (bf16: its sums' 15 bits
are 2^-15 W).
"""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from test_gpu_kv4 import World, stands_for

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "float16", "bfloat16"]
LN2 = float(np.log(2.0))


@pytest.fixture(scope="module")
def torch():
    return importlib.import_module("torch")


@pytest.fixture(scope="module")
def kv4():
    return importlib.import_module("cis2-lab-archive_b200.kv4")


# ---------------------------------------------------------------- plain restatements

def random_parents(g, new, reach=6, roots=False):
    """Each row hangs on one of the `reach` before it; with `roots` some hang on the cached tokens."""
    out = []
    for n in new:
        for i in range(n):
            p = i - 1 - int(g.integers(0, min(i, reach))) if i else -1
            out.append(-1 if roots and i and g.random() < 0.2 else p)
    return np.array(out, np.int32).reshape(-1)


def plain_plan(parent, lengths, new, rows, words):
    mask, position = np.zeros((rows, words), np.uint32), np.full(rows, -1, np.int64)
    at = 0
    for r, n in enumerate(new):
        for i in range(n):
            if i < 32 * words and at + i < rows:
                j, depth = i, -1
                while j >= 0:
                    mask[at + i, j // 32] |= np.uint32(1 << (j % 32))
                    depth += 1
                    j = parent[at + j] if -1 <= parent[at + j] < j else -1
                position[at + i] = lengths[r] - n + depth
        at += n
    return mask, position


def sees_tree(mask, position, lengths, new, window=0, sinks=0):
    """see(r, i): the tokens of request r that its row i sees."""
    start = np.concatenate([[0], np.cumsum(new)])

    def see(r, i):
        n, cached = lengths[r], lengths[r] - new[r]
        j = np.arange(n)
        old = j < cached
        if window:
            old &= (j > position[start[r] + i] - window) | (j < sinks)
        b = np.clip(j - cached, 0, 32 * mask.shape[1] - 1)
        named = (mask[start[r] + i, b // 32] >> (b % 32).astype(np.uint32)) & 1
        return np.where(j < cached, old, (named == 1) & (j - cached < 32 * mask.shape[1]))
    return see


def plain_rows(q, k, v, new, scale, see):
    out = np.zeros(q.shape)
    at = 0
    for r, n in enumerate(new):
        group = q.shape[1] // k[r].shape[1]
        for i in range(n):
            j = np.flatnonzero(see(r, i))
            if len(j):
                for h in range(q.shape[1]):
                    s = k[r][j, h // group] @ q[at + i, h] * scale
                    w = np.exp(s - s.max())
                    out[at + i, h] = (w / w.sum()) @ v[r][j, h // group]
        at += n
    return out


def tolerance(w, q, scale):
    """Of a World's queries (the module's comment), relative to the largest |value|."""
    name = str(w.dtype).split(".")[1]
    if name == "float32":
        return 4e-5
    x, at, most = np.abs(q.double().cpu().numpy()), 0, 0.0
    for r, n in enumerate(w.new):
        group = q.shape[1] // w.k[r].shape[1]
        for h in range(q.shape[1]):
            if n and len(w.k[r]):
                most = max(most, (x[at:at + n, h] @ np.abs(w.k[r][:, h // group]).T).max() * abs(scale))
        at += n
    return 2 * (2.0 ** -11 * most + 2.0 ** -11) + 2.0 ** -11 + 2.0 ** -15 + (2.0 ** -11 if name == "float16" else 2.0 ** -8)


def check(w, q, out, see, scale=None, top=None):
    used = sum(w.new)
    scale = q.shape[2] ** -0.5 if scale is None else scale
    want = plain_rows(q[:used].double().cpu().numpy(), w.k, w.v, w.new, scale, see)
    got = out.double().cpu().numpy()
    assert np.all(np.isfinite(got))
    top = max((np.abs(v).max() for v in w.v if v.size), default=1.0) if top is None else top
    off = np.abs(got[:used] - want).max(initial=0.0)
    assert off <= tolerance(w, q, scale) * top, (off / top, tolerance(w, q, scale))
    assert not np.any(got[used:])  # rows of no request


def i32(torch, x):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(x)).astype(np.int64)).int().cuda()


def bits(torch, mask):
    return torch.from_numpy(np.ascontiguousarray(mask).view(np.int32)).cuda()


class Trees:
    """A World with a random tree per request, planned on the host."""

    def __init__(self, torch, kv4, lengths, new, kv_heads, head_dim, page, dtype, seed=0, words=None, roots=True, **more):
        self.w = World(torch, kv4, lengths, new, kv_heads, head_dim, page, dtype, seed=seed, **more)
        self.parent = random_parents(np.random.default_rng(seed + 50), new, roots=roots)
        words = words or max(1, -(-max(new) // 32))
        self.mask, self.position = plain_plan(self.parent, lengths, new, self.w.rows, words)
        self.args = dict(mask=bits(torch, self.mask), position=i32(torch, self.position))

    def see(self, window=0, sinks=0):
        return sees_tree(self.mask, self.position, self.w.lengths, self.w.new, window, sinks)


# ---------------------------------------------------------------- tree attention

TREES = [  # lengths, new, heads, kv_heads, head_dim, page, window, sinks
    ([1], [1], 1, 1, 64, 16, 0, 0),
    ([16], [16], 9, 3, 64, 16, 0, 0),                  # nothing cached
    ([333], [16], 9, 3, 64, 16, 0, 0),
    ([130, 17, 65], [1, 2, 3], 4, 4, 128, 16, 0, 0),
    ([127, 128, 129, 300], [4, 0, 9, 12], 8, 2, 128, 32, 0, 0),   # tiles that end around the tree
    ([700, 64, 33], [33, 64, 32], 32, 8, 128, 64, 0, 0),          # words that end in a tree
    ([400], [100], 6, 2, 64, 16, 0, 0),                # several tiles of query columns, a tree over several tiles of keys
    ([500, 20], [7, 5], 32, 1, 64, 16, 0, 0),          # a group of 32
    ([50, 300], [3, 6], 24, 1, 128, 16, 0, 0),         # a group of 24: columns left over
    ([9000], [20], 4, 2, 64, 32, 0, 0),                # cut over its keys
    ([5000, 300], [16, 13], 16, 2, 128, 64, 0, 0),
    ([600, 450, 90], [30, 33, 40], 8, 2, 128, 64, 100, 4),
    ([900], [40], 4, 1, 64, 16, 37, 21),               # sinks that end inside a record
    ([300], [12], 6, 2, 64, 16, 50, 270),              # the sinks reach into the window
    ([200, 30], [10, 4], 4, 2, 128, 16, 1, 0),         # of the cached tokens the window has none
    ([6000], [5], 2, 1, 64, 256, 3500, 4),
    ([80], [80], 3, 3, 64, 16, 20, 2),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", range(len(TREES)))
def test_trees_match_64_bits(torch, kv4, dtype, shape):
    lengths, new, heads, kv_heads, d, page, window, sinks = TREES[shape]
    t = Trees(torch, kv4, lengths, new, kv_heads, d, page, dtype, seed=200 + shape, rows=sum(new) + shape % 3)
    w = t.w
    q = w.queries(heads, d)
    more = dict(window=window, sinks=sinks, max_new=max(new), **t.args)
    out = w.cache.tree_attention(q, w.batch, **more)
    check(w, q, out, t.see(window, sinks))
    assert torch.equal(out, w.cache.tree_attention(q, w.batch, **more))
    check(w, q, w.cache.tree_attention(q, w.batch, whole=True, **more), t.see(window, sinks))
    assert w.cache.errors() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [2, 6, 16, 32])
def test_any_mask_over_the_new_tokens(torch, kv4, dtype, heads):
    """Bits in any order: a row that sees nothing at all, one that sees all, itself left out, bits past the tokens
    (which name nothing), and fewer words than tokens."""
    n, d = 45, 64
    w = World(torch, kv4, [n, 200], [n, 40], 2, d, 16, dtype, seed=8)
    g = np.random.default_rng(4)
    mask = g.integers(0, 2 ** 32, (85, 2), dtype=np.uint32)
    mask[3], mask[4], mask[60] = 0, 2 ** 32 - 1, 0
    q = w.queries(heads, d)
    position = np.zeros(85, np.int64)
    for words in (2, 1, 3):
        m = np.concatenate([mask, g.integers(0, 2 ** 32, (85, 1), dtype=np.uint32)], 1)[:, :words]
        out = w.cache.tree_attention(q, w.batch, mask=bits(torch, m), max_new=n)
        check(w, q, out, sees_tree(m, position, w.lengths, w.new))
        assert not out[3].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_chain_is_causal_attention(torch, kv4, dtype):
    """Tokens that each continue the last: the same rows as attention()'s, within both kernels' tolerances."""
    lengths, new, d = [300, 41], [20, 3], 64
    w = World(torch, kv4, lengths, new, 2, d, 16, dtype, seed=9)
    batch = kv4.Batch.of(w.table, w.batch.length, w.batch.row_start, 16, rows=23, tree=20)
    batch.plan_tree(i32(torch, np.concatenate([np.arange(n) - 1 for n in new])))
    q = w.queries(8, d)
    for more in (dict(), dict(window=33, sinks=2)):
        a, b = w.cache.attention(q, w.batch, max_new=20, **more), w.cache.tree_attention(q, batch, max_new=20, **more)
        if more:  # a tree's own tokens are all inside a window longer than it is deep
            assert 20 < more["window"]
        top = max(np.abs(v).max() for v in w.v)
        assert (a.double() - b.double()).abs().max().item() <= 2 * tolerance(w, q, d ** -0.5) * top
    assert batch.tree_errors() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [2, 12])
def test_positions_outside_the_tree_count_as_the_nearest_inside(torch, kv4, dtype, heads):
    t = Trees(torch, kv4, [300], [10], 2, 64, 16, dtype, seed=12)
    w, q = t.w, t.w.queries(heads, 64)
    got = w.cache.tree_attention(q, w.batch, mask=t.args["mask"], window=30, max_new=10,
                                 position=i32(torch, [0, 299, 5000, -7, 290, 2 ** 31 - 1, -2 ** 31, 295, 289, 300]))
    want = w.cache.tree_attention(q, w.batch, mask=t.args["mask"], window=30, max_new=10,
                                  position=i32(torch, [290, 299, 299, 290, 290, 299, 290, 295, 290, 299]))
    assert torch.equal(got, want)


# ---------------------------------------------------------------- cross attention

CROSS = [  # lengths of the encoders, rows, heads, kv_heads, head_dim, page
    ([1], [1], 1, 1, 64, 16),
    ([40], [1], 9, 3, 64, 16),
    ([97, 1500, 0, 16], [1, 1, 1, 1], 12, 12, 64, 16),   # one encoder is empty
    ([0, 0], [3, 7], 4, 2, 128, 16),                     # all are
    ([128, 129, 127, 5], [5, 5, 0, 5], 9, 3, 64, 32),
    ([20, 333], [300, 9], 8, 2, 128, 64),                # more rows than states
    ([300], [70], 32, 1, 64, 16),
    ([9000], [1], 16, 8, 128, 64),                       # cut over its keys
    ([7000, 100], [6, 3], 16, 2, 64, 256),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", range(len(CROSS)))
def test_cross_attention_matches_64_bits(torch, kv4, dtype, shape):
    lengths, new, heads, kv_heads, d, page = CROSS[shape]
    w = World(torch, kv4, lengths, new, kv_heads, d, page, dtype, seed=300 + shape, rows=sum(new) + shape % 3)
    q = w.queries(heads, d)
    see = lambda r, i: np.ones(lengths[r], bool)  # noqa: E731
    out = w.cache.cross_attention(q, w.batch, max_new=max(new))
    check(w, q, out, see)
    assert torch.equal(out, w.cache.cross_attention(q, w.batch, max_new=max(new)))
    check(w, q, w.cache.cross_attention(q, w.batch, max_new=max(new), whole=True), see)
    check(w, q, w.cache.cross_attention(q, w.batch), see)
    assert w.cache.errors() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_beams_share_an_encoder(torch, kv4, dtype):
    """Requests on the same pages: each row as with pages of its own."""
    w = World(torch, kv4, [217], [4], 2, 64, 16, dtype, seed=2)
    q = w.queries(6, 64)
    alone = w.cache.cross_attention(q, w.batch, max_new=4, whole=True)
    beams = kv4.Batch.of(w.table.expand(4, -1).contiguous(), i32(torch, [217] * 4), i32(torch, range(5)), 16)
    got = w.cache.cross_attention(q, beams, max_new=4, whole=True)
    assert torch.equal(got, alone)


# ---------------------------------------------------------------- both, at their edges

def write(torch, w, x, y, request=0):
    at = np.arange(len(x))
    slots = w.table[request].cpu().numpy()[at // w.page] * w.page + at % w.page
    w.cache.append(torch.from_numpy(x.astype(np.float32)).cuda(), torch.from_numpy(y.astype(np.float32)).cuda(),
                   i32(torch, slots))
    w.k[request], w.v[request] = stands_for(x.astype(np.float32)), stands_for(y.astype(np.float32))


def everyone(w):
    return lambda r, i: np.ones(w.lengths[r], bool)


NEW = [1, 3, 5, 14, 30, 60]  # of 4 heads of one KV head: 4, 12, 20, 56, 120 and 240 query columns


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("rise", [5.0, 12.0, 18.0, 33.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_the_maximum_rises(torch, kv4, dtype, rise, new):
    """Scores that stand `rise` powers of two above those of the 32 keys before, over and over."""
    d, n = 64, 700
    w = World(torch, kv4, [n], [new], 1, d, 16, dtype)
    j = np.arange(n)
    t = (j % 128 // 32) * rise + (j // 128) * rise * 2
    write(torch, w, np.broadcast_to((t / d)[:, None, None], (n, 1, d)), w.y[0])
    q = torch.ones((new, 4, d), device="cuda").to(w.dtype)
    # The largest score is at most 20 rise <= 660 powers of two, one key of base t / d: rounded to bfloat16 in the
    # cache (which stands_for knows) and exact as an operand, so scores are sums of 64 equal products: exact to 2^-24.
    out = w.cache.cross_attention(q, w.batch, scale=LN2, max_new=new)
    want = plain_rows(q.double().cpu().numpy(), w.k, w.v, w.new, LN2, everyone(w))
    limit = {"float32": 4e-5 + 700 * 2.0 ** -22, "float16": 6e-3, "bfloat16": 1e-2}[dtype]
    assert np.abs(out.double().cpu().numpy() - want).max() <= limit * np.abs(w.v[0]).max()


@pytest.mark.parametrize("kind", ["append", "bytes"])
@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("dtype", DTYPES)
def test_what_stands_in_unseen_places_changes_no_bit(torch, kv4, dtype, new, kind):
    from test_gpu_kv4_edges import junk
    d, page, n = 64, 64, 333
    t = Trees(torch, kv4, [n, 70], [new, 1], 1, d, page, dtype, seed=21)
    w = t.w
    q = w.queries(4, d)
    tree = lambda **k: w.cache.tree_attention(q, w.batch, max_new=new, **t.args, **k)  # noqa: E731
    cross = lambda: w.cache.cross_attention(q, w.batch, max_new=new)  # noqa: E731
    clean, windowed, crossed = tree(), tree(window=40, sinks=20), cross()
    check(w, q, clean, t.see())
    check(w, q, windowed, t.see(40, 20))
    check(w, q, crossed, everyone(w))
    for seed in range(3):
        junk(torch, w, 0, n, 384, kind, seed), junk(torch, w, 1, 70, 128, kind, seed)
        assert torch.equal(tree(), clean) and torch.equal(cross(), crossed)
        junk(torch, w, 0, 20, n - new - 39, kind, seed)
        assert torch.equal(tree(window=40, sinks=20), windowed)
        for r in range(2):
            write(torch, w, w.x[r], w.y[r], r)
        if new > 1:  # another new token: rows that it is no ancestor of
            last = n - new + new // 2
            junk(torch, w, 0, last, last + 1, kind, seed)
            b = new // 2
            blind = torch.from_numpy((t.mask[:new, b // 32] >> np.uint32(b % 32)) & 1 == 0).cuda()
            assert torch.equal(tree()[:new][blind], clean[:new][blind])
            write(torch, w, w.x[0], w.y[0])
    assert w.cache.errors() == 0


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e-3, 1e5, 1e12, 1e30])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_query_of_another_size_changes_no_other_row(torch, kv4, dtype, size, new):
    d = 64
    w = World(torch, kv4, [200, 90], [new, 1], 1, d, 16, dtype)
    q = w.queries(4, d)
    clean = w.cache.cross_attention(q, w.batch, max_new=new)
    check(w, q, clean, everyone(w))
    other = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    other[0, 1] = other[new // 2, 3] = True
    q[other] = (q[other].float() * size).to(w.dtype)
    got = w.cache.cross_attention(q, w.batch, max_new=new)
    assert torch.equal(got[~other], clean[~other]) and torch.isfinite(got).all()
    q[~other] = 0
    write(torch, w, w.x[0] / size, w.y[0])  # keys that bring the scores back
    check(w, q, w.cache.cross_attention(q, w.batch, max_new=new), everyone(w))


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("power", [-117, -108, -90, -30, 30, 90, 95, 117])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_queries_and_keys_at_the_ends_of_the_range(torch, kv4, dtype, power, new):
    d = 64
    w = World(torch, kv4, [200, 90], [new, 1], 1, d, 16, dtype)
    for r in range(2):
        write(torch, w, w.x[r] * np.float32(2.0 ** -power), w.y[r], r)
    q = (w.queries(4, d).float() * 2.0 ** power).to(w.dtype)
    check(w, q, w.cache.cross_attention(q, w.batch, max_new=new), everyone(w))


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("gain", [1e-12, 1e-20, 1e-27, 3e-29, 1e15, 1e30])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_values_of_any_size(torch, kv4, dtype, gain, new):
    w = World(torch, kv4, [300, 90], [new, 1], 1, 64, 16, dtype, gain=gain)
    q = w.queries(4, 64)
    check(w, q, w.cache.cross_attention(q, w.batch, max_new=new), everyone(w))


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("size", [1e20, 2e22, 1e33, 2e37])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_constant_groups_of_any_size(torch, kv4, dtype, size, new):
    """Values that are one number in a whole group (a step of 0), alone or beside others 2^60 smaller."""
    w = World(torch, kv4, [200, 90], [new, 1], 1, 64, 16, dtype)
    g = np.random.default_rng(6)
    for every in (1, 2):
        for r, n in enumerate(w.lengths):
            y = w.y[r] * np.float32(size if every == 1 else size * 2.0 ** -60)
            y[::every] = np.float32(size) * (g.integers(1, 128, (len(range(0, n, every)), 1, 1)) / np.float32(64))
            write(torch, w, w.x[r], (y.view(np.uint32) & 0xffff0000).view(np.float32), r)
        q = w.queries(4, 64)
        check(w, q, w.cache.cross_attention(q, w.batch, max_new=new), everyone(w))


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("dtype", DTYPES)
def test_an_outlier_does_not_coarsen_its_neighbours(torch, kv4, dtype, new):
    """Tokens whose values are 2^22 times the others', 80 powers of two lighter: they do not show."""
    d, n = 64, 600
    w = World(torch, kv4, [n], [new], 1, d, 16, dtype)
    y = np.random.default_rng(4).standard_normal((n, 1, d)).astype(np.float32)
    top = np.abs(stands_for(y)).max()
    big = np.arange(n) % 32 == 9
    y[big] *= np.float32(2.0 ** 22)
    t = np.where(big, -80.0, 0.0)
    write(torch, w, np.broadcast_to((t / d)[:, None, None], (n, 1, d)), y)
    q = torch.ones((new, 4, d), device="cuda").to(w.dtype)
    check(w, q, w.cache.cross_attention(q, w.batch, scale=LN2, max_new=new), everyone(w), scale=LN2, top=top)


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("dtype", DTYPES)
def test_numbers_that_are_none_stay_in_their_rows(torch, kv4, dtype, new):
    """A query row with an infinity or a NaN is NaN; a group that reads NaN makes NaN of the rows that see it, and
    of no other; every other row keeps its bits."""
    d, n = 64, 150
    t = Trees(torch, kv4, [n, 40], [new, 1], 1, d, 16, dtype, seed=31)
    w, q = t.w, t.w.queries(4, d)
    call = lambda: w.cache.tree_attention(q, w.batch, max_new=new, **t.args)  # noqa: E731
    clean = call()
    for bad in (float("inf"), float("-inf"), float("nan")):
        keep = q[0, 2, 7].clone()
        q[0, 2, 7] = bad
        got = call()
        assert torch.isnan(got[0, 2]).all()
        got[0, 2] = clean[0, 2]
        assert torch.equal(got, clean)
        q[0, 2, 7] = keep
    for name in "xy":
        x, y = w.x[0].copy(), w.y[0].copy()
        (x if name == "x" else y)[n - 1, 0, 3] = np.nan  # the last drafted token
        write(torch, w, x, y)
        got, b = call(), new - 1
        sees = torch.from_numpy((t.mask[:new, b // 32] >> np.uint32(b % 32)) & 1 == 1).cuda()
        assert torch.isnan(got[:new][sees]).all() and sees.any()
        assert torch.equal(got[:new][~sees], clean[:new][~sees]) and torch.equal(got[new:], clean[new:])
        write(torch, w, w.x[0], w.y[0])


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_far_below_zero(torch, kv4, dtype, new):
    """Every score below -10^31: the first key has all the weight."""
    d, n = 64, 400
    w = World(torch, kv4, [n], [new], 1, d, 16, dtype)
    write(torch, w, np.broadcast_to((-1e31 * (1 + np.arange(n)) / d)[:, None, None], (n, 1, d)), w.y[0])
    q = torch.ones((new, 4, d), device="cuda").to(w.dtype)
    out = w.cache.cross_attention(q, w.batch, scale=LN2, max_new=new).double().cpu().numpy()
    assert np.abs(out - w.v[0][0, 0]).max() <= {"float32": 4e-5, "float16": 6e-3, "bfloat16": 1e-2}[dtype] * np.abs(w.v[0][0]).max()


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("dtype", DTYPES)
def test_scales(torch, kv4, dtype, new, scale):
    w = World(torch, kv4, [200, 90], [new, 1], 1, 64, 16, dtype)
    q = (w.queries(4, 64).float() * 0.2).to(w.dtype)
    check(w, q, w.cache.cross_attention(q, w.batch, max_new=new, scale=scale), everyone(w), scale=scale)


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("dtype", DTYPES)
def test_any_strides(torch, kv4, dtype, new):
    """Rows read and written in the midst of wider ones, on boundaries of 2 bytes, heads before rows."""
    d, heads = 64, 4
    t = Trees(torch, kv4, [150, 40], [new, 1], 1, d, 16, dtype, seed=41)
    w = t.w
    q = w.queries(heads, d)
    call = lambda x, o: w.cache.tree_attention(x, w.batch, max_new=new, out=o, **t.args)  # noqa: E731
    want = call(q, None)
    wide = torch.full((w.rows, heads * d + 5), 7.0, dtype=w.dtype, device="cuda")
    x = wide[:, 3:3 + heads * d].unflatten(1, (heads, d))
    x.copy_(q)
    o_wide = torch.full_like(wide, 9.0)
    o = o_wide[:, 1:1 + heads * d].unflatten(1, (heads, d))
    assert torch.equal(call(x, o), want)
    assert (o_wide[:, 0] == 9).all() and (o_wide[:, 1 + heads * d:] == 9).all()
    turned = torch.empty((heads, w.rows, d), dtype=w.dtype, device="cuda").transpose(0, 1)
    assert torch.equal(call(turned.copy_(q), torch.empty_like(turned)), want)


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("dtype", DTYPES)
def test_missing_pages_are_not_seen(torch, kv4, dtype, new):
    d, n, page = 64, 300, 16
    t = Trees(torch, kv4, [n], [new], 1, d, page, dtype, seed=51)
    w, q = t.w, t.w.queries(4, d)
    w.table[0, 2], w.table[0, 5] = -1, 2 ** 30
    gone = np.isin(np.arange(n) // page, (2, 5))
    out = w.cache.tree_attention(q, w.batch, max_new=new, **t.args)
    assert w.cache.errors() == kv4.BAD_PAGE
    see = t.see()
    check(w, q, out, lambda r, i: see(r, i) & ~gone)
    check(w, q, w.cache.cross_attention(q, w.batch, max_new=new), lambda r, i: ~gone)
    assert w.cache.errors() == kv4.BAD_PAGE
    w.table[:] = -1
    assert not w.cache.cross_attention(q, w.batch, max_new=new).any()


@pytest.mark.parametrize("max_new", [1, 8, 64])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_row_starts_and_lengths_that_do_not_belong_together(torch, kv4, dtype, max_new):
    """Lengths past the table and below 0, row starts out of order, overlapping or past the rows: rows that have a
    request see what its table holds, nothing else is touched, and the next call is as it should be."""
    d, n = 64, 200
    w = World(torch, kv4, [n, 50], [8, 8], 1, d, 16, dtype)
    q = w.queries(4, d)
    good = w.cache.cross_attention(q, w.batch, max_new=max_new)
    mask = torch.full((16, 2), -1, dtype=torch.int32, device="cuda")
    for lengths in ([n, 50], [2 ** 31 - 1, 50], [-5, 50], [n, 0], [10 ** 6, -2 ** 31]):
        for start in ([0, 8, 16], [0, 16, 16], [5, 3, 16], [-4, 8, 16], [0, 8, 4000], [12, 20, 2 ** 31 - 1], [0, 0, 0]):
            batch = kv4.Batch.of(w.table, i32(torch, lengths), i32(torch, start), 16)
            for more in (dict(), dict(window=20, sinks=3)):
                position = torch.arange(16, dtype=torch.int32, device="cuda")
                out = w.cache.tree_attention(q, batch, mask=mask, position=position, max_new=max_new, **more)
                assert out.shape == q.shape
            w.cache.cross_attention(q, batch, max_new=max_new)
    assert w.cache.errors() & ~kv4.BAD_PAGE == 0
    assert torch.equal(w.cache.cross_attention(q, w.batch, max_new=max_new), good)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_many_requests(torch, kv4, dtype):
    """More requests than a block looks at in one go."""
    g = np.random.default_rng(3)
    new = g.integers(0, 4, 600)
    new[7] = 12
    lengths = new + g.integers(0, 60, 600)
    t = Trees(torch, kv4, list(lengths), list(new), 1, 64, 16, dtype, seed=3)
    q = t.w.queries(2, 64)
    check(t.w, q, t.w.cache.tree_attention(q, t.w.batch, max_new=12, **t.args), t.see())
    check(t.w, q, t.w.cache.cross_attention(q, t.w.batch, max_new=12), everyone(t.w))
    assert t.w.cache.errors() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_request_alone_gives_the_bits_it_gives_in_a_batch(torch, kv4, dtype):
    t = Trees(torch, kv4, [3000, 700, 41], [6, 20, 9], 2, 128, 32, dtype, seed=61)
    w, q = t.w, t.w.queries(8, 128)
    both = w.cache.tree_attention(q, w.batch, max_new=20, whole=True, **t.args)
    one = kv4.Batch.of(w.table[1:2], w.batch.length[1:2].clone(), i32(torch, [0, 20]), 32)
    got = w.cache.tree_attention(q[6:26], one, mask=t.args["mask"][6:26].contiguous(), max_new=20, whole=True)
    assert torch.equal(got, both[6:26])


def test_offsets_past_32_bits(torch, kv4):
    """The last pages of a pool of more than 2^32 bytes."""
    pages, page, kv, d = 2 ** 15 + 9, 64, 16, 128
    cache = kv4.Cache(pages, page, kv, d)
    assert cache.pool.numel() > 2 ** 32
    g = np.random.default_rng(1)
    n, table = 130, [pages - 1, pages - 5, pages - 2]
    x, y = (g.standard_normal((n, kv, d)).astype(np.float32) for _ in range(2))
    slot = np.array([table[p // page] * page + p % page for p in range(n)])
    cache.append(torch.from_numpy(x).cuda(), torch.from_numpy(y).cuda(), i32(torch, slot))
    batch = kv4.Batch.of(i32(torch, [table]), i32(torch, [n]), i32(torch, [0, 6]), page, slot=i32(torch, slot[-6:]), tree=6)
    parent = [-1, 0, 0, 1, 2, 3]
    batch.plan_tree(i32(torch, parent))
    for dtype in (torch.float32, torch.bfloat16):
        q = torch.from_numpy(g.standard_normal((6, 64, d)).astype(np.float32)).cuda().to(dtype)
        out = cache.tree_attention(q, batch, max_new=6)
        mask, position = plain_plan(np.array(parent), [n], [6], 6, 1)
        want = plain_rows(q.double().cpu().numpy(), [stands_for(x)], [stands_for(y)], [6], d ** -0.5,
                          sees_tree(mask, position, [n], [6]))
        # W <= 40 here: |q| and |k| of 128 normal numbers, scaled
        limit = 4e-5 if dtype is torch.float32 else 2 * 41 * 2.0 ** -11 + 2.0 ** -7
        assert np.abs(out.double().cpu().numpy() - want).max() <= limit * np.abs(stands_for(y)).max()
    before = cache.gather(batch.slot)[0].clone()
    batch.accept(i32(torch, [0, 1, 2, 3, 4, 5]), i32(torch, parent), i32(torch, [2, 9, 4, 9, 9, 9]))  # 0, 2, 4
    batch.keep([cache])
    after = cache.gather(batch.slot)[0]
    assert torch.equal(after, before[[0, 2, 4, 3, 4, 5]])


# ---------------------------------------------------------------- plan_tree, accept, keep

@pytest.mark.parametrize("new,pad,roots", [([1], 0, False), ([0, 5, 0], 3, True), ([31, 32, 33, 64, 65], 0, True),
                                           ([1024, 3], 7, False), ([7] * 700, 100, True), ([257, 0, 100], 1, True)])
def test_plan_tree_matches_the_loops(torch, kv4, new, pad, roots):
    g = np.random.default_rng(len(new))
    rows, tree = sum(new) + pad, max(new)
    lengths = np.array(new) + g.integers(0, 1000, len(new))
    for parent in (random_parents(g, new, roots=roots), np.concatenate([np.arange(n) - 1 for n in new])):
        given = np.concatenate([parent, g.integers(-5, 5, pad)])
        batch = kv4.Batch.of(i32(torch, np.zeros((len(new), 1))), i32(torch, lengths),
                             i32(torch, np.concatenate([[0], np.cumsum(new)])), 16, rows=rows, tree=tree)
        batch.plan_tree(i32(torch, given))
        mask, position = plain_plan(parent, lengths, new, rows, (tree + 31) // 32)
        assert np.array_equal(batch.mask.cpu().numpy().view(np.uint32), mask)
        assert np.array_equal(batch.position.cpu().numpy(), position)
        assert batch.tree_errors() == 0


def test_plan_tree_reports_what_does_not_fit(torch, kv4):
    start = i32(torch, [0, 40, 44])
    batch = kv4.Batch.of(i32(torch, [[0], [0]]), i32(torch, [100, 4]), start, 16, rows=42, tree=32)
    parent = np.full(42, -1)
    parent[40:] = [-1, 0]
    batch.plan_tree(i32(torch, parent))  # 40 rows, masks of 32; and two of the second request's rows have no place
    assert batch.tree_errors() == kv4.TREE_ROWS and batch.tree_errors() == 0
    assert batch.position.tolist() == [60] * 32 + [-1] * 8 + [0, 1] and not batch.mask[32:40].any()
    assert batch.mask[40:].tolist() == [[1], [3]]
    parent[5], parent[6], parent[7], parent[41] = 5, 2 ** 31 - 1, -2, 4
    batch.plan_tree(i32(torch, parent))
    assert batch.tree_errors() == kv4.TREE_ROWS | kv4.TREE_PARENT
    assert batch.mask[5:8].flatten().tolist() == [32, 64, 128] and batch.mask[41].tolist() == [2]


def plain_accept(new, lengths, token, parent, target, rows):
    path, accepted, following = np.full(rows, -1), [], []
    at = 0
    for r, n in enumerate(new):
        cur, k = 0, 0
        while n:
            path[at + k] = cur
            k += 1
            nxt = [i for i in range(n) if parent[at + i] == cur and i > cur and token[at + i] == target[at + cur]]
            if not nxt:
                break
            cur = nxt[0]
        accepted.append(k)
        following.append(target[at + cur] if n else -1)
        at += n
    return path, accepted, following, np.array(lengths) - np.array(new) + accepted


@pytest.mark.parametrize("new", [[1], [6, 0, 3], [1024], [40] * 300, [0]])
def test_accept_matches_the_loops(torch, kv4, new):
    g = np.random.default_rng(sum(new))
    rows = sum(new) + 2
    lengths = np.array(new) + g.integers(0, 50, len(new))
    for vocabulary in (1, 2, 3, 1000):  # with 1 everything agrees; with few, siblings have the same token
        parent = random_parents(g, new, roots=True)
        token, target = (g.integers(0, vocabulary, rows) for _ in range(2))
        batch = kv4.Batch.of(i32(torch, np.zeros((len(new), 1))), i32(torch, lengths),
                             i32(torch, np.concatenate([[0], np.cumsum(new)])), 16)
        batch.accept(i32(torch, token), i32(torch, np.concatenate([parent, [0, 0]])), i32(torch, target))
        want = plain_accept(new, lengths, token, parent, target, rows)
        for name, x in zip(("path", "accepted", "next_token", "kept"), want):
            assert np.array_equal(getattr(batch, name).cpu().numpy(), x), name
        assert batch.tree_errors() == 0


def test_accept_at_its_edges(torch, kv4):
    """Parents that are none, a request whose rows do not all have a place, one with more rows than a tree has, and
    a request whose rows begin past the last."""
    batch = kv4.Batch.of(i32(torch, [[0], [0]]), i32(torch, [9, 9]), i32(torch, [0, 3, 6]), 16)
    batch.accept(i32(torch, [7, 1, 2, 7, 5]), i32(torch, [-1, 0, 2, -1, 0]), i32(torch, [1, 2, 2, 5, 8]))
    assert batch.tree_errors() == kv4.TREE_PARENT
    assert batch.accepted.tolist() == [2, 2] and batch.path.tolist() == [0, 1, -1, 0, 1]
    assert batch.next_token.tolist() == [2, 8] and batch.kept.tolist() == [8, 8]
    n = 1030
    batch = kv4.Batch.of(i32(torch, [[0], [0]]), i32(torch, [n, 20]), i32(torch, [0, n, n + 4]), 16)
    same = torch.zeros(n, dtype=torch.int32, device="cuda")
    batch.accept(same, torch.arange(-1, n - 1, dtype=torch.int32, device="cuda"), same)
    assert batch.tree_errors() == kv4.TREE_ROWS
    assert batch.accepted.tolist() == [1024, 0] and batch.path.tolist() == list(range(1024)) + [-1] * 6
    assert batch.next_token.tolist() == [0, -1] and batch.kept.tolist() == [1024, 16]
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    batch.accept(empty, empty, empty)
    assert batch.accepted.tolist() == [0, 0] and batch.kept.tolist() == [0, 16] and batch.path.shape == (0,)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("layers", [1, 3, 70])
def test_keep_moves_bit_for_bit(torch, kv4, head_dim, layers):
    """Paths whose places overlap (a token moves to where another one left), long ones, none; every other byte of
    every layer's pool stays as it is."""
    g = np.random.default_rng(layers)
    kv, page, pages = 3, 16, 40
    new = [9, 0, 1, 60, 33, 5]
    start = np.concatenate([[0], np.cumsum(new)])
    slot = g.permutation(pages * page)[:start[-1] + 2].astype(np.int32)
    slot[start[-1]:] = -1
    slot[start[5]:start[5] + 5] = [-1, slot[start[5] + 1], -1, slot[start[5] + 3], slot[start[5] + 4]]
    path = np.full(len(slot), -1)
    accepted = np.zeros(len(new), np.int64)
    for r, p in enumerate([[0, 2, 3, 4, 8], [], [0], list(range(0, 2)) + list(range(4, 60)), list(range(0, 33, 2)), [0, 2, 3, 4]]):
        path[start[r]:start[r] + len(p)], accepted[r] = p, len(p)
    caches = [kv4.Cache(pages + i % 2, page, kv, head_dim) for i in range(layers)]
    want = []
    for c in caches:
        c.pool.copy_(torch.randint(0, 256, c.pool.shape, dtype=torch.uint8, device="cuda"))
        old = c.pool.cpu().numpy()
        now = old.copy()
        for r in range(len(new)):
            for k in range(accepted[r]):
                a, b = slot[start[r] + path[start[r] + k]], slot[start[r] + k]
                if a < 0 or b < 0:
                    continue
                for lo, size in ((0, head_dim // 2), (8 * head_dim, head_dim // 2), (16 * head_dim, 8)):
                    i, j = lo + a % 16 * size, lo + b % 16 * size
                    now[b // page, :, b % page // 16, j:j + size] = old[a // page, :, a % page // 16, i:i + size]
        want.append(now)
    batch = kv4.Batch.of(i32(torch, np.zeros((len(new), 1))), i32(torch, np.array(new) + 3), i32(torch, start), page,
                         slot=i32(torch, slot))
    none = torch.zeros(len(slot), dtype=torch.int32, device="cuda")
    batch.accept(none, none, none)
    batch.path.copy_(i32(torch, path)), batch.accepted.copy_(i32(torch, accepted))
    batch.tree_errors()
    batch.keep(caches)
    for c, x in zip(caches, want):
        assert np.array_equal(c.pool.cpu().numpy(), x)
        assert c.errors() == 0


def test_keep_reports_and_skips_what_is_out_of_range(torch, kv4):
    cache = kv4.Cache(2, 16, 1, 64)
    cache.pool.copy_(torch.randint(0, 256, cache.pool.shape, dtype=torch.uint8, device="cuda"))
    old = cache.pool.clone()
    batch = kv4.Batch.of(i32(torch, [[0]]), i32(torch, [4]), i32(torch, [0, 4]), 16, slot=i32(torch, [0, 1, 2, 32]))
    none = torch.zeros(4, dtype=torch.int32, device="cuda")
    batch.accept(none, none, none)
    batch.accepted.fill_(2 ** 31 - 1)  # no more than the request has rows
    for path, bit in (([0, 0, 4, 3], kv4.BAD_PATH), ([0, 3, -1, 3], kv4.BAD_SLOT | kv4.BAD_PATH), ([0, 1, 2 ** 31 - 1, 3], kv4.BAD_PATH)):
        batch.path.copy_(i32(torch, path))
        batch.keep([cache])
        assert cache.errors() == bit
        assert torch.equal(cache.pool, old)


# ---------------------------------------------------------------- together

def test_speculative_steps(torch, kv4):
    """Steps of drafted trees through all operators, two layers of self attention and one to an encoder.  After
    each, the caches hold what a cache without any drafts would: the accepted tokens in order, bit for bit, and
    causal attention of the last accepted token gives the tree's row within the tolerance of both."""
    g = np.random.default_rng(7)
    kv, d, heads, page, requests, tree = 2, 64, 8, 16, 3, 11
    caches = [kv4.Cache(60, page, kv, d) for _ in range(2)]
    plain = [kv4.Cache(60, page, kv, d) for _ in range(2)]
    states = World(torch, kv4, [90, 0, 33], [tree] * 3, kv, d, page, "bfloat16", seed=1)
    batch = kv4.Batch(requests, 52, width=20, page_size=page, tree=tree)
    cached, free = np.array([37, 0, 15]), list(range(60))
    texts = [[(g.standard_normal((n, kv, d)), g.standard_normal((n, kv, d))) for n in cached] for _ in range(2)]
    batch.plan(i32(torch, [0] * 3), i32(torch, cached), i32(torch, free))
    free = free[int(batch.counts[1]):]
    for c, p, text in zip(caches, plain, texts):
        k, v = (torch.from_numpy(np.concatenate([t[i] for t in text]).astype(np.float32)).cuda().bfloat16() for i in range(2))
        c.append(k, v, batch.slot[:52])
        p.append(k, v, batch.slot[:52])
    for step in range(6):
        new = [tree, 4, tree] if step % 2 else [tree, tree, 1]
        rows, start = sum(new), np.concatenate([[0], np.cumsum(new)])
        batch.plan(i32(torch, cached), i32(torch, new), i32(torch, free))
        assert batch.errors() == 0
        used = int(batch.counts[1])
        parent = random_parents(g, new, 4)
        given = i32(torch, np.concatenate([parent, np.zeros(52 - rows, np.int64)]))
        batch.plan_tree(given)
        token, target = (i32(torch, g.integers(0, 2, 52)) for _ in range(2))
        batch.accept(token, given, target)
        accepted, path = batch.accepted.tolist(), batch.path.cpu().numpy()
        q = torch.from_numpy(g.standard_normal((rows, heads, d)).astype(np.float32)).cuda().bfloat16()
        encoder = kv4.Batch.of(states.table, states.batch.length, i32(torch, start), page)
        states.new, crossed = new, states.cache.cross_attention(q, encoder, max_new=tree)
        check(states, q, crossed, everyone(states))
        outs = []
        for c, p in zip(caches, plain):
            k, v = (torch.from_numpy(g.standard_normal((rows, kv, d)).astype(np.float32)).cuda().bfloat16() for _ in range(2))
            c.append(k, v, batch.slot[:rows])
            outs.append(c.tree_attention(q, batch, max_new=tree))
            for r in range(3):  # the text without drafts: the accepted rows one after another
                take = torch.from_numpy(start[r] + path[start[r]:start[r] + accepted[r]]).cuda()
                p.append(k[take], v[take], batch.slot[int(start[r]):int(start[r]) + accepted[r]].contiguous())
        batch.keep(caches)
        assert batch.kept.tolist() == list(cached + accepted)
        for c, p, out in zip(caches, plain, outs):
            for r in range(3):
                n = int(cached[r]) + accepted[r]
                pages = batch.table[r].cpu().numpy()
                slots = i32(torch, [pages[j // page] * page + j % page for j in range(n)])
                for a, b in zip(c.gather(slots), p.gather(slots)):
                    assert torch.equal(a, b)
                at = start[r] + path[start[r] + accepted[r] - 1]
                one = kv4.Batch.of(batch.table[r:r + 1], i32(torch, [n]), i32(torch, [0, 1]), page)
                alone = p.attention(q[at:at + 1], one, max_new=1)
                # W <= 12 (64 products of normal numbers, scaled), twice its tolerance
                assert (alone.double() - out[at].double()).abs().max().item() <= 2 * (2 * 13 * 2.0 ** -11 + 2.0 ** -7) * 4
        # pages that only drafts were on go back
        free = free[used:]
        cached = cached + accepted
        for r in range(3):
            last = -(-int(cached[r] - accepted[r] + new[r]) // page)
            free += batch.table[r, -(-int(cached[r]) // page):last].tolist()
    assert batch.tree_errors() == 0 and not any(c.errors() for c in caches + plain)


@pytest.mark.parametrize("new", [2, 8, 40])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_graphs_and_streams(torch, kv4, dtype, new):
    """The step captured once and replayed on other inputs, on another stream, beside calls on this one."""
    d = 64
    t = Trees(torch, kv4, [1500, 90], [new, 1], 2, d, 16, dtype, seed=71)
    w, q = t.w, t.w.queries(8, d)
    batch = kv4.Batch.of(w.table, w.batch.length, w.batch.row_start, 16, rows=new + 1, tree=new)
    parent = i32(torch, t.parent)
    token = torch.zeros(new + 1, dtype=torch.int32, device="cuda")
    want = w.cache.tree_attention(q, w.batch, max_new=new, **t.args).clone()
    crossed = w.cache.cross_attention(q, w.batch, max_new=new).clone()
    x, graphs, outs = q.clone(), [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            batch.plan_tree(parent)
            outs.append((w.cache.tree_attention(x, batch, max_new=new), w.cache.cross_attention(x, w.batch, max_new=new)))
            batch.accept(token, parent, token)
        graphs.append(graph)
    x.zero_()
    graphs[0].replay()
    assert not torch.equal(outs[0][1], crossed)
    x.copy_(q)
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for s, graph in zip(side, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        got = w.cache.tree_attention(q, w.batch, max_new=new, **t.args), w.cache.cross_attention(q, w.batch, max_new=new)
        torch.cuda.synchronize()
        for a, b in [got] + outs:
            assert torch.equal(a, want) and torch.equal(b, crossed)
    assert w.cache.errors() == 0


def test_one_workspace_serves_all_forms(torch, kv4):
    """Calls of every kind and size on one stream, one after another: each as it is alone."""
    w = World(torch, kv4, [2500, 300], [40, 33], 2, 128, 32, "bfloat16", seed=5)
    f = World(torch, kv4, [1800], [70], 1, 64, 16, "float32", seed=6)
    full = torch.full((73, 3), -1, dtype=torch.int32, device="cuda")
    calls = []
    for x, heads, d in ((w, 8, 128), (f, 3, 64), (w, 2, 128)):
        q = x.queries(heads, d)
        for new in (1, 3, 8, 70):
            calls += [lambda x=x, q=q, n=new: x.cache.attention(q, x.batch, max_new=n),
                      lambda x=x, q=q, n=new: x.cache.tree_attention(q, x.batch, mask=full, max_new=n),
                      lambda x=x, q=q, n=new: x.cache.cross_attention(q, x.batch, max_new=n)]
    first = [c() for c in calls]
    for seed in range(3):
        for i in np.random.default_rng(seed).permutation(len(calls)):
            assert torch.equal(calls[i](), first[i])
    assert w.cache.errors() == 0 and f.cache.errors() == 0


def test_refusals(torch, kv4):
    cache = kv4.Cache(8, 16, 2, 64)
    batch = kv4.Batch(2, 6, 4, 16, tree=3)
    ints = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.zeros(6, 4, 64, device="cuda")
    for call in [
        lambda: cache.tree_attention(q, kv4.Batch(2, 6, 4, 16)),                      # no masks
        lambda: cache.tree_attention(q, batch, mask=ints(5, 1)),                      # too few
        lambda: cache.tree_attention(q, batch, mask=ints(6, 2)[:, :1]),               # not contiguous
        lambda: cache.tree_attention(q, batch, mask=ints(6, 1).long()),
        lambda: cache.tree_attention(q, batch, mask=ints(6, 1).cpu()),
        lambda: cache.tree_attention(q, batch, window=4, position=ints(5)),
        lambda: cache.tree_attention(q, batch, window=4, position=ints(6).long()),
        lambda: cache.tree_attention(q, batch, window=-1),
        lambda: cache.tree_attention(q[:, :3], batch),                                # heads
        lambda: cache.tree_attention(q.double(), batch),
        lambda: cache.tree_attention(q.requires_grad_(), batch),
        lambda: cache.cross_attention(q, batch),                                      # q still asks for a gradient
        lambda: cache.cross_attention(q.detach()[..., :32], batch),
        lambda: cache.cross_attention(q.detach(), batch, scale=float("nan")),
        lambda: cache.cross_attention(q.detach(), batch, out=torch.empty(6, 4, 64, device="cuda", dtype=torch.half)),
        lambda: kv4.Batch(2, 6, 4, 16).plan_tree(ints(6)),
        lambda: batch.plan_tree(ints(5)),
        lambda: batch.plan_tree(ints(6).cpu()),
        lambda: kv4.Batch(2, 6, 4, 16, tree=1025),
        lambda: kv4.Batch(2, 6, 4, 16, tree=-1),
        lambda: kv4.Batch.of(ints(2, 1), ints(2), ints(3), 16, tree=4),               # how many rows
        lambda: kv4.Batch.of(ints(2, 1), ints(2), ints(3), 16, slot=ints(4), rows=5),
        lambda: kv4.Batch.of(ints(2, 1), ints(2), ints(3), 16, slot=ints(4).long()),
        lambda: batch.accept(ints(6), ints(5), ints(6)),
        lambda: batch.accept(ints(6), ints(6), ints(6).float()),
        lambda: batch.keep([cache]),                                                  # before accept
    ]:
        with pytest.raises((ValueError, kv4.Cis2Error)):
            call()
    batch.plan(ints(2), ints(2) + 3, torch.arange(8, dtype=torch.int32, device="cuda"))
    batch.accept(ints(6), ints(6), ints(6))
    for caches in ([], [cache, cache], [cache, kv4.Cache(8, 16, 1, 64)], [kv4.Cache(8, 32, 2, 64)], [cache, kv4.Cache(8, 16, 2, 128)]):
        with pytest.raises((ValueError, kv4.Cis2Error)):
            batch.keep(caches)
    batch.keep([cache])
    assert cache.errors() == 0
