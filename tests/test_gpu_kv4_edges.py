"""The 4-bit cache at its edges: jumps of the running maximum, what stands in
places that no row sees, the ends of the number range, arguments that do not
belong together, streams and graphs.

Tolerances are those of test_gpu_kv4.py (errors relative to the largest
|value| that the rows see); where a test needs another one its comment derives it."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from test_gpu_kv4 import TOL, World, plain_attention, stands_for

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "float16", "bfloat16"]


@pytest.fixture(scope="module")
def torch():
    return importlib.import_module("torch")


@pytest.fixture(scope="module")
def kv4():
    return importlib.import_module("cis2-lab-archive_b200.kv4")


def write(torch, w, x, y, request=0, first=0):
    """Keys x and values y [n, kv_heads, head_dim] into the request's tokens first .. of a World."""
    at = np.arange(first, first + len(x))
    slots = (w.table[request].cpu().numpy()[at // w.page] * w.page + at % w.page).astype(np.int32)
    w.cache.append(torch.from_numpy(x.astype(np.float32)).cuda(), torch.from_numpy(y.astype(np.float32)).cuda(),
                   torch.from_numpy(slots).cuda())
    if first + len(x) <= len(w.k[request]):
        w.k[request][at], w.v[request][at] = stands_for(x), stands_for(y)


def along(t, d, kv_heads=1):
    """Keys whose product with a query of ones is t (log2 units where the scale is ln 2)."""
    return np.broadcast_to((np.asarray(t, np.float64) / d)[:, None, None], (len(t), kv_heads, d)).astype(np.float32)


LN2 = float(np.log(2.0))


# ---------------------------------------------------------------- the running maximum

@pytest.mark.parametrize("rise", [5.0, 12.0, 18.0])
@pytest.mark.parametrize("dtype", DTYPES)
def test_the_maximum_rises_inside_a_tile(torch, kv4, dtype, rise):
    """The scores of every 32 keys stand `rise` above those before them (and start again with each 128),
    so the weights of a tile that are already written have to be scaled, several times over."""
    d, n, m = 64, 600, 70
    w = World(torch, kv4, [n], [m], 1, d, 16, dtype)
    g = np.random.default_rng(2)
    j = np.arange(n)
    x = along((j % 128 // 32) * rise + (j // 128) * rise * 2, d)
    write(torch, w, x, g.standard_normal((n, 1, d)))
    q = torch.ones((m, 2, d), device="cuda").to(w.dtype)
    for _ in range(20):
        out = w.cache.attention(q, w.batch, scale=LN2, max_new=m)
    w.check(q, out, scale=LN2)
    assert w.cache.errors() == 0


# ---------------------------------------------------------------- hand-offs between warps

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("head_dim", [64, 128])
def test_many_tiles_hand_over(torch, kv4, dtype, head_dim):
    """Requests of one to many key tiles behind one another in each block, many times over: no wait runs out
    and every call has the same bits."""
    new = [40, 33, 300, 1, 129]
    w = World(torch, kv4, [9000, 300, 700, 129, 129], new, 2, head_dim, 64, dtype)
    q = w.queries(4, head_dim)
    want = w.cache.attention(q, w.batch, max_new=300)
    whole = w.cache.attention(q, w.batch, max_new=300, whole=True)
    for _ in range(100):
        assert torch.equal(w.cache.attention(q, w.batch, max_new=300), want)
        assert torch.equal(w.cache.attention(q, w.batch, max_new=300, whole=True), whole)
    assert w.cache.errors() == 0
    w.check(q, want), w.check(q, whole)


# ---------------------------------------------------------------- lengths and row starts

@pytest.mark.parametrize("heads", [2, 16])  # one kernel or the other for the 20 rows below
def test_a_request_that_reaches_past_the_rows(torch, kv4, heads):
    """A step with more new tokens than rows (PLAN_ROWS): the rows that there are stand at their own
    positions, p = length - (row_start[r + 1] - row_start[r]) + i."""
    lengths, new = [30, 100, 9], [4, 80, 9]
    w = World(torch, kv4, lengths, new, 1, 64, 16, "float32", rows=20)
    q = w.queries(heads, 64)
    for max_new in (1, 16):
        out = w.cache.attention(q, w.batch, max_new=max_new)
        # request 1's first 16 rows are the last of a request of 36 tokens
        cut = plain_attention(q.double().cpu().numpy(), [w.k[0], w.k[1][:36]], [w.v[0], w.v[1][:36]], [30, 36], [4, 16], 0.125, 0, 0)
        assert np.abs(out.double().cpu().numpy() - cut).max() <= TOL["float32"] * np.abs(w.v[1]).max()
    assert w.cache.errors() == 0


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("max_new,new", [(1, [1, 1]), (3, [3, 2]), (600, [600, 500])])
@pytest.mark.parametrize("length", [2 ** 31 - 1, 2 ** 31 - 16, 2 ** 31 - 700, 10 ** 6])
def test_a_length_past_the_table(torch, kv4, dtype, max_new, new, length):
    """Every key of the table is seen by every row, what is past it is reported, and with a window that
    lies past the table nothing is seen.  The sums over so many tiles stay in range."""
    w = World(torch, kv4, [64, 48], [1, 1], 2, 64, 16, dtype)
    table = torch.cat([w.table[:, :3], w.table[:, :3]]).contiguous()[:2]  # three full pages each
    n = sum(new)
    start = torch.tensor([0, new[0], n], dtype=torch.int32, device="cuda")
    b = kv4.Batch.of(table, torch.tensor([length, 48 + new[1]], dtype=torch.int32, device="cuda"), start, 16)
    q = torch.randn(n, 4, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(w.dtype)
    k, v = [w.k[0][:48], w.k[1]], [w.v[0][:48], w.v[1]]
    out = w.cache.attention(q, b, max_new=max_new)
    assert w.cache.errors() == kv4.BAD_PAGE
    # all 48 keys before every row: the same as one row of a request of 48 tokens, row by row
    rows = [0, 1, new[0] - 1, new[0], n - 1]
    for i in rows:
        r = int(i >= new[0])
        want = plain_attention(q[i:i + 1].double().cpu().numpy(), [k[r]], [v[r]], [48], [1], 0.125, 0, 0)
        assert np.abs(out[i].double().cpu().numpy() - want).max() <= TOL[dtype] * np.abs(v[r]).max(), i
    out = w.cache.attention(q, b, max_new=max_new, window=40, sinks=0)
    assert not out[:new[0]].any() and w.cache.errors() == kv4.BAD_PAGE
    assert torch.equal(out, w.cache.attention(q, b, max_new=max_new, window=40, sinks=0))
    w.cache.errors()
    # the counters of the workspace are as they were
    w2 = World(torch, kv4, [3000, 900], [40, 1], 2, 64, 16, dtype)
    w2.cache._work = w.cache._work
    q2 = w2.queries(4, 64)
    for m in (1, 40):
        w2.check(q2, w2.cache.attention(q2, w2.batch, max_new=m))


@pytest.mark.parametrize("max_new", [1, 64])
def test_requests_that_overlap_in_their_rows(torch, kv4, max_new):
    """More query tiles than the host counts with: nothing is written outside out, and the workspace's
    counters are as they were."""
    n, rows = 300, 257
    w = World(torch, kv4, [3000, 900], [40, 1], 2, 64, 16, "float32")
    q = torch.randn(rows, 4, 64, device="cuda")
    guard = torch.full((rows + 2, 4, 64), 3.0, device="cuda")
    start = torch.tensor([0, 2 ** 31 - 1] * (n // 2) + [2 ** 31 - 1], dtype=torch.int32, device="cuda")
    b = kv4.Batch.of(w.table[:1].expand(n, -1).contiguous(), torch.full((n,), 2 ** 31 - 1, dtype=torch.int32, device="cuda"), start, 16)
    w.cache.attention(q, b, max_new=max_new, out=guard[1:-1])
    assert (guard[0] == 3.0).all() and (guard[-1] == 3.0).all()
    w.cache.errors()
    q = w.queries(4, 64)
    for m in (1, 40):
        w.check(q, w.cache.attention(q, w.batch, max_new=m))
    with pytest.raises(kv4.Cis2Error):  # more query tiles than can be counted
        a = kv4._Attn(0, 2, 2 ** 30, 2 ** 30, 4, 1, 0, 0, 0.125, 0, *([256] * 2), 256, 64, 256, 64, *([256] * 4), 2 ** 60)
        kv4._check(kv4._lib().cis2b_kv4_attention(kv4.ctypes.byref(kv4._Cache(0, 4, 16, 2, 64, 0, 256, None)), kv4.ctypes.byref(a), None))


# ---------------------------------------------------------------- streams and graphs

@pytest.mark.parametrize("max_new", [1, 40])
def test_graphs_run_beside_their_capture_stream(torch, kv4, max_new):
    """Two graphs captured on a stream that has called before, replayed on two other streams beside calls
    on the first: each has a workspace of its own."""
    w = World(torch, kv4, [9000, 7000], [max_new, 1], 2, 64, 16, "float32")
    q = w.queries(4, 64)
    side, one, two = (torch.cuda.Stream() for _ in range(3))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = w.cache.attention(q, w.batch, max_new=max_new)
    torch.cuda.synchronize()
    w.check(q, want)
    graphs, outs = [], []
    for _ in range(2):
        out = torch.zeros_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            w.cache.attention(q, w.batch, max_new=max_new, out=out)
            w.cache.attention(q, w.batch, max_new=max_new, out=out)
        graphs.append(graph), outs.append(out)
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for stream, graph in zip((one, two), graphs):
            with torch.cuda.stream(stream):
                for _ in range(5):
                    graph.replay()
        with torch.cuda.stream(side):
            for _ in range(10):
                got.append(w.cache.attention(q, w.batch, max_new=max_new))
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in [*got, *outs])
    assert w.cache.errors() == 0


# ---------------------------------------------------------------- numbers of very different sizes

@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_scores_that_underflow(torch, kv4, dtype, new):
    """Queries and keys around 1e-25: every score is 0 in 32 bits, every row the mean of what it sees."""
    w = World(torch, kv4, [150, 40], [new, 40], 1, 64, 16, dtype)
    g = np.random.default_rng(3)
    for r, n in enumerate(w.lengths):
        write(torch, w, 1e-25 * g.standard_normal((n, 1, 64)), w.y[r], request=r)
    q = (w.queries(2, 64).float() * 1e-25).to(w.dtype)
    w.check(q, w.cache.attention(q, w.batch, max_new=40 if new > 1 else 1))


@pytest.mark.parametrize("size", [2.0 ** 14, 2.0 ** 22])
@pytest.mark.parametrize("dtype", DTYPES)
def test_an_outlier_does_not_coarsen_its_neighbours(torch, kv4, dtype, size):
    """One token in every 32 has values `size` times the others' and a score 80 powers of two below them:
    its share of a result is at most 20 * 2^(22 - 80), so errors are relative to the others' values."""
    d, n, m = 64, 600, 70
    w = World(torch, kv4, [n], [m], 1, d, 16, dtype)
    g = np.random.default_rng(4)
    y = g.standard_normal((n, 1, d))
    top = np.abs(stands_for(y.astype(np.float32))).max()
    big = np.arange(n) % 32 == 9
    y[big] *= size
    write(torch, w, along(np.where(big, -80.0, 0.0), d), y)
    q = torch.ones((m, 2, d), device="cuda").to(w.dtype)
    out = w.cache.attention(q, w.batch, scale=LN2, max_new=m)
    want = plain_attention(q.double().cpu().numpy(), w.k, w.v, [n], [m], LN2, 0, 0)
    assert np.abs(out.double().cpu().numpy() - want).max() <= TOL[dtype] * top


def junk(torch, w, request, first, last, kind, seed=7):
    """Other contents, all finite, for the tokens first .. last - 1 (slots of the request's pages)."""
    n, (kv, d) = last - first, (w.cache.kv_heads, w.cache.head_dim)
    if n <= 0:
        return
    if kind == "append":  # what an earlier request of large values leaves
        g = np.random.default_rng(seed)
        x = (g.standard_normal((2, n, kv, d)) * 10.0 ** g.integers(-30, 31, (2, n, 1, 1))).astype(np.float32)
        saved = w.k[request].copy(), w.v[request].copy()
        write(torch, w, x[0], x[1], request, first)
        w.k[request], w.v[request] = saved
        return
    g = torch.Generator("cuda").manual_seed(seed)  # any bytes, as in a pool that was never set
    pool = w.cache.pool.view(*w.cache.pool.shape[:3], 16 * (d + 8))
    for p in range(first, last):
        page, rec, row = int(w.table[request, p // w.page]), p % w.page // 16, p % 16
        at = pool[page, :, rec]
        for a, b in ((row * d // 2, d // 2), (8 * d + row * d // 2, d // 2), (16 * d + 8 * row, 8)):
            at[:, a:a + b] = torch.randint(0, 256, (kv, b), dtype=torch.uint8, device="cuda", generator=g)


@pytest.mark.parametrize("kind", ["append", "bytes"])
@pytest.mark.parametrize("new", [1, 5, 90])
@pytest.mark.parametrize("dtype", DTYPES)
def test_what_stands_in_unseen_places_changes_no_bit(torch, kv4, dtype, new, kind):
    """The rest of the last page, tokens before the window, and tokens after a row: whatever finite numbers
    (or bytes) stand there, every row has the bits that it has without them."""
    d, page, n = 64, 64, 333
    w = World(torch, kv4, [n, 70], [new, 1], 2, d, page, dtype)
    q = w.queries(4, d)
    clean = w.cache.attention(q, w.batch, max_new=new)
    w.check(q, clean)
    windowed = w.cache.attention(q, w.batch, max_new=new, window=40, sinks=20)
    w.check(q, windowed, window=40, sinks=20)
    for seed in range(4):
        junk(torch, w, 0, n, 384, kind, seed), junk(torch, w, 1, 70, 128, kind, seed)
        assert torch.equal(w.cache.attention(q, w.batch, max_new=new), clean)
        junk(torch, w, 0, 20, n - new - 39, kind, seed)  # the first row is at n - new
        assert torch.equal(w.cache.attention(q, w.batch, max_new=new, window=40, sinks=20), windowed)
        for r in range(2):  # as it was
            write(torch, w, w.x[r], w.y[r], r)
        if new > 1:
            cut = new // 2  # tokens from here on are changed: the rows before are not
            junk(torch, w, 0, n - new + cut, n, kind, seed)
            assert torch.equal(w.cache.attention(q, w.batch, max_new=new)[:cut], clean[:cut])
            assert torch.equal(w.cache.attention(q, w.batch, max_new=new, window=40, sinks=20)[:cut], windowed[:cut])
            write(torch, w, w.x[0], w.y[0])
    assert w.cache.errors() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_later_and_lighter_tokens_of_any_size(torch, kv4, dtype):
    """The last token of a prompt is 10^12 times the others: the rows before it are as they are without it.
    And a token of that size that is seen, with 2^-150 of the weight, costs the rows nothing either."""
    d, n, m = 64, 300, 120
    w = World(torch, kv4, [n], [m], 1, d, 16, dtype)
    y = w.y[0].copy()
    y[n - 1] *= 1e12
    write(torch, w, w.x[0], y)
    q = w.queries(2, d)
    out = w.cache.attention(q, w.batch, max_new=m)
    want = plain_attention(q.double().cpu().numpy(), w.k, w.v, [n], [m], d ** -0.5, 0, 0)
    top = np.abs(w.v[0][:n - 1]).max()
    assert np.abs(out[:-1].double().cpu().numpy() - want[:-1]).max() <= TOL[dtype] * top
    y = np.random.default_rng(8).standard_normal((n, 1, d))
    y[7::40] *= 1e12
    write(torch, w, along(np.where(np.arange(n) % 40 == 7, -150.0, 0.0), d), y)
    q = torch.ones((m, 2, d), device="cuda").to(w.dtype)
    out = w.cache.attention(q, w.batch, scale=LN2, max_new=m)
    want = plain_attention(q.double().cpu().numpy(), w.k, w.v, [n], [m], LN2, 0, 0)
    assert np.abs(out.double().cpu().numpy() - want).max() <= TOL[dtype] * 5


@pytest.mark.parametrize("jump", [17.0, 19.2, 20.3, 21.0, 25.0, 33.0])
def test_the_maximum_jumps_inside_a_tile(torch, kv4, jump):
    """96 keys just below the bound of their weights, then one of the same tile `jump` powers of two above
    them, where the factor for what is written is below half precision's least: their share, 96 * 2^-jump
    of values of +-1 beside one of +-1/2, is not lost (it is up to 1.8 times the tolerance)."""
    d, n, m = 64, 326, 70
    w = World(torch, kv4, [n], [m], 1, d, 16, "float32")
    t = np.full(n, -100.0)
    t[:128] = 0.0
    t[128:224] = 6.5
    t[224] = 6.5 + jump
    y = np.broadcast_to(np.where(np.arange(d) % 3 > 0, 1.0, -1.0), (n, 1, d)).astype(np.float32).copy()
    y[224] = np.where(np.arange(d) % 2 > 0, 0.5, -0.5)
    write(torch, w, along(t, d), y)
    q = torch.ones((m, 2, d), device="cuda")
    out = w.cache.attention(q, w.batch, scale=LN2, max_new=m)
    want = plain_attention(q.double().cpu().numpy(), w.k, w.v, [n], [m], LN2, 0, 0)
    assert np.abs(out.double().cpu().numpy() - want).max() <= TOL["float32"]


@pytest.mark.parametrize("new", [1, 5, 60])
@pytest.mark.parametrize("gain", [1e-4, 1e-5, 1e6])
@pytest.mark.parametrize("dtype", DTYPES)
def test_an_infinite_query_stays_in_its_row(torch, kv4, dtype, gain, new):
    """Rows with an infinity or a NaN are NaN; the other heads and tokens of their tile, 1 / gain in size,
    are as they are without them."""
    if dtype == "float16" and gain == 1e-5:
        pytest.skip("queries of 1e5 are outside half precision")
    d = 64
    w = World(torch, kv4, [200, 90], [new, 1], 1, d, 16, dtype)
    for r, x in enumerate(w.x):
        write(torch, w, x * gain, w.y[r], r)
    q = (w.queries(4, d).float() / gain).to(w.dtype)
    clean = w.cache.attention(q, w.batch, max_new=new)
    w.check(q, clean)
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[new // 2, 3] = bad[new, 0] = True
    q[0, 1, 5], q[new // 2, 3, 60], q[new, 0, 0] = float("inf"), float("nan"), -float("inf")
    got = w.cache.attention(q, w.batch, max_new=new)
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], clean[~bad])
    # rows that see nothing are zero whatever their query is
    got = w.cache.attention(q, kv4.Batch.of(torch.full_like(w.table, -1), w.batch.length, w.batch.row_start, 16), max_new=new)
    assert not got.any() and w.cache.errors() == kv4.BAD_PAGE


@pytest.mark.parametrize("new", [1, 5, 60])
@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e12, 1e30])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_query_of_another_size_changes_no_other_row(torch, kv4, dtype, size, new):
    d = 64
    w = World(torch, kv4, [200, 90], [new, 1], 1, d, 16, dtype)
    q = w.queries(4, d)
    clean = w.cache.attention(q, w.batch, max_new=new)
    w.check(q, clean)
    other = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    other[0, 1] = other[new // 2, 3] = True
    q[other] = (q[other].float() * size).to(w.dtype)
    got = w.cache.attention(q, w.batch, max_new=new)
    assert torch.equal(got[~other], clean[~other]) and torch.isfinite(got).all()
    # and the rows of that size alone, over keys that bring their scores back
    q[~other] = 0
    w.cache.append(*(torch.from_numpy(a).cuda() for a in ((w.x[0] / size).astype(np.float32), w.y[0])),
                   (w.table[0, torch.arange(200, device="cuda") // 16] * 16 + torch.arange(200, device="cuda") % 16).int())
    w.k[0] = stands_for((w.x[0] / size).astype(np.float32))
    w.check(q, w.cache.attention(q, w.batch, max_new=new))


@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_largest_queries(torch, kv4, dtype, new):
    """Queries up to 2^121 over keys that bring their scores back."""
    d, size = 64, 2.0 ** 119
    w = World(torch, kv4, [200], [new], 1, d, 16, dtype)
    write(torch, w, w.x[0] / np.float32(size), w.y[0])
    q = (w.queries(4, d).float() * size).to(w.dtype)
    assert torch.isfinite(q).all()
    w.check(q, w.cache.attention(q, w.batch, max_new=new))


@pytest.mark.parametrize("new", [1, 5, 60])
@pytest.mark.parametrize("size", [1e20, 2e22, 1e27, 1e33, 2e37])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_constant_groups_of_any_size(torch, kv4, dtype, size, new):
    """Values that are the same number in a whole group have a step of 0 and no weight but p itself; with
    others, or alone, they come out as they are."""
    d = 64
    w = World(torch, kv4, [200, 90], [new, 1], 1, d, 16, dtype)
    g = np.random.default_rng(6)
    for every in (1, 2):  # all of them, or every other one
        for r, n in enumerate(w.lengths):
            y = w.y[r] * np.float32(size if every == 1 else size * 2.0 ** -60)
            # bfloat16 numbers, so that a group's base is the value
            y[::every] = np.float32(size) * (g.integers(1, 128, (len(range(0, n, every)), 1, 1)) / np.float32(64))
            y = (y.view(np.uint32) & 0xffff0000).view(np.float32)
            write(torch, w, w.x[r], y, r)
        q = w.queries(4, d)
        w.check(q, w.cache.attention(q, w.batch, max_new=new))


@pytest.mark.parametrize("lengths,new", [([200], 1), ([6000], 1), ([200], 60), ([6000], 60)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_scores_far_below_zero(torch, kv4, dtype, lengths, new):
    """Every score below -10^31: the first key, whose score is the largest by far, has all the weight."""
    d, n = 64, lengths[0]
    w = World(torch, kv4, lengths, [new], 1, d, 16, dtype)
    write(torch, w, along(-1e31 * (1 + np.arange(n)), d), w.y[0])
    q = torch.ones((new, 4, d), device="cuda").to(w.dtype)
    for whole in (False, True):
        w.check(q, w.cache.attention(q, w.batch, scale=LN2, max_new=new, whole=whole), scale=LN2)


@pytest.mark.parametrize("max_new", [1, 4, 80])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 30, 41, 40])
def test_windows_of_any_length_with_rows_before_the_first_token(torch, kv4, max_new, window):
    """More new rows than tokens, so that the first stand before position 0, and a window up to the largest."""
    w = World(torch, kv4, [40], [80], 2, 64, 16, "float32")
    q = w.queries(4, 64)
    out = w.cache.attention(q, w.batch, window=window, max_new=max_new)
    assert not out[:40].any()
    want = plain_attention(q[40:].double().cpu().numpy(), w.k, w.v, [40], [40], 0.125, 0, 0)
    assert np.abs(out[40:].double().cpu().numpy() - want).max() <= TOL["float32"] * np.abs(w.v[0]).max()


# ---------------------------------------------------------------- planning

def plan_case(torch, kv4, requests):
    """A batch of many requests, its inputs, and what it has to give (by prefix sums)."""
    g = np.random.default_rng(requests)
    page, width = 16, 4
    cached, new = g.integers(0, 40, requests), g.integers(0, 3, requests)
    have, need = -(-cached // page), -(-(cached + new) // page)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
    batch = kv4.Batch(requests, int(new.sum()), width, page, table=i32(np.arange(requests * width).reshape(-1, width)))
    row = np.concatenate([[0], np.cumsum(new)])
    first = np.concatenate([[0], np.cumsum(need - have)])
    req = np.repeat(np.arange(requests), new)
    pos = cached[req] + np.arange(row[-1]) - row[req]
    col = pos // page
    fresh = col >= have[req]
    page_of = np.where(fresh, 10 ** 6 + first[req] + col - have[req], req * width + col)
    want = dict(row_start=row, request=req, position=pos, slot=page_of * page + pos % page)
    free = i32(10 ** 6 + np.arange(first[-1]))
    return batch, (i32(cached), i32(new), free), want, [int(row[-1]), int(first[-1]), 0, 0]


@pytest.mark.parametrize("requests", [6013, 6014, 6016, 12000, 16384])
def test_plan_of_many_requests(torch, kv4, requests):
    batch, args, want, counts = plan_case(torch, kv4, requests)
    batch.plan(*args)
    assert batch.counts.tolist() == counts
    for name, x in want.items():
        assert np.array_equal(getattr(batch, name).cpu().numpy(), x), name


def test_plans_of_two_threads(torch, kv4):
    """Batches of different sizes planned by two threads at once: neither takes the other's shared memory away."""
    import threading
    errors = []

    def plan(requests, stream):
        try:
            with torch.cuda.stream(stream):
                batch, args, want, _ = plan_case(torch, kv4, requests)
                for _ in range(4000):
                    batch.plan(*args)
                assert np.array_equal(batch.slot.cpu().numpy(), want["slot"])
        except Exception as e:  # noqa: BLE001 -- of another thread
            errors.append(e)

    threads = [threading.Thread(target=plan, args=(n, torch.cuda.Stream())) for n in (16384, 6100, 9000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors


# ---------------------------------------------------------------- what a user holds

def test_layers_share_a_workspace(torch, kv4):
    """The caches of a model's layers hold one workspace per stream between them, and none once they are gone."""
    import gc
    n = 12
    worlds = [World(torch, kv4, [2000 + 100 * i], [40], 2, 128, 64, "bfloat16", seed=i) for i in range(n)]
    qs = [w.queries(8, 128) for w in worlds]
    torch.cuda.synchronize()
    gc.collect()
    before = torch.cuda.memory_allocated()
    outs = [[torch.empty_like(q) for q in qs] for _ in range(2)]
    held = sum(o.numel() * o.element_size() for o in outs[0] + outs[1])
    for m, some in zip((1, 40), outs):  # each kernel, the layers one after another
        for w, q, out in zip(worlds, qs, some):
            w.cache.attention(q, w.batch, max_new=m, out=out)
    after = torch.cuda.memory_allocated()
    assert len({id(w.cache._work) for w in worlds}) == 1
    largest = max(work.numel() for work in worlds[0].cache._work.values())
    assert after - before <= held + 1.1 * largest + (1 << 20)
    for w, q, a, b in zip(worlds, qs, *outs):
        w.check(q, a), w.check(q, b)
        assert w.cache.errors() == 0
    del w, worlds
    gc.collect()
    assert not kv4._workspaces.get(torch.cuda.current_device())


# ---------------------------------------------------------------- arguments

@pytest.mark.parametrize("dtype", DTYPES)
def test_a_decode_batch_takes_the_one_row_kernel_by_itself(torch, kv4, dtype):
    """Without max_new, a batch with no more rows than requests is taken for decode: the bits of max_new=1."""
    lengths = list(range(20, 660, 40))
    w = World(torch, kv4, lengths, [1] * len(lengths), 2, 64, 16, dtype)
    q = w.queries(16, 64)
    out = w.cache.attention(q, w.batch)
    w.check(q, out)
    assert torch.equal(out, w.cache.attention(q, w.batch, max_new=1))
    assert not torch.equal(out, w.cache.attention(q, w.batch, max_new=len(lengths)))  # the other kernel's
    # and one request with all the rows of such a batch is still right
    w = World(torch, kv4, [500, 9, 9, 9], [4, 0, 0, 0], 2, 64, 16, dtype)
    q = w.queries(16, 64)
    w.check(q, w.cache.attention(q, w.batch))
    assert torch.equal(w.cache.attention(q, w.batch, max_new=0), w.cache.attention(q, w.batch, max_new=1))


def test_numbers_past_32_bits_are_refused(torch, kv4):
    w = World(torch, kv4, [100], [1], 1, 64, 16, "float32")
    q = w.queries(2, 64)
    want = w.cache.attention(q, w.batch)
    for kw in [dict(window=2 ** 32 + 5), dict(window=2 ** 31), dict(window=5, sinks=2 ** 32), dict(sinks=-2 ** 40)]:
        with pytest.raises(ValueError):
            w.cache.attention(q, w.batch, **kw)
    w.check(q, w.cache.attention(q, w.batch, max_new=2 ** 32 + 1))  # a bound may be anything
    for args in [(2 ** 32 + 4, 16, 1, 64), (4, 2 ** 32 + 16, 1, 64), (4, 16, 2 ** 32 + 1, 64), (4, 16, 1, 2 ** 32 + 64)]:
        with pytest.raises(ValueError):
            kv4.Cache(*args)
    with pytest.raises(ValueError):
        kv4.Batch(1, 4, 4, 2 ** 32 + 16)
    assert torch.equal(w.cache.attention(q, w.batch, window=0), want)


def test_errors_waits_for_every_stream(torch, kv4):
    """errors() of calls that still run on another stream, and of one that follows it there."""
    cache = kv4.Cache(2, 16, 1, 64)
    x = torch.randn(1, 1, 64, device="cuda")
    bad = torch.tensor([10 ** 6], dtype=torch.int32, device="cuda")
    batch = kv4.Batch(1, 4, 1, 16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    args = i32(0), i32(17), i32(0, 1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)  # about 10 ms
            cache.append(x, x, bad)
            batch.plan(*args)
        assert cache.errors() == kv4.BAD_SLOT
        with torch.cuda.stream(side):
            cache.append(x, x, bad)  # not wiped by the read before
        assert cache.errors() == kv4.BAD_SLOT and cache.errors() == 0
        with torch.cuda.stream(side):
            batch.counts.fill_(0)
            torch.cuda._sleep(20_000_000)
            batch.plan(*args)
        assert batch.errors() == kv4.PLAN_WIDTH | kv4.PLAN_ROWS


# ---------------------------------------------------------------- small values

@pytest.mark.parametrize("new", [1, 5, 60])
@pytest.mark.parametrize("gain", [1e-12, 1e-16, 1e-20, 1e-24, 1e-27, 3e-29])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_values_of_any_small_size(torch, kv4, dtype, gain, new):
    """Values down to the format's least steps (2^-96 here) keep their codes."""
    w = World(torch, kv4, [300, 90], [new, 1], 1, 64, 16, dtype, gain=gain)
    q = w.queries(4, 64)
    w.check(q, w.cache.attention(q, w.batch, max_new=new))


@pytest.mark.parametrize("new", [1, 5, 60])
@pytest.mark.parametrize("power", [-117, -108, -90, 90, 95])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_queries_and_keys_at_the_ends_of_the_range(torch, kv4, dtype, power, new):
    """Queries of 2^power over keys that bring their scores back (steps below 2^-100 are 0 in the format)."""
    d = 64
    w = World(torch, kv4, [200, 90], [new, 1], 1, d, 16, dtype)
    for r in range(2):
        write(torch, w, w.x[r] * np.float32(2.0 ** -power), w.y[r], r)
    q = (w.queries(4, d).float() * 2.0 ** power).to(w.dtype)
    w.check(q, w.cache.attention(q, w.batch, max_new=new))
