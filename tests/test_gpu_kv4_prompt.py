"""Many new rows per request over the 4-bit cache (more than 32 query columns
of a KV head: the tensor-memory kernel), against the 64-bit restatements and
with the tolerances of test_gpu_kv4.py."""
from __future__ import annotations

import importlib

import numpy as np
import pytest

from test_gpu_kv4 import TOL, World, stands_for

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    return importlib.import_module("torch")


@pytest.fixture(scope="module")
def kv4():
    return importlib.import_module("cis2-lab-archive_b200.kv4")


SHAPES = [  # lengths, new, heads, kv_heads, head_dim, page, window, sinks
    ([33], [33], 1, 1, 64, 16, 0, 0),
    ([128], [128], 1, 1, 128, 128, 0, 0),             # one full tile
    ([129, 127], [129, 127], 1, 1, 64, 16, 0, 0),      # one key and one row past a tile, one short of it
    ([300, 40, 9], [257, 0, 9], 9, 3, 64, 32, 0, 0),   # 3 heads a group: 126 of 128 rows used
    ([700, 64, 1], [90, 64, 1], 32, 8, 128, 64, 0, 0),
    ([257], [200], 32, 1, 64, 16, 0, 0),               # a group of 32
    ([5000], [40], 4, 2, 64, 32, 0, 0),                # cut over its keys
    ([4100, 300], [50, 60], 16, 2, 128, 64, 0, 0),     # one of two cut
    ([600, 450], [300, 33], 8, 2, 128, 64, 100, 4),
    ([900], [400], 4, 1, 64, 16, 37, 21),              # sinks that end inside a record
    ([400], [400], 4, 2, 128, 16, 1, 0),               # rows see themselves only
    ([300], [120], 6, 2, 64, 16, 50, 270),             # the sinks reach into the window
    ([6000], [64], 2, 1, 64, 256, 3500, 4),            # a window long enough to be cut
]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_prompts_match_64_bits(torch, kv4, dtype, shape):
    lengths, new, heads, kv_heads, d, page, window, sinks = SHAPES[shape]
    w = World(torch, kv4, lengths, new, kv_heads, d, page, dtype, seed=100 + shape, rows=sum(new) + shape % 2)
    q = w.queries(heads, d)
    out = w.cache.attention(q, w.batch, window=window, sinks=sinks, max_new=max(new))
    w.check(q, out, window, sinks)
    assert w.cache.errors() == 0
    again = w.cache.attention(q, w.batch, window=window, sinks=sinks, max_new=max(new))
    assert torch.equal(out, again)
    w.check(q, w.cache.attention(q, w.batch, window=window, sinks=sinks, max_new=max(new), whole=True), window, sinks)


@pytest.mark.parametrize("max_new", [1, 45])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_many_requests(torch, kv4, dtype, max_new):
    """More requests than a block has threads, and more query tiles than are put in order."""
    g = np.random.default_rng(max_new)
    n = 600
    new = np.ones(n, int) if max_new == 1 else g.integers(0, 4, n)
    new[7] = max_new
    lengths = new + g.integers(0, 30, n)
    w = World(torch, kv4, list(lengths), list(new), 1, 64, 16, dtype, seed=3)
    q = w.queries(1, 64)
    w.check(q, w.cache.attention(q, w.batch, max_new=max_new))
    assert w.cache.errors() == 0


@pytest.mark.parametrize("scale,gain,q_gain", [(0.0, 1.0, 1.0), (None, 1e-6, 1.0), (None, 1e6, 1.0), (-0.3, 1.0, 1.0),
                                               (None, 1.0, 0.0), (None, 1e30, 1e-30), (1e-20, 1e-30, 1e20)])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_prompts_over_the_range_of_numbers(torch, kv4, dtype, scale, gain, q_gain):
    if dtype == "float16" and (gain not in (1.0,) or q_gain not in (0.0, 1.0)):
        pytest.skip("outside half precision")
    w = World(torch, kv4, [300, 70], [50, 70], 1, 64, 16, dtype, gain=gain)
    q = w.queries(2, 64) * q_gain
    w.check(q, w.cache.attention(q, w.batch, scale=scale, max_new=70), scale=scale)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_prompts_follow_a_rising_maximum(torch, kv4, dtype):
    """Scores that grow along the keys, so that the running maximum moves in every tile, beside values
    of very different sizes."""
    d, n, m = 64, 700, 60
    w = World(torch, kv4, [n], [m], 1, d, 16, dtype)
    g = np.random.default_rng(1)
    x = (np.linspace(-1, 1, n)[:, None] * np.ones(d) + 0.01 * g.standard_normal((n, d))).astype(np.float32)
    y = g.standard_normal((n, d)).astype(np.float32)
    y[::97] *= 1e-3
    slots = (w.table[0].cpu().numpy()[np.arange(n) // 16] * 16 + np.arange(n) % 16).astype(np.int32)
    w.cache.append(torch.from_numpy(x[:, None]).cuda(), torch.from_numpy(y[:, None]).cuda(), torch.from_numpy(slots).cuda())
    w.k, w.v = [stands_for(x[:, None])], [stands_for(y[:, None])]
    for factor in (4.0, -4.0):
        q = torch.full((m, 1, d), factor, device="cuda").to(w.dtype)
        w.check(q, w.cache.attention(q, w.batch, scale=0.25, max_new=m), scale=0.25)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_masked_nan_leaves_no_trace_in_prompts(torch, kv4, dtype):
    """A NaN key and an infinite value reach exactly the rows that see their token."""
    d, page = 64, 16
    w = World(torch, kv4, [200], [90], 1, d, page, dtype)
    q = w.queries(2, d)
    clean = w.cache.attention(q, w.batch, window=40, max_new=90)
    w.check(q, clean, window=40)
    bad = torch.full((1, 1, d), float("nan"), device="cuda")
    p = 150  # rows stand at 110 .. 199; with a window of 40 those at 150 .. 189 see it
    slot = w.table[0, p // page] * page + p % page
    w.cache.append(bad, torch.full_like(bad, float("inf")), slot.view(1))
    got = w.cache.attention(q, w.batch, window=40, max_new=90)
    seen = torch.zeros(90, dtype=torch.bool, device="cuda")
    seen[40:80] = True
    assert torch.isnan(got[seen]).all() and torch.isfinite(got[~seen]).all()
    top = np.abs(w.v[0]).max()
    assert (got[~seen].double() - clean[~seen].double()).abs().max() <= TOL[dtype] * top
    # a page that is not there: its keys are not seen
    table = w.table.clone()
    table[0, 2] = -1
    b = kv4.Batch.of(table, w.batch.length, w.batch.row_start, page)
    out = w.cache.attention(q, b, window=40, sinks=64, max_new=90)
    assert torch.isfinite(out[~seen]).all() and w.cache.errors() == kv4.BAD_PAGE


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_prompts_with_any_strides_and_alone(torch, kv4, dtype):
    w = World(torch, kv4, [150, 260], [60, 100], 2, 64, 16, dtype)
    q = w.queries(6, 64)
    want = w.cache.attention(q, w.batch, max_new=100, whole=True)
    w.check(q, want)
    wide = torch.full((160, 6 * 64 + 129), 9.0, dtype=w.dtype, device="cuda")
    wide[:, 1:385] = q.view(160, -1)  # rows on no 16-byte boundary
    dest = torch.full((6, 162, 67), 5.0, dtype=w.dtype, device="cuda")
    out = dest[:, 1:161, 2:66].transpose(0, 1)
    w.cache.attention(wide[:, 1:385].unflatten(1, (6, 64)), w.batch, max_new=100, whole=True, out=out)
    assert torch.equal(out, want)
    dest[:, 1:161, 2:66] = 5.0
    assert torch.equal(dest, torch.full_like(dest, 5.0))
    one = kv4.Batch.of(w.table[1:].contiguous(), w.batch.length[1:].clone(),
                       torch.tensor([0, 100], dtype=torch.int32, device="cuda"), 16)
    assert torch.equal(w.cache.attention(q[60:], one, max_new=100, whole=True), want[60:])


def test_prompts_in_a_graph_and_on_streams(torch, kv4):
    w = World(torch, kv4, [3000, 500], [40, 90], 2, 64, 16, "bfloat16")
    q = w.queries(4, 64)
    want = w.cache.attention(q, w.batch, max_new=90)
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(w.cache.attention(q, w.batch, max_new=90))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs) and w.cache.errors() == 0
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.cache.attention(q, w.batch, max_new=90, out=out)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
