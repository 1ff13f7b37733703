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
