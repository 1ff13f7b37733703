"""The 4-bit key/value cache on the device against plain 64-bit restatements.

Tolerances.  A row's result is a weighted mean of values, so errors are
bounded relative to the largest |value| that the row can see:
  fp32   22-bit weights and query limbs, fp32 scores: a relative error of
         2^-21 for the weights, and of |score| * 2^-22 <= 64 * 2^-22 in an
         exponent, for numerator and denominator: 2 (2^-21 + 2^-16) < 4e-5
  fp16   weights of 11 bits (2^-11), the sums' 15 bits in scores up to 64
         (64 * 2^-15 = 2^-9) and the result's own rounding (2^-11), the first
         two twice: < 6e-3
  bf16   the same with a result rounded to 8 bits (2^-8): < 1e-2
"""
from __future__ import annotations

import ctypes
import importlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TOL = {"float32": 4e-5, "float16": 6e-3, "bfloat16": 1e-2}


@pytest.fixture(scope="module")
def torch():
    return importlib.import_module("torch")


@pytest.fixture(scope="module")
def kv4():
    return importlib.import_module("cis2-lab-archive_b200.kv4")


# ---------------------------------------------------------------- plain restatements

def bf16_bound(x, rounded):
    x = np.asarray(x, np.float64)
    unit = np.ldexp(1.0, np.frexp(x)[1] - 8)
    return rounded(x / unit) * unit


def quantise(x):
    """[..., D] float32 -> (codes, step, base) by the definition, fp32 operations; NaN for a group
    that holds a NaN or an infinity."""
    x = np.asarray(x, np.float32)
    bad = ~np.isfinite(x).all(-1)
    x = np.where(bad[..., None], np.float32(0), x)
    base = bf16_bound(x.min(-1), np.floor).astype(np.float32)
    step = bf16_bound((x.max(-1) - base) / np.float32(15), np.ceil).astype(np.float32)
    step[step < 2.0 ** -100] = 0
    inv = np.divide(np.float32(1), step, out=np.zeros_like(step), where=step > 0)
    codes = np.clip(np.rint((x - base[..., None]) * inv[..., None]), 0, 15)
    step[bad] = base[bad] = np.nan
    return codes, step, base


def stands_for(x):
    codes, step, base = quantise(x)
    return base[..., None].astype(np.float64) + step[..., None].astype(np.float64) * codes


def plain_attention(q, k, v, lengths, new, scale, window, sinks):
    """q [rows, H, D], k and v: per request [len, KV, D], all float64."""
    out = np.zeros(q.shape)
    at = 0
    for r, n in enumerate(new):
        for i in range(n):
            p = lengths[r] - n + i
            j = np.arange(lengths[r])
            see = j <= p
            if window:
                see &= (j > p - window) | (j < sinks)
            j = j[see]
            group = q.shape[1] // k[r].shape[1]
            for h in range(q.shape[1]):
                if len(j):
                    s = k[r][j, h // group] @ q[at + i, h] * scale
                    w = np.exp(s - s.max())
                    out[at + i, h] = (w / w.sum()) @ v[r][j, h // group]
        at += n
    return out


def plain_plan(cached, new, free, table, page, rows):
    table = table.copy()
    slot, pos, req = (np.full(rows, -1, np.int64) for _ in range(3))
    row, taken = 0, 0
    width = table.shape[1]
    for r, (c, n) in enumerate(zip(cached, new)):
        have, need = -(-c // page), -(-(c + n) // page)
        for col in range(have, need):
            if col < width:
                table[r, col] = free[taken] if taken < len(free) else -1
            taken += 1
        for p in range(c, c + n):
            if row < rows:
                pg = table[r, p // page] if p // page < width else -1
                slot[row] = pg * page + p % page if pg >= 0 else -1
                pos[row], req[row] = p, r
            row += 1
    return table, slot, pos, req, row, taken


# ---------------------------------------------------------------- a cache with known contents

class World:
    """Requests with random keys and values in a cache whose other bytes are 0xff (NaN parameters)."""

    def __init__(self, torch, kv4, lengths, new, kv_heads, head_dim, page, dtype="float32", seed=0, spare=3, rows=None,
                 pages=None, gain=1.0):
        g = np.random.default_rng(seed)
        self.torch, self.lengths, self.new, self.page = torch, lengths, new, page
        need = [-(-n // page) for n in lengths]
        pages = pages or sum(need) + spare
        width = max(1, max(need)) + 1
        order = pages - 1 - g.permutation(sum(need) + spare)[:sum(need)]
        table = np.full((len(lengths), width), -1, np.int32)
        at = 0
        for r, n in enumerate(need):
            table[r, :n] = order[at:at + n]
            at += n
        pool = torch.empty(pages * kv_heads * page * (head_dim + 8), dtype=torch.uint8, device="cuda")
        self.cache = kv4.Cache(pages, page, kv_heads, head_dim, pool=pool)
        self.cache.pool[torch.from_numpy(table[table >= 0].astype(np.int64)).cuda()] = 255
        self.cache.pool[0] = 255
        self.x = [(g.standard_normal((n, kv_heads, head_dim)) + 0.3).astype(np.float32) for n in lengths]
        self.y = [(g.standard_normal((n, kv_heads, head_dim)) * gain).astype(np.float32) for n in lengths]
        slots = [table[r, p // page] * page + p % page for r, n in enumerate(lengths) for p in range(n)]
        if slots:
            self.cache.append(torch.from_numpy(np.concatenate(self.x)).cuda(),
                              torch.from_numpy(np.concatenate(self.y)).cuda(),
                              torch.tensor(slots, dtype=torch.int32, device="cuda"))
        self.k, self.v = [stands_for(x) for x in self.x], [stands_for(y) for y in self.y]
        self.table = torch.from_numpy(table).cuda()
        start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.rows = int(start[-1]) if rows is None else rows
        self.batch = kv4.Batch.of(self.table, torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                                  torch.from_numpy(start).cuda(), page)
        self.dtype, self.g = getattr(torch, dtype), g

    def queries(self, heads, head_dim):
        return self.torch.from_numpy(self.g.standard_normal((self.rows, heads, head_dim)).astype(np.float32)).cuda().to(self.dtype)

    def check(self, q, out, window=0, sinks=0, scale=None):
        used = sum(self.new)
        want = plain_attention(q[:used].double().cpu().numpy(), self.k, self.v, self.lengths, self.new,
                               q.shape[2] ** -0.5 if scale is None else scale, window, sinks)
        got = out.double().cpu().numpy()
        assert np.all(np.isfinite(got))
        top = max((np.abs(v).max() for v in self.v if v.size), default=1.0)
        assert np.abs(got[:used] - want).max(initial=0.0) <= TOL[str(self.dtype).split(".")[1]] * top
        assert not np.any(got[used:])  # rows of no request


# ---------------------------------------------------------------- append and gather

@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("rows,kv_heads,page,layout", [(1, 1, 16, "plain"), (37, 3, 32, "fused"), (130, 5, 256, "odd")])
def test_append_matches_the_definition(torch, kv4, head_dim, dtype, rows, kv_heads, page, layout):
    g = np.random.default_rng(rows)
    dt = getattr(torch, dtype)
    d = head_dim

    def tensor():
        x = torch.from_numpy((g.standard_normal((rows, kv_heads, d)) * np.exp(g.standard_normal((rows, kv_heads, 1)) * 4))
                             .astype(np.float32)).cuda().to(dt)
        if layout == "plain":
            return x
        wide = torch.zeros(rows, kv_heads * d + (3 * d if layout == "fused" else 3), dtype=dt, device="cuda")
        at = d if layout == "fused" else 1  # "odd": no row on a 16-byte boundary
        wide[:, at:at + kv_heads * d] = x.view(rows, -1)
        return wide[:, at:at + kv_heads * d].unflatten(1, (kv_heads, d))

    k, v = tensor(), tensor()
    pages = -(-rows // page) + 2
    cache = kv4.Cache(pages, page, kv_heads, d)
    slot = torch.from_numpy(g.permutation(pages * page)[:rows].astype(np.int32)).cuda()
    cache.append(k, v, slot)
    for got, x in zip(cache.gather(slot), (k, v)):
        want = stands_for(x.float().cpu().numpy())
        # base + step * code in one fp32 rounding
        got, fine = got.double().cpu().numpy(), ~np.isnan(want)
        assert np.array_equal(~np.isnan(got), fine)
        assert np.abs(got - want)[fine].max() <= 2.0 ** -24 * np.abs(want[fine]).max()
        _, step, _ = quantise(x.float().cpu().numpy())
        off = np.abs(want - x.double().cpu().numpy())
        assert np.all((off <= step[..., None] * 0.5001)[fine])
    got = cache.gather(slot, dtype=dt)
    for a, b in zip(got, cache.gather(slot)):
        assert torch.equal(a.nan_to_num(7.0), b.to(dt).nan_to_num(7.0))
    # the bytes, as documented: codes of element 2b low and 2b + 1 high, then the parameters
    codes, step, base = quantise(k.float().cpu().numpy())
    s = int(slot[0])
    rec = cache.pool[s // page, 0, s % page // 16].cpu().numpy()
    i = s % 16
    row = rec[i * d // 2:(i + 1) * d // 2]
    assert np.array_equal(row & 15, codes[0, 0, 0::2]) and np.array_equal(row >> 4, codes[0, 0, 1::2])
    par = rec[16 * d + 8 * i:16 * d + 8 * i + 4].view(np.uint16).astype(np.uint32) << 16
    assert np.array_equal(par.view(np.float32), [step[0, 0], base[0, 0]])
    assert cache.errors() == 0


def test_append_skips_and_reports_slots(torch, kv4):
    cache = kv4.Cache(2, 16, 1, 64)
    x = torch.randn(4, 1, 64, device="cuda")
    cache.append(x, x, torch.tensor([-1, 3, 32, 2 ** 31 - 1], dtype=torch.int32, device="cuda"))
    assert cache.errors() == kv4.BAD_SLOT and cache.errors() == 0
    assert torch.count_nonzero(cache.pool.view(2, -1).sum(1)) == 1
    k, v = cache.gather(torch.tensor([3, -1, 4], dtype=torch.int32, device="cuda"))
    assert torch.equal(k, v) and k[0].abs().max() > 0 and not k[1:].any()
    cache.gather(torch.tensor([32], dtype=torch.int32, device="cuda"))
    assert cache.errors() == kv4.BAD_SLOT
    cache.append(x[:0], x[:0], torch.empty(0, dtype=torch.int32, device="cuda"))
    assert cache.gather(torch.empty(0, dtype=torch.int32, device="cuda"))[0].shape == (0, 1, 64)
    assert cache.errors() == 0


def test_append_groups_at_the_edges_of_the_format(torch, kv4):
    """Constant, zero, tiny, huge and mixed groups; a group with a NaN or an infinity reads NaN and no other does."""
    d = 64
    g = np.random.default_rng(5)
    x = np.zeros((9, 1, d), np.float32)
    x[1] = 0.3
    x[2] = -7.77
    x[3] = 1e-38 * g.standard_normal(d)
    x[4] = 1e37 * g.uniform(-1, 1, d)
    x[5] = 100 + 1e-3 * g.standard_normal(d)
    x[6] = g.standard_normal(d)
    x[6, 0, 9] = np.nan
    x[7] = g.standard_normal(d)
    x[7, 0, 63] = -np.inf
    x[8] = g.standard_normal(d)
    x[8, 0, 0] = np.inf
    cache = kv4.Cache(1, 16, 1, d)
    slot = torch.arange(9, dtype=torch.int32, device="cuda")
    t = torch.from_numpy(x).cuda()
    cache.append(t, t, slot)
    for got in cache.gather(slot):
        got = got.double().cpu().numpy()
        assert np.all(np.isnan(got[6:]))
        want = stands_for(x[:6])
        assert np.all(np.abs(got[:6] - want) <= 2.0 ** -23 * np.abs(want))
        assert not got[0].any()


# ---------------------------------------------------------------- plan

@pytest.mark.parametrize("requests,page,top,most,pad", [(1, 16, 0, 1, 0), (1, 256, 1000, 700, 5), (3, 16, 40, 1, 0),
                                                         (64, 32, 300, 5, 9), (700, 16, 90, 3, 100), (5000, 64, 50, 2, 1)])
def test_plan_matches_the_loops(torch, kv4, requests, page, top, most, pad):
    g = np.random.default_rng(requests)
    cached, new = g.integers(0, top + 1, requests), g.integers(0, most + 1, requests)
    have = [-(-c // page) for c in cached]
    width = max(-(-(c + n) // page) for c, n in zip(cached, new)) + 1
    ids = g.permutation(sum(have) + requests * (most // page + 1) + 7).astype(np.int32)
    table = np.full((requests, width), -1, np.int32)
    at = 0
    for r, h in enumerate(have):
        table[r, :h] = ids[at:at + h]
        at += h
    free, rows = ids[at:], int(new.sum()) + pad
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731
    batch = kv4.Batch(requests, rows, width, page, table=i32(table))
    for _ in range(2):  # again on its own result: the same
        batch.plan(i32(cached), i32(new), i32(free))
        want = plain_plan(cached, new, free, table, page, rows)
        for name, w in zip(("table", "slot", "position", "request"), want):
            assert np.array_equal(getattr(batch, name).cpu().numpy(), w), name
        assert batch.counts.tolist() == [want[4], want[5], 0, 0] and batch.errors() == 0
        assert np.array_equal(batch.length.cpu().numpy(), cached + new)
        assert np.array_equal(batch.row_start.cpu().numpy(), np.concatenate([[0], np.cumsum(new)]))


def test_plan_reports_what_does_not_fit(torch, kv4):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    batch = kv4.Batch(3, 20, 2, 16)
    batch.plan(i32([0, 0, 0]), i32([5, 17, 1]), i32([7, 8]))  # 4 pages needed, 23 rows
    assert batch.errors() == kv4.PLAN_FREE | kv4.PLAN_ROWS
    want = plain_plan([0, 0, 0], [5, 17, 1], [7, 8], np.full((3, 2), -1, np.int32), 16, 20)
    assert np.array_equal(batch.table.cpu().numpy(), want[0]) and np.array_equal(batch.slot.cpu().numpy(), want[1])
    assert batch.counts.tolist()[:2] == [20, 4]
    batch = kv4.Batch(2, 8, 1, 16)
    batch.plan(i32([15, -3]), i32([2, 2]), i32([4, 5, 6]))
    assert batch.errors() == kv4.PLAN_WIDTH | kv4.PLAN_NEGATIVE
    assert batch.slot.tolist()[1] == -1 and batch.slot.tolist()[2:4] == [5 * 16, 5 * 16 + 1]
    batch = kv4.Batch(2, 4, 1, 16)
    batch.plan(i32([2 ** 31 - 1, 2 ** 31 - 1]), i32([2 ** 31 - 1, 2 ** 31 - 1]), i32([]))  # sums past 32 bits
    assert batch.errors() == kv4.PLAN_WIDTH | kv4.PLAN_ROWS | kv4.PLAN_FREE and batch.slot.tolist() == [-1] * 4


# ---------------------------------------------------------------- attention

SHAPES = [  # lengths, new, heads, kv_heads, head_dim, page, window, sinks
    ([1], [1], 1, 1, 64, 16, 0, 0),
    ([1], [1], 32, 1, 128, 16, 0, 0),
    ([15, 16, 17, 33], [1, 1, 1, 1], 9, 3, 64, 16, 0, 0),
    ([317], [1], 9, 3, 64, 16, 0, 0),
    ([5, 0, 260, 64], [1, 0, 1, 1], 16, 8, 128, 64, 0, 0),
    ([129, 1, 700], [1, 1, 1], 8, 1, 128, 256, 0, 0),
    ([2500], [1], 4, 1, 128, 32, 0, 0),           # split over its keys
    ([2061, 900], [3, 1], 6, 2, 64, 16, 0, 0),    # several rows, split
    ([40, 7, 20], [5, 7, 0], 9, 3, 64, 16, 0, 0),
    ([100, 3], [70, 3], 4, 2, 128, 32, 0, 0),
    ([90], [90], 12, 12, 64, 16, 0, 0),
    ([150, 40], [33, 40], 10, 2, 128, 16, 0, 0),
    ([130, 257], [130, 200], 16, 8, 128, 64, 0, 0),
    ([600], [300], 8, 2, 128, 64, 100, 4),
    ([500, 20], [1, 1], 4, 2, 64, 16, 1, 0),      # sees itself only
    ([500, 20, 90], [1, 1, 1], 4, 2, 128, 16, 33, 4),
    ([300], [1], 4, 2, 64, 32, 7, 290),           # the sinks reach into the window
    ([300, 100], [1, 2], 4, 2, 128, 32, 1000, 5),  # the window is longer than the request
    ([2000, 1500], [1, 1], 8, 2, 64, 16, 1100, 37),
    ([77], [60], 6, 2, 64, 16, 9, 3),
    ([64], [64], 3, 1, 128, 16, 16, 16),
]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_matches_64_bits(torch, kv4, dtype, shape):
    lengths, new, heads, kv_heads, d, page, window, sinks = SHAPES[shape]
    w = World(torch, kv4, lengths, new, kv_heads, d, page, dtype, seed=shape, rows=sum(new) + shape % 3)
    q = w.queries(heads, d)
    out = w.cache.attention(q, w.batch, window=window, sinks=sinks, max_new=max(new))
    w.check(q, out, window, sinks)
    assert w.cache.errors() == 0
    # the same bits again, and with a bound on max_new in place of its value
    assert torch.equal(out, w.cache.attention(q, w.batch, window=window, sinks=sinks, max_new=max(new)))
    w.check(q, w.cache.attention(q, w.batch, window=window, sinks=sinks), window, sinks)
    w.check(q, w.cache.attention(q, w.batch, window=window, sinks=sinks, whole=True), window, sinks)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_attention_reads_and_writes_any_strides(torch, kv4, dtype):
    w = World(torch, kv4, [40, 23], [3, 4], 2, 64, 16, dtype)
    q = w.queries(6, 64)
    want = w.cache.attention(q, w.batch, max_new=4)
    wide = torch.full((7, 6 * 64 + 129), 9.0, dtype=w.dtype, device="cuda")
    wide[:, 1:385] = q.view(7, -1)  # rows on no 16-byte boundary
    dest = torch.full((6, 9, 67), 5.0, dtype=w.dtype, device="cuda")
    out = dest[:, 1:8, 2:66].transpose(0, 1)  # heads first in memory
    assert w.cache.attention(wide[:, 1:385].unflatten(1, (6, 64)), w.batch, max_new=4, out=out) is out
    assert torch.equal(out, want)
    dest[:, 1:8, 2:66] = 5.0
    assert torch.equal(dest, torch.full_like(dest, 5.0))  # and nothing beside it


@pytest.mark.parametrize("scale,gain,q_gain", [(0.0, 1.0, 1.0), (None, 1e-6, 1.0), (None, 1e6, 1.0), (-0.3, 1.0, 1.0),
                                               (None, 1.0, 0.0), (None, 1e30, 1e-30), (1e-20, 1e-30, 1e20)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_attention_over_the_range_of_numbers(torch, kv4, dtype, scale, gain, q_gain):
    w = World(torch, kv4, [700, 33], [1, 9], 2, 64, 16, dtype, gain=gain)
    q = w.queries(4, 64) * q_gain
    w.check(q, w.cache.attention(q, w.batch, scale=scale, max_new=9), scale=scale)


def test_attention_follows_a_rising_maximum(torch, kv4):
    """Scores that grow along the keys, so that the running maximum has to move many times, one
    value far larger than the rest, and one that is masked."""
    d = 64
    w = World(torch, kv4, [1200], [1], 1, d, 16, "float32")
    g = np.random.default_rng(1)
    x = (np.linspace(-1, 1, 1200)[:, None] * np.ones(d) + 0.01 * g.standard_normal((1200, d))).astype(np.float32)
    y = g.standard_normal((1200, d)).astype(np.float32)
    y[5] *= 1e12  # outside the window below
    y[1100] *= 1e-9
    slots = (w.table[0].cpu().numpy()[np.arange(1200) // 16] * 16 + np.arange(1200) % 16).astype(np.int32)
    w.cache.append(torch.from_numpy(x[:, None]).cuda(), torch.from_numpy(y[:, None]).cuda(), torch.from_numpy(slots).cuda())
    w.k, w.v = [stands_for(x[:, None])], [stands_for(y[:, None])]
    for factor in (40.0, -40.0):
        q = torch.full((1, 1, d), factor / 8, device="cuda")
        out = w.cache.attention(q, w.batch, scale=1.0, window=1150, max_new=1)
        w.v[0][:50] = 0.0  # not seen
        w.check(q, out, window=1150, scale=1.0)


def test_keys_that_are_not_seen_leave_no_trace(torch, kv4):
    """NaN and infinities in masked places (pages of other requests, the rest of a page, keys after a row or
    before its window) reach no row; a NaN that is seen reaches exactly the rows that see it."""
    d, page = 64, 16
    w = World(torch, kv4, [60], [30], 1, d, page, "float32")
    q = w.queries(3, d)
    clean = w.cache.attention(q, w.batch, window=20, max_new=30)
    w.check(q, clean, window=20)
    bad = torch.full((1, 1, d), float("nan"), device="cuda")
    p = 45  # seen by positions 45 .. 59 without a window, 45 .. 64 with one of 20
    slot = w.table[0, p // page] * page + p % page
    w.cache.append(bad, torch.full_like(bad, float("inf")), slot.view(1))
    got = w.cache.attention(q, w.batch, window=20, max_new=30)
    assert torch.equal(got[:15], clean[:15])  # positions 30 .. 44
    assert torch.isnan(got[15:]).all()
    got = w.cache.attention(q, w.batch, window=5, max_new=30)
    assert torch.isnan(got[15:20]).all() and torch.isfinite(got[:15]).all() and torch.isfinite(got[20:]).all()


def test_missing_pages_are_not_seen(torch, kv4):
    w = World(torch, kv4, [50], [1], 1, 64, 16, "float32")
    q = w.queries(2, 64)
    for bad in (-1, 10 ** 6):
        table = w.table.clone()
        table[0, 1] = bad
        b = kv4.Batch.of(table, w.batch.length, w.batch.row_start, 16)
        out = w.cache.attention(q, b, max_new=1)
        keep = np.r_[0:16, 32:50]
        want = plain_attention(q.double().cpu().numpy(), [w.k[0][keep]], [w.v[0][keep]], [34], [1], 0.125, 0, 0)
        assert np.abs(out.double().cpu().numpy() - want).max() <= TOL["float32"] * np.abs(w.v[0]).max()
        assert w.cache.errors() == kv4.BAD_PAGE
    table = torch.full_like(w.table, -1)
    out = w.cache.attention(q, kv4.Batch.of(table, w.batch.length, w.batch.row_start, 16), max_new=1)
    assert not out.any()
    # more new rows than tokens: the first stand before position 0 and see nothing
    b = kv4.Batch.of(w.table, torch.tensor([2], dtype=torch.int32, device="cuda"),
                     torch.tensor([0, 4], dtype=torch.int32, device="cuda"), 16)
    out = w.cache.attention(w.torch.ones(4, 2, 64, device="cuda"), b, max_new=4)
    assert not out[:2].any() and out[2:].abs().min() > 0


def test_a_request_alone_gives_the_bits_it_gives_in_a_batch(torch, kv4):
    lengths, new = [3000, 17, 900, 64, 1999], [1, 1, 1, 1, 1]
    w = World(torch, kv4, lengths, new, 2, 128, 32, "bfloat16")
    q = w.queries(8, 128)
    both = w.cache.attention(q, w.batch, max_new=1, whole=True)
    w.check(q, both)
    for r in range(len(lengths)):
        one = kv4.Batch.of(w.table[r:r + 1].contiguous(), w.batch.length[r:r + 1].clone(),
                           torch.tensor([0, 1], dtype=torch.int32, device="cuda"), 32)
        assert torch.equal(w.cache.attention(q[r:r + 1], one, max_new=1, whole=True)[0], both[r])


def test_offsets_past_32_bits(torch, kv4):
    """A pool of 4.4 GB with the request's pages at its end."""
    w = World(torch, kv4, [600], [2], 8, 128, 256, "bfloat16", pages=16000)
    assert w.cache.pool.numel() > 2 ** 32 and int(w.table[0].max()) > 15000
    q = w.queries(16, 128)
    w.check(q, w.cache.attention(q, w.batch, max_new=2))
    k, _ = w.cache.gather((w.table[0, :1] * 256).int())
    assert np.abs(k[0].double().cpu().numpy() - w.k[0][0]).max() < 1e-5


def test_one_workspace_serves_calls_of_all_sizes(torch, kv4):
    """Batches of other sizes, and both kernels, one after another on one cache: nothing that one call
    leaves in the workspace is taken for a counter by the next."""
    lengths, new = [3000, 2500, 40, 900, 1700, 33, 2100], [1, 60, 40, 1, 3, 33, 1]
    w = World(torch, kv4, lengths, new, 2, 64, 16, "float32")
    start = np.concatenate([[0], np.cumsum(new)])
    q = w.queries(6, 64)

    def part(first, last, max_new):
        b = kv4.Batch.of(w.table[first:last].contiguous(), w.batch.length[first:last].clone(),
                         (w.batch.row_start[first:last + 1] - int(start[first])).contiguous(), 16)
        return w.cache.attention(q[start[first]:start[last]], b, max_new=max_new)

    calls = [(0, 1, 1), (3, 5, 3), (0, 7, 60), (0, 7, 1), (1, 3, 60), (6, 7, 1), (2, 7, 40), (0, 4, 2), (0, 1, 1)]
    first = [part(*c) for c in calls]
    again = [part(*c) for c in calls[::-1]][::-1]
    w.cache._work.clear()
    for c, a, b in zip(calls, first, again):
        fresh = part(*c)
        w.cache._work.clear()
        assert torch.equal(a, fresh) and torch.equal(b, fresh), c
    w.check(q, first[2])
    assert w.cache.errors() == 0


def test_streams_and_graphs(torch, kv4):
    """Calls on two streams of one cache do not share a workspace; a captured step replays."""
    lengths = [2500, 1800]
    w = World(torch, kv4, lengths, [1, 1], 2, 64, 16, "float32")
    q = w.queries(4, 64)
    want = w.cache.attention(q, w.batch, max_new=1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(w.cache.attention(q, w.batch, max_new=1))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    out = torch.zeros_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.cache.attention(q, w.batch, max_new=1, out=out)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_a_first_call_inside_a_graph(torch, kv4):
    """A call that makes its workspace while a graph is captured leaves nothing unzeroed to others, and a
    workspace that is outgrown stays with the graph that holds it."""
    w = World(torch, kv4, [2500, 1800], [1, 1], 2, 64, 16, "float32")
    q = w.queries(4, 64)
    out = torch.zeros_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        w.cache.attention(q, w.batch, max_new=1, out=out)
    with torch.cuda.stream(side):  # before any replay
        want = w.cache.attention(q, w.batch, max_new=1)
        w.check(q, want)
        second = torch.cuda.CUDAGraph()
    out2 = torch.zeros_like(q)
    with torch.cuda.graph(second, stream=side):
        w.cache.attention(q, w.batch, max_new=1, out=out2)
    with torch.cuda.stream(side):  # a larger workspace on the same stream
        w.cache.attention(q, w.batch, max_new=16)
    torch.cuda.synchronize()
    for _ in range(2):
        for g, o in ((graph, out), (second, out2)):
            o.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want)


def test_a_step_through_all_operators(torch, kv4):
    """plan, append and attention as a serving loop calls them, against the restatements: a prompt chunk,
    then decode steps, pages taken from a free list."""
    g = np.random.default_rng(9)
    page, kv, h, d, n = 16, 2, 6, 64, 3
    cache = kv4.Cache(40, page, kv, d)
    free = torch.randperm(40, device="cuda").to(torch.int32)
    batch = kv4.Batch(n, 64, 8, page)
    ks, vs = [np.zeros((0, kv, d)) for _ in range(n)], [np.zeros((0, kv, d)) for _ in range(n)]
    cached = np.zeros(n, np.int32)
    for new in ([20, 1, 17], [1, 30, 0], [1, 1, 1], [0, 1, 1], [3, 1, 2]):
        rows = 64
        batch.plan(torch.from_numpy(cached).cuda(), torch.tensor(new, dtype=torch.int32, device="cuda"), free)
        assert batch.errors() == 0
        x, y, q = (g.standard_normal((rows, m, d)).astype(np.float32) for m in (kv, kv, h))
        cache.append(torch.from_numpy(x).cuda(), torch.from_numpy(y).cuda(), batch.slot)
        out = cache.attention(torch.from_numpy(q).cuda(), batch, max_new=max(new))
        at = 0
        for r, m in enumerate(new):
            ks[r], vs[r] = np.concatenate([ks[r], stands_for(x[at:at + m])]), np.concatenate([vs[r], stands_for(y[at:at + m])])
            at += m
        cached = cached + np.array(new, np.int32)
        want = plain_attention(q[:at].astype(np.float64), ks, vs, list(cached), new, d ** -0.5, 0, 0)
        got = out.double().cpu().numpy()
        assert np.abs(got[:at] - want).max() <= TOL["float32"] * max(np.abs(v).max() for v in vs) and not got[at:].any()
        free = free[int(batch.counts[1].item()):].contiguous()
    assert cache.errors() == 0


def test_refusals(torch, kv4):
    cache = kv4.Cache(4, 16, 2, 64)
    t = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    for args in [(0, 16, 1, 64), (1, 24, 1, 64), (1, 16, 0, 64), (1, 16, 1, 80), (2 ** 27, 16, 1, 64)]:
        with pytest.raises(kv4.Cis2Error):
            kv4.Cache(*args)
    with pytest.raises(ValueError):
        kv4.Cache(4, 16, 2, 64, pool=t(10, dtype=torch.uint8))
    with pytest.raises(ValueError):
        kv4.Cache(4, 16, 2, 64, device="cpu")
    for k, v, s in [(t(3, 2, 64), t(2, 2, 64), i(3)), (t(3, 2, 64), t(3, 2, 64).half(), i(3)), (t(3, 2, 32), t(3, 2, 32), i(3)),
                    (t(3, 2, 64), t(3, 2, 64), i(2)), (t(3, 2, 64), t(3, 2, 64), i(3).long()),
                    (t(3, 2, 64).double(), t(3, 2, 64).double(), i(3)), (t(3, 64, 2).mT, t(3, 64, 2).mT, i(3)),
                    (t(3, 2, 64).cpu(), t(3, 2, 64).cpu(), i(3))]:
        with pytest.raises(ValueError):
            cache.append(k, v, s)
    with pytest.raises(ValueError):
        cache.gather(i(3), dtype=torch.float64)
    batch = kv4.Batch.of(i(1, 4), i(1), i(2), 16)
    q = t(1, 4, 64)
    for kw in [dict(window=-1), dict(sinks=-1), dict(scale=float("nan"))]:
        with pytest.raises(kv4.Cis2Error):
            cache.attention(q, batch, **kw)
    for bad in [t(1, 3, 64), t(1, 66, 64)]:
        with pytest.raises(kv4.Cis2Error):
            cache.attention(bad, batch)
    for bad in [t(1, 4, 32), t(4, 64), q.double(), q.clone().requires_grad_(), q.cpu(), t(1, 64, 4).mT]:
        with pytest.raises(ValueError):
            cache.attention(bad, batch)
    with pytest.raises(ValueError):
        cache.attention(q, batch, out=t(1, 4, 64).half())
    with pytest.raises(ValueError):
        cache.attention(q, kv4.Batch.of(i(1, 4), i(1), i(2), 32))
    with pytest.raises(ValueError):
        batch.plan(i(1), i(1), i(1))
    with pytest.raises(ValueError):
        kv4.Batch.of(i(1, 4), i(2), i(2), 16)
    b = kv4.Batch(2, 4, 2, 16)
    for args in [(i(1), i(2), i(2)), (i(2), i(2).long(), i(2)), (i(2), i(2), i(2).cpu())]:
        with pytest.raises(ValueError):
            b.plan(*args)
    with pytest.raises(kv4.Cis2Error):
        kv4.Batch(2, 4, 2, 20).plan(i(2), i(2), i(2))
    assert cache.errors() == 0
    # too small a workspace is an argument error, not an overrun
    a = kv4._Attn(0, 4, 1, 1, 4, 1, 0, 0, 0.125, 0, q.data_ptr(), q.data_ptr(), 256, 64, 256, 64, batch.table.data_ptr(),
                  batch.length.data_ptr(), batch.row_start.data_ptr(), q.data_ptr(), 1)
    assert kv4._lib().cis2b_kv4_attention(cache._ref, ctypes.byref(a), None) == 1


@pytest.mark.parametrize("max_new", [1, 64])
def test_row_starts_and_lengths_that_do_not_belong_together(torch, kv4, max_new):
    """Row starts that go back, leave the rows or overlap, and negative lengths: the call ends, writes only
    inside out, and the next call is right."""
    w = World(torch, kv4, [300, 40, 500], [1, 1, 1], 2, 64, 16, "float32")
    q = w.queries(4, 64)
    want = w.cache.attention(q, w.batch, max_new=1)
    guard = torch.full((5, 4, 64), 3.0, device="cuda")
    for starts, lengths in [([2, 1, 0, 3], [300, 40, 500]), ([0, 100, 100, 200], [300, 40, 500]),
                            ([-50, 1, 2, 1000], [300, 40, 500]), ([0, 1, 2, 3], [-5, 40, -1])]:
        b = kv4.Batch.of(w.table, torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                         torch.tensor(starts, dtype=torch.int32, device="cuda"), 16)
        w.cache.attention(q, b, max_new=max_new, out=guard[1:4])
        assert (guard[0] == 3.0).all() and (guard[4] == 3.0).all()
    w.cache.errors()
    w.cache._work.clear()
    assert torch.equal(w.cache.attention(q, w.batch, max_new=1), want)
