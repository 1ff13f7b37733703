"""Operators around the 4-bit key/value cache for rows that do not see by their place alone, as cases
that can be timed and compared.

Four operators work on the paged cache that holds keys and values in 4 bits:

  tree       attention of drafted tokens: a row sees the request's cached tokens (all, or a window of
             them and a few first ones) and, of the new tokens, those that a mask of bits names
  cross      attention to the cached states of an encoder: a row sees all of them, however many rows
             there are
  plan_tree  from each drafted token's parent, the mask of its ancestors and its position
  commit     after the model has spoken: the longest path of drafted tokens that it agrees with, and the
             path's keys and values moved to the places that follow the cached tokens, in every
             layer's cache

`run` computes a case in its plain form (elementary torch operations in 32 bits) where `own` is
false, and through the package's entry points where it is true.

The cache.  A pool of pages; a page holds `page` tokens of every KV head; per head it is a run of
records of 16 tokens.  A record of head size D is 16 rows of D/2 key bytes, 16 rows of D/2 value
bytes (byte b holds element 2b in its low four bits and 2b+1 in its high four), then 16 times four
bfloat16 numbers: key step, key base, value step, value base.  Code c stands for base + step * c.
Of a group (one token's D elements of one head) base is the minimum rounded down to bfloat16, step
the range over 15 rounded up to bfloat16, and c the nearest of 0 .. 15.

The new tokens of a step stand behind a request's cached ones: token i of request r in slot
slot[row_start[r] + i], at place cached + i of the cache, whatever its position in the text.
"""
import importlib
import math

import numpy as np
import torch

own = False

REC = 16  # tokens in a record
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
GOLD = 0.6180339887498949  # spreads the lengths of a batch evenly, whatever its size
MOST = 8e9  # bounds what is drawn, see _weight: less than the largest listed cases have
VOCAB = 49152


def _kv4():
    return importlib.import_module("cis2-lab-archive_b200.kv4")


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # One request drafts 16 tokens at batch 1, SmolLM2 shape, float32 as this decoder computes:
        # latency is what counts.
        dict(name="tree 1x16 over 317 f32", op="tree", requests=1, min_len=333, max_len=333, min_new=16, max_new=16,
             heads=9, kv_heads=3, head_dim=64, page=16, window=0, sinks=0, dtype="f32", pool=2),
        # A loaded server that verifies 16 drafted tokens a request, ragged lengths up to 16K, over a
        # pool of more than 2^32 bytes.
        dict(name="tree 64x16 ragged bf16", op="tree", requests=64, min_len=1500, max_len=16384, min_new=16,
             max_new=16, heads=32, kv_heads=8, head_dim=128, page=32, window=0, sinks=0, dtype="bf16", pool=10),
        # One very long context and a wide tree: the work is split over the keys.
        dict(name="tree 1x64 over 130K bf16", op="tree", requests=1, min_len=130051, max_len=130051, min_new=64,
             max_new=64, heads=16, kv_heads=8, head_dim=128, page=64, window=0, sinks=0, dtype="bf16", pool=2),
        # Sliding-window layers with sinks, odd trees of up to 61 tokens, some requests with few.
        dict(name="tree 24x61 window f16", op="tree", requests=24, min_len=700, max_len=30011, min_new=3, max_new=61,
             heads=16, kv_heads=8, head_dim=128, page=16, window=1000, sinks=4, dtype="f16", pool=1),
        # Decoding one token a sequence against encoders of up to 1,500 states, a KV head per head.
        dict(name="cross decode 64x1 f16", op="cross", requests=64, min_len=97, max_len=1500, min_new=1, max_new=1,
             heads=12, kv_heads=12, head_dim=64, page=16, dtype="f16", pool=2),
        # Beam search: five rows share each encoder, float32; some encoders are empty.
        dict(name="cross beams 16x5 f32", op="cross", requests=16, min_len=0, max_len=1024, min_new=5, max_new=5,
             heads=9, kv_heads=3, head_dim=64, page=32, dtype="f32", pool=2),
        # A few long documents, one row each: the work is split over the keys.
        dict(name="cross 8x1 long bf16", op="cross", requests=8, min_len=5003, max_len=30011, min_new=1, max_new=1,
             heads=16, kv_heads=8, head_dim=128, page=64, dtype="bf16", pool=2),
        # Decoder prompts, or a whole teacher-forced batch: about 1,000 rows a request.
        dict(name="cross prompts 8x1000 bf16", op="cross", requests=8, min_len=1024, max_len=6000, min_new=777,
             max_new=1024, heads=16, kv_heads=8, head_dim=128, page=64, dtype="bf16", pool=2),
        # The masks of one decode step of the 64-sequence batch, 16 drafted tokens each.
        dict(name="plan_tree 64x16", op="plan_tree", requests=64, min_len=64, max_len=320, min_new=16, max_new=16,
             reach=8),
        # Many requests with large trees, some idle.
        dict(name="plan_tree 1021x257", op="plan_tree", requests=1021, min_len=0, max_len=20000, min_new=0,
             max_new=257, reach=24),
        # The end of that decode step in a model of two layers of the SmolLM2 shape.
        dict(name="commit 64x16 f32", op="commit", requests=64, min_len=64, max_len=320, min_new=16, max_new=16,
             reach=8, heads=9, kv_heads=3, head_dim=64, page=16, dtype="f32", layers=2),
        # The end of a step with large trees, four layers of the Qwen3 shape.
        dict(name="commit 250x61 bf16", op="commit", requests=250, min_len=1, max_len=2000, min_new=0, max_new=61,
             reach=24, heads=16, kv_heads=8, head_dim=128, page=64, dtype="bf16", layers=4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _weight(case):
    """Values that the plain form of a case goes through, which bounds what is drawn."""
    if case["op"] == "plan_tree":
        return case["requests"] * case["max_new"] * 64
    if case["op"] == "commit":
        return case["requests"] * case["max_new"] * case["kv_heads"] * case["head_dim"] * case["layers"] * 16
    keys = _visible_width(case)
    kv = case["requests"] * keys * case["kv_heads"] * case["head_dim"]
    return kv * 8 + case["requests"] * case["max_new"] * keys * case["heads"] * 16


def draw(rng):
    """A case of the ranges that the listed ones stand for."""
    while True:
        op = rng.choice(["tree", "tree", "tree", "cross", "cross", "cross", "plan_tree", "commit"])
        case = dict(op=op)
        if op in ("plan_tree", "commit"):
            few = op == "commit"
            top = _log_int(rng, 16, 2000 if few else 20000)
            new = _log_int(rng, 1, 61 if few else 257)
            case.update(requests=_log_int(rng, 1, 250 if few else 1021), min_new=rng.choice([0, 1, new]), max_new=new,
                        min_len=min(top, rng.choice([0, 1, 17, 64])), max_len=top, reach=rng.choice([1, 3, 8, 24]))
            case["max_len"] = max(top, new)
            if case["requests"] == 1:
                case["min_new"] = new
        if op != "plan_tree":
            heads, kv_heads, head_dim = rng.choice([(9, 3, 64), (12, 12, 64), (16, 8, 128), (32, 8, 128)])
            case.update(heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=rng.choice([16, 32, 64]),
                        dtype=rng.choice(["f32", "bf16", "bf16", "f16"]))
        if op == "commit":
            case["layers"] = rng.randint(1, 4)
        elif op == "tree":
            new = _log_int(rng, 1, 100)
            top = max(new, _log_int(rng, 16, 130051))
            case.update(requests=_log_int(rng, 1, 64), min_len=min(top, max(new, _log_int(rng, 1, top))), max_len=top,
                        min_new=rng.choice([0, 1, new]), max_new=new, window=0, sinks=0, pool=rng.choice([1, 2]))
            if rng.random() < 0.3:
                case.update(window=_log_int(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 33]))
            if case["requests"] < 3:
                case["min_new"] = new
        elif op == "cross":
            kind = rng.choice(["decode", "beams", "prompt"])
            new = 1 if kind == "decode" else _log_int(rng, 2, 16) if kind == "beams" else _log_int(rng, 17, 1024)
            top = _log_int(rng, 1, 6000 if kind == "prompt" else 30011)
            case.update(requests=_log_int(rng, 1, 8 if kind == "prompt" else 96), min_len=rng.choice([0, 1, top]),
                        max_len=top, min_new=rng.choice([1, new]), max_new=new, pool=rng.choice([1, 2]))
        if _weight(case) < MOST:
            return case


def _spread(n, lo, hi, phase):
    """n whole numbers from lo to hi, spread over their logarithm, both ends among them if n > 1."""
    u = [(0.5 * phase + (i + 1) * GOLD) % 1.0 for i in range(n)]
    if n > 1:
        u[0], u[1] = 0.0, 1.0
    a, b = math.log(lo + 1), math.log(hi + 1)
    return [min(hi, max(lo, round(math.exp(a + x * (b - a))) - 1)) for x in u]


def _lengths(case):
    """Tokens in the cache (a tree's new ones among them) and rows of every request; they go by the
    case alone."""
    n = case["requests"]
    new = _spread(n, case["min_new"], case["max_new"], 1)
    total = _spread(n, case["min_len"], case["max_len"], 0)
    if case["op"] == "cross":
        return total, new
    if n > 1:
        new[1], new[-1] = new[-1], new[1]  # the longest request is not always the one with most rows
    return [max(t, f) for t, f in zip(total, new)], new


def _visible_width(case):
    """The most keys that the rows of one request see between them."""
    if case.get("window"):
        return min(max(case["max_len"], case["max_new"]), case["sinks"] + case["window"] + case["max_new"] - 1)
    return max(case["max_len"], case["max_new"] if case["op"] == "tree" else 1, 1)


def _geometry(case):
    d = case["head_dim"]
    return case["kv_heads"], d, REC * (d + 8), case["page"] // REC


def _words(case):
    return (case["max_new"] + 31) // 32


# ---------------------------------------------------------------- what has to be moved and computed

def work(case):
    total, new = _lengths(case)
    n, rows = len(new), sum(new)
    if case["op"] == "plan_tree":
        return {"bytes": 4 * (rows + 2 * n + 1 + rows * (_words(case) + 1)), "flops": rows * 2 * math.log2(2 + case["max_new"])}
    kv, d, _, _ = _geometry(case)
    if case["op"] == "commit":
        # Token, parent and target in, path out; about half of a path moves; every row is read back.
        moved = sum(min(f, 4) // 2 for f in new)
        record = kv * (d + 8)
        back = rows * (record + 2 * kv * d * SIZE[case["dtype"]])
        return {"bytes": 4 * (4 * rows + 4 * n) + case["layers"] * (2 * moved * record + back),
                "flops": 3 * rows + case["layers"] * rows * kv * d * 4}
    keys = pairs = table = 0
    w, s = case.get("window", 0), case.get("sinks", 0)
    for t, f in zip(total, new):
        if not f:
            continue
        c = t - f if case["op"] == "tree" else t
        seen = c
        if w and c > w - 1:
            first = c - w + 1
            seen = c - first + min(s, first)
        own_rows = f if case["op"] == "tree" else 0
        keys += seen + own_rows
        table += -(-(seen + own_rows) // case["page"])
        # A drafted token sees about as many of its like as a tree of f nodes is deep.
        pairs += f * seen + (f * math.log2(1 + f) if own_rows else 0)
    mask = 4 * rows * (_words(case) + (1 if w else 0)) if case["op"] == "tree" else 0
    return {"bytes": keys * kv * (d + 8) + 2 * rows * case["heads"] * d * SIZE[case["dtype"]] + 4 * table + 8 * n + mask,
            "flops": 4 * d * case["heads"] * pairs}


# ---------------------------------------------------------------- the format, in 32 bits

def _round_down(x):
    """float32 to the next bfloat16 value at or below it, as float32."""
    bits = x.contiguous().view(torch.int32)
    cut = bits & -65536
    low = torch.where((bits < 0) & (bits != cut), cut + 65536, cut)
    return low.view(torch.float32)


def _round_up(x):
    """A float32 >= 0 to the next bfloat16 value at or above it, as float32."""
    return ((x.contiguous().view(torch.int32) + 65535) & -65536).view(torch.float32)


def _quantise(x):
    """[..., D] float32 -> codes [..., D] (whole numbers), step and base [...]."""
    base = _round_down(x.amin(-1))
    step = _round_up((x.amax(-1) - base) / torch.full_like(base, 15.0))  # a tensor: a number is multiplied by 1/15
    step = torch.where(step < 2.0 ** -100, torch.zeros_like(step), step)
    inv = torch.where(step > 0, 1.0 / step, torch.zeros_like(step))
    codes = torch.round((x - base.unsqueeze(-1)) * inv.unsqueeze(-1)).clamp(0, 15)
    return codes, step, base


def _pack(codes):
    c = codes.to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _records(pool, case):
    kv, d, size, _ = _geometry(case)
    recs = pool.view(-1, size)
    keys = recs[:, :8 * d].unflatten(1, (REC, d // 2))
    values = recs[:, 8 * d:16 * d].unflatten(1, (REC, d // 2))
    params = recs.view(torch.bfloat16)[:, 8 * d:].unflatten(1, (REC, 4))
    return keys, values, params


def _places(slot, case):
    """Record and row of every slot, for every KV head: [..., KV]."""
    kv, _, _, per_page = _geometry(case)
    page, off = slot // case["page"], slot % case["page"]
    head = torch.arange(kv, device=slot.device)
    rec = (page.unsqueeze(-1) * kv + head) * per_page + (off // REC).unsqueeze(-1)
    return rec, (off % REC).unsqueeze(-1).expand_as(rec)


def _store(pool, case, slot, k, v):
    keys, values, params = _records(pool, case)
    rec, row = _places(slot, case)
    kc, ks, kb = _quantise(k.float())
    vc, vs, vb = _quantise(v.float())
    keys[rec, row] = _pack(kc)
    values[rec, row] = _pack(vc)
    params[rec, row] = torch.stack([ks, kb, vs, vb], -1).to(torch.bfloat16)


def _unpack(codes, step, base):
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    return c.mul_(step.unsqueeze(-1)).add_(base.unsqueeze(-1))


def _load(pool, case, slot):
    """The values of the slots' keys and values in float32: two of [..., KV, D]."""
    keys, values, params = _records(pool, case)
    rec, row = _places(slot, case)
    p = params[rec, row].float()
    return _unpack(keys[rec, row], p[..., 0], p[..., 1]), _unpack(values[rec, row], p[..., 2], p[..., 3])


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 29)
    return g


def _kv_rows(g, shape):
    """Keys with a few large channels and an offset, as they are after rotary positions; plain values."""
    kv, d = shape[-2:]
    gain = torch.exp(0.5 * torch.randn(kv, d, generator=g, device="cuda"))
    shift = 0.5 * torch.randn(kv, d, generator=g, device="cuda")
    k = torch.randn(shape, generator=g, device="cuda").mul_(gain).add_(shift)
    v = torch.randn(shape, generator=g, device="cuda")
    return k, v


def _table(g, total, case):
    """Distinct pages for every request, at random places of the pool: the table and the pool's pages."""
    p = case["page"]
    need = [-(-t // p) for t in total]
    width = max(1, max(need))
    pages = max(1, sum(need)) * case.get("pool", 1)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    have = torch.tensor(need, device="cuda")
    start = torch.cumsum(have, 0) - have
    at = torch.arange(width, device="cuda")
    table = torch.where(at < have.unsqueeze(1), order[(start.unsqueeze(1) + at).clamp(max=pages - 1)], -1)
    return table.to(torch.int32).contiguous(), pages


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _starts(new):
    start = [0]
    for f in new:
        start.append(start[-1] + f)
    return start


def _parents(case, seed, new):
    """A drafted tree per request: each token hangs on one of the `reach` before it, nearer ones more
    often; the first on the request's cached tokens."""
    rng = np.random.default_rng([int(seed), 11])
    i = np.concatenate([np.arange(f) for f in new]) if sum(new) else np.zeros(0, np.int64)
    back = np.floor(rng.random(i.size) ** 2 * np.minimum(i, case.get("reach", 8))).astype(np.int64)
    return np.where(i > 0, i - 1 - back, -1)


def _mask_and_depth(parent, new, words):
    """Each row's ancestors and itself as bits of `words` numbers of 32, and its depth, on the host."""
    mask, depth, at = np.zeros((parent.size, words), np.uint32), np.zeros(parent.size, np.int64), 0
    for f in new:
        for i in range(f):
            p = parent[at + i]
            if p >= 0:
                mask[at + i], depth[at + i] = mask[at + p], depth[at + p] + 1
            mask[at + i, i // 32] |= np.uint32(1 << (i % 32))
        at += f
    return mask, depth


def _attention_inputs(case, seed):
    g = _gen(seed)
    kv, d, size, per_page = _geometry(case)
    total, new = _lengths(case)
    table, pages = _table(g, total, case)
    pool = torch.empty(pages, kv, per_page, size, dtype=torch.uint8, device="cuda")
    lens = torch.tensor(total, device="cuda")
    req = torch.repeat_interleave(torch.arange(len(total), device="cuda"), lens)
    pos = torch.arange(req.numel(), device="cuda") - torch.repeat_interleave(torch.cumsum(lens, 0) - lens, lens)
    slot = table[req, pos // case["page"]].long() * case["page"] + pos % case["page"]
    piece = max(1, (1 << 27) // (kv * d))
    for at in range(0, slot.numel(), piece):  # in pieces: the float rows need not all be there at once
        part = slot[at:at + piece]
        k, v = _kv_rows(g, (part.numel(), kv, d))
        _store(pool, case, part, k, v)
    start = _starts(new)
    q = (1.5 * torch.randn(start[-1], case["heads"], d, generator=g, device="cuda")).to(DTYPES[case["dtype"]])
    state = dict(q=q, pool=pool, pages=pages, table=table, length=_i32(total), row_start=_i32(start), max_new=max(new))
    if case["op"] == "tree":
        mask, depth = _mask_and_depth(_parents(case, seed, new), new, _words(case))
        state["mask"] = torch.from_numpy(mask.view(np.int32)).cuda()
        cached = np.repeat(np.array(total) - np.array(new), new)
        state["position"] = torch.from_numpy((cached + depth).astype(np.int32)).cuda()
    return state


def _plan_inputs(case, seed):
    total, new = _lengths(case)
    return dict(parent=_i32(_parents(case, seed, new)), length=_i32(total), row_start=_i32(_starts(new)), rows=sum(new))


def _commit_inputs(case, seed):
    """Drafted tokens, what the model says after each, and every layer's cache with the drafted tokens'
    keys and values.  Along a random path of each tree the model agrees; siblings with the same token
    are among them."""
    g = _gen(seed)
    total, new = _lengths(case)
    rng = np.random.default_rng([int(seed), 13])
    parent = _parents(case, seed, new)
    token, target = rng.integers(0, VOCAB, (2, parent.size))
    at = 0
    for f in new:
        children = [[] for _ in range(f)]
        for i in range(1, f):
            children[parent[at + i]].append(i)
        path = [0] if f else []
        while path and children[path[-1]]:
            kids = children[path[-1]]
            pick = int(rng.integers(len(kids)))
            target[at + path[-1]] = token[at + kids[pick]]
            if pick and rng.random() < 0.25:  # an earlier sibling with the same token is the one that counts
                token[at + kids[0]] = token[at + kids[pick]]
            path.append(next(i for i in kids if token[at + i] == target[at + path[-1]]))
        # The pass can be repeated on what it has left: no place that receives a token gives one, too.
        most = len(path)
        while any(i != k and i < most for k, i in enumerate(path[:most])):
            most -= 1
        if path:
            target[at + path[most - 1]] = VOCAB
        at += f
    kv, d, size, per_page = _geometry(case)
    table, pages = _table(g, total, case)
    fresh = torch.tensor(new, device="cuda")
    req = torch.repeat_interleave(torch.arange(len(new), device="cuda"), fresh)
    first = torch.tensor([t - f for t, f in zip(total, new)], device="cuda")
    row = torch.arange(req.numel(), device="cuda")
    pos = first[req] + row - torch.tensor(_starts(new), device="cuda")[req]
    slot = table[req, pos // case["page"]].long() * case["page"] + pos % case["page"]
    pools = []
    for _ in range(case["layers"]):
        pool = torch.zeros(pages, kv, per_page, size, dtype=torch.uint8, device="cuda")
        k, v = _kv_rows(g, (slot.numel(), kv, d))
        _store(pool, case, slot, k, v)
        pools.append(pool)
    return dict(token=_i32(token), parent=_i32(parent), target=_i32(target), length=_i32(total),
                row_start=_i32(_starts(new)), slot=slot.to(torch.int32), table=table, pools=pools, pages=pages,
                rows=int(parent.size))


def prepare(case, seed):
    op = case["op"]
    state = _plan_inputs(case, seed) if op == "plan_tree" else _commit_inputs(case, seed) if op == "commit" else \
        _attention_inputs(case, seed)
    if own:
        kv4 = _kv4()
        made = dict(page_size=case.get("page", 16), length=state["length"], row_start=state["row_start"])
        if op == "plan_tree":
            none = torch.full((case["requests"], 1), -1, dtype=torch.int32, device="cuda")
            state["batch"] = kv4.Batch.of(table=none, rows=state["rows"], tree=case["max_new"], **made)
        elif op == "commit":
            state["batch"] = kv4.Batch.of(table=state["table"], slot=state["slot"], **made)
            state["caches"] = [_cache(kv4, case, state, pool) for pool in state["pools"]]
        else:
            state["batch"] = kv4.Batch.of(table=state["table"], **made)
            state["cache"] = _cache(kv4, case, state, state["pool"])
            state["out"] = torch.empty_like(state["q"])
    state["case"] = case
    return state


def _cache(kv4, case, state, pool):
    return kv4.Cache(pages=state["pages"], page_size=case["page"], kv_heads=case["kv_heads"],
                     head_dim=case["head_dim"], pool=pool)


# ---------------------------------------------------------------- one pass

def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return _plain_plan(state, case) if op == "plan_tree" else _plain_commit(state, case) if op == "commit" else \
            _plain_attention(state, case)
    batch = state["batch"]
    if op == "plan_tree":
        batch.plan_tree(state["parent"])
        return dict(mask=batch.mask, position=batch.position)
    if op == "commit":
        batch.accept(state["token"], state["parent"], state["target"])
        batch.keep(state["caches"])
        back = [cache.gather(batch.slot, dtype=DTYPES[case["dtype"]]) for cache in state["caches"]]
        return dict(accepted=batch.accepted, path=batch.path, next_token=batch.next_token, kept=batch.kept,
                    k=[k for k, _ in back], v=[v for _, v in back])
    if op == "tree":
        return state["cache"].tree_attention(state["q"], batch, mask=state["mask"], position=state["position"],
                                             window=case["window"], sinks=case["sinks"], max_new=state["max_new"],
                                             out=state["out"])
    return state["cache"].cross_attention(state["q"], batch, max_new=state["max_new"], out=state["out"])


def _rows_of(state):
    """The request of every row, and its number in it."""
    start = state["row_start"].long()
    row = torch.arange(state["rows"], device="cuda")
    req = torch.searchsorted(start[1:], row, right=True)
    return req, row - start[req]


def _plain_plan(state, case):
    """Twice as many ancestors each time: a row's mask takes in that of the nearest one it lacks."""
    req, i = _rows_of(state)
    start, words = state["row_start"].long(), _words(case)
    cached = (state["length"].long() - (start[1:] - start[:-1]))[req]
    bit = torch.zeros(i.numel(), words, dtype=torch.int64, device="cuda")
    bit[torch.arange(i.numel(), device="cuda"), i // 32] = 1 << (i % 32)
    parent = state["parent"].long()
    up = torch.where(parent >= 0, start[req] + parent, -1)  # the nearest ancestor that is not in the mask yet
    mask, depth = bit.clone(), torch.zeros_like(i)
    for _ in range(case["max_new"].bit_length()):  # twice as many ancestors each time
        has, at = up >= 0, up.clamp(min=0)
        mask |= torch.where(has.unsqueeze(1), mask[at], 0)
        up = torch.where(has, up[at], -1)
    for b in range(32):
        depth += ((mask >> b) & 1).sum(1)
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask)
    return dict(mask=mask.to(torch.int32), position=(cached + depth - 1).to(torch.int32))


def _plain_commit(state, case):
    req, i = _rows_of(state)
    rows, n, most = i.numel(), case["requests"], case["max_new"]
    start = state["row_start"].long()
    new = start[1:] - start[:-1]
    parent, row = state["parent"].long(), torch.arange(rows, device="cuda")
    up = start[req] + parent.clamp(min=0)
    fits = (parent >= 0) & (state["token"] == state["target"][up])
    # The lowest row that a row agrees with; `rows` where there is none.
    follow = torch.full((rows + 1,), rows, dtype=torch.int64, device="cuda")
    follow.scatter_reduce_(0, torch.where(fits, up, rows), torch.where(fits, row, rows), "amin")
    follow[rows] = rows
    cur = torch.where(new > 0, start[:-1], rows)
    steps = [cur]
    for _ in range(most - 1):
        steps.append(follow[steps[-1]])
    steps = torch.stack(steps, 1)  # [requests, most]
    on = steps < rows
    accepted = on.sum(1)
    last = steps.gather(1, (accepted - 1).clamp(min=0).unsqueeze(1)).squeeze(1).clamp(max=max(rows - 1, 0))
    next_token = torch.where(accepted > 0, state["target"][last], -1) if rows else accepted.to(torch.int32) - 1
    path = torch.where(i < accepted[req], steps[req, i] - start[req], -1)
    slot = state["slot"].long()
    move = path >= 0
    source, place = slot[(start[req] + path)[move]], slot[move]
    ks, vs = [], []
    for pool in state["pools"]:
        rec, at = _places(source, case)
        to, to_at = _places(place, case)
        for part in _records(pool, case):
            part[to, to_at] = part[rec, at]
        k, v = _load(pool, case, slot)
        ks.append(k.to(DTYPES[case["dtype"]]))
        vs.append(v.to(DTYPES[case["dtype"]]))
    return dict(accepted=accepted.to(torch.int32), path=path.to(torch.int32), next_token=next_token.to(torch.int32),
                kept=(state["length"] - new + accepted).to(torch.int32), k=ks, v=vs)


def _plain_attention(state, case):
    q, table = state["q"], state["table"]
    h, kv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    window, sinks, tree = case.get("window", 0), case.get("sinks", 0), case["op"] == "tree"
    length, row_start, most = state["length"].long(), state["row_start"].long(), state["max_new"]
    new = row_start[1:] - row_start[:-1]
    n, width = new.numel(), _visible_width(case)
    cached = length - new if tree else length
    # The keys that any row of a request sees: the sinks, then those from the window's first on.
    i = torch.arange(width, device=q.device)
    if window:
        low = (cached - window + 1).clamp(min=sinks)
        key = torch.where(i < sinks, i, low.unsqueeze(1) + i - sinks)
    else:
        key = i.expand(n, width)
    held = key < length.unsqueeze(1)
    slot = table.gather(1, torch.where(held, key // page, 0)).long().clamp(min=0) * page + key % page
    k, v = _load(state["pool"], case, torch.where(held, slot, slot[:, :1]))
    # The rows of every request, padded to the most.
    j = torch.arange(most, device=q.device)
    row = (row_start[:-1].unsqueeze(1) + j).clamp(max=q.shape[0] - 1)
    x = q.float()[row].view(n, most, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, d)
    score = torch.matmul(x, k.permute(0, 2, 3, 1)).view(n, kv, h // kv, most, width)
    see = held.unsqueeze(1).expand(n, most, width)
    if tree:
        fresh = (key - cached.unsqueeze(1)).clamp(0, 32 * _words(case) - 1)  # the bit, where it is a new token
        bits = state["mask"].long()[row].gather(2, (fresh // 32).unsqueeze(1).expand(n, most, width))
        named = ((bits >> (fresh % 32).unsqueeze(1)) & 1) == 1
        old = (key < cached.unsqueeze(1)).unsqueeze(1)
        if window:
            pos = state["position"].long()[row].unsqueeze(2)
            old = old & ((key.unsqueeze(1) > pos - window) | (key < sinks).unsqueeze(1))
        see = see & torch.where((key >= cached.unsqueeze(1)).unsqueeze(1), named, old)
    score = score.mul_(d ** -0.5).masked_fill_(~see[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    prob = score.sub_(top).exp_()
    total = prob.sum(-1, keepdim=True)
    v = v.masked_fill(~held[:, :, None, None], 0.0)
    out = torch.matmul(prob.view(n, kv, -1, width), v.permute(0, 2, 1, 3)).view(n, kv, h // kv, most, d)
    out = (out / total.clamp(min=torch.finfo(torch.float32).tiny)).permute(0, 3, 1, 2, 4).reshape(n, most, h, d)
    return out[j < new.unsqueeze(1)].to(q.dtype)


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_values(codes, step, base):  # bytes [L, D/2], parameters [L] -> [L, D]
    c = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    c[:, 0::2] = (codes % 16).double()
    c[:, 1::2] = (codes // 16).double()
    return base[:, None].double() + step[:, None].double() * c


def _exact_rows(pool, case, pages, head, n):
    """The first n tokens on those pages, of one head: two of [n, D]."""
    _, d, size, _ = _geometry(case)
    recs = pool[pages, head].reshape(-1, size)
    par = recs[:, 16 * d:].contiguous().view(torch.bfloat16).view(-1, 4)[:n]
    kc, vc = recs[:, :8 * d].reshape(-1, d // 2)[:n], recs[:, 8 * d:16 * d].reshape(-1, d // 2)[:n]
    return _exact_values(kc, par[:, 0], par[:, 1]), _exact_values(vc, par[:, 2], par[:, 3])


def exact(case, seed):
    if case["op"] == "plan_tree":
        return None
    total, new = _lengths(case)
    kv = case["kv_heads"]
    if case["op"] == "commit":
        s = _commit_inputs(case, seed)
        token, parent, target, slot = (s[x].tolist() for x in ("token", "parent", "target", "slot"))
        source, at = list(slot), 0
        for f in new:
            cur, k = 0, 0
            while f:
                source[at + k] = slot[at + cur]
                follow = [i for i in range(cur + 1, f)
                          if parent[at + i] == cur and token[at + i] == target[at + cur]]
                if not follow:
                    break
                cur, k = follow[0], k + 1
            at += f
        src = torch.tensor(source, dtype=torch.int64, device="cuda")
        out = dict(accepted=None, path=None, next_token=None, kept=None, k=[], v=[])
        for pool in s["pools"]:
            k = torch.empty(len(source), kv, case["head_dim"], dtype=torch.float64, device="cuda")
            v = torch.empty_like(k)
            for hd in range(kv):
                every = _exact_rows(pool, case, torch.arange(s["pages"], device="cuda"), hd, s["pages"] * case["page"])
                k[:, hd], v[:, hd] = every[0][src], every[1][src]
            out["k"].append(k)
            out["v"].append(v)
        return out
    s = _attention_inputs(case, seed)
    group, window, sinks = case["heads"] // kv, case.get("window", 0), case.get("sinks", 0)
    bounds, tree = s["row_start"].tolist(), case["op"] == "tree"
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    if tree:
        parents = _parents(case, seed, new)
    for r, n in enumerate(total):
        a, b = bounds[r], bounds[r + 1]
        if a == b or not n:
            continue
        see = torch.ones(b - a, n, dtype=torch.bool, device="cuda")
        if tree:
            cached, up = n - (b - a), parents[a:b]
            among = np.zeros((b - a, b - a), bool)
            depth = np.zeros(b - a, np.int64)
            for i in range(b - a):
                x = i
                while x >= 0:
                    among[i, x] = True
                    x = up[x]
                depth[i] = among[i].sum() - 1
            see[:, cached:] = torch.from_numpy(among).cuda()
            if window:
                pos = cached + torch.from_numpy(depth).cuda()[:, None]
                j = torch.arange(cached, device="cuda")[None, :]
                see[:, :cached] = (pos - j < window) | (j < sinks)
        pages = s["table"][r, :-(-n // case["page"])].long()
        for hd in range(kv):
            k, v = _exact_rows(s["pool"], case, pages, hd, n)
            for g in range(group):
                x = s["q"][a:b, hd * group + g].double()
                logit = (x @ k.T) / math.sqrt(case["head_dim"])
                out[a:b, hd * group + g] = torch.softmax(logit.masked_fill(~see, -math.inf), -1) @ v
    return out
