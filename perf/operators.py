"""The operators of the 4-bit key/value cache, as cases that can be timed and compared.

Three operators work on one paged cache that holds keys and values in 4 bits:

  plan       block tables, slot maps and row offsets built on the GPU from the requests' lengths
  append     new key/value rows quantised to 4 bits and written to their slots, and the same
             rows read back as the values that they stand for
  attention  causal attention over the cache for one or many new tokens per request, with an
             optional sliding window and a few first tokens that stay visible (sinks)

`run` computes a case in its plain form (elementary torch operations in 32 bits) where `own` is
false, and through the package's entry points where it is true.

The cache.  A pool of pages; a page holds `page` tokens of every KV head; per head it is a run of
records of 16 tokens.  A record of head size D is 16 rows of D/2 key bytes, 16 rows of D/2 value
bytes (byte b holds element 2b in its low four bits and 2b+1 in its high four), then 16 times four
bfloat16 numbers: key step, key base, value step, value base.  Code c stands for base + step * c.
A group is one token's D elements of one head:

  base = min(x) rounded down to bfloat16
  step = (max(x) - base) / 15 rounded up to bfloat16 (0 if below 2^-100)
  c    = round((x - base) * (1 / step)) clamped to 0 .. 15, ties to even (0 if the step is 0)

with every step of it in 32 bits.
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


def _kv4():
    return importlib.import_module("cis2-lab-archive_b200.kv4")


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # One decode step of the 64-sequence batch: every request adds one token. A serving loop
        # pays this once a step, so its latency is what counts.
        dict(name="plan decode step", op="plan", requests=64, min_len=64, max_len=320, min_new=1, max_new=1,
             page=16, pad=0),
        # A continuous batch of many requests, most of them decoding, some with a chunk of their
        # prompt, some idle; the token rows are padded to the capacity that a captured graph has.
        dict(name="plan mixed batch", op="plan", requests=1021, min_len=0, max_len=20000, min_new=0, max_new=257,
             page=32, pad=1999),
        # The rows that one decode step of the SmolLM2 shape adds: 64 tokens, 3 KV heads of 64,
        # float32 as this decoder computes.
        dict(name="append decode step f32", op="append", tokens=64, heads=9, kv_heads=3, head_dim=64, page=16,
             dtype="f32", pool=2),
        # A prompt pass of 8,192 rows (the decoder's largest) of the Qwen3 shape, read out of the
        # fused q/k/v rows of a bfloat16 model.
        dict(name="append prompt bf16", op="append", tokens=8192, heads=16, kv_heads=8, head_dim=128, page=64,
             dtype="bf16", pool=2),
        # The prompts of a whole batch at once, an odd number of rows, half precision.
        dict(name="append prompts f16", op="append", tokens=40009, heads=16, kv_heads=8, head_dim=128, page=32,
             dtype="f16", pool=1),
        # Decode at batch 1 (the single-sequence configuration): 320 positions at most.
        dict(name="decode 1x317 f32", op="attention", requests=1, min_len=317, max_len=317, min_new=1, max_new=1,
             heads=9, kv_heads=3, head_dim=64, page=16, window=0, sinks=0, dtype="f32", pool=2),
        # Decode of the 64-sequence batch of the SmolLM2 shape, at the positions that it has.
        dict(name="decode 64x320 f32", op="attention", requests=64, min_len=64, max_len=320, min_new=1, max_new=1,
             heads=9, kv_heads=3, head_dim=64, page=16, window=0, sinks=0, dtype="f32", pool=2),
        # One request with a very long context: the work has to be split over its keys.
        dict(name="decode 1x130051 bf16", op="attention", requests=1, min_len=130051, max_len=130051, min_new=1,
             max_new=1, heads=16, kv_heads=8, head_dim=128, page=64, window=0, sinks=0, dtype="bf16", pool=2),
        # A loaded server: ragged requests of up to 16K tokens, spread over a pool of more than
        # 2^32 bytes.
        dict(name="decode 64 ragged bf16", op="attention", requests=64, min_len=1500, max_len=16384, min_new=1,
             max_new=1, heads=32, kv_heads=8, head_dim=128, page=32, window=0, sinks=0, dtype="bf16", pool=12),
        # Sliding-window layers with sinks over long requests: only 4 + 1,000 keys are visible.
        dict(name="decode window f16", op="attention", requests=96, min_len=700, max_len=30011, min_new=1,
             max_new=1, heads=16, kv_heads=8, head_dim=128, page=16, window=1000, sinks=4, dtype="f16", pool=1),
        # Chunked prompts: about 1,000 new tokens a request, some on top of a cached prefix.
        dict(name="prompt chunks bf16", op="attention", requests=5, min_len=1024, max_len=6000, min_new=777,
             max_new=1024, heads=16, kv_heads=8, head_dim=128, page=64, window=0, sinks=0, dtype="bf16", pool=2),
        # The 1,024-token prompts of the long-context configuration, float32.
        dict(name="prompts 8x1024 f32", op="attention", requests=8, min_len=1024, max_len=1024, min_new=1024,
             max_new=1024, heads=9, kv_heads=3, head_dim=64, page=16, window=0, sinks=0, dtype="f32", pool=2),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _weight(case):
    """Values that the plain form of a case goes through, which bounds what is drawn."""
    if case["op"] == "plan":
        return case["requests"] * (case["max_new"] + 64)
    if case["op"] == "append":
        return case["tokens"] * case["kv_heads"] * case["head_dim"]
    keys = _visible_width(case)
    kv = case["requests"] * keys * case["kv_heads"] * case["head_dim"]
    return kv * 8 + case["requests"] * case["max_new"] * keys * case["heads"] * 16


def draw(rng):
    """A case of the ranges that the listed ones stand for."""
    while True:
        op = rng.choice(["plan", "append", "attention", "attention", "attention"])
        if op == "plan":
            many = rng.random() < 0.5
            top = _log_int(rng, 16, 20000)
            case = dict(op=op, requests=_log_int(rng, 1, 1021), min_len=min(top, rng.choice([0, 1, 17, 64])),
                        max_len=top, min_new=rng.choice([0, 1]), max_new=_log_int(rng, 2, 257) if many else 1,
                        page=rng.choice([16, 32, 64]), pad=rng.choice([0, 0, rng.randint(1, 1999)]))
        else:
            heads, kv_heads, head_dim = rng.choice([(9, 3, 64), (12, 12, 64), (16, 8, 128), (32, 8, 128)])
            case = dict(op=op, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=rng.choice([16, 32, 64]),
                        dtype=rng.choice(["f32", "bf16", "bf16", "f16"]), pool=rng.choice([1, 2]))
            if op == "append":
                case["tokens"] = _log_int(rng, 1, 40009)
            else:
                kind = rng.choice(["decode", "decode", "window", "few", "prompt"])
                top = _log_int(rng, 16, 130051 if kind == "decode" else 30011)
                new = 1 if kind in ("decode", "window") else _log_int(rng, 2, 8) if kind == "few" else \
                    _log_int(rng, 9, 1024)
                top = max(top, new) if kind != "prompt" else min(max(top, new), 6000)
                case.update(requests=_log_int(rng, 1, 96) if kind != "prompt" else _log_int(rng, 1, 8),
                            min_len=min(top, max(new, _log_int(rng, 1, top))), max_len=top, min_new=1,
                            max_new=new, window=0, sinks=0)
                if new > 1 and case["requests"] > 2:
                    case["min_new"] = rng.choice([0, 1])  # some requests may have nothing to add
                if kind == "window" or rng.random() < 0.2:
                    case.update(window=_log_int(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 33]))
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
    """Cached and new tokens of every request; they go by the case alone."""
    n = case["requests"]
    new = _spread(n, case["min_new"], case["max_new"], 1)
    total = _spread(n, case["min_len"], case["max_len"], 0)
    if case["op"] == "plan":
        return total, new
    if case["max_new"] > 1:  # the longest prompts arrive whole, the others on a cached prefix
        new = new[::-1]
    total = [max(t, f) for t, f in zip(total, new)]
    return [t - f for t, f in zip(total, new)], new


def _visible_width(case):
    """The most keys that the rows of one request see between them."""
    if case["window"]:
        return min(case["max_len"], case["sinks"] + case["window"] + case["max_new"] - 1)
    return max(case["max_len"], case["max_new"])


def _geometry(case):
    d = case["head_dim"]
    return case["kv_heads"], d, REC * (d + 8), case["page"] // REC


# ---------------------------------------------------------------- what has to be moved and computed

def work(case):
    if case["op"] == "plan":
        cached, new = _lengths(case)
        p = case["page"]
        taken = sum(-(-(c + f) // p) - -(-c // p) for c, f in zip(cached, new))
        rows = sum(new) + case["pad"]
        return {"bytes": 4 * (4 * len(new) + 1 + 3 * rows + 2 * taken + len(new)), "flops": 4 * rows}
    kv, d, _, _ = _geometry(case)
    if case["op"] == "append":
        n = case["tokens"] * kv
        # Rows in, record out, record in, rows out, and the slots once for each way.
        return {"bytes": n * (4 * d * SIZE[case["dtype"]] + 2 * (d + 8)) + 8 * case["tokens"],
                "flops": n * 2 * d * 6}
    cached, new = _lengths(case)
    keys = pairs = table = 0
    w, s = case["window"], case["sinks"]
    for c, f in zip(cached, new):
        if not f:
            continue
        total = c + f
        first = max(0, c - w + 1) if w else 0
        seen = total - first + min(s, first) if w else total
        keys += seen
        table += -(-seen // case["page"])
        for_all = f * c + f * (f + 1) // 2
        if w:
            for_all = sum((p + 1) if p + 1 <= w else w + min(s, p + 1 - w) for p in range(c, total))
        pairs += for_all
    rows = sum(new)
    return {"bytes": keys * kv * (d + 8) + 2 * rows * case["heads"] * d * SIZE[case["dtype"]] + 4 * table
            + 8 * len(new), "flops": 4 * d * case["heads"] * pairs}


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
    return (page.unsqueeze(-1) * kv + head) * per_page + (off // REC).unsqueeze(-1), (off % REC).unsqueeze(-1)


def _store(pool, case, slot, k, v):
    keys, values, params = _records(pool, case)
    rec, row = _places(slot, case)
    row = row.expand_as(rec)
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
    row = row.expand_as(rec)
    p = params[rec, row].float()
    return _unpack(keys[rec, row], p[..., 0], p[..., 1]), _unpack(values[rec, row], p[..., 2], p[..., 3])


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 17)
    return g


def _kv_rows(g, shape):
    """Keys with a few large channels and an offset, as they are after rotary positions; plain values."""
    kv, d = shape[-2:]
    gain = torch.exp(0.5 * torch.randn(kv, d, generator=g, device="cuda"))
    shift = 0.5 * torch.randn(kv, d, generator=g, device="cuda")
    k = torch.randn(shape, generator=g, device="cuda").mul_(gain).add_(shift)
    v = torch.randn(shape, generator=g, device="cuda")
    return k, v


def _pages(g, cached, new, case, spare):
    """Distinct pages for every request, at random places of the pool: the table and its width."""
    p = case["page"]
    need = [-(-(c + f) // p) for c, f in zip(cached, new)]
    width = max(1, max(need)) + spare
    pages = max(1, sum(need)) * case.get("pool", 1)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    have = torch.tensor(need, device="cuda")
    start = torch.cumsum(have, 0) - have
    at = torch.arange(width, device="cuda")
    inside = at < have.unsqueeze(1)
    table = torch.where(inside, order[(start.unsqueeze(1) + at).clamp(max=pages - 1)], -1)
    return table.to(torch.int32).contiguous(), pages


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _plan_inputs(case, seed):
    g = _gen(seed)
    cached, new = _lengths(case)
    p = case["page"]
    have = [-(-c // p) for c in cached]
    need = [-(-(c + f) // p) for c, f in zip(cached, new)]
    taken = sum(need) - sum(have)
    order = torch.randperm(sum(need) + 64, generator=g, device="cuda").to(torch.int32)
    width = max(1, max(need)) + 3
    held = torch.tensor(have, device="cuda")
    start = torch.cumsum(held, 0) - held
    at = torch.arange(width, device="cuda")
    table = torch.where(at < held.unsqueeze(1), order[(start.unsqueeze(1) + at).clamp(max=order.numel() - 1)], -1)
    return dict(cached=_i32(cached), new=_i32(new), free=order[sum(have):].contiguous(), width=width,
                rows=sum(new) + case["pad"], table=table.to(torch.int32).contiguous(), taken=taken)


def _append_inputs(case, seed):
    """Fused q/k/v rows, as a decoder's first product of a layer leaves them, and their slots."""
    g = _gen(seed)
    n, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"]
    k, v = _kv_rows(g, (n, kv, d))
    fused = torch.empty(n, (h + 2 * kv) * d, dtype=DTYPES[case["dtype"]], device="cuda").normal_(generator=g)
    fused[:, h * d:(h + kv) * d] = k.reshape(n, -1).to(fused.dtype)
    fused[:, (h + kv) * d:] = v.reshape(n, -1).to(fused.dtype)
    table, pages = _pages(g, [0], [n], case, 0)
    at = torch.arange(n, device="cuda")
    slot = table[0][at // case["page"]] * case["page"] + at % case["page"]
    return dict(k=fused[:, h * d:(h + kv) * d].unflatten(1, (kv, d)), v=fused[:, (h + kv) * d:].unflatten(1, (kv, d)),
                slot=slot.to(torch.int32).contiguous(), pages=pages)


def _attention_inputs(case, seed):
    g = _gen(seed)
    kv, d, size, per_page = _geometry(case)
    cached, new = _lengths(case)
    table, pages = _pages(g, cached, new, case, 0)
    total = [c + f for c, f in zip(cached, new)]
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
    rows = sum(new)
    q = (1.5 * torch.randn(rows, case["heads"], d, generator=g, device="cuda")).to(DTYPES[case["dtype"]])
    start = [0]
    for f in new:
        start.append(start[-1] + f)
    return dict(q=q, pool=pool, pages=pages, table=table, length=_i32(total), row_start=_i32(start), max_new=max(new))


def prepare(case, seed):
    if case["op"] == "plan":
        state = _plan_inputs(case, seed)
        if own:
            kv4 = _kv4()
            state["batch"] = kv4.Batch(requests=case["requests"], tokens=state["rows"], width=state["width"],
                                       page_size=case["page"], table=state["table"])
    elif case["op"] == "append":
        state = _append_inputs(case, seed)
        kv, d, size, per_page = _geometry(case)
        state["pool"] = torch.zeros(state["pages"], kv, per_page, size, dtype=torch.uint8, device="cuda")
    else:
        state = _attention_inputs(case, seed)
        if own:
            state["batch"] = _kv4().Batch.of(table=state["table"], length=state["length"],
                                             row_start=state["row_start"], page_size=case["page"])
            state["out"] = torch.empty_like(state["q"])
    if own and case["op"] != "plan":
        state["cache"] = _kv4().Cache(pages=state["pages"], page_size=case["page"], kv_heads=case["kv_heads"],
                                      head_dim=case["head_dim"], pool=state["pool"])
    state["case"] = case
    return state


# ---------------------------------------------------------------- one pass

def run(state):
    case = state["case"]
    if own:
        if case["op"] == "plan":
            b = state["batch"]
            b.plan(state["cached"], state["new"], state["free"])
            return dict(table=b.table, length=b.length, row_start=b.row_start, slot=b.slot, position=b.position,
                        request=b.request, counts=b.counts)
        if case["op"] == "append":
            state["cache"].append(state["k"], state["v"], state["slot"])
            k, v = state["cache"].gather(state["slot"], dtype=state["k"].dtype)
            return dict(k=k, v=v)
        return state["cache"].attention(state["q"], state["batch"], window=case["window"], sinks=case["sinks"],
                                        max_new=state["max_new"], out=state["out"])
    if case["op"] == "plan":
        return _plain_plan(state, case["page"])
    if case["op"] == "append":
        slot = state["slot"].long()
        _store(state["pool"], case, slot, state["k"], state["v"])
        k, v = _load(state["pool"], case, slot)
        return dict(k=k.to(state["k"].dtype), v=v.to(state["v"].dtype))
    return _plain_attention(state, case)


def _plain_plan(state, page):
    cached, new, free = state["cached"], state["new"], state["free"]
    n, rows = cached.numel(), state["rows"]
    length = cached + new
    have = (cached + (page - 1)) // page
    need = (length + (page - 1)) // page - have
    row_start = torch.cat([new.new_zeros(1), torch.cumsum(new, 0, dtype=torch.int32)])
    first = torch.cumsum(need, 0) - need
    t = torch.arange(rows, dtype=torch.int32, device=new.device)
    inside = t < row_start[-1]
    req = torch.searchsorted(row_start[1:], t, right=True).clamp(max=n - 1)
    pos = cached[req] + t - row_start[req]
    col = torch.where(inside, pos // page, 0)
    fresh = col >= have[req]
    taken = free[torch.where(fresh & inside, first[req] + col - have[req], 0)]
    chosen = torch.where(fresh, taken, state["table"][req, col])
    state["table"][req[inside], col[inside].long()] = chosen[inside]
    slot = chosen * page + pos % page
    none = torch.full_like(t, -1)
    counts = torch.stack([row_start[-1].long(), need.sum(), torch.zeros_like(first[0]), torch.zeros_like(first[0])])
    return dict(table=state["table"], length=length, row_start=row_start, slot=torch.where(inside, slot, none),
                position=torch.where(inside, pos, none), request=torch.where(inside, req.to(torch.int32), none),
                counts=counts.to(torch.int32))


def _plain_attention(state, case):
    q, table = state["q"], state["table"]
    h, kv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    length, row_start, most = state["length"].long(), state["row_start"].long(), state["max_new"]
    new = row_start[1:] - row_start[:-1]
    n, width = new.numel(), _visible_width(case)
    # The keys that any row of a request sees: the sinks, then those from the first row's window on.
    i = torch.arange(width, device=q.device)
    if case["window"]:
        low = (length - new - case["window"] + 1).clamp(min=case["sinks"])
        key = torch.where(i < case["sinks"], i, low.unsqueeze(1) + i - case["sinks"])
    else:
        key = i.expand(n, width)
    held = key < length.unsqueeze(1)
    slot = table.gather(1, torch.where(held, key // page, 0)).long() * page + key % page
    k, v = _load(state["pool"], case, torch.where(held, slot, slot[:, :1]))
    # The rows of every request, padded to the longest.
    j = torch.arange(most, device=q.device)
    pos = (length - new).unsqueeze(1) + j
    row = (row_start[:-1].unsqueeze(1) + j).clamp(max=q.shape[0] - 1)
    x = q.float()[row].view(n, most, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, d)
    score = torch.matmul(x, k.permute(0, 2, 3, 1)).view(n, kv, h // kv, most, width)
    see = held.unsqueeze(1) & (key.unsqueeze(1) <= pos.unsqueeze(2))
    if case["window"]:
        see &= (key.unsqueeze(1) > pos.unsqueeze(2) - case["window"]) | (key.unsqueeze(1) < case["sinks"])
    score = score.mul_(d ** -0.5).masked_fill_(~see[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    prob = score.sub_(top).exp_()
    total = prob.sum(-1, keepdim=True)
    out = torch.matmul(prob.view(n, kv, -1, width), v.permute(0, 2, 1, 3)).view(n, kv, h // kv, most, d)
    out = (out / total.clamp(min=torch.finfo(torch.float32).tiny)).permute(0, 3, 1, 2, 4).reshape(n, most, h, d)
    return out[j < new.unsqueeze(1)].to(q.dtype)


# ---------------------------------------------------------------- the definition in 64 bits

def _bf16_bound(x, rounded):
    """float64 values to the bfloat16 ones below (rounded = floor) or above (ceil) them."""
    unit = np.ldexp(1.0, np.frexp(x)[1] - 8)
    return rounded(x / unit) * unit


def _exact_group(x):
    """One tensor [N, KV, D] through the format: what its codes stand for, in 64 bits.
    The definition rounds the difference, the quotient and the product to 32 bits."""
    x = x.double().cpu().numpy()

    def r32(a):
        return a.astype(np.float32).astype(np.float64)

    base = _bf16_bound(x.min(-1), np.floor)
    step = _bf16_bound(r32(r32(x.max(-1) - base) / 15.0), np.ceil)
    flat = step < 2.0 ** -100
    inv = np.where(flat, 0.0, r32(1.0 / np.where(flat, 1.0, step)))
    codes = np.clip(np.rint(r32(r32(x - base[..., None]) * inv[..., None])), 0, 15)
    return torch.from_numpy(base[..., None] + np.where(flat, 0.0, step)[..., None] * codes)


def exact(case, seed):
    if case["op"] == "plan":
        return None
    if case["op"] == "append":
        s = _append_inputs(case, seed)
        return dict(k=_exact_group(s["k"]).cuda(), v=_exact_group(s["v"]).cuda())
    s = _attention_inputs(case, seed)
    kv, d, size, per_page = _geometry(case)
    group = case["heads"] // kv
    raw = s["pool"].view(s["pages"], kv, per_page, size)
    bounds, lens = s["row_start"].tolist(), s["length"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")

    def values(codes, step, base):  # [L, D/2] bytes -> [L, D]
        c = torch.empty(codes.shape[0], d, dtype=torch.float64, device="cuda")
        c[:, 0::2] = (codes % 16).double()
        c[:, 1::2] = (codes // 16).double()
        return base[:, None] + step[:, None] * c

    for r, n in enumerate(lens):
        a, b = bounds[r], bounds[r + 1]
        if a == b:
            continue
        pages = s["table"][r, :-(-n // case["page"])].long()
        for hd in range(kv):
            recs = raw[pages, hd].reshape(-1, size)
            kc = recs[:, :8 * d].reshape(-1, d // 2)[:n]
            vc = recs[:, 8 * d:16 * d].reshape(-1, d // 2)[:n]
            par = recs[:, 16 * d:].contiguous().view(torch.bfloat16).view(-1, 4)[:n].double()
            k = values(kc, par[:, 0], par[:, 1])
            v = values(vc, par[:, 2], par[:, 3])
            pos = torch.arange(n - (b - a), n, device="cuda")[:, None]
            j = torch.arange(n, device="cuda")[None, :]
            seen = j <= pos
            if case["window"]:
                seen = seen & ((pos - j < case["window"]) | (j < case["sinks"]))
            for g in range(group):
                x = s["q"][a:b, hd * group + g].double()
                logit = (x @ k.T) / math.sqrt(d)
                weight = torch.softmax(logit.masked_fill(~seen, -math.inf), -1)
                out[a:b, hd * group + g] = weight @ v
    return out
