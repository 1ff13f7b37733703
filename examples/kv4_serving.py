"""A small serving loop over the 4-bit key/value cache.

Requests of different lengths share one pool of pages.  Every step plans the
batch on the GPU (a chunk of a prompt for new requests, one token for the
others), and every layer appends the step's keys and values and attends over
its cache; one layer has a sliding window with sinks.  Finished requests give
their pages back.  The layers are random projections: what is shown is how the
operators fit together, and how far 4 bits are from an uncompressed cache.

    python examples/kv4_serving.py
"""
from __future__ import annotations

import importlib
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
kv4 = importlib.import_module("cis2-lab-archive_b200.kv4")

HIDDEN, HEADS, KV_HEADS, HEAD_DIM, PAGE = 576, 9, 3, 64, 16  # the SmolLM2 shape's attention
WINDOWS = [(0, 0), (64, 4)]  # (window, sinks) of each layer


def make_layers(generator):
    def weight(*shape):
        return torch.randn(*shape, generator=generator, device="cuda") * shape[-1] ** -0.5

    return [dict(qkv=weight((HEADS + 2 * KV_HEADS) * HEAD_DIM, HIDDEN), out=weight(HIDDEN, HEADS * HEAD_DIM))
            for _ in WINDOWS]


def plain_rows(q, k, v, first, window, sinks):
    """Rows q [n, heads, d] at positions first .. over plain k, v [len, kv heads, d]."""
    group = HEADS // KV_HEADS
    score = torch.einsum("nhd,lhd->hnl", q, k.repeat_interleave(group, 1)) * HEAD_DIM ** -0.5
    pos = torch.arange(first, first + q.shape[0], device=q.device)[:, None]
    key = torch.arange(k.shape[0], device=q.device)
    see = key <= pos
    if window:
        see &= (key > pos - window) | (key < sinks)
    return torch.einsum("hnl,lhd->nhd", score.masked_fill(~see, float("-inf")).softmax(-1), v.repeat_interleave(group, 1))


def serve(prompts=(70, 9, 150, 33, 1), tokens=12, chunk=48, pages=96, seed=0):
    """Runs every request to prompt + tokens.  Returns the number of steps and
    the relative difference of all attention outputs from an uncompressed cache."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    layers = make_layers(gen)
    caches = [kv4.Cache(pages, PAGE, KV_HEADS, HEAD_DIM) for _ in layers]
    slots = 4  # requests that run at a time
    batch = kv4.Batch(slots, slots * chunk, width=pages, page_size=PAGE)
    waiting, running = list(range(len(prompts))), {}
    inputs = [torch.randn(n + tokens, HIDDEN, generator=gen, device="cuda") for n in prompts]
    plain = {}  # (request, layer): uncompressed keys and values
    free = list(range(pages))
    off = total = 0.0
    steps = 0
    while waiting or running:
        for slot in range(slots):
            if slot not in running and waiting:
                running[slot] = dict(request=waiting.pop(0), cached=0)
        new = [0] * slots
        for slot, r in running.items():
            left = prompts[r["request"]] - r["cached"]
            new[slot] = min(left, chunk) if left > 0 else 1
        cached = [running[s]["cached"] if s in running else 0 for s in range(slots)]
        batch.plan(torch.tensor(cached, dtype=torch.int32, device="cuda"), torch.tensor(new, dtype=torch.int32, device="cuda"),
                   torch.tensor(free, dtype=torch.int32, device="cuda"))
        if batch.errors():
            raise RuntimeError("the pool is too small for these requests")
        free = free[int(batch.counts[1]):]

        rows = sum(new)
        x = torch.cat([inputs[r["request"]][r["cached"]:r["cached"] + new[s]] for s, r in sorted(running.items())])
        for i, (layer, cache, (window, sinks)) in enumerate(zip(layers, caches, WINDOWS)):
            q, k, v = (x @ layer["qkv"].T).unflatten(1, (-1, HEAD_DIM)).split([HEADS, KV_HEADS, KV_HEADS], 1)
            cache.append(k, v, batch.slot[:rows])
            y = cache.attention(q, batch, window=window, sinks=sinks, max_new=max(new))
            at = 0
            for s, r in sorted(running.items()):  # the same rows over an uncompressed cache
                part = slice(at, at + new[s])
                old = plain.get((r["request"], i))
                pair = [torch.cat([o, n[part]]) for o, n in zip(old, (k, v))] if old else [k[part], v[part]]
                plain[r["request"], i] = pair
                want = plain_rows(q[part], *pair, r["cached"], window, sinks)
                off, total = off + float((y[part] - want).square().sum()), total + float(want.square().sum())
                at += new[s]
            x = x + y.flatten(1) @ layer["out"].T

        for slot in list(running):
            r = running[slot]
            r["cached"] += new[slot]
            if r["cached"] == prompts[r["request"]] + tokens:
                free += batch.table[slot, :-(-r["cached"] // PAGE)].tolist()
                del running[slot]
        steps += 1
    if any(cache.errors() for cache in caches):
        raise RuntimeError("a kernel reported an error")
    if sorted(free) != list(range(pages)):
        raise RuntimeError("pages were lost")
    return steps, (off / total) ** 0.5


if __name__ == "__main__":
    n, difference = serve()
    print(f"{n} steps; attention over 4 bits differs from an uncompressed cache by {difference:.3f} (relative)")
