"""4-bit paged key/value cache on the GPU: planning, append, read-back and
attention, over torch tensors (C ABI: the cis2b_kv4_* part of
include/cis2b.h, where the format and every rule is written down).

    kv4 = importlib.import_module("cis2-lab-archive_b200.kv4")
    cache = kv4.Cache(pages=4096, page_size=64, kv_heads=8, head_dim=128)  # one per layer
    batch = kv4.Batch(requests=64, tokens=64, width=256, page_size=64)     # one per step, all layers
    batch.plan(cached, new, free_pages)        # block table, slots, positions
    cache.append(k, v, batch.slot)             # rows -> 4 bits
    out = cache.attention(q, batch, window=0, sinks=0, max_new=1)

Everything runs on torch's current stream and returns without waiting for
it.  attention keeps a workspace per stream, which the caches of a device
share; each call captured in a CUDA graph has its own, so graphs may be
replayed on any streams, and beside other calls (not one graph beside itself).
Nothing here has a gradient.  This module needs torch for its tensors; the
rest of the package does not.

A step that verifies a tree of drafted tokens, and attention to an encoder's
states, whose keys and values another cache holds:

    batch = kv4.Batch(requests=64, tokens=64 * 16, width=256, page_size=64, tree=16)
    batch.plan(cached, new, free_pages)
    batch.plan_tree(parent)                    # batch.mask, batch.position; with a window: plan_tree(parent, window, sinks)
    cache.append(k, v, batch.slot)             # in every layer
    out = cache.tree_attention(q, batch, max_new=16)
    out = encoder.cross_attention(q, encoder_batch, max_new=16)
    batch.accept(token, parent, target)        # batch.accepted, .path, .next_token, .kept
    batch.keep(caches)                         # the accepted rows, in all layers at once
"""
from __future__ import annotations

import ctypes
import importlib
import weakref

import torch

_pkg = importlib.import_module(__package__)
Cis2Error = _pkg.Cis2Error

_I32, _I64, _U64, _P = ctypes.c_int32, ctypes.c_int64, ctypes.c_uint64, ctypes.c_void_p

BAD_SLOT, BAD_PAGE, STUCK, BAD_PATH = 1, 2, 4, 8  # CIS2B_KV4_*
_WORK_ZERO = 266240  # CIS2B_KV4_WORK_ZERO
PLAN_FREE, PLAN_WIDTH, PLAN_ROWS, PLAN_NEGATIVE = 1, 2, 4, 8  # CIS2B_KV4_PLAN_*
TREE_PARENT, TREE_ROWS = 1, 2  # CIS2B_KV4_TREE_*
TREE_MOST = 1024  # CIS2B_KV4_TREE_MOST
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # CIS2B_F32, _F16, _BF16


class _Cache(ctypes.Structure):
    _fields_ = [("device", _I32), ("pages", _I32), ("page_size", _I32), ("kv_heads", _I32), ("head_dim", _I32),
                ("reserved", _I32), ("pool", _P), ("status", _P)]


class _Step(ctypes.Structure):
    _fields_ = [("device", _I32), ("requests", _I32), ("rows", _I32), ("width", _I32), ("page_size", _I32),
                ("free_count", _I32), ("cached", _P), ("new_tokens", _P), ("free_pages", _P), ("table", _P),
                ("length", _P), ("row_start", _P), ("slot", _P), ("position", _P), ("request", _P), ("counts", _P)]


class _Attn(ctypes.Structure):
    _fields_ = [("dtype", _I32), ("heads", _I32), ("requests", _I32), ("rows", _I32), ("width", _I32),
                ("max_new", _I32), ("window", _I32), ("sinks", _I32), ("scale", ctypes.c_float), ("flags", _I32),
                ("q", _P), ("out", _P), ("q_row_stride", _I64), ("q_head_stride", _I64), ("out_row_stride", _I64),
                ("out_head_stride", _I64), ("table", _P), ("length", _P), ("row_start", _P), ("work", _P),
                ("work_bytes", _U64)]


class _Tree(ctypes.Structure):
    _fields_ = [("device", _I32), ("requests", _I32), ("rows", _I32), ("words", _I32), ("length", _P), ("row_start", _P),
                ("parent", _P), ("mask", _P), ("position", _P), ("status", _P)]


class _Draft(ctypes.Structure):
    _fields_ = [("device", _I32), ("requests", _I32), ("rows", _I32), ("reserved", _I32), ("length", _P), ("row_start", _P),
                ("token", _P), ("parent", _P), ("target", _P), ("accepted", _P), ("path", _P), ("next_token", _P),
                ("kept", _P), ("status", _P)]


class _Kept(ctypes.Structure):
    _fields_ = [("device", _I32), ("requests", _I32), ("rows", _I32), ("reserved", _I32), ("row_start", _P),
                ("accepted", _P), ("path", _P), ("slot", _P)]


_funcs = None


def _lib():
    global _funcs
    if _funcs is None:
        L = _pkg.lib()
        L.cis2b_kv4_bytes.argtypes = [_P, _P]
        L.cis2b_kv4_plan.argtypes = [_P, _P]
        L.cis2b_kv4_append.argtypes = [_P, _I32, _P, _P, _I64, _I64, _I64, _I64, _P, _I32, _P]
        L.cis2b_kv4_gather.argtypes = [_P, _I32, _P, _P, _P, _I32, _P]
        L.cis2b_kv4_workspace.argtypes = [_P, _P, _P]
        L.cis2b_kv4_attention.argtypes = [_P, _P, _P]
        L.cis2b_kv4_plan_tree_window.argtypes = [_P, _I32, _I32, _P]
        L.cis2b_kv4_plan_tree.argtypes = [_P, _P]
        L.cis2b_kv4_accept.argtypes = [_P, _P]
        L.cis2b_kv4_keep.argtypes = [_P, _I32, _P, _P]
        L.cis2b_kv4_tree_workspace.argtypes = [_P, _P, _P]
        L.cis2b_kv4_tree_attention.argtypes = [_P, _P, _P, _I32, _P, _P]
        L.cis2b_kv4_cross_attention.argtypes = [_P, _P, _P]
        _funcs = L
    return _funcs


def _check(rc: int) -> None:
    if rc:
        _pkg._check(rc)


_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice
_capturing = torch._C._cuda_isCurrentStreamCapturing


def _call(device: int, fn, *args) -> None:
    """fn(*args, torch's current stream), leaving the current device as it
    was: the C entry points make theirs current."""
    if _current_device() == device:
        rc = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(device))
    if rc:
        _pkg._check(rc)


def _device_index(device) -> int:
    d = torch.device(device)
    if d.type != "cuda":
        raise ValueError(f"device must be a CUDA device, not {d}")
    return torch.cuda.current_device() if d.index is None else d.index


def _ints(t, name: str, device: int, shape: tuple | None = None):
    if t.dtype is not torch.int32 or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor on cuda:{device}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, not {tuple(t.shape)}")
    return t


def _int32(*named) -> None:
    """Refuses numbers that a field of 32 bits would cut: (name, number) pairs."""
    for name, x in named:
        if not -2 ** 31 <= x < 2 ** 31:
            raise ValueError(f"{name} must fit in 32 bits, not {x}")


class Batch:
    """One step's block tables and slot maps, shared by every layer's cache.

    table [requests, width], length [requests], row_start [requests + 1],
    slot, position and request [tokens], counts [4]: int32 on the device.
    `plan` fills them; a batch made by `of` takes a table, lengths and row
    starts that the caller has built.

    Of drafted trees: mask [tokens, ceil(tree / 32)], which `plan_tree` fills
    (and position with it), if `tree`, the most rows of one request, is given;
    accepted, next_token and kept [requests] and path [tokens], which `accept`
    fills and which are None before."""

    mask = accepted = path = next_token = kept = None

    def __init__(self, requests: int, tokens: int, width: int, page_size: int, table=None, device="cuda", tree: int = 0):
        if requests < 1 or tokens < 0 or width < 1:
            raise ValueError("requests and width must be >= 1 and tokens >= 0")
        _int32(("requests", requests), ("tokens", tokens), ("width", width), ("page_size", page_size))
        self.device = _device_index(device if table is None else table.device)
        self.page_size = page_size

        def ints(*shape):
            return torch.full(shape, -1, dtype=torch.int32, device=f"cuda:{self.device}")

        self.table = ints(requests, width) if table is None else _ints(table, "table", self.device, (requests, width))
        self.length, self.row_start = ints(requests), ints(requests + 1)
        self.slot, self.position, self.request = ints(tokens), ints(tokens), ints(tokens)
        self.counts = ints(4)
        self._step = _Step(self.device, requests, tokens, width, page_size, 0, None, None, None,
                           self.table.data_ptr(), self.length.data_ptr(), self.row_start.data_ptr(),
                           self.slot.data_ptr(), self.position.data_ptr(), self.request.data_ptr(),
                           self.counts.data_ptr())
        self._ref = ctypes.byref(self._step)
        self._trees(tree, tokens)

    def _trees(self, tree: int, rows: int) -> None:
        if not 0 <= tree <= TREE_MOST:
            raise ValueError(f"tree must be in 0..{TREE_MOST}")
        self._tree = self._draft = self._kept = self._bits = None
        if tree:
            words = (tree + 31) // 32
            self.mask = torch.zeros((rows, words), dtype=torch.int32, device=f"cuda:{self.device}")
            self._tree = _Tree(self.device, self.length.numel(), rows, words, None, None, None, None, None, self._tree_bits())
            self._tree_ref = ctypes.byref(self._tree)

    def _tree_bits(self) -> int:
        """The status word of plan_tree and accept, made by the first that needs it."""
        if self._bits is None:
            self._bits = torch.zeros(1, dtype=torch.int32, device=f"cuda:{self.device}")
        return self._bits.data_ptr()

    @classmethod
    def of(cls, table, length, row_start, page_size: int, slot=None, rows: int | None = None, tree: int = 0) -> "Batch":
        """A batch over the caller's own table, lengths and row starts.  `keep`
        needs slot [rows], plan_tree `tree` and the number of rows (slot's, if
        that is given)."""
        self = cls.__new__(cls)
        self.device = _device_index(table.device)
        self.page_size = page_size
        if table.dim() != 2 or not table.numel():
            raise ValueError("table must be [requests, width]")
        n = table.shape[0]
        self.table = _ints(table, "table", self.device)
        self.length = _ints(length, "length", self.device, (n,))
        self.row_start = _ints(row_start, "row_start", self.device, (n + 1,))
        self.slot = self.position = self.request = self.counts = self._step = None
        if slot is not None:
            if slot.dim() != 1 or rows not in (None, slot.shape[0]):
                raise ValueError("slot must be [rows]")
            self.slot, rows = _ints(slot, "slot", self.device), slot.shape[0]
        if tree:
            if rows is None or rows < 0:
                raise ValueError("a batch with trees needs the number of its rows")
            _int32(("rows", rows))
            self.position = torch.full((rows,), -1, dtype=torch.int32, device=f"cuda:{self.device}")
        self._trees(tree, rows or 0)
        return self

    def plan(self, cached, new, free_pages) -> None:
        """cached, new [requests] and free_pages [any]: int32 on the device.
        Fills the batch's tensors (cis2b_kv4_plan); nothing is returned and
        nothing waited for.  `errors` reads what went wrong, if anything."""
        s = self._step
        if s is None:
            raise ValueError("this batch was made from a finished table; make one with Batch(...) to plan")
        dev, n = self.device, s.requests
        _ints(cached, "cached", dev, (n,)), _ints(new, "new", dev, (n,)), _ints(free_pages, "free_pages", dev)
        s.cached, s.new_tokens = cached.data_ptr(), new.data_ptr()
        _int32(("the number of free pages", free_pages.numel()))
        s.free_pages, s.free_count = free_pages.data_ptr(), free_pages.numel()
        _call(dev, _lib().cis2b_kv4_plan, self._ref)

    def errors(self) -> int:
        """PLAN_* bits of the last plan, 0 if all is well.  Waits for the GPU."""
        torch.cuda.synchronize(self.device)  # on whichever stream it was
        return int(self.counts[2].item())

    def plan_tree(self, parent, window: int = 0, sinks: int = 0, mask=None) -> None:
        """Masks and positions of drafted trees (cis2b_kv4_plan_tree_window):
        parent [rows], int32, the row of the same request that each row
        continues, -1 for the cached tokens.  Fills mask and position.  Give it
        the window and sinks of the layers that the masks are for: a row does
        not see ancestors outside them.  That matters only where a path is
        longer than the window; then layers with other windows need masks of
        their own: another call with `mask`, which is filled in place of the
        batch's and passed to tree_attention.  `tree_errors` reads what went
        wrong, if anything."""
        t = self._tree
        if t is None:
            raise ValueError("this batch was made without trees; give it `tree`, the most rows of one request")
        _ints(parent, "parent", self.device, (t.rows,))
        t.length, t.row_start, t.parent = self.length.data_ptr(), self.row_start.data_ptr(), parent.data_ptr()
        mask = self.mask if mask is None else _ints(mask, "mask", self.device, tuple(self.mask.shape))
        if window or sinks:
            _int32(("window", window), ("sinks", sinks))
        t.mask, t.position = mask.data_ptr(), self.position.data_ptr()
        _call(self.device, _lib().cis2b_kv4_plan_tree_window, self._tree_ref, window, sinks)

    def accept(self, token, parent, target) -> None:
        """The longest path of drafted tokens that the model agrees with
        (cis2b_kv4_accept): token, parent and target [rows], int32; target is
        the model's next token after each row.  Fills accepted, path, next_token
        and kept, the tokens that the request has cached from now on: the same
        tensors each time (path: the first rows of one that is made larger when
        it has to be; a captured call keeps the one it was captured with)."""
        dev = self.device
        if token.dim() != 1:
            raise ValueError("token must be [rows]")
        rows, n = token.shape[0], self.length.numel()
        for t, name in ((token, "token"), (parent, "parent"), (target, "target")):
            _ints(t, name, dev, (rows,))
        d = self._draft
        if d is None or d.rows != rows:
            _int32(("rows", rows))
            if self.accepted is None:
                self.accepted, self.next_token, self.kept = (
                    torch.full((n,), -1, dtype=torch.int32, device=f"cuda:{dev}") for _ in range(3))
                self._paths = []  # all of them: captured calls may write to any
            most = self._paths[-1].shape[0] if self._paths else -1
            if rows > most:
                size = max(rows, 2 * most, self.slot.shape[0] if self.slot is not None else 0)
                self._paths.append(torch.full((size,), -1, dtype=torch.int32, device=f"cuda:{dev}"))
            self.path = self._paths[-1][:rows]
            d = self._draft = _Draft(dev, n, rows, 0, None, None, None, None, None, self.accepted.data_ptr(),
                                     self.path.data_ptr(), self.next_token.data_ptr(), self.kept.data_ptr(),
                                     self._tree_bits())
        d.length, d.row_start = self.length.data_ptr(), self.row_start.data_ptr()
        d.token, d.parent, d.target = token.data_ptr(), parent.data_ptr(), target.data_ptr()
        _call(dev, _lib().cis2b_kv4_accept, ctypes.byref(d))

    def keep(self, caches) -> None:
        """Moves the accepted rows of every request to the places that follow
        its cached tokens, in each of `caches` (cis2b_kv4_keep), one launch for
        up to 64 layers.  They are cached from then on: kept[r] tokens.  What
        stands in the other rows' places is left as it is."""
        caches = list(caches)
        if self._draft is None or self.slot is None:
            raise ValueError("keep follows accept, and needs the batch's slots")
        if not caches or any(c.device != self.device or c.page_size != self.page_size for c in caches):
            raise ValueError(f"the caches must be on cuda:{self.device}, with pages of {self.page_size} tokens")
        if len({c.pool.data_ptr() for c in caches}) != len(caches):
            raise ValueError("a cache may be given once")
        rows = self.path.shape[0]
        if self.slot.shape[0] < rows:
            raise ValueError(f"the batch has slots for {self.slot.shape[0]} rows, not {rows}")
        every = self._kept
        if every is None or every[0] != caches:
            every = self._kept = (caches, (_Cache * len(caches))(*(c._c for c in caches)))
        k = _Kept(self.device, self.length.numel(), rows, 0, self.row_start.data_ptr(), self.accepted.data_ptr(),
                  self.path.data_ptr(), self.slot.data_ptr())
        _call(self.device, _lib().cis2b_kv4_keep, every[1], len(caches), ctypes.byref(k))

    def tree_errors(self) -> int:
        """TREE_* bits that plan_tree and accept have left since the last time,
        0 if all is well.  Waits for the GPU.  (Of a batch without `tree`, if its
        first accept was captured: those of the last replay.)"""
        if self._bits is None:
            return 0
        torch.cuda.synchronize(self.device)
        bits = int(self._bits.item())
        if bits:
            self._bits.zero_()
            torch.cuda.synchronize(self.device)
        return bits


class _Workspaces(dict):
    """A device's workspaces, by stream: calls on one stream follow one another,
    whichever layer's cache they are of.  Kept by the caches of the device."""


_workspaces = weakref.WeakValueDictionary()  # by device


class Cache:
    """One layer's keys and values in 4 bits: a pool of pages on the device.
    Like a model handle, it belongs to one thread at a time.

    pool  uint8 [pages, kv_heads, page_size // 16, 16 * (head_dim + 8)];
          pass your own to place it, else it is allocated (zeroed)."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, pool=None, device="cuda"):
        self.device = _device_index(device if pool is None else pool.device)
        _int32(("pages", pages), ("page_size", page_size), ("kv_heads", kv_heads), ("head_dim", head_dim))
        self._c = _Cache(self.device, pages, page_size, kv_heads, head_dim, 0, None, None)
        self._ref = ctypes.byref(self._c)
        size = _U64()
        _check(_lib().cis2b_kv4_bytes(self._ref, ctypes.byref(size)))
        shape = (pages, kv_heads, page_size // 16, 16 * (head_dim + 8))
        if pool is None:
            pool = torch.zeros(shape, dtype=torch.uint8, device=f"cuda:{self.device}")
        elif pool.dtype is not torch.uint8 or not pool.is_contiguous() or pool.numel() != size.value:
            raise ValueError(f"pool must be a contiguous uint8 tensor of {size.value} bytes")
        self.pool = pool.view(shape)
        self.page_size, self.kv_heads, self.head_dim = page_size, kv_heads, head_dim
        self.status = torch.zeros(1, dtype=torch.int32, device=f"cuda:{self.device}")
        self._c.pool, self._c.status = self.pool.data_ptr(), self.status.data_ptr()
        self._work = _workspaces.setdefault(self.device, _Workspaces())
        self._calls = {}  # by shape: filled-in arguments

    def errors(self) -> int:
        """BAD_* and STUCK bits that calls have left since the last time, 0 if all is well.  Waits for the GPU."""
        torch.cuda.synchronize(self.device)  # calls may be on any stream, and those that follow too
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            if bits & STUCK:  # counters may have been left in the middle
                for work in list(self._work.values()):
                    work[:_WORK_ZERO].zero_()
            torch.cuda.synchronize(self.device)
        return bits

    def _rows(self, t, name: str):
        if t.dim() != 3 or t.shape[1] != self.kv_heads or t.shape[2] != self.head_dim:
            raise ValueError(f"{name} must be [rows, {self.kv_heads}, {self.head_dim}]")
        if t.get_device() != self.device or t.dtype not in _DTYPES:
            raise ValueError(f"{name} must be float32, float16 or bfloat16 on cuda:{self.device}")
        s = t.stride()
        if s[2] != 1:
            raise ValueError(f"the elements of a head of {name} must be contiguous")
        return s

    def append(self, k, v, slot) -> None:
        """Quantises rows k, v [rows, kv_heads, head_dim] (any row and head
        strides) into the slots slot [rows]; negative slots are skipped."""
        ks, vs = self._rows(k, "k"), self._rows(v, "v")
        n = k.shape[0]
        if v.shape[0] != n or v.dtype is not k.dtype:
            raise ValueError("k and v must have the same rows and type")
        _ints(slot, "slot", self.device, (n,))
        _call(self.device, _lib().cis2b_kv4_append, self._ref, _DTYPES[k.dtype], k.data_ptr(), v.data_ptr(), ks[0], ks[1],
              vs[0], vs[1], slot.data_ptr(), n)

    def gather(self, slot, dtype=torch.float32):
        """The keys and values of the slots as the values that their codes
        stand for: two [rows, kv_heads, head_dim]; zeros for negative slots."""
        _ints(slot, "slot", self.device)
        if dtype not in _DTYPES or slot.dim() != 1:
            raise ValueError("dtype must be float32, float16 or bfloat16 and slot [rows]")
        n = slot.shape[0]
        k, v = torch.empty((2, n, self.kv_heads, self.head_dim), dtype=dtype, device=slot.device).unbind(0)
        _call(self.device, _lib().cis2b_kv4_gather, self._ref, _DTYPES[dtype], k.data_ptr(), v.data_ptr(), slot.data_ptr(), n)
        return k, v

    def attention(self, q, batch: Batch, scale: float | None = None, window: int = 0, sinks: int = 0,
                  max_new: int | None = None, out=None, whole: bool = False):
        """Causal attention of the step's rows q [rows, heads, head_dim] over
        the cache; their own keys and values are appended before.  With
        window > 0 a row sees its last `window` keys and the first `sinks`.
        max_new is the most rows that one request has in this step (a bound
        will do; it only chooses the kernel).  If None, a batch with no more
        rows than requests is taken to have one each, any other may have all
        rows in one request.  whole: a request's result does not depend on the
        rest of the batch, given the same max_new (slower over long requests).
        Returns out (made if None)."""
        ref, out = self._arguments("attention", q, batch, out, scale, window, sinks, max_new, whole)
        _call(self.device, _lib().cis2b_kv4_attention, self._ref, ref)
        return out

    def tree_attention(self, q, batch: Batch, mask=None, position=None, scale: float | None = None, window: int = 0,
                       sinks: int = 0, max_new: int | None = None, out=None, whole: bool = False):
        """Attention of drafted tokens q [rows, heads, head_dim], whose own
        keys and values are appended before.  A row sees the request's cached
        tokens (with window > 0 those less than `window` before its position,
        and the first `sinks`), and of its new ones those whose bits mask
        [rows, words] has: bit b % 32 of word b // 32 for row b of the request.
        The window hides no new token: where a path is longer than it, the mask
        has to be one that plan_tree made for that window.  mask and position
        [rows] are the batch's own (plan_tree) if None; any mask may be given;
        position is read with a window only.  The rest is as in `attention`."""
        mask = batch.mask if mask is None else mask
        position = batch.position if position is None else position
        if mask is None or mask.dim() != 2 or mask.shape[0] < q.shape[0] or not mask.shape[1]:
            raise ValueError("mask must be [rows, words], with a row for each of q; plan_tree makes the batch's own")
        _ints(mask, "mask", self.device)
        at = None
        if window:
            if position is None or position.dim() != 1 or position.shape[0] < q.shape[0]:
                raise ValueError("with a window, position must be [rows], with one for each row of q")
            at = _ints(position, "position", self.device).data_ptr()
        ref, out = self._arguments("tree_attention", q, batch, out, scale, window, sinks, max_new, whole)
        _call(self.device, _lib().cis2b_kv4_tree_attention, self._ref, ref, mask.data_ptr(), mask.shape[1], at)
        return out

    def cross_attention(self, q, batch: Batch, scale: float | None = None, max_new: int | None = None, out=None,
                        whole: bool = False):
        """Attention of rows q [rows, heads, head_dim] to the states of an
        encoder that this cache holds: batch.length[r] of them, 0 or more, on
        the pages of batch.table[r], all seen by every row of request r
        (batch.row_start), however many rows that are.  Requests may share
        pages, as beams do.  The rest is as in `attention`."""
        ref, out = self._arguments("cross_attention", q, batch, out, scale, 0, 0, max_new, whole)
        _call(self.device, _lib().cis2b_kv4_cross_attention, self._ref, ref)
        return out

    def _arguments(self, kind, q, batch, out, scale, window, sinks, max_new, whole):
        """The filled-in arguments of a call, and its output."""
        if q.requires_grad and torch.is_grad_enabled():
            raise ValueError("attention over the 4-bit cache has no gradient")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        key = (kind, q.dtype, q.shape, q.stride(), out.dtype, out.shape, out.stride(), batch.table.shape, batch.page_size,
               scale, window, sinks, max_new, whole)
        call = self._calls.get(key)
        if call is None:
            call = self._prepare(kind, q, out, batch, scale, window, sinks, max_new, whole)
            if len(self._calls) >= 64:
                self._calls.clear()
            self._calls[key] = call
        a, ref, need = call
        dev = self.device
        if q.get_device() != dev or out.get_device() != dev or batch.device != dev:
            raise ValueError(f"q, out and the batch must be on cuda:{dev}")
        work = self._workspace(need)
        a.q, a.out, a.work, a.work_bytes = q.data_ptr(), out.data_ptr(), work.data_ptr(), work.numel()
        a.table, a.length, a.row_start = batch.table.data_ptr(), batch.length.data_ptr(), batch.row_start.data_ptr()
        return ref, out

    def _workspace(self, need: int):
        """The current stream's workspace.  A call that is captured gets one of
        its own, zeroed by each replay: a graph may run beside this stream."""
        dev = self.device
        if _current_device() != dev:
            with torch.cuda.device(dev):
                return self._workspace(need)
        capturing, stream = _capturing(), _raw_stream(dev)
        work = None if capturing else self._work.get(stream)
        if work is None or work.numel() < need:
            work = torch.empty(need, dtype=torch.uint8, device=f"cuda:{dev}")
            work[:_WORK_ZERO].zero_()
            if not capturing:
                self._work[stream] = work  # an outgrown one is free for what follows on this stream
        return work

    def _prepare(self, kind, q, out, batch, scale, window, sinks, max_new, whole):
        if q.dim() != 3 or q.shape[2] != self.head_dim:
            raise ValueError(f"q must be [rows, heads, {self.head_dim}]")
        if q.dtype not in _DTYPES:
            raise ValueError("q must be float32, float16 or bfloat16")
        if out.shape != q.shape or out.dtype is not q.dtype:
            raise ValueError("out must have q's shape and type")
        if q.stride(2) != 1 or out.stride(2) != 1:
            raise ValueError("the elements of a head of q and out must be contiguous")
        if batch.page_size != self.page_size:
            raise ValueError(f"the batch was made for pages of {batch.page_size} tokens, not {self.page_size}")
        rows, heads = q.shape[0], q.shape[1]
        _int32(("window", window), ("sinks", sinks))
        if max_new is None:
            max_new = 1 if rows <= batch.table.shape[0] else rows
        a = _Attn(_DTYPES[q.dtype], heads, batch.table.shape[0], rows, batch.table.shape[1],
                  min(max(1, max_new), 2 ** 31 - 1), window, sinks,
                  self.head_dim ** -0.5 if scale is None else scale, int(whole), None, None, q.stride(0), q.stride(1),
                  out.stride(0), out.stride(1), None, None, None, None, 0)
        need = _U64()
        size = _lib().cis2b_kv4_workspace if kind == "attention" else _lib().cis2b_kv4_tree_workspace
        _check(size(self._ref, ctypes.byref(a), ctypes.byref(need)))
        return a, ctypes.byref(a), need.value
