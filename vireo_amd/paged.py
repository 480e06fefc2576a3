"""Serving many sequences from one paged 16-bit key-value cache
(include/vireo_paged.h) on torch device tensors:

    table = PagedTable.create(max_seqs, max_blocks, n_blocks, block_tokens)
    caches = [PagedCache.create(table, n_kv_heads, head_size) for each layer]
    plan = PagedPlan(table, caches[0], n, n_heads)
    each step:
        table.extend(n_new, start, positions, slots, status, ids=ids)
        plan.update(ids=ids)
        each layer:
            cache.append(q, k, v, positions, slots, q_out, rope)
            cache.attend(q_out, out, plan)

As with every call of the library, a call on the default stream waits for its
work; on a stream (the current one, or `stream=`) it is only enqueued. Where
`stream=` is not the current one, the call's tensors are recorded on it, so that
they may be dropped before its work is done (tensors made on the current stream
need nothing, as with torch's own calls); that inputs are there when it begins
and that outputs are read after it is the caller's to order, and so is that the
tensors of a captured graph live as long as it. Every tensor must be on the
table's or cache's device, which need not be the current one. Arguments that the
library would misread raise ValueError here; what it refuses itself raises
VireoError.
"""
import ctypes as C
import math

import torch

from . import _lib

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_I32 = torch.int32


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _count(v, name):
    """v, which a C int would otherwise hold the low bits of."""
    if not -2 ** 31 <= v < 2 ** 31:
        raise ValueError(f"{name}: a count within 32 bits is needed")
    return v


def _ints(t, shape, dev, name):
    """The address of a contiguous int32 tensor of this shape; dev: the device's index."""
    if t.dtype is not _I32 or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous int32 tensor of shape {tuple(shape)} on GPU {dev} is needed")
    return t.data_ptr()


def _floats(t, n, dev, name):
    if t.dtype is not torch.float32 or t.numel() != n or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{name}: a contiguous float32 tensor of {n} values on GPU {dev} is needed")
    return t.data_ptr()


def _rows(t, shape, dev, name):
    """Address, type and row stride of [rows, heads, d] rows whose heads are consecutive."""
    kind = _TYPES.get(t.dtype)
    if kind is None or t.shape != shape or t.get_device() != dev:
        raise ValueError(f"{name}: a float32, float16 or bfloat16 tensor of shape {tuple(shape)} on GPU {dev} is needed")
    rows, heads, d = shape
    row, head, one = t.stride()
    if one != 1 or (head != d and heads > 1):
        raise ValueError(f"{name}: the heads of a row have to be consecutive")
    return t.data_ptr(), kind, row if rows > 1 else heads * d


class _On:
    """A device's calls: on the given or current stream, with that device current."""

    def __init__(self, device):
        _need(device.type == "cuda", "a tensor on a GPU is needed")
        self.lib = _lib.load()
        self.device = device
        self.index = device.index
        self.alone = torch.cuda.device_count() == 1

    def call(self, name, stream, tensors, handles, *args):
        """tensors: the call's (or None); handles: the objects whose own tensors it uses."""
        fn = getattr(self.lib, name)
        if stream is None:
            stream = torch.cuda.current_stream(self.device)
        elif stream.device_index != self.index:
            raise ValueError(f"a stream of {self.device} is needed")
        elif torch.accelerator.current_stream(self.index).stream_id != stream.stream_id:
            # the tensors' memory is not to be given to others before this stream's work is done (0.3 us each)
            for t in tensors:
                if t is not None:
                    t.record_stream(stream)
            for h in handles:
                if stream.cuda_stream not in h.streams:
                    h.streams.add(stream.cuda_stream)
                    for t in h.own:
                        t.record_stream(stream)
        if self.alone or torch.cuda.current_device() == self.index:
            rc = fn(*args, stream.cuda_stream)
        else:
            with torch.cuda.device(self.device):
                rc = fn(*args, stream.cuda_stream)
        if rc:
            _lib.check(rc, name)


class PagedTable:
    """Block tables [max_seqs, max_blocks], lengths [max_seqs], the free blocks
    (a stack in [n_blocks]) and their number [1], int32 tensors that the caller
    keeps and may read; block_tokens is 16, 32, 64 or 128."""

    def __init__(self, blocks, length, free_blocks, n_free, block_tokens):
        _need(blocks.dim() == 2 and free_blocks.dim() == 1, "blocks is [max_seqs, max_blocks], free_blocks [n_blocks]")
        self.on = _On(blocks.device)
        self.device = blocks.device
        self.index = dev = blocks.get_device()
        self.max_seqs, self.max_blocks = blocks.shape
        self.n_blocks, self.block_tokens = free_blocks.numel(), _count(block_tokens, "block_tokens")
        self.blocks, self.len, self.free_blocks, self.n_free = blocks, length, free_blocks, n_free
        self.c = _lib.PagedTableC(self.max_seqs, self.max_blocks, self.n_blocks, block_tokens,
                                  _ints(blocks, blocks.shape, dev, "blocks"),
                                  _ints(length, (self.max_seqs,), dev, "len"),
                                  _ints(free_blocks, free_blocks.shape, dev, "free_blocks"),
                                  _ints(n_free, (1,), dev, "n_free"))
        self._p = C.pointer(self.c)
        self.own, self.streams = (blocks, length, free_blocks, n_free), set()

    @classmethod
    def create(cls, max_seqs, max_blocks, n_blocks, block_tokens, device="cuda", stream=None):
        """A table of empty sequences with every block free."""
        dev = torch.device(device)
        if dev.index is None:
            dev = torch.device(dev.type, torch.cuda.current_device())
        new = lambda *shape: torch.zeros(shape, dtype=_I32, device=dev)  # noqa: E731
        t = cls(new(max_seqs, max_blocks), new(max_seqs), new(n_blocks), new(1), block_tokens)
        if stream is not None:  # the zeros are written on the current stream
            stream.wait_stream(torch.cuda.current_stream(dev))
        t.reset(stream=stream)
        return t

    def reset(self, stream=None):
        self.on.call("vireo_paged_reset", stream, (), (self,), self._p)

    def _ids(self, ids, n):
        if ids is None:
            return None
        return _ints(ids, (n,), self.index, "ids")

    def extend(self, n_new, start, positions, slots, status, ids=None, stream=None):
        """Room for n_new [n] more tokens (None: one each) of sequences ids [n] (None:
        0 .. n - 1): fills start [n + 1], positions and slots [max_rows] and status
        [n] (0 or a negative errno, per sequence: see the header)."""
        n, rows, dev = status.numel(), slots.numel(), self.index
        self.on.call("vireo_paged_extend", stream, (ids, n_new, start, positions, slots, status), (self,), self._p,
                     self._ids(ids, n), None if n_new is None else _ints(n_new, (n,), dev, "n_new"), n, rows,
                     _ints(start, (n + 1,), dev, "start"), _ints(positions, (rows,), dev, "positions"),
                     _ints(slots, (rows,), dev, "slots"), _ints(status, (n,), dev, "status"))

    def truncate(self, new_len=None, ids=None, stream=None):
        """Sequences ids cut back to new_len tokens (None: to none, which ends them);
        ids None: as many as new_len has, or every sequence."""
        n = ids.numel() if ids is not None else new_len.numel() if new_len is not None else self.max_seqs
        self.on.call("vireo_paged_truncate", stream, (ids, new_len), (self,), self._p, self._ids(ids, n),
                     None if new_len is None else _ints(new_len, (n,), self.index, "new_len"), n)


class PagedPlan:
    """The split of a batch's attention over the device, for n sequences of
    `table` and caches shaped like `cache`; list_blocks > 0: over lists of that
    many blocks (PagedCache.select). update() once per step: before the first one
    attend and select leave their outputs as they were. Its memory serves one
    stream at a time."""

    def __init__(self, table, cache, n, n_heads, list_blocks=0):
        self.table, self.n, self.n_heads = table, _count(n, "n"), _count(n_heads, "n_heads")
        self.list_blocks = _count(list_blocks, "list_blocks")
        self.n_kv_heads, self.head_size = cache.n_kv_heads, cache.head_size
        self.ids = None  # of the last update
        self._shape = (n, n_heads, cache.head_size)
        self._lists = (n, cache.n_kv_heads, list_blocks)
        self.index = table.index
        self.c = _lib.PagedPlanC(table._p, None, n, n_heads, cache.n_kv_heads, cache.head_size, list_blocks, None)
        self._p = C.pointer(self.c)
        nbytes = table.on.lib.vireo_paged_plan_bytes(self._p)
        if nbytes < 0:
            _lib.check(int(nbytes), "vireo_paged_plan_bytes")
        self.mem = torch.zeros(int(nbytes), dtype=torch.uint8, device=table.device)
        self.c.mem = self.mem.data_ptr()
        self.own, self.streams = (self.mem,), set()
        # zeroed on the current stream; the plan may serve on another
        torch.cuda.current_stream(table.device).synchronize()

    def update(self, ids=None, stream=None):
        """By the table's lengths now; ids [n]: the batch's sequences (None: 0 .. n - 1)."""
        self.c.ids = self.table._ids(ids, self.n)
        self.ids = ids
        self.table.on.call("vireo_paged_plan_update", stream, (ids,), (self, self.table), self._p)


class PagedCache:
    """One layer's keys [n_blocks, n_kv_heads, block_tokens, head_size], values
    [n_blocks, n_kv_heads, head_size, block_tokens] and, for select, mean keys of
    full blocks [n_blocks, n_kv_heads, head_size]: float16 or bfloat16."""

    def __init__(self, k, v, means=None):
        _need(k.dim() == 4 and k.dtype in (torch.float16, torch.bfloat16), "k: a 4-dimensional 16-bit float tensor")
        nb, kv, G, d = k.shape
        _need(v.shape == (nb, kv, d, G) and v.dtype is k.dtype and v.device == k.device,
              "v: [n_blocks, n_kv_heads, head_size, block_tokens] beside k [n_blocks, n_kv_heads, block_tokens, head_size]")
        _need(k.is_contiguous() and v.is_contiguous(), "k and v have to be contiguous")
        _need(means is None or (means.shape == (nb, kv, d) and means.dtype is k.dtype and means.device == k.device and
                                means.is_contiguous()), "means: [n_blocks, n_kv_heads, head_size] like k")
        self.on = _On(k.device)
        self.device, self.dtype, self.index = k.device, k.dtype, k.get_device()
        self.n_blocks, self.n_kv_heads, self.block_tokens, self.head_size = nb, kv, G, d
        self.k, self.v, self.means = k, v, means
        self.c = _lib.PagedCacheC(_TYPES[k.dtype], nb, G, kv, d, k.data_ptr(), v.data_ptr(),
                                  None if means is None else means.data_ptr())
        self._p = C.pointer(self.c)
        self.own, self.streams = (k, v) if means is None else (k, v, means), set()

    @classmethod
    def create(cls, table, n_kv_heads, head_size, dtype=torch.bfloat16, means=False):
        """An empty cache for the blocks of `table`."""
        nb, G = table.n_blocks, table.block_tokens
        new = lambda *shape: torch.empty(shape, dtype=dtype, device=table.device)  # noqa: E731
        return cls(new(nb, n_kv_heads, G, head_size), new(nb, n_kv_heads, head_size, G),
                   new(nb, n_kv_heads, head_size) if means else None)

    def append(self, q, k, v, positions, slots, q_out, rope=None, q_norm=None, k_norm=None, q_bias=None, k_bias=None,
               v_bias=None, eps=1e-6, stream=None):
        """A step's rows: q [T, n_heads, head_size], k and v [T, n_kv_heads, head_size]
        (views of one projection's output will do) with positions and slots [T] from
        PagedTable.extend; norms and biases in fp32; rope: [max_pos, rotary] from
        vireo_rope_table (None: no rotation). q_out [T, n_heads, head_size] receives
        the queries for attend; k and v go into the cache."""
        dev, d, KV = self.index, self.head_size, self.n_kv_heads
        T, H = slots.numel(), q.shape[1]
        qp, qt, qs = _rows(q, (T, H, d), dev, "q")
        kp, kt, ks = _rows(k, (T, KV, d), dev, "k")
        vp, vt, vs = _rows(v, (T, KV, d), dev, "v")
        op, ot, os_ = _rows(q_out, (T, H, d), dev, "q_out")
        _need(qt == kt == vt, "q, k and v have to be of one type")
        max_pos, rotary = (0, 0) if rope is None else rope.shape
        r = _lib.PagedRowsC(T, H, qt, qp, kp, vp, qs, ks, vs,
                            None if q_bias is None else _floats(q_bias, H * d, dev, "q_bias"),
                            None if k_bias is None else _floats(k_bias, KV * d, dev, "k_bias"),
                            None if v_bias is None else _floats(v_bias, KV * d, dev, "v_bias"),
                            None if q_norm is None else _floats(q_norm, d, dev, "q_norm"),
                            None if k_norm is None else _floats(k_norm, d, dev, "k_norm"), eps,
                            None if rope is None else _floats(rope, max_pos * rotary, dev, "rope"), rotary, max_pos,
                            _ints(positions, (T,), dev, "positions"), _ints(slots, (T,), dev, "slots"), op, ot, os_)
        self.on.call("vireo_paged_append", stream,
                     (q, k, v, positions, slots, q_out, rope, q_norm, k_norm, q_bias, k_bias, v_bias), (self,), self._p,
                     C.byref(r))

    def _plan(self, plan):
        if plan.index != self.index:
            raise ValueError(f"a plan on {self.device} is needed")
        return plan._p

    def attend(self, q, out, plan, lists=None, scale=None, stream=None):
        """out [n, n_heads, head_size] = attention of q (each sequence's newest token; of
        a prompt appended at once only the last can be attended) over the sequences' blocks, or over lists [n, n_kv_heads,
        list_blocks] of them; scale: 1 / sqrt(head_size) if None."""
        qp, qt, qs = _rows(q, plan._shape, self.index, "q")
        op, ot, os_ = _rows(out, plan._shape, self.index, "out")
        if qt != ot:
            raise ValueError("q and out have to be of one type")
        if (lists is not None) != (plan.list_blocks > 0):
            raise ValueError("lists go with a plan for lists, and only with one")
        lp = None if lists is None else _ints(lists, plan._lists, self.index, "lists")
        self.on.call("vireo_paged_attend", stream, (q, out, lists), (self, plan, plan.table), self._p, self._plan(plan),
                     qp, qt, qs, 1.0 / math.sqrt(self.head_size) if scale is None else scale, lp, op, os_)

    def select(self, q, plan, lists, sinks=0, window=1, stream=None):
        """lists [n, n_kv_heads, plan.list_blocks]: the first `sinks` blocks of each
        sequence, its last `window` and the best of those between by mean key, in
        ascending order, -1 behind them."""
        qp, qt, qs = _rows(q, plan._shape, self.index, "q")
        lp = _ints(lists, plan._lists, self.index, "lists")
        if not (-2 ** 31 <= sinks < 2 ** 31 and -2 ** 31 <= window < 2 ** 31):
            raise ValueError("sinks and window: counts within 32 bits are needed")
        self.on.call("vireo_paged_select", stream, (q, lists), (self, plan, plan.table), self._p, self._plan(plan),
                     qp, qt, qs, sinks, window, lp)
