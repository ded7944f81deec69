"""8-bit paged KV cache on the engine: e4m3 codes with one power-of-two scale for each block of 16
tokens and head, in pages that sequences name through a page table.

`Kv8Cache` holds the pages of every layer and runs the engine's operators on them: `append` (RoPE
and quantisation of new tokens), `attention_decode` (one query per sequence), `attention_prefill`
(ragged causal chunks) and `copy_pages`. Attention takes grouped heads and a sliding window with
first tokens that stay visible. `PageTable` is the host's bookkeeping for it: which pages a
sequence has, shared pages of forks, freed pages, compaction.

Launches go to PyTorch's current stream of the cache's device; outputs come from its allocator on
that stream, and the decode workspace is kept, one per stream; threads may share a cache and a
stream. The reference has no KV cache; the functions are stated in include/jax4j_b200.h.
"""
from __future__ import annotations

import ctypes
import heapq
import threading
from array import array

import torch

from . import _lib
from ._lib import BF16, F32, call
from .backend import CUDA_STREAM_LEGACY

BLOCK = 16  # tokens that share a scale
_TYPES = {torch.float32: F32, torch.bfloat16: BF16}


def rope_table(positions: int, head_dim: int, theta: float = 10000.0, device=None) -> torch.Tensor:
    """(cos, sin) of pos * theta^(-2i / head_dim), angles formed in float64: f32 [positions, head_dim / 2, 2]."""
    freq = theta ** (-torch.arange(0, head_dim, 2, dtype=torch.float64, device=device) / head_dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.stack((angle.cos(), angle.sin()), -1).float()


def _rows(t: torch.Tensor, what: str) -> int:
    """Row stride of a tensor [rows, heads, dim] (or [rows, width]) whose rows are dense."""
    if t.is_contiguous() and t.shape[0] > 1:  # the stride of a row alone may be anything
        return t.stride(0)
    inner = 1
    for size, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        if size != 1 and stride != inner:
            raise ValueError(f"{what} must be dense within a row")
        inner *= size
    return t.stride(0) if t.shape[0] > 1 else inner


class Kv8Cache:
    """Pages of `layers` layers: codes k, v float8_e4m3fn [layers, pages, kv_heads, page, head_dim],
    scales k_scale, v_scale float32 [layers, pages, kv_heads, page / 16]."""

    def __init__(self, pages: int, kv_heads: int, page: int = 64, head_dim: int = 128, layers: int = 1, device=0):
        dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        codes, scales = (layers, pages, kv_heads, page, head_dim), (layers, pages, kv_heads, page // BLOCK)
        self._set(*(torch.zeros(codes, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn) for _ in range(2)),
                  *(torch.zeros(scales, dtype=torch.float32, device=dev) for _ in range(2)))

    @classmethod
    def wrap(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> "Kv8Cache":
        """A cache over tensors that the caller made (shapes above, contiguous)."""
        cache = cls.__new__(cls)
        cache._set(k, v, k_scale, v_scale)
        return cache

    def _set(self, k, v, k_scale, v_scale) -> None:
        if k.dim() != 5 or k.shape != v.shape or k.dtype != torch.float8_e4m3fn or v.dtype != k.dtype:
            raise ValueError("codes must be two float8_e4m3fn tensors [layers, pages, kv_heads, page, head_dim]")
        layers, pages, kv_heads, page, dim = k.shape
        if page % BLOCK or page == 0:
            raise ValueError(f"page must be a positive multiple of {BLOCK}, got {page}")
        if dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {dim}")
        want = (layers, pages, kv_heads, page // BLOCK)
        if tuple(k_scale.shape) != want or tuple(v_scale.shape) != want or k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise ValueError(f"scales must be two float32 tensors {want}")
        for t in (k, v, k_scale, v_scale):
            if not t.is_contiguous() or t.device != k.device:
                raise ValueError("codes and scales must be contiguous and on one device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.layers, self.pages, self.kv_heads, self.page, self.head_dim = layers, pages, kv_heads, page, dim
        self.device = k.device
        self._index = k.device.index if k.device.type == "cuda" else -1
        self._need = {}  # (heads, batch) -> bytes of the decode workspace
        self._work = {}  # stream -> workspace
        self._lock = threading.Lock()  # of the two
        self._desc = _lib.Kv8CacheDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), layers, pages, kv_heads, page, dim)
        self._ref = ctypes.byref(self._desc)

    def _ints(self, t: torch.Tensor, what: str, n: int) -> int:
        if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != n or t.get_device() != self._index or not t.is_contiguous():
            raise ValueError(f"{what} must be a contiguous int32 tensor ({n},) on {self.device}")
        return t.data_ptr()

    def _table(self, table: torch.Tensor) -> tuple:
        shape, strides = table.shape, table.stride()
        if len(shape) != 2 or table.dtype is not torch.int32 or table.get_device() != self._index or (strides[1] != 1 and shape[1] > 1):
            raise ValueError(f"the page table must be an int32 tensor [batch, pages of a sequence] on {self.device}, dense within a row")
        batch, width = shape
        return table.data_ptr(), strides[0] if batch > 1 else width, batch, width

    def _queries(self, q: torch.Tensor, out: torch.Tensor | None, out_dtype) -> torch.Tensor:
        if q.dim() != 3 or q.shape[2] != self.head_dim or q.get_device() != self._index:
            raise ValueError(f"q must be [rows, heads, {self.head_dim}] on {self.device}, got {tuple(q.shape)}")
        if q.dtype not in _TYPES or (out_dtype is not None and out_dtype not in _TYPES):
            raise ValueError(f"q and the output must be float32 or bfloat16, got {q.dtype} and {out_dtype or q.dtype}")
        if out is None:
            same = (out_dtype is None or out_dtype is q.dtype) and q.is_contiguous()
            return torch.empty_like(q) if same else q.new_empty(q.shape, dtype=out_dtype)  # the former takes half the time
        if out.shape != q.shape or not out.is_contiguous() or out.get_device() != self._index or out.dtype not in _TYPES:
            raise ValueError("out must be contiguous, float32 or bfloat16, and of q's shape and device")
        return out

    def _stream(self) -> int:
        """The current stream, as backend.torch_stream gives it."""
        return torch._C._cuda_getCurrentRawStream(self._index) or CUDA_STREAM_LEGACY

    def _workspace(self, heads: int, batch: int, stream: int) -> torch.Tensor:
        """Of a decode call. One per stream, since calls on different streams may run at the same time;
        a graph gets one of its own, which lives as long as the graph's memory."""
        need = self._need.get((heads, batch))
        if need is None:
            n = ctypes.c_int64()
            call("j4b_kv8_decode_workspace", self._ref, heads, batch, ctypes.byref(n))
            need = self._need[heads, batch] = n.value
        if torch._C._cuda_isCurrentStreamCapturing():
            return torch.empty(need, dtype=torch.uint8, device=self.device)
        work = self._work.get(stream)
        if work is None or work.shape[0] < need:
            work = self._work[stream] = torch.empty(need, dtype=torch.uint8, device=self.device)
        return work

    def append(self, qkv: torch.Tensor, rope: torch.Tensor, table: torch.Tensor, starts: torch.Tensor, heads: int,
               offsets: torch.Tensor | None = None, layer: int = 0, q_dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """Rotates the queries and keys of new tokens and writes keys and values into their pages.

        qkv f32 [tokens, (heads + 2 kv_heads) * head_dim] (q | k | v); sequence b's rows are
        offsets[b] .. offsets[b + 1] - 1 (no offsets: row b alone) and go to positions starts[b], ...;
        rope f32 [positions, head_dim / 2, 2] (`rope_table`). Returns the rotated queries
        [tokens, heads, head_dim]."""
        if qkv.dim() != 2 or qkv.dtype != torch.float32 or qkv.shape[1] != (heads + 2 * self.kv_heads) * self.head_dim or qkv.get_device() != self._index:
            raise ValueError(f"qkv must be float32 [tokens, {(heads + 2 * self.kv_heads) * self.head_dim}] on {self.device}")
        if rope.dim() != 3 or rope.dtype != torch.float32 or rope.shape[1] != self.head_dim // 2 or rope.shape[2] != 2 or not rope.is_contiguous() or rope.get_device() != self._index:
            raise ValueError(f"rope must be a contiguous float32 tensor [positions, {self.head_dim // 2}, 2] on {self.device}")
        if q_dtype not in _TYPES:
            raise ValueError(f"q must be float32 or bfloat16, got {q_dtype}")
        at, stride, batch, width = self._table(table)
        tokens = qkv.shape[0]
        if q_dtype is torch.float32:
            q = qkv.new_empty((tokens, heads, self.head_dim))
        else:
            q = qkv.new_empty((tokens, heads, self.head_dim), dtype=q_dtype)
        call("j4b_kv8_append", self._ref, layer, qkv.data_ptr(), _rows(qkv, "qkv"), tokens, heads, rope.data_ptr(), rope.shape[0], at, stride,
             width, self._ints(starts, "starts", batch), 0 if offsets is None else self._ints(offsets, "offsets", batch + 1), batch,
             q.data_ptr(), _TYPES[q_dtype], self._stream())
        return q

    def attention_decode(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, window: int = 0, sinks: int = 0,
                         scale: float | None = None, layer: int = 0, out: torch.Tensor | None = None,
                         out_dtype: torch.dtype | None = None) -> torch.Tensor:
        """softmax(scale q k^T) v of one query per sequence, q [batch, heads, head_dim], at position
        lengths[b] - 1 over its cached tokens (with window > 0: the last `window` and the first
        `sinks`). Sequences that see nothing give zeros."""
        out = self._queries(q, out, out_dtype)
        at, stride, batch, width = self._table(table)
        rows, heads, _ = q.shape
        if rows != batch:
            raise ValueError(f"q has {rows} rows for {batch} sequences")
        stream = self._stream()
        # A call may be two launches that share the workspace. ctypes runs it without the interpreter's
        # lock, so another thread's call on the same stream could come between them.
        with self._lock:
            work = self._workspace(heads, batch, stream)
            call("j4b_kv8_attention_decode", self._ref, layer, q.data_ptr(), _TYPES[q.dtype], _rows(q, "q"), heads, at, stride, width,
                 self._ints(lengths, "lengths", batch), batch, window, sinks, self.head_dim ** -0.5 if scale is None else scale,
                 out.data_ptr(), _TYPES[out.dtype], work.data_ptr(), work.shape[0], stream)
        return out

    def attention_prefill(self, q: torch.Tensor, offsets: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, window: int = 0,
                          sinks: int = 0, scale: float | None = None, layer: int = 0, out: torch.Tensor | None = None,
                          out_dtype: torch.dtype | None = None) -> torch.Tensor:
        """Causal attention of ragged chunks: sequence b's queries, the rows offsets[b] ..
        offsets[b + 1] - 1 of q [tokens, heads, head_dim], are its last tokens (lengths[b] counts
        them). Window, sinks and empty rows as in attention_decode."""
        out = self._queries(q, out, out_dtype)
        at, stride, batch, width = self._table(table)
        rows, heads, _ = q.shape
        call("j4b_kv8_attention_prefill", self._ref, layer, q.data_ptr(), _TYPES[q.dtype], _rows(q, "q"), rows, heads,
             self._ints(offsets, "offsets", batch + 1), at, stride, width, self._ints(lengths, "lengths", batch), batch, window, sinks,
             self.head_dim ** -0.5 if scale is None else scale, out.data_ptr(), _TYPES[out.dtype], self._stream())
        return out

    def copy_pages(self, src: list, dst: list, tokens: list | None = None) -> None:
        """Copies the blocks that hold the first tokens[i] tokens (default: all) of page src[i] to
        page dst[i], in every layer. The lists are host integers; no page may be written twice, or
        read and written."""
        n = len(src)
        if len(dst) != n or (tokens is not None and len(tokens) != n):
            raise ValueError("src, dst and tokens must have one entry per move")
        try:  # ctypes would take what 32 bits hold of a number
            lists = [None if x is None else (ctypes.c_int32 * n).from_buffer(array("i", x)) for x in (src, dst, tokens)]
        except OverflowError:
            raise ValueError("pages and tokens must be numbers of 32 bits") from None
        call("j4b_kv8_copy_pages", self._ref, n, *lists, self._stream())


class PageTable:
    """The host's bookkeeping of a `Kv8Cache`: `slots` sequences of up to `max_tokens` tokens (counted from
    their first one, under a window too), each a list of pages in token order. Full pages of a fork are shared (counted), its partly filled last page
    is copied. The device sees it through `table` (int32 [slots, pages of a sequence], -1: none),
    one tensor, which a read of the attribute and `extend` bring up to date on the current stream, and
    the arrays that `extend` returns."""

    def __init__(self, cache: Kv8Cache, slots: int, max_tokens: int):
        if slots <= 0 or max_tokens <= 0:
            raise ValueError("slots and max_tokens must be positive")
        self.cache, self.slots = cache, slots
        self.width = -(-max_tokens // cache.page)
        self.pages = [[] for _ in range(slots)]  # -1: freed by trim
        self.lengths = [0] * slots
        self.refs = [0] * cache.pages
        self._free = list(range(cache.pages))  # a heap: the lowest page first, so what is in use stays low
        self._table = torch.full((slots, self.width), -1, dtype=torch.int32, device=cache.device)
        self._dirty = False
        self._ropes = {}  # theta -> table
        # of the last extend, for a model's other layers: what it returned, (starts, lengths) of decode's
        # rows, one a slot, and what it was given
        self.step = self.rows = self.counts = None

    def _slot(self, slot: int) -> int:
        if not 0 <= slot < self.slots:
            raise ValueError(f"slot {slot} outside [0, {self.slots})")
        return slot

    def _take(self, n: int) -> list:
        if n > len(self._free):
            raise MemoryError(f"{n} pages are needed and {len(self._free)} are free")
        got = [heapq.heappop(self._free) for _ in range(n)]
        for p in got:
            self.refs[p] = 1
        return got

    def _drop(self, page: int) -> None:
        if page < 0:
            return
        self.refs[page] -= 1
        if self.refs[page] == 0:
            heapq.heappush(self._free, page)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def extend(self, counts: list) -> tuple:
        """Room for counts[slot] new tokens in each slot. Returns device int32 arrays (starts, lengths,
        offsets): where each slot's new tokens begin, its length with them, and the rows of the new
        tokens, slot by slot. Raises MemoryError, changing nothing, where pages do not suffice."""
        if len(counts) != self.slots or any(n < 0 for n in counts):
            raise ValueError(f"one count for each of {self.slots} slots, none negative")
        page = self.cache.page
        need = [max(0, -(-(m + n) // page) - len(p)) for m, n, p in zip(self.lengths, counts, self.pages)]
        for slot, (m, n) in enumerate(zip(self.lengths, counts)):
            if m + n > self.width * page:
                raise ValueError(f"slot {slot} holds at most {self.width * page} tokens, {m} + {n} asked for")
        fresh = self._take(sum(need))
        starts = list(self.lengths)
        for slot, n in enumerate(need):
            if n:
                self.pages[slot] += fresh[:n]
                del fresh[:n]
                self._dirty = True
            self.lengths[slot] += counts[slot]
        self._upload()
        offsets = [0]
        for n in counts:
            offsets.append(offsets[-1] + n)
        # for a row each of decode: slots without a new token start nowhere and see nothing
        busy = [(m, n) if k else (-1, 0) for m, n, k in zip(starts, self.lengths, counts)]
        rows = [m for m, _ in busy] + [n for _, n in busy]
        packed = torch.tensor(starts + self.lengths + rows + offsets, dtype=torch.int32).to(self.cache.device)
        starts, lengths, *rows, offsets = packed.split([self.slots] * 4 + [self.slots + 1])
        self.step, self.rows, self.counts = (starts, lengths, offsets), tuple(rows), list(counts)
        return self.step

    def _upload(self) -> None:
        if self._dirty:
            rows = [p + [-1] * (self.width - len(p)) for p in self.pages]
            self._table.copy_(torch.tensor(rows, dtype=torch.int32))
            self._dirty = False

    @property
    def table(self) -> torch.Tensor:
        self._upload()
        return self._table

    def rope(self, theta: float = 10000.0) -> torch.Tensor:
        """The `rope_table` of all positions that a slot can have, made once for all layers."""
        if theta not in self._ropes:
            self._ropes[theta] = rope_table(self.width * self.cache.page, self.cache.head_dim, theta, self.cache.device)
        return self._ropes[theta]

    def release(self, slot: int) -> None:
        """Ends a slot's sequence: its pages that no other shares are free again."""
        for p in self.pages[self._slot(slot)]:
            self._drop(p)
        self.pages[slot], self.lengths[slot], self._dirty = [], 0, True
        self.step = self.rows = self.counts = None

    def trim(self, window: int, sinks: int = 0) -> int:
        """Frees the pages that no later query sees under a window with sinks; returns how many."""
        if window <= 0 or sinks < 0:
            raise ValueError("trim needs a positive window and no negative sinks")
        page, freed = self.cache.page, len(self._free)
        for slot in range(self.slots):
            first = self.lengths[slot] - window + 1  # of the next query's window
            for i in range(-(-sinks // page), max(0, first) // page):
                if self.pages[slot][i] >= 0:
                    self._drop(self.pages[slot][i])
                    self.pages[slot][i] = -1
                    self._dirty = True
        return len(self._free) - freed

    def fork(self, parent: int, children: list) -> None:
        """Makes each child (a slot without a sequence) a copy of the parent's sequence: full pages are
        shared, the partly filled last one is copied, in every layer, by one call."""
        self._slot(parent)
        for c in children:
            if self.pages[self._slot(c)] or c == parent:
                raise ValueError(f"slot {c} is in use")
        if len(set(children)) != len(children):
            raise ValueError("a slot is named twice")
        rest = self.lengths[parent] % self.cache.page
        shared, last = (self.pages[parent][:-1], self.pages[parent][-1]) if rest else (self.pages[parent], -1)
        fresh = self._take(len(children)) if last >= 0 else []
        if fresh:
            try:
                self.cache.copy_pages([last] * len(children), fresh, [rest] * len(children))
            except BaseException:
                for p in fresh:
                    self._drop(p)
                raise
        for i, c in enumerate(children):
            for p in shared:
                if p >= 0:
                    self.refs[p] += 1
            self.pages[c] = list(shared) + ([fresh[i]] if last >= 0 else [])
            self.lengths[c] = self.lengths[parent]
        self._dirty = True
        self.step = self.rows = self.counts = None

    def compact(self) -> int:
        """Moves pages so that the ones in use are the lowest (a pool that can then be cut, or saved
        whole); returns how many moved."""
        used = sum(r > 0 for r in self.refs)
        src = [p for p in range(used, self.cache.pages) if self.refs[p] > 0]
        dst = [p for p in range(used) if self.refs[p] == 0]
        if src:
            self.cache.copy_pages(src, dst)
            to = dict(zip(src, dst))
            self.pages = [[to.get(p, p) for p in pages] for pages in self.pages]
            for a, b in to.items():
                self.refs[b], self.refs[a] = self.refs[a], 0
            self._free = list(range(used, self.cache.pages))  # ascending: a heap
            self._dirty = True
        return len(src)
