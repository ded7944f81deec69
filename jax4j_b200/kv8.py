"""8-bit paged KV cache on the engine: e4m3 codes with one power-of-two scale for each block of 16
tokens and head, in pages that sequences name through a page table.

`Kv8Cache` holds the pages of every layer and runs the engine's operators on them: `append` (RoPE
and quantisation of new tokens), `attention_decode` (one query per sequence), `attention_prefill`
(ragged causal chunks) and `copy_pages`. Attention takes grouped heads and a sliding window with
first tokens that stay visible. `PageTable` is the host's bookkeeping for it: which pages a
sequence has, shared pages of forks, freed pages, compaction.

Launches go to PyTorch's current stream of the cache's device; outputs and the decode workspace
come from its allocator on that stream. The reference has no KV cache; the functions are stated in
include/jax4j_b200.h.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import BF16, F32, call
from .backend import torch_stream

BLOCK = 16  # tokens that share a scale
_TYPES = {torch.float32: F32, torch.bfloat16: BF16}


def rope_table(positions: int, head_dim: int, theta: float = 10000.0, device=None) -> torch.Tensor:
    """(cos, sin) of pos * theta^(-2i / head_dim), angles formed in float64: f32 [positions, head_dim / 2, 2]."""
    freq = theta ** (-torch.arange(0, head_dim, 2, dtype=torch.float64, device=device) / head_dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.stack((angle.cos(), angle.sin()), -1).float()


def _type(t: torch.Tensor, what: str) -> int:
    if t.dtype not in _TYPES:
        raise ValueError(f"{what} must be float32 or bfloat16, got {t.dtype}")
    return _TYPES[t.dtype]


def _rows(t: torch.Tensor, what: str) -> int:
    """Row stride of a tensor [rows, heads, dim] (or [rows, width]) whose rows are dense."""
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
        self._desc = _lib.Kv8CacheDesc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), layers, pages, kv_heads, page, dim)
        self._ref = ctypes.byref(self._desc)
        self._workspace = {}  # (heads, batch) -> bytes

    def _ints(self, t: torch.Tensor, what: str, shape: tuple) -> int:
        if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != self.device:
            raise ValueError(f"{what} must be a contiguous int32 tensor {shape} on {self.device}")
        return t.data_ptr()

    def _table(self, table: torch.Tensor) -> tuple:
        if table.dtype != torch.int32 or table.dim() != 2 or table.device != self.device or (table.shape[1] > 1 and table.stride(1) != 1):
            raise ValueError(f"the page table must be an int32 tensor [batch, pages of a sequence] on {self.device}, dense within a row")
        return table.data_ptr(), table.stride(0) if table.shape[0] > 1 else table.shape[1], table.shape[1]

    def _queries(self, q: torch.Tensor, out: torch.Tensor | None, out_dtype, scale) -> tuple:
        if q.dim() != 3 or q.shape[2] != self.head_dim or q.device != self.device:
            raise ValueError(f"q must be [rows, heads, {self.head_dim}] on {self.device}, got {tuple(q.shape)}")
        if out is None:
            out = torch.empty(q.shape, dtype=out_dtype or q.dtype, device=self.device)
        elif out.shape != q.shape or not out.is_contiguous() or out.device != self.device:
            raise ValueError("out must be contiguous and of q's shape and device")
        return out, self.head_dim ** -0.5 if scale is None else float(scale)

    def append(self, qkv: torch.Tensor, rope: torch.Tensor, table: torch.Tensor, starts: torch.Tensor, heads: int,
               offsets: torch.Tensor | None = None, layer: int = 0, q_dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """Rotates the queries and keys of new tokens and writes keys and values into their pages.

        qkv f32 [tokens, (heads + 2 kv_heads) * head_dim] (q | k | v); sequence b's rows are
        offsets[b] .. offsets[b + 1] - 1 (no offsets: row b alone) and go to positions starts[b], ...;
        rope f32 [positions, head_dim / 2, 2] (`rope_table`). Returns the rotated queries
        [tokens, heads, head_dim]."""
        if qkv.dim() != 2 or qkv.dtype != torch.float32 or qkv.shape[1] != (heads + 2 * self.kv_heads) * self.head_dim or qkv.device != self.device:
            raise ValueError(f"qkv must be float32 [tokens, {(heads + 2 * self.kv_heads) * self.head_dim}] on {self.device}")
        if rope.dim() != 3 or rope.dtype != torch.float32 or tuple(rope.shape[1:]) != (self.head_dim // 2, 2) or not rope.is_contiguous() or rope.device != self.device:
            raise ValueError(f"rope must be a contiguous float32 tensor [positions, {self.head_dim // 2}, 2] on {self.device}")
        if q_dtype not in _TYPES:
            raise ValueError(f"q must be float32 or bfloat16, got {q_dtype}")
        tokens, batch = qkv.shape[0], table.shape[0]
        at, stride, width = self._table(table)
        q = torch.empty(tokens, heads, self.head_dim, dtype=q_dtype, device=self.device)
        call("j4b_kv8_append", self._ref, layer, qkv.data_ptr(), _rows(qkv, "qkv"), tokens, heads, rope.data_ptr(), rope.shape[0], at, stride,
             width, self._ints(starts, "starts", (batch,)), 0 if offsets is None else self._ints(offsets, "offsets", (batch + 1,)), batch,
             q.data_ptr(), _TYPES[q_dtype], torch_stream(self.device))
        return q

    def attention_decode(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, window: int = 0, sinks: int = 0,
                         scale: float | None = None, layer: int = 0, out: torch.Tensor | None = None,
                         out_dtype: torch.dtype | None = None) -> torch.Tensor:
        """softmax(scale q k^T) v of one query per sequence, q [batch, heads, head_dim], at position
        lengths[b] - 1 over its cached tokens (with window > 0: the last `window` and the first
        `sinks`). Sequences that see nothing give zeros."""
        batch, heads = table.shape[0], q.shape[1] if q.dim() == 3 else 0
        out, scale = self._queries(q, out, out_dtype, scale)
        if q.shape[0] != batch:
            raise ValueError(f"q has {q.shape[0]} rows for {batch} sequences")
        at, stride, width = self._table(table)
        if (heads, batch) not in self._workspace:
            n = ctypes.c_int64()
            call("j4b_kv8_decode_workspace", self._ref, heads, batch, ctypes.byref(n))
            self._workspace[heads, batch] = n.value
        n = self._workspace[heads, batch]
        work = torch.empty(n, dtype=torch.uint8, device=self.device)
        call("j4b_kv8_attention_decode", self._ref, layer, q.data_ptr(), _type(q, "q"), _rows(q, "q"), heads, at, stride, width,
             self._ints(lengths, "lengths", (batch,)), batch, window, sinks, scale, out.data_ptr(), _type(out, "out"), work.data_ptr(), n,
             torch_stream(self.device))
        return out

    def attention_prefill(self, q: torch.Tensor, offsets: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, window: int = 0,
                          sinks: int = 0, scale: float | None = None, layer: int = 0, out: torch.Tensor | None = None,
                          out_dtype: torch.dtype | None = None) -> torch.Tensor:
        """Causal attention of ragged chunks: sequence b's queries, the rows offsets[b] ..
        offsets[b + 1] - 1 of q [tokens, heads, head_dim], are its last tokens (lengths[b] counts
        them). Window, sinks and empty rows as in attention_decode."""
        batch, heads = table.shape[0], q.shape[1] if q.dim() == 3 else 0
        out, scale = self._queries(q, out, out_dtype, scale)
        at, stride, width = self._table(table)
        call("j4b_kv8_attention_prefill", self._ref, layer, q.data_ptr(), _type(q, "q"), _rows(q, "q"), q.shape[0], heads,
             self._ints(offsets, "offsets", (batch + 1,)), at, stride, width, self._ints(lengths, "lengths", (batch,)), batch, window, sinks,
             scale, out.data_ptr(), _type(out, "out"), torch_stream(self.device))
        return out

    def copy_pages(self, src: list, dst: list, tokens: list | None = None) -> None:
        """Copies the blocks that hold the first tokens[i] tokens (default: all) of page src[i] to
        page dst[i], in every layer. The lists are host integers; no page may be written twice, or
        read and written."""
        n = len(src)
        if len(dst) != n or (tokens is not None and len(tokens) != n):
            raise ValueError("src, dst and tokens must have one entry per move")
        ints = ctypes.c_int32 * n
        call("j4b_kv8_copy_pages", self._ref, n, ints(*src), ints(*dst), None if tokens is None else ints(*tokens), torch_stream(self.device))
