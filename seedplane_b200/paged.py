"""K / V in pages that requests share: the append of a pass's keys and values (with the position rotation
on the way) and attention of a batch over a shared prefix and each request's own pages.

The reference keeps one contiguous cache per session (`seedplane/qwen_engine.py:18-29`) and decodes
requests one at a time (`README.md:67-68`); here many requests can start from the same pages, and the
attention of a batch reads those once. Three pieces:

* `PagedKV`: the pages of every layer, [layers][n_pages][kv_heads][page_size][head_dim] for K and for V;
* `PageBatch`: which rows of a call belong to which request, how many keys each request has, its pages,
  and the prefix all of them start with;
* `append` and `attention` (`sp_pages_append`, `sp_pages_attention`), which the engine's passes over pages
  (`CudaQwen2.forward_pages`, `decode_pages`, `batch.generate_shared`) run for every layer.

All of a batch's arrays are device memory that the kernels read, so a CUDA graph captured over them serves
their later contents. PyTorch only holds memory and streams. The kernels never trap: a bad page number,
length or position is recorded and raised by `PagedKV.status`.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch

from . import _native as N

# the current stream's handle by device index, without a Stream object around it
_raw_stream = torch._C._cuda_getCurrentRawStream
# The checks below cost as much as a small call's kernels: the common case of each is tested first, in few steps.
_TYPES = {torch.float32: N.SP_F32, torch.float16: N.SP_F16, torch.bfloat16: N.SP_BF16}


def _int32(t: torch.Tensor, name: str, device, dim: int) -> torch.Tensor:
    if t.dtype != torch.int32 or t.device != device or t.dim() != dim or (t.numel() > 0 and t.stride(-1) != 1):
        raise ValueError(f"{name}: int32 with {dim} dimension(s) on {device}, unit stride in the last, expected")
    return t


class PagedKV:
    """The pages of `layers` layers on one device. K and V are zeroed; `k`, `v` are the tensors."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, n_pages: int, page_size: int = 64,
                 dtype: torch.dtype = torch.float16, device="cuda"):
        shape = (layers, n_pages, kv_heads, page_size, head_dim)
        self._set(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))

    @classmethod
    def wrap(cls, k: torch.Tensor, v: torch.Tensor) -> "PagedKV":
        """Pages in the caller's tensors, [layers][n_pages][kv_heads][page_size][head_dim] or one layer's
        [n_pages][kv_heads][page_size][head_dim]; any strides that are multiples of 8, the last 1 (the
        same for both)."""
        self = cls.__new__(cls)
        self._set(k, v)
        return self

    def _set(self, k, v):
        if k.dim() == 4:
            k, v = k[None], v[None]
        if k.dim() != 5 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.device != v.device:
            raise ValueError("K and V pages must be alike: [layers][n_pages][kv_heads][page_size][head_dim]")
        if k.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("pages are fp16 or bf16")
        if not k.is_cuda or (k.numel() > 0 and k.stride(4) != 1):
            raise ValueError("pages must be CUDA tensors with unit stride in the last dimension")
        self.k, self.v, self.device = k, v, k.device
        self._index = k.get_device()
        self.layers, self.n_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self._word = torch.zeros(1, dtype=torch.int32, device=k.device)
        self._layer = []
        for i in range(self.layers):
            self._layer.append(N.SpPages(
                k_dev=k[i].data_ptr(), v_dev=v[i].data_ptr(), page_stride=k.stride(1), head_stride=k.stride(2),
                slot_stride=k.stride(3), n_pages=self.n_pages, page_size=self.page_size, kv_heads=self.kv_heads,
                head_dim=self.head_dim, dtype=_TYPES[k.dtype], status_dev=self._word.data_ptr()))
        self.layer_array = (N.SpPages * self.layers)(*self._layer)
        self._ref = [C.byref(c) for c in self._layer]
        # what a workspace's size depends on
        self._key = (self.n_pages, self.page_size, self.kv_heads, self.head_dim, k.dtype, k.stride()[1:])

    def status(self):
        """Raise if a kernel met a bad page number, length or position since the last check (waits
        for the current stream)."""
        bad = int(self._word.item())
        if bad:
            self._word.zero_()
            raise N.EngineError(N.SP_ERR_DEVICE, f"device error {bad}: page, length or position outside its table")


class PageBatch:
    """A ragged batch (`sp_page_batch`): request b's rows are q_start[b] .. q_start[b + 1] - 1 (None: max_q
    rows each), it has lens[b] own keys, these rows' among them, in the pages tables[b], and sees
    `prefix_len` keys in the pages `prefix_table` before them. `tokens` and `max_q` bound the rows of a call
    and of one request from above."""

    def __init__(self, tables: torch.Tensor, lens: torch.Tensor, *, q_start: Optional[torch.Tensor] = None,
                 tokens: Optional[int] = None, max_q: int = 1, prefix_table: Optional[torch.Tensor] = None,
                 prefix_len: int = 0):
        dev = lens.device
        self.device, self._index = dev, lens.get_device()
        self.lens = _int32(lens, "lens", dev, 1)
        self.tables = _int32(tables, "tables", dev, 2)
        b = lens.numel()
        if tables.shape[0] != b:
            raise ValueError(f"{tables.shape[0]} tables for {b} requests")
        if q_start is not None and _int32(q_start, "q_start", dev, 1).numel() != b + 1:
            raise ValueError(f"q_start of {q_start.numel()} entries for {b} requests")
        if tokens is None:
            if q_start is not None:
                raise ValueError("q_start needs `tokens`, the rows of a call at most")
            tokens = b * max_q
        self.q_start, self.prefix_table = q_start, prefix_table
        if prefix_table is not None:
            _int32(prefix_table, "prefix_table", dev, 1)
        self.prefix_pages = 0 if prefix_table is None else prefix_table.numel()
        self.batch, self.tokens, self.max_q, self.prefix_len = b, int(tokens), int(max_q), int(prefix_len)
        self._c = N.SpPageBatch(
            batch=b, tokens=self.tokens, max_q=self.max_q, q_start_dev=None if q_start is None else q_start.data_ptr(),
            lens_dev=lens.data_ptr(), tables_dev=tables.data_ptr(), table_stride=tables.stride(0) if b > 1 else tables.shape[1],
            table_width=tables.shape[1], prefix_dev=None if prefix_table is None else prefix_table.data_ptr(),
            prefix_len=self.prefix_len)
        self._ref = C.byref(self._c)
        self._ws = {}                          # workspace bytes by (pages' sizes, heads, type)

    def _check(self, pages: PagedKV, layer: int):
        if not 0 <= layer < pages.layers:
            raise ValueError(f"layer {layer} of {pages.layers}")
        if pages._index != self._index:
            raise ValueError(f"pages on {pages.device}, batch on {self.device}")
        if self.prefix_len > self.prefix_pages * pages.page_size:
            raise ValueError(f"a prefix of {self.prefix_len} keys in {self.prefix_pages} pages of {pages.page_size}")


def _rows(t: torch.Tensor, name: str, batch: PageBatch, cols: int) -> int:
    """The row stride of a [rows, ...] matrix of `cols` values a row (heads and dims contiguous)."""
    if t.get_device() != batch._index or t.dtype not in _TYPES:
        raise ValueError(f"{name}: fp32, fp16 or bf16 on {batch.device} expected")
    if t.dim() < 2 or t.size(0) < batch.tokens or t.numel() != t.size(0) * cols:
        raise ValueError(f"{name}: [{batch.tokens}, {cols}] expected, not {tuple(t.shape)}")
    if t.is_contiguous():
        return cols
    if t.numel() > 0 and (t.stride(-1) != 1 or (t.dim() == 3 and t.size(1) > 1 and t.stride(1) != t.size(2)) or t.dim() > 3):
        raise ValueError(f"{name}: the values of a row must be contiguous")
    return t.stride(0) if t.size(0) > 1 else cols


def append(pages: PagedKV, layer: int, batch: PageBatch, qkv: torch.Tensor, heads: int, rope: torch.Tensor, *,
           bias: Optional[torch.Tensor] = None, interleaved: bool = False, positions: Optional[torch.Tensor] = None,
           q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Keys and values of a pass into their pages (`sp_pages_append`): qkv [tokens, (heads + 2 kv_heads)
    * head_dim] in the fused q | k | v order, plus `bias` (fp32); the first rot_dim dims of every q and k
    head rotated by `rope` (fp32 [positions, rot_dim / 2, 2] of cos, sin; `engine.rope_table`'s layout) at
    `positions` (int32 [tokens]; None: prefix_len + own key). Returns q [tokens, heads, head_dim] in
    qkv's type (fp32 rows into bf16 pages: round it to bf16 for `attention`)."""
    hd = pages.head_dim
    batch._check(pages, layer)
    cols = (heads + 2 * pages.kv_heads) * hd
    xs = _rows(qkv, "qkv", batch, cols)
    if q_out is None:
        q_out = torch.empty((qkv.shape[0], heads, hd), dtype=qkv.dtype, device=batch.device)
    qs = _rows(q_out, "q_out", batch, heads * hd)
    if q_out.dtype != qkv.dtype:
        raise ValueError("q_out must have qkv's type")
    if rope.dtype != torch.float32 or rope.get_device() != batch._index or rope.dim() != 3 or rope.size(2) != 2 or \
            not rope.is_contiguous():
        raise ValueError("rope: contiguous fp32 [positions, rot_dim / 2, 2] expected")
    if bias is not None and (bias.dtype != torch.float32 or bias.get_device() != batch._index or bias.numel() != cols or
                             not bias.is_contiguous()):
        raise ValueError(f"bias: contiguous fp32 [{cols}] expected")
    if positions is not None and _int32(positions, "positions", batch.device, 1).numel() < batch.tokens:
        raise ValueError(f"positions: {batch.tokens} entries expected")
    N.check(N.load().sp_pages_append(
        batch._index, pages._ref[layer], batch._ref, heads, qkv.data_ptr(), _TYPES[qkv.dtype], xs,
        None if bias is None else bias.data_ptr(), rope.data_ptr(), rope.size(0), 2 * rope.size(1), int(interleaved),
        None if positions is None else positions.data_ptr(), q_out.data_ptr(), qs, _raw_stream(batch._index)))
    return q_out


def attention(pages: PagedKV, layer: int, batch: PageBatch, q: torch.Tensor, *, scale: Optional[float] = None,
              out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale * q K) V of every row over the shared prefix and the row's request's own keys up to its
    own (`sp_pages_attention`). q [tokens, heads, head_dim]: fp32 over fp16 pages, or the pages' type;
    scale: default 1 / sqrt(head_dim); lse: fp32 [tokens, heads] that receives the log-sum-exps. Returns
    out, in q's shape and type. The workspace is allocated here, on the current stream."""
    batch._check(pages, layer)
    if q.dim() != 3 or q.size(2) != pages.head_dim:
        raise ValueError(f"q: [{batch.tokens}, heads, {pages.head_dim}] expected, not {tuple(q.shape)}")
    heads = q.size(1)
    qs = _rows(q, "q", batch, heads * pages.head_dim)
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    os_ = _rows(out, "out", batch, heads * pages.head_dim)
    if out.dtype != q.dtype:
        raise ValueError("out must have q's type")
    if lse is not None and (lse.dtype != torch.float32 or lse.get_device() != batch._index or lse.shape != (q.size(0), heads) or
                            not lse.is_contiguous()):
        raise ValueError(f"lse: contiguous fp32 [{q.shape[0]}, {heads}] expected")
    lib, c, dt = N.load(), pages._ref[layer], _TYPES[q.dtype]
    key = (pages._key, heads, dt)
    need = batch._ws.get(key)
    if need is None:
        need = lib.sp_pages_attention_workspace(c, batch._ref, heads, dt)
        if need < 0:
            N.check(need)
        batch._ws[key] = need
    ws = torch.empty(need, dtype=torch.uint8, device=batch.device) if need else None
    N.check(lib.sp_pages_attention(
        batch._index, c, batch._ref, heads, q.data_ptr(), dt, qs, scale if scale is not None else pages.head_dim ** -0.5,
        out.data_ptr(), os_, None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), need,
        _raw_stream(batch._index)))
    return out
