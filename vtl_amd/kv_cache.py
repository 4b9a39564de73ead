"""Int8 key/value cache in pages and attention over it: what stands between the int8 linear layers of a decoder.

Keys and values of new tokens are quantized into the cache (`kv_write_hip`) with the arithmetic of
`HipTensor.quantize_i8(0)`, a row for each token and head; they come back as f32 (`kv_read_hip`), and
queries attend over them where they lie (`attention_i8_hip`).  include/vtl_hip.h has the layout of a page and the
contract of each call.  As everywhere in this package the work is enqueued on the library's stream.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import capi
from .storage import HipParams, HipStorage
from .tensor import HipTensor


class HipKVCache:
    """Pages for the keys and values of `kv_heads` heads of `head_dim` values each, `page_size` tokens a page."""

    def __init__(self, num_pages: int, page_size: int, kv_heads: int, head_dim: int, params: HipParams | None = None):
        nbytes = capi.lib().vtl_hip_kv_cache_bytes(num_pages, page_size, kv_heads, head_dim)
        if not nbytes:
            raise ValueError(f"HipKVCache: no cache of {num_pages} pages of {page_size} tokens, {kv_heads} heads of {head_dim}")
        self.num_pages, self.page_size = num_pages, page_size
        self.kv_heads, self.head_dim = kv_heads, head_dim
        self.pages = HipStorage.empty(nbytes, np.uint8, params)
        self.handle = capi.KVCache(self.pages.ptr, num_pages, page_size, kv_heads, head_dim)

    def release(self) -> None:
        self.pages.release()
        self.handle.pages = None


class HipKVBatch:
    """The sequences of a call: `page_table` [batch, max_pages], `lengths` [batch] and `starts` [batch + 1], int32 tensors on the
    device.  Rows starts[b] .. starts[b + 1] - 1 of a call's tensors are the last tokens of sequence b; without `starts` row b is
    the last token of sequence b.  `rows` is needed with `starts` only; `most_rows` and `most_length` tell the host the largest of
    each (0: not known)."""

    def __init__(self, page_table: HipTensor, lengths: HipTensor, starts: HipTensor | None = None, rows: int | None = None,
                 most_rows: int = 0, most_length: int = 0):
        page_table._assert(np.int32, what="page_table")
        lengths._assert(np.int32, matrix=False, what="lengths")
        batch, max_pages = page_table.shape
        if lengths.size != batch:
            raise ValueError(f"lengths: expected {batch} entries, got {lengths.size}")
        if starts is not None:
            starts._assert(np.int32, matrix=False, what="starts")
            if starts.size != batch + 1:
                raise ValueError(f"starts: expected {batch + 1} entries, got {starts.size}")
            if rows is None:
                raise ValueError("HipKVBatch: the number of rows is needed with starts")
        elif rows not in (None, batch):
            raise ValueError(f"HipKVBatch: {rows} rows without starts, {batch} sequences")
        self.page_table, self.lengths, self.starts = page_table, lengths, starts
        self.rows = batch if rows is None else rows
        self.handle = capi.KVBatch(batch, max_pages, page_table.ptr, lengths.ptr, starts.ptr if starts is not None else None,
                                   self.rows, most_rows, most_length)


def _rows(t: HipTensor, batch: HipKVBatch, width: int, first: int, what: str):
    """Address of column `first` of the f32 rows of t ([rows, columns], or [rows, heads, head_dim]), and their stride."""
    t._assert(np.float32, matrix=False, what=what)
    stride = t.size // t.shape[0] if t.shape and t.shape[0] else width
    if t.rank() < 2 or t.shape[0] != batch.rows or first < 0 or first + width > stride:
        raise ValueError(f"{what}: {batch.rows} rows with columns {first} to {first + width} expected, got shape {t.shape}")
    return t.ptr + 4 * first if t.ptr else None, stride


def kv_write_hip(cache: HipKVCache, batch: HipKVBatch, k: HipTensor, v: HipTensor, k_first: int = 0, v_first: int = 0) -> None:
    """`kv_write_hip(cache, batch, k, v) !`: the rows' keys and values into the cache.  They may be columns of one tensor, a fused
    projection's output, from k_first and v_first on."""
    width = cache.kv_heads * cache.head_dim
    kp, ks = _rows(k, batch, width, k_first, "kv_write_hip k")
    vp, vs = _rows(v, batch, width, v_first, "kv_write_hip v")
    capi.call("vtl_hip_kv_write_f32", C.byref(cache.handle), C.byref(batch.handle), kp, ks, vp, vs)


def kv_read_hip(cache: HipKVCache, batch: HipKVBatch):
    """`kv_read_hip(cache, batch) !(&HipTensor[f32], &HipTensor[f32])`: the rows' keys and values, [rows, kv_heads, head_dim] each.
    Rows of no sequence are not written: what they hold is undefined."""
    p = cache.pages.params
    k = HipTensor.empty([batch.rows, cache.kv_heads, cache.head_dim], np.float32, p)
    v = HipTensor.empty(k.shape, np.float32, p)
    stride = cache.kv_heads * cache.head_dim
    capi.call("vtl_hip_kv_read_f32", C.byref(cache.handle), C.byref(batch.handle), k.ptr or None, stride, v.ptr or None, stride)
    return k, v


def attention_i8_workspace(cache: HipKVCache, batch: HipKVBatch, heads: int) -> int:
    """Bytes of the workspace that `attention_i8_hip` takes for these arguments (0: none is needed): for calls that may overlap on a device, and
    for calls recorded into a graph, `HipStorage.empty(bytes, np.uint8)` each."""
    return capi.lib().vtl_hip_attention_i8_workspace(C.byref(cache.handle), C.byref(batch.handle), heads)


def attention_i8_hip(cache: HipKVCache, batch: HipKVBatch, q: HipTensor, heads: int, scale: float | None = None, causal: bool = True,
                     q_first: int = 0, workspace: HipStorage | None = None) -> HipTensor:
    """`attention_i8_hip(cache, batch, q, heads, scale, causal) !&HipTensor[f32]`: softmax(scale * q . k^T) . v of every row over
    its sequence, [rows, heads, head_dim]; scale is 1 / sqrt(head_dim) unless given.  The rows' own tokens have been written before.
    q may be columns of a fused projection's output, from q_first on; workspace, of `attention_i8_workspace` bytes, is the library's own
    unless given.  Rows of no sequence are not written: what they hold is undefined."""
    width = heads * cache.head_dim
    qp, qs = _rows(q, batch, width, q_first, "attention_i8_hip q")
    if scale is None:
        scale = cache.head_dim ** -0.5
    out = HipTensor.empty([batch.rows, heads, cache.head_dim], np.float32, q.data.params)
    capi.call("vtl_hip_attention_i8_f32", C.byref(cache.handle), C.byref(batch.handle), qp, qs, heads, scale, int(causal),
              out.ptr or None, width, workspace.ptr if workspace is not None else None, workspace.size if workspace is not None else 0)
    return out
