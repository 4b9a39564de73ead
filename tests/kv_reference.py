"""The int8 key/value cache and the attention over it from their definitions, in 64 bits and with numpy: what the tests of both
compare with.  Pages are taken apart and put together here by the layout that the header states, value by value."""
from __future__ import annotations

import numpy as np

from vtl_amd import HipKVBatch, HipKVCache, capi
from vtl_amd.tensor import HipTensor


def padded(dim: int) -> int:
    return -(-dim // 16) * 16


def parts(pages: np.ndarray, page_size: int, kv_heads: int, dim: int):
    """Views of raw pages: codes of the keys [pages, heads, D / 16, P, 16], of the values [pages, heads, P / 16, D, 16], scales [pages, heads, P]."""
    d = padded(dim)
    half = d * page_size
    raw = pages.reshape(-1, kv_heads, page_size * (2 * d + 8))
    k = raw[..., :half].view(np.int8).reshape(*raw.shape[:2], d // 16, page_size, 16)
    v = raw[..., half:2 * half].view(np.int8).reshape(*raw.shape[:2], page_size // 16, d, 16)
    scales = raw[..., 2 * half:].view(np.float32)
    return k, v, scales[..., :page_size], scales[..., page_size:]


def quantize(x: np.ndarray):
    """Codes and scales of the last axis: absmax / 127, half to even, both quotients f32."""
    finite = np.where(np.isnan(x), np.float32(0), np.abs(x))
    scale = (finite.max(-1) / np.float32(127)).astype(np.float32)
    with np.errstate(all="ignore"):
        r = np.rint((x / scale[..., None]).astype(np.float32))
    r = np.where(np.isnan(r) | (scale[..., None] == 0), 0, np.clip(r, -127, 127))
    return r.astype(np.int8), scale


class Cache:
    """A cache on the device and what its bytes are on the host."""

    def __init__(self, lengths, page_size, kv_heads, dim, spare=3, seed=0, most_pages=None, fill=True):
        rng = np.random.default_rng(seed)
        self.lengths = np.asarray(lengths, np.int32)
        need = -(-np.maximum(self.lengths, 0) // page_size)
        self.num_pages = max(1, int(need.sum()) + spare)
        self.page_size, self.kv_heads, self.dim = page_size, kv_heads, dim
        width = max(1, int(need.max(initial=1))) if most_pages is None else most_pages
        order = rng.permutation(self.num_pages).astype(np.int32)
        self.table = np.full((len(self.lengths), width), -1, np.int32)     # places behind a sequence's end are no pages
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        size = self.num_pages * kv_heads * page_size * (2 * padded(dim) + 8)
        # what nobody has written: any bytes, among them scales that are NaN or infinite
        self.host = rng.integers(0, 256, size, dtype=np.uint8)
        if fill:
            k, v, ks, vs = self.parts()
            for b, n in enumerate(np.maximum(self.lengths, 0)):
                for j in range(n):
                    page, slot = self.table[b, j // page_size], j % page_size
                    k[page, :, :, slot] = rng.integers(-127, 128, (kv_heads, padded(dim) // 16, 16))
                    v[page, :, slot // 16, :, slot % 16] = rng.integers(-127, 128, (kv_heads, padded(dim)))
                    ks[page, :, slot] = rng.uniform(0.2, 1.5, kv_heads) * (3 / 127)
                    vs[page, :, slot] = rng.uniform(0.2, 1.5, kv_heads) * (3 / 127)

    def parts(self):
        return parts(self.host, self.page_size, self.kv_heads, self.dim)

    def to_device(self):
        self.cache = HipKVCache(self.num_pages, self.page_size, self.kv_heads, self.dim)
        assert self.cache.pages.size == self.host.size
        capi.call("vtl_hip_memcpy_h2d", self.cache.pages.ptr, self.host.ctypes.data, self.host.nbytes)
        return self

    def batch(self, counts=None, rows=None, starts=None, hints=True):
        """Rows counts[b] of each sequence, behind each other; counts None: one row each, without starts."""
        if counts is None:
            self.starts, rows = None, len(self.lengths)
        else:
            self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32) if starts is None else np.asarray(starts, np.int32)
            rows = int(self.starts[-1]) if rows is None else rows
        hint = (int(np.max(counts if counts is not None else 1, initial=0)), int(max(0, self.lengths.max(initial=0)))) if hints else (0, 0)
        dev = HipTensor.from_host
        return HipKVBatch(dev(self.table), dev(self.lengths), None if self.starts is None else dev(self.starts), rows, *hint)

    def fetch(self) -> np.ndarray:
        got = np.empty_like(self.host)
        capi.call("vtl_hip_memcpy_d2h", got.ctypes.data, self.cache.pages.ptr, got.nbytes)
        return got

    def place(self, b, j):
        """Page and slot of token j of sequence b, or None."""
        if j < 0 or j // self.page_size >= self.table.shape[1]:
            return None
        page = self.table[b, j // self.page_size]
        return (page, j % self.page_size) if 0 <= page < self.num_pages else None

    def rows_of(self, b):
        if self.starts is None:
            return b, b + 1
        return int(self.starts[b]), int(self.starts[b + 1])

    def length(self, b):
        return int(min(max(self.lengths[b], 0), self.table.shape[1] * self.page_size))

    def written(self, k, v) -> np.ndarray:
        """The bytes of the pages once rows k, v [rows, heads, dim] are in them."""
        self.host = self.host.copy()
        kc, vc, ks, vs = self.parts()
        pad = [(0, 0), (0, 0), (0, padded(self.dim) - self.dim)]
        (qk, sk), (qv, sv) = quantize(k), quantize(v)
        qk, qv = np.pad(qk, pad), np.pad(qv, pad)
        for b in range(len(self.lengths)):
            lo, hi = self.rows_of(b)
            for r in range(lo, hi):
                at = self.place(b, self.length(b) - (hi - r))
                if at is not None:
                    page, slot = at
                    kc[page, :, :, slot] = qk[r].reshape(self.kv_heads, -1, 16)
                    vc[page, :, slot // 16, :, slot % 16] = qv[r]
                    ks[page, :, slot], vs[page, :, slot] = sk[r], sv[r]
        return self.host

    def tokens(self, b, j):
        """Keys and values [n, heads, dim] of tokens j of sequence b as f32 (code times scale), and which of them have a page."""
        kc, vc, ks, vs = self.parts()
        k = np.zeros((len(j), self.kv_heads, self.dim), np.float32)
        v, there = k.copy(), np.zeros(len(j), bool)
        for i, t in enumerate(j):
            at = self.place(b, t)
            if at is not None:
                page, slot = at
                there[i] = True
                with np.errstate(all="ignore"):
                    k[i] = kc[page, :, :, slot].reshape(self.kv_heads, -1)[:, :self.dim].astype(np.float32) * ks[page, :, slot, None]
                    v[i] = vc[page, :, slot // 16, :, slot % 16][:, :self.dim].astype(np.float32) * vs[page, :, slot, None]
        return k, v, there

    def read(self, rows):
        k = np.zeros((rows, self.kv_heads, self.dim), np.float32)
        v = k.copy()
        for b in range(len(self.lengths)):
            lo, hi = self.rows_of(b)
            if hi > lo:
                k[lo:hi], v[lo:hi], _ = self.tokens(b, np.arange(lo, hi) - hi + self.length(b))
        return k, v

    def attend(self, q, heads, scale, causal):
        """out [rows, heads, dim] in 64 bits, and how far f32 sums may be from it.

        A score's error: q has 22 bits and is scaled in f32 (2^-22 + 2^-23 of sum |q k|), dim products are added up in f32 (dim 2^-24 of the
        same sum), and the score is rounded three times (3 2^-24 of it) and once more when the maximum is taken off (the size of both).  A weight
        is off by twice the largest such error (its own and the sum's), relatively, and by 2^-20 for the exponential, the 22 bits of the weight
        and the scales; adding up n tokens, 8 or more at a time, costs (n / 8 + 64) 2^-24.  The weight times the value's scale is two fp16 numbers once
        the sequence's largest scale so far is brought to 2^9 at least, beside weights of up to 2^5: fp16 has no steps below 2^-24, so
        each such product is off by up to 2^-25 / 2^9 of that scale, and n of them, times codes of up to 127, over a sum of weights that is 1 at least, by
        n 127 2^-34 of it."""
        out = np.zeros((q.shape[0], heads, self.dim))
        far = np.full(out.shape, 1e-30)
        group = heads // self.kv_heads
        for b in range(len(self.lengths)):
            lo, hi = self.rows_of(b)
            n = self.length(b)
            if hi <= lo or n == 0:
                continue
            k, v, there = self.tokens(b, np.arange(n))
            finite = np.where(np.isfinite(v), np.abs(v), 0).max((0, 2))      # 127 times the largest scale, about, of each head
            k, v = k.astype(np.float64), v.astype(np.float64)
            last = np.arange(lo, hi) - hi + n if causal else np.full(hi - lo, n - 1)
            seen = there[None] & (np.arange(n)[None] <= last[:, None])
            for h in range(heads):
                g = h // group
                x = q[lo:hi, h].astype(np.float64)
                with np.errstate(all="ignore"):
                    s = x @ k[:, g].T * scale
                    size = np.abs(x) @ np.abs(k[:, g]).T * abs(scale)
                    s = np.where(seen, s, -np.inf)
                    top = np.where(seen.any(1), s.max(1), 0)
                    w = np.where(seen, np.exp(s - top[:, None]), 0)
                    total = w.sum(1)
                    w = w / np.where(total > 0, total, 1)[:, None]
                    w = np.where(seen, w, 0)
                    vg = np.where(there[:, None], v[:, g], 0)
                    none = ~np.isfinite(vg).all(1)              # such a token is no number for the rows that see it, and nothing for the others
                    vg[none] = 0
                    w[(seen & none).any(1)] = np.nan
                    out[lo:hi, h] = w @ vg
                    score_off = np.where(seen, size * (2.0 ** -22 + 2.0 ** -23 + self.dim * 2.0 ** -24) + 3 * 2.0 ** -24 * np.abs(s)
                                         + 2.0 ** -23 * (np.abs(s) + np.abs(top[:, None])), 0).max(1)
                    far[lo:hi, h] += (w @ np.abs(vg)) * (2 * score_off + 2.0 ** -20 + (n / 8 + 64) * 2.0 ** -24)[:, None]
                    far[lo:hi, h] += n * 2.0 ** -34 * finite[g] * 127 / 64      # random codes come to half of 127 at least
        return out, far
