"""A paged cache of keys and values held in INT8, with one scale for each page and head, and attention over it.

A page holds ``page`` rows of each cached head.  Sequence b's row i lies in page ``tables[b, i // page]``, place
``i % page``; tables and lengths are int32 tensors on the device, so that a captured graph can be replayed while they
change.  The reference's cache is bf16; this one takes half its bytes, which is what a single-token step is bound by.
The kernels are ``reax_kv8_append``, ``reax_kv8_read`` and ``reax_kv8_attend`` in ``include/reax_b200.h``.
"""
from __future__ import annotations

import torch

from . import _native

PAGES = (16, 32, 64)
DIMS = (64, 128, 256)


def _ints(t, shape, name):
    assert t.dtype is torch.int32 and t.shape == shape and t.is_contiguous(), f"{name} is contiguous int32 {shape}"


def _rows(x, heads, dim, name):
    """Checks packed rows [rows, heads, dim] of bf16 and returns their row stride."""
    n, *rest = x.shape
    assert x.dtype is torch.bfloat16 and rest == [heads, dim], f"{name} is bf16 [rows, {heads}, {dim}]"
    s0, s1, s2 = x.stride()
    assert s2 == 1 and (s1 == dim or heads == 1), f"the heads of a row of {name} must lie one after the other"
    return s0 if n > 1 else heads * dim       # (torch leaves the stride of a dimension of one row undefined)


class Int8Cache:
    """The pool: codes ``k``, ``v`` int8 [pages, heads, page, dim] and ``k_scale``, ``v_scale`` float32 [pages, heads]."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "pages", "heads", "page", "dim")

    def __init__(self, k, v, k_scale, v_scale):
        self.pages, self.heads, self.page, self.dim = k.shape
        assert self.page in PAGES and self.dim in DIMS, f"pages have {PAGES} rows, heads {DIMS} values"
        assert k.dtype is torch.int8 and v.dtype is torch.int8 and v.shape == k.shape, \
            "codes are int8 [pages, heads, page, dim]"
        two = (self.pages, self.heads)
        assert k_scale.dtype is torch.float32 and v_scale.dtype is torch.float32 and k_scale.shape == two and \
            v_scale.shape == two, "scales are float32 [pages, heads]"
        assert k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous(), \
            "the cache must be contiguous"
        _native.require_one_device(k, v, k_scale, v_scale)
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale

    @classmethod
    def empty(cls, pages, heads, dim, page=64, device="cuda"):
        """A pool of `pages` pages of zeros."""
        codes = [torch.zeros((pages, heads, page, dim), dtype=torch.int8, device=device) for _ in "kv"]
        return cls(*codes, *[torch.zeros((pages, heads), dtype=torch.float32, device=device) for _ in "kv"])

    def _cache(self):
        return self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr()

    def _sequences(self, tables, counts, cu_seqlens, rows, name):
        batch, width = tables.shape
        _ints(tables, (batch, width), "tables")
        _ints(counts, (batch,), name)
        if cu_seqlens is not None:
            _ints(cu_seqlens, (batch + 1,), "cu_seqlens")
        else:
            assert rows == batch, "without cu_seqlens each sequence has one row"
        return batch, width

    def append(self, k, v, tables, lengths, *, cu_seqlens=None):
        """Rows ``cu_seqlens[b]`` up to ``cu_seqlens[b + 1]`` of k and v (bf16 [rows, heads, dim]; without
        ``cu_seqlens`` row b alone) become sequence b's rows ``lengths[b]`` on.  ``lengths`` is not changed."""
        ldk, ldv = _rows(k, self.heads, self.dim, "k"), _rows(v, self.heads, self.dim, "v")
        n = k.shape[0]
        assert n == v.shape[0], "k and v have the same rows"
        batch, width = self._sequences(tables, lengths, cu_seqlens, n, "lengths")
        index = _native.require_one_device(self.k, k, v, tables, lengths, cu_seqlens)
        _native.launch(
            index, "reax_kv8_append", k.data_ptr(), v.data_ptr(), *self._cache(), tables.data_ptr(), lengths.data_ptr(),
            None if cu_seqlens is None else cu_seqlens.data_ptr(), n, batch, width, self.pages, self.heads, self.page, self.dim,
            ldk, ldv)

    def read(self, tables, starts, cu_seqlens, rows):
        """Sequence b's rows ``starts[b]`` on, ``cu_seqlens[b + 1] - cu_seqlens[b]`` of them and ``rows`` in all, as bf16
        k and v [rows, heads, dim]."""
        batch, width = self._sequences(tables, starts, cu_seqlens, rows, "starts")
        assert cu_seqlens is not None, "read needs cu_seqlens"
        index = _native.require_one_device(self.k, tables, starts, cu_seqlens)
        k = torch.empty((rows, self.heads, self.dim), dtype=torch.bfloat16, device=self.k.device)
        v = torch.empty_like(k)
        _native.launch(
            index, "reax_kv8_read", *self._cache(), tables.data_ptr(), starts.data_ptr(), cu_seqlens.data_ptr(), k.data_ptr(),
            v.data_ptr(), rows, batch, width, self.pages, self.heads, self.page, self.dim)
        return k, v

    def attend(self, q, tables, lengths, *, cu_seqlens=None, max_rows=None, scale=None, return_lse=False, out=None):
        """Softmax attention of q (bf16 [rows, heads * group, dim]; query head h reads cached head h // group).

        Sequence b has ``lengths[b]`` cached rows, of which its query rows are the last ones: row i of n sees cached
        rows 0 .. lengths[b] - n + i.  A row that sees none gives zeros (and -inf), one that holds a NaN or an infinity
        gives NaN (in both).  ``max_rows``: at least the most query rows of a sequence, where the caller knows it (a hint: it
        picks the kernel, not the result; without it ``cu_seqlens`` means the form for many rows, the slow one where each
        sequence has one).  Rows of no sequence are not written.  Returns out bf16 [rows, heads * group, dim], with the
        float32 log-sum-exp [rows, heads * group] beside it if asked."""
        assert q.dim() == 3 and q.shape[1] % self.heads == 0, "the query heads are a multiple of the cached heads"
        n, heads_q, _ = q.shape
        ldq = _rows(q, heads_q, self.dim, "q")
        batch, width = self._sequences(tables, lengths, cu_seqlens, n, "lengths")
        if out is None:
            out = torch.empty_like(q)         # (contiguous: q's heads are)
        else:
            assert out.dtype is torch.bfloat16 and out.shape == q.shape and out.is_contiguous(), \
                "out is contiguous bf16 like q"
        index = _native.require_one_device(self.k, q, tables, lengths, cu_seqlens, out)
        lse = torch.empty((n, heads_q), dtype=torch.float32, device=q.device) if return_lse else None
        if max_rows is None:
            max_rows = 1 if cu_seqlens is None else n
        ws = _native.kv8_workspace(q.device)
        _native.launch(
            index, "reax_kv8_attend", q.data_ptr(), *self._cache(), tables.data_ptr(), lengths.data_ptr(),
            None if cu_seqlens is None else cu_seqlens.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(), n,
            max_rows, batch, width, self.pages, self.heads, heads_q // self.heads, self.page, self.dim, ldq,
            self.dim ** -0.5 if scale is None else scale, ws.data_ptr(), ws.numel())
        return (out, lse) if return_lse else out
