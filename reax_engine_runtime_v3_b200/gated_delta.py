"""The gated delta rule: the token mixer between the split q, k, v projection and the output projection.

For each value head, with a float32 state ``S [Dk, Dv]`` and row by row:

    S <- exp(g) S;   u = beta (v - k^T S);   S <- S + k u^T;   out = scale q^T S

``prefill`` takes the rows of any number of sequences packed one after the other, ``decode`` one row of each.  Both
update the states in place in a pool ``state [n_slots, v_heads, Dk, Dv]``, of which sequence b uses slot ``slots[b]``
(b itself without ``slots``).  A slot outside the pool marks a padding sequence, whose outputs are zeros.  The
reference's engine calls a library for this operator; here it runs in this package's own kernels
(``reax_gdn_prefill`` and ``reax_gdn_decode`` in ``include/reax_b200.h``), forward only.
"""
from __future__ import annotations

import torch

from . import _native

_WIDTHS = (64, 128)


def _check(q, k, v, g, beta, state, slots, out, batch):
    """The checks that both forms share: shapes, types and layouts the kernels take; returns the output."""
    assert q.dtype == k.dtype == v.dtype == torch.bfloat16, "q, k and v are bf16"
    n, k_heads, dk = q.shape
    n_v, v_heads, dv = v.shape
    assert k.shape == q.shape and n_v == n, "q, k [rows, k_heads, Dk] and v [rows, v_heads, Dv] disagree"
    assert v_heads % k_heads == 0, "the value heads are a multiple of the key heads"
    assert dk in _WIDTHS and dv in _WIDTHS, "head widths are 64 or 128"
    for t in (q, k, v):
        _, heads, width = t.shape
        _, s1, s2 = t.stride()
        assert s2 == 1 and (s1 == width or heads == 1), "a row's heads must lie one after the other"
    assert g.dtype == beta.dtype == torch.float32 and g.shape == beta.shape == (n, v_heads), \
        "g and beta are float32 [rows, v_heads]"
    assert g.is_contiguous() and beta.is_contiguous(), "g and beta must be contiguous"
    assert state.dtype == torch.float32 and state.is_contiguous() and state.shape[1:] == (v_heads, dk, dv), \
        "state is contiguous float32 [slots, v_heads, Dk, Dv]"
    if slots is None:
        assert len(state) >= batch, "fewer states than sequences"
    else:
        assert slots.dtype == torch.int32 and slots.shape == (batch,) and slots.is_contiguous(), \
            "slots is int32, one for each sequence"
    if out is None:
        out = torch.empty((n, v_heads, dv), dtype=torch.bfloat16, device=q.device)
    else:
        assert out.dtype == torch.bfloat16 and out.shape == v.shape and out.is_contiguous(), \
            "out is contiguous bf16 [rows, v_heads, Dv]"
    _native.require_cuda(q, k, v, g, beta, state, slots, out)
    return out


def _ld(t):
    """Row stride of packed rows (torch leaves the stride of a dimension of one row undefined)."""
    return t.stride(0) if len(t) > 1 else t.shape[1] * t.shape[2]


def prefill(q, k, v, g, beta, state, *, cu_seqlens=None, slots=None, carry=True, scale=None, normalize=True, out=None):
    """Rows of packed sequences: q, k bf16 [rows, k_heads, Dk], v bf16 [rows, v_heads, Dv], g (log of the decay) and
    beta float32 [rows, v_heads]; sequence b has rows ``cu_seqlens[b]`` up to ``cu_seqlens[b + 1]`` (int32 on the
    device; without it all rows are one sequence).  ``carry``: start from the states kept, else from zeros.
    ``normalize``: divide q and k by the root of their sum of squares first; ``scale`` is Dk ** -0.5 if not given.
    Returns out bf16 [rows, v_heads, Dv]; the states are updated in place."""
    batch = 1 if cu_seqlens is None else len(cu_seqlens) - 1
    out = _check(q, k, v, g, beta, state, slots, out, batch)
    if cu_seqlens is not None:
        assert cu_seqlens.dtype == torch.int32 and cu_seqlens.dim() == 1 and cu_seqlens.is_contiguous(), \
            "cu_seqlens is contiguous int32"
        _native.require_cuda(cu_seqlens)
    n, k_heads, dk = q.shape
    _native.check(_native.load().reax_gdn_prefill(
        _native.ptr(q), _native.ptr(k), _native.ptr(v), _native.ptr(g), _native.ptr(beta), _native.ptr(state),
        _native.ptr(cu_seqlens), _native.ptr(slots), _native.ptr(out), n, batch, k_heads, v.shape[1], dk, v.shape[2],
        len(state), _ld(q), _ld(k), _ld(v), dk ** -0.5 if scale is None else scale, bool(normalize), bool(carry),
        _native.stream_handle(q.device)))
    return out


def decode(q, k, v, g, beta, state, *, slots=None, scale=None, normalize=True, out=None):
    """One row of each sequence, from the states kept: arguments and result as ``prefill``, row b is sequence b's."""
    n, k_heads, dk = q.shape
    out = _check(q, k, v, g, beta, state, slots, out, n)
    _native.check(_native.load().reax_gdn_decode(
        _native.ptr(q), _native.ptr(k), _native.ptr(v), _native.ptr(g), _native.ptr(beta), _native.ptr(state),
        _native.ptr(slots), _native.ptr(out), n, k_heads, v.shape[1], dk, v.shape[2], len(state), _ld(q), _ld(k), _ld(v),
        dk ** -0.5 if scale is None else scale, bool(normalize), _native.stream_handle(q.device)))
    return out
