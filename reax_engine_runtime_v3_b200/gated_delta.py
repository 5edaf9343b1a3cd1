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


def _rows(x, name):
    """Checks packed rows [rows, heads, width] of bf16, a row's heads one after the other, and returns their stride."""
    assert x.dtype is torch.bfloat16, f"{name} is bf16"
    n, heads, width = x.shape
    s0, s1, s2 = x.stride()
    assert s2 == 1 and (s1 == width or heads == 1), f"the heads of a row of {name} must lie one after the other"
    return s0 if n > 1 else heads * width     # (torch leaves the stride of a dimension of one row undefined)


def _check(q, k, v, g, beta, state, slots, out, batch):
    """The checks that both forms share: shapes, types and layouts the kernels take.  Returns the output, the row strides
    of q, k and v, the sizes and the device."""
    n, k_heads, dk = q.shape
    n_v, v_heads, dv = v.shape
    assert k.shape == q.shape and n_v == n, "q, k [rows, k_heads, Dk] and v [rows, v_heads, Dv] disagree"
    assert v_heads % k_heads == 0, "the value heads are a multiple of the key heads"
    assert dk in _WIDTHS and dv in _WIDTHS, "head widths are 64 or 128"
    strides = _rows(q, "q"), _rows(k, "k"), _rows(v, "v")
    assert g.dtype is torch.float32 and beta.dtype is torch.float32 and g.shape == (n, v_heads) and beta.shape == (n, v_heads), \
        "g and beta are float32 [rows, v_heads]"
    assert g.is_contiguous() and beta.is_contiguous(), "g and beta must be contiguous"
    n_slots, *rest = state.shape
    assert state.dtype is torch.float32 and state.is_contiguous() and rest == [v_heads, dk, dv], \
        "state is contiguous float32 [slots, v_heads, Dk, Dv]"
    if slots is None:
        assert n_slots >= batch, "fewer states than sequences"
    else:
        assert slots.dtype is torch.int32 and slots.shape == (batch,) and slots.is_contiguous(), \
            "slots is int32, one for each sequence"
    if out is None:
        out = torch.empty_like(v)             # (contiguous: v's heads are)
    else:
        assert out.dtype is torch.bfloat16 and out.shape == v.shape and out.is_contiguous(), \
            "out is contiguous bf16 [rows, v_heads, Dv]"
    index = _native.require_one_device(q, k, v, g, beta, state, slots, out)
    return out, strides, (k_heads, v_heads, dk, dv, n_slots), index


def prefill(q, k, v, g, beta, state, *, cu_seqlens=None, slots=None, carry=True, scale=None, normalize=True, out=None):
    """Rows of packed sequences: q, k bf16 [rows, k_heads, Dk], v bf16 [rows, v_heads, Dv], g (log of the decay) and
    beta float32 [rows, v_heads]; sequence b has rows ``cu_seqlens[b]`` up to ``cu_seqlens[b + 1]`` (int32 on the
    device; without it all rows are one sequence).  ``carry``: start from the states kept, else from zeros.
    ``normalize``: divide q and k by the root of their sum of squares first; ``scale`` is Dk ** -0.5 if not given.
    A sequence without rows keeps its state, or gets zeros without ``carry``; a call without any rows does nothing.  Returns
    out bf16 [rows, v_heads, Dv] (rows of no sequence are not written); the states are updated in place."""
    batch = 1 if cu_seqlens is None else cu_seqlens.shape[0] - 1
    out, strides, sizes, index = _check(q, k, v, g, beta, state, slots, out, batch)
    if cu_seqlens is not None:
        assert cu_seqlens.dtype is torch.int32 and cu_seqlens.dim() == 1 and cu_seqlens.is_contiguous(), \
            "cu_seqlens is contiguous int32"
        _native.require_one_device(q, cu_seqlens)
    # scratch memory of this call: torch's allocator keeps it for the next one on this stream
    size = _native.load().reax_gdn_workspace_bytes(q.shape[0], batch, sizes[0], sizes[1], sizes[2])
    scratch = torch.empty(size, dtype=torch.uint8, device=q.device)
    _native.launch(
        index, "reax_gdn_prefill", q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), state.data_ptr(),
        None if cu_seqlens is None else cu_seqlens.data_ptr(), None if slots is None else slots.data_ptr(), out.data_ptr(),
        q.shape[0], batch, *sizes, *strides, sizes[2] ** -0.5 if scale is None else scale, normalize, carry,
        scratch.data_ptr(), size)
    return out


def decode(q, k, v, g, beta, state, *, slots=None, scale=None, normalize=True, out=None):
    """One row of each sequence, from the states kept: arguments and result as ``prefill``, row b is sequence b's."""
    n = q.shape[0]
    out, strides, sizes, index = _check(q, k, v, g, beta, state, slots, out, n)
    _native.launch(
        index, "reax_gdn_decode", q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), state.data_ptr(),
        None if slots is None else slots.data_ptr(), out.data_ptr(), n, *sizes, *strides,
        sizes[2] ** -0.5 if scale is None else scale, normalize)
    return out
