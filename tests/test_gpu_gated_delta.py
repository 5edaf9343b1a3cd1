"""GPU checks of the gated delta rule (prompt and single-row forms) against its definition in 64 bits.

Tolerances.  State (float32): relative 2-norm error of a head's state at most 8e-6.  The chunked form splits each
product's inexact operand into two 11-bit halves (2^-22 = 2.4e-7 of the operand left out), and a state collects
a handful of such errors through the solve of each chunk.  Output (bf16): half a bf16 unit is 2^-9 of the value; its
operands are rounded to 11 bits (2^-12 each) before sums whose terms may cancel, which is measured against the
root mean square of the head's row: |error| <= 2^-8 |o| + 2^-8 rms.
"""
import math

import pytest
import torch

from tests import helpers as H

pytestmark = pytest.mark.gpu


def inputs(seed, rows, hk, hv, dk, dv, slots, normalize=True, g_scale=1.0, shared=0.5):
    gen = H.gen(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen)
    size = 1.0 if normalize else dk ** -0.5
    q = ((rnd(rows, hk, dk) + shared * rnd(1, hk, dk)) * size).bfloat16()
    k = ((rnd(rows, hk, dk) + shared * rnd(1, hk, dk)) * size).bfloat16()
    v = rnd(rows, hv, dv).bfloat16()
    g = -torch.exp(rnd(rows, hv)) * 0.1 * g_scale
    beta = torch.sigmoid(rnd(rows, hv))
    state = rnd(slots, hv, dk, dv)
    return q, k, v, g, beta, state


def definition(q, k, v, g, beta, state, spans, slots, scale=None, normalize=True, carry=True):
    """Row by row in 64 bits; returns (out, state)."""
    q, k, v, g, beta, state = (x.double() for x in (q, k, v, g, beta, state))
    hv, dk = v.shape[1], q.shape[2]
    each = hv // q.shape[1]
    if normalize:
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + 1e-6)
        k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    q, k = q.repeat_interleave(each, 1) * (dk ** -0.5 if scale is None else scale), k.repeat_interleave(each, 1)
    out, state = torch.zeros_like(v), state.clone()
    for (lo, hi), slot in zip(spans, slots):
        if not 0 <= slot < len(state):
            continue
        s = state[slot].clone() if carry else torch.zeros_like(state[slot])
        for r in range(lo, hi):
            s = s * torch.exp(g[r])[:, None, None]
            u = beta[r][:, None] * (v[r] - torch.einsum("hk,hkv->hv", k[r], s))
            s = s + k[r][:, :, None] * u[:, None, :]
            out[r] = torch.einsum("hk,hkv->hv", q[r], s)
        state[slot] = s
    return out, state


def compare(out, state, want_out, want_state, spans=None):
    out, state = out.cpu().double(), state.cpu().double()
    assert torch.isfinite(out).all() and torch.isfinite(state).all()
    err = (state - want_state).flatten(2).norm(dim=-1)
    size = want_state.flatten(2).norm(dim=-1)
    assert (err <= 8e-6 * size + 1e-30).all(), f"state error {(err / size.clamp(min=1e-30)).max():.2e}"
    rms = want_out.square().mean(-1, keepdim=True).sqrt()
    excess = (out - want_out).abs() - (want_out.abs() + rms) * 2.0 ** -8
    assert (excess <= 1e-30).all(), f"output off by {(out - want_out).abs().max():.3g}, beyond bound by {excess.max():.3g}"


def run_prefill(x, lens, slots, **kw):
    from reax_engine_runtime_v3_b200 import gated_delta
    q, k, v, g, beta, state = (t.cuda() for t in x)
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    cu = torch.tensor(at, dtype=torch.int32).cuda()
    sl = torch.tensor(slots, dtype=torch.int32).cuda()
    out = gated_delta.prefill(q, k, v, g, beta, state, cu_seqlens=cu, slots=sl, **kw)
    torch.cuda.synchronize()
    return out, state, list(zip(at, at[1:]))


@pytest.mark.parametrize("hk,hv,dk,dv", [(2, 4, 128, 128), (1, 1, 128, 64), (2, 2, 64, 128), (3, 9, 64, 64), (16, 32, 128, 128)])
@pytest.mark.parametrize("batch", [1, 5])
def test_decode(hk, hv, dk, dv, batch):
    from reax_engine_runtime_v3_b200 import gated_delta
    x = inputs(batch * 7 + dk, batch, hk, hv, dk, dv, batch + 2)
    slots = [(3 * i + 1) % (batch + 2) for i in range(batch)] if batch > 1 else [1]
    if batch == 5:
        slots = [6, -1, 0, 3, 99]                      # two padding rows
    want = definition(*x, [(i, i + 1) for i in range(batch)], slots)
    q, k, v, g, beta, state = (t.cuda() for t in x)
    out = gated_delta.decode(q, k, v, g, beta, state, slots=torch.tensor(slots, dtype=torch.int32).cuda())
    torch.cuda.synchronize()
    compare(out, state, *want)
    for i, s in enumerate(slots):
        if not 0 <= s < batch + 2:
            assert not out[i].any()


def test_decode_strided_rows_given_out_and_another_stream():
    """q, k, v as slices of one projection's rows, a caller's out, default slots, and a stream of its own."""
    from reax_engine_runtime_v3_b200 import gated_delta
    hk, hv, d, n = 4, 8, 128, 7
    x = inputs(3, n, hk, hv, d, d, n)
    want = definition(*x, [(i, i + 1) for i in range(n)], range(n), scale=0.3)
    row = torch.cat([t.reshape(n, -1) for t in x[:3]], 1).cuda()
    q, k, v = row[:, :hk * d].view(n, hk, d), row[:, hk * d:2 * hk * d].view(n, hk, d), row[:, 2 * hk * d:].view(n, hv, d)
    g, beta, state = (t.cuda() for t in x[3:])
    out = torch.full((n, hv, d), 7.0, dtype=torch.bfloat16, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = gated_delta.decode(q, k, v, g, beta, state, out=out, scale=0.3)
    stream.synchronize()
    assert got is out
    compare(out, state, *want)


@pytest.mark.parametrize("lens", [[1], [2], [17], [63], [64], [65], [128], [200], [1, 64, 0, 130, 3], [0], [0, 0, 5]])
@pytest.mark.parametrize("carry", [True, False])
def test_prefill_lengths(lens, carry):
    x = inputs(sum(lens) + 5, sum(lens), 2, 4, 128, 128, len(lens) + 1)
    slots = [(i + 1) % (len(lens) + 1) for i in range(len(lens))]
    out, state, spans = run_prefill(x, lens, slots, carry=carry)
    if sum(lens) == 0:                                  # nothing to do: nothing is touched
        assert torch.equal(state.cpu(), x[5])
        return
    compare(out, state, *definition(*x, spans, slots, carry=carry))


@pytest.mark.parametrize("hk,hv,dk,dv", [(1, 1, 64, 64), (1, 3, 64, 128), (2, 2, 128, 64), (16, 32, 128, 128)])
def test_prefill_heads(hk, hv, dk, dv):
    lens = [70, 129]
    x = inputs(hk + dk, sum(lens), hk, hv, dk, dv, 2)
    out, state, spans = run_prefill(x, lens, [1, 0])
    compare(out, state, *definition(*x, spans, [1, 0]))


@pytest.mark.parametrize("normalize,g_scale,shared", [(False, 1.0, 0.5), (True, 0.0, 0.5), (True, 300.0, 0.5), (True, 0.01, 4.0)])
def test_prefill_decays_and_keys(normalize, g_scale, shared):
    """Keys as they come; no decay; decays whose products underflow within a chunk; keys that nearly agree."""
    lens = [150, 33]
    x = inputs(11, sum(lens), 2, 4, 128, 128, 2, normalize=normalize, g_scale=g_scale, shared=shared)
    out, state, spans = run_prefill(x, lens, [0, 1], normalize=normalize)
    compare(out, state, *definition(*x, spans, [0, 1], normalize=normalize))


def test_prefill_beta_ends_zero_rows_and_sizes():
    """beta of 0 and 1, rows of zeros, a decay of exp(-inf), and rows and states of very different sizes."""
    lens = [100]
    x = list(inputs(12, 100, 2, 2, 128, 128, 1))
    x[4][10:20], x[4][20:30] = 0.0, 1.0
    x[0][40:44], x[1][42:46], x[2][44:50] = 0, 0, 0
    x[3][60] = -math.inf
    x[1][70:75] *= 2.0 ** 20
    x[1][75:80] *= 2.0 ** -20
    x[0][80:85] *= 2.0 ** 30
    x[2][85:90] *= 2.0 ** 12
    x[5] *= 2.0 ** -14
    out, state, spans = run_prefill(x, lens, [0])
    want = definition(*x, spans, [0])
    compare(out, state, *want)


def test_prefill_padding_sequence_and_untouched_slots():
    lens = [65, 70, 3]
    slots = [2, -1, 0]
    x = inputs(13, sum(lens), 2, 4, 128, 128, 4)
    out, state, spans = run_prefill(x, lens, slots)
    want = definition(*x, spans, slots)
    compare(out, state, *want)
    assert not out[65:135].any()
    assert torch.equal(state[[1, 3]].cpu(), x[5][[1, 3]])


def test_prefill_in_two_calls_and_steps_agree_with_one():
    """A sequence cut into two prompts and five steps against the definition of the whole."""
    from reax_engine_runtime_v3_b200 import gated_delta
    n = 105
    x = inputs(14, n, 2, 4, 128, 128, 1)
    want = definition(*x, [(0, n)], [0])
    q, k, v, g, beta, state = (t.cuda() for t in x)
    outs = [gated_delta.prefill(*(t[a:b] for t in (q, k, v, g, beta)), state) for a, b in ((0, 41), (41, 100))]
    outs += [gated_delta.decode(*(t[i:i + 1] for t in (q, k, v, g, beta)), state) for i in range(100, n)]
    compare(torch.cat(outs), state, *want)


def test_prefill_repeats_bit_for_bit_and_in_a_graph():
    x = inputs(15, 333, 4, 8, 128, 128, 2)
    a = run_prefill(x, [300, 33], [0, 1])
    b = run_prefill(x, [300, 33], [0, 1])
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    from reax_engine_runtime_v3_b200 import gated_delta
    q, k, v, g, beta, state = (t.cuda() for t in x)
    cu = torch.tensor([0, 300, 333], dtype=torch.int32).cuda()
    out = torch.empty_like(v)
    graph = torch.cuda.CUDAGraph()
    gated_delta.prefill(q, k, v, g, beta, state.clone(), cu_seqlens=cu)
    with torch.cuda.graph(graph):
        gated_delta.prefill(q, k, v, g, beta, state, cu_seqlens=cu, out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, a[0]) and torch.equal(state, a[1])


def test_long_sequence():
    """1500 rows of one sequence: 24 chunks, the last of 28 rows."""
    x = inputs(16, 1500, 1, 2, 128, 128, 1, g_scale=0.05)
    out, state, spans = run_prefill(x, [1500], [0])
    compare(out, state, *definition(*x, spans, [0]))


def test_more_chunks_than_the_scratch_memory_holds():
    """A batch that takes several launches gives what its sequences give alone, bit for bit."""
    from reax_engine_runtime_v3_b200 import _native, gated_delta
    heads, lens = 512, [2500, 0, 1300, 65]
    n = sum(lens)
    size = _native.load().reax_gdn_workspace_bytes
    assert size(n, len(lens), heads, heads, 128) == size(2 * n, len(lens), heads, heads, 128)     # (one launch holds no more)
    assert size(max(lens), 1, heads, heads, 128) < size(n, len(lens), heads, heads, 128)
    gen = torch.Generator(device="cuda").manual_seed(9)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    q, k, v = rnd(n, heads, 128).bfloat16(), rnd(n, heads, 128).bfloat16(), rnd(n, heads, 64).bfloat16()
    g, beta, state = -torch.rand(n, heads, generator=gen, device="cuda"), torch.rand(n, heads, generator=gen, device="cuda"), \
        rnd(len(lens), heads, 128, 64)
    alone, outs, at = state.clone(), [], 0
    for b, m in enumerate(lens):
        rows = slice(at, at + m)
        if m:
            outs.append(gated_delta.prefill(q[rows], k[rows], v[rows], g[rows], beta[rows], alone[b:b + 1]))
        at += m
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    out = gated_delta.prefill(q, k, v, g, beta, state, cu_seqlens=cu)
    assert torch.equal(out, torch.cat(outs)) and torch.equal(state, alone)


def test_refusals():
    from reax_engine_runtime_v3_b200 import gated_delta
    x = [t.cuda() for t in inputs(17, 4, 2, 4, 128, 128, 4)]
    with pytest.raises(AssertionError, match="bf16"):
        gated_delta.decode(x[0].float(), *x[1:])
    with pytest.raises(AssertionError, match="multiple"):
        gated_delta.decode(*x[:2], x[2][:, :3].contiguous(), x[3][:, :3].contiguous(), x[4][:, :3].contiguous(),
                           x[5][:, :3].contiguous())
    with pytest.raises(AssertionError, match="64 or 128"):
        gated_delta.decode(x[0][:, :, :96], x[1][:, :, :96], *x[2:])
    with pytest.raises(AssertionError, match="fewer states"):
        gated_delta.decode(*x[:5], x[5][:3])
    with pytest.raises(AssertionError, match="slots"):
        gated_delta.decode(*x, slots=torch.arange(4).cuda())
    with pytest.raises(AssertionError, match="one after the other"):
        gated_delta.decode(x[0].transpose(0, 1).contiguous().transpose(0, 1), *x[1:])
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        gated_delta.decode(x[0].cpu(), *x[1:])
    odd = torch.empty(4 * 256 + 4, dtype=torch.bfloat16, device="cuda")[4:].view(4, 2, 128)
    with pytest.raises(RuntimeError, match="status 2"):
        gated_delta.decode(odd, *x[1:])


def test_expired_wait_is_reported_and_the_next_call_is_right():
    """With waits bounded by a nanosecond a block gives up, ends and says so; with the default it works again."""
    from reax_engine_runtime_v3_b200 import _native
    x = inputs(18, 300, 2, 4, 128, 128, 1)
    assert _native.mixer_status(clear=True) == 0
    _native.load().reax_set_wait_timeout_ns(1)
    try:
        run_prefill(x, [300], [0])
        assert _native.mixer_status(clear=True) != 0
    finally:
        _native.load().reax_set_wait_timeout_ns(0)
    out, state, spans = run_prefill(x, [300], [0])
    compare(out, state, *definition(*x, spans, [0]))
    assert _native.mixer_status() == 0


def test_example_runs():
    """The example's prompt and steps through both mixers."""
    import os
    import runpy
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "token_mixers.py")
    outs, state, cached = runpy.run_path(path)["main"]()
    torch.cuda.synchronize()
    assert cached.tolist() == [74, 5, 204] and torch.isfinite(state).all() and state.any()
    for mixed, seen in outs:
        assert torch.isfinite(mixed).all() and torch.isfinite(seen).all() and mixed.any() and seen.any()
