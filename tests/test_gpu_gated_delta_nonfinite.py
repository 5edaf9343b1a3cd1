"""GPU checks of the gated delta rule's prompt form where a value is not finite.

By the definition, row by row, a value that is not finite in row j touches no row before j: in v it spoils its column of the
state, in k, g or beta the whole state of the heads that read it, and with the state every output from row j on; in q only
row j's outputs.  What it does not touch keeps the tolerances that hold without it (state: 8e-6 of a head's 2-norm; output:
2^-8 of itself and of its row's root mean square).
"""
import math

import pytest
import torch

from tests.test_gpu_gated_delta import definition, inputs, run_prefill

pytestmark = pytest.mark.gpu

HK, HV, D = 2, 4, 128
LENS = [150, 70, 3]


def check(x, spoil, rows, columns, heads, slot_bad=True, lens=LENS, dv=D, **kw):
    """Runs x with `spoil` applied; rows `rows`, columns `columns` of value heads `heads` must not be finite, nor the state
    of those heads and columns of sequence 0 (`slot_bad`); all else is as defined."""
    x = [t.clone() for t in x]
    clean = definition(*x, *_spans(lens), **kw)
    spoil(x)
    out, state, spans = run_prefill(x, lens, list(range(len(lens))), **kw)
    out, state = out.cpu().double(), state.cpu().double()
    bad = torch.zeros(out.shape, dtype=torch.bool)
    for r in rows:
        for h in heads:
            bad[r, h, columns] = True
    bad_state = torch.zeros(state.shape, dtype=torch.bool)
    if slot_bad:
        for h in heads:
            bad_state[0, h, :, columns] = True
    assert not out[bad].isfinite().any() and not state[bad_state].isfinite().any()
    assert out[~bad].isfinite().all() and state[~bad_state].isfinite().all()
    want, want_state = (torch.where(b, 0.0, y) for b, y in zip((bad, bad_state), clean))
    out, state = torch.where(bad, 0.0, out), torch.where(bad_state, 0.0, state)
    error, size = (state - want_state).flatten(2).norm(dim=-1), want_state.flatten(2).norm(dim=-1)
    assert (error <= 8e-6 * size + 1e-30).all(), f"state error {(error / size.clamp(min=1e-30)).max():.2e}"
    rms = clean[0].square().mean(-1, keepdim=True).sqrt()
    excess = (out - want).abs() - (want.abs() + rms) * 2.0 ** -8
    assert (excess <= 1e-30).all(), f"output beyond its bound by {excess.max():.3g}"


def _spans(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return list(zip(at, at[1:])), range(len(lens))


# rows of sequence 0: the first, either half of a chunk, a chunk's first, the last
ROWS = pytest.mark.parametrize("row", [0, 37, 64, 73, 101, 149])


@ROWS
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dv", [64, 128])
def test_v(row, value, dv):
    def spoil(x):
        x[2][row, 2, 5] = value
    check(inputs(31 + row, sum(LENS), HK, HV, D, dv, 3), spoil, range(row, 150), [5], [2], dv=dv)


@ROWS
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("normalize", [True, False])
def test_k(row, value, normalize):
    def spoil(x):
        x[1][row, 1, 77] = value
    check(inputs(32 + row, sum(LENS), HK, HV, D, D, 3, normalize=normalize), spoil, range(row, 150), slice(None), [2, 3],
          normalize=normalize)


@ROWS
@pytest.mark.parametrize("which,value", [("g", math.nan), ("g", math.inf), ("beta", math.nan), ("beta", math.inf)])
def test_g_and_beta(row, which, value):
    def spoil(x):
        x[3 if which == "g" else 4][row, 1] = value
    check(inputs(33 + row, sum(LENS), HK, HV, D, D, 3), spoil, range(row, 150), slice(None), [1])


@ROWS
@pytest.mark.parametrize("value", [math.nan, -math.inf])
def test_q(row, value):
    def spoil(x):
        x[0][row, 0, 9] = value
    check(inputs(34 + row, sum(LENS), HK, HV, D, D, 3), spoil, [row], slice(None), [0, 1], slot_bad=False)


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_state(value):
    """A column of the state that comes in is not finite: its outputs are not from the first row on."""
    def spoil(x):
        x[5][0, 3, 100, 7] = value
    check(inputs(35, sum(LENS), HK, HV, D, D, 3), spoil, range(150), [7], [3])


def test_several_rows_and_heads():
    """Each head and column goes by its own first row."""
    x = inputs(36, sum(LENS), HK, HV, D, D, 3)
    x[2][90, 0, 3] = x[2][100, 0, 3] = x[2][80, 0, 4] = math.nan
    x[4][70, 3] = math.nan
    out, state, _ = run_prefill(x, LENS, [0, 1, 2])
    fine = out.cpu().isfinite()
    bad = torch.zeros_like(fine)
    bad[90:150, 0, 3] = bad[80:150, 0, 4] = bad[70:150, 3] = True
    assert torch.equal(fine, ~bad)
    fine = state.cpu().isfinite()
    bad = torch.zeros_like(fine)
    bad[0, 0, :, 3] = bad[0, 0, :, 4] = bad[0, 3] = True
    assert torch.equal(fine, ~bad)


@pytest.mark.parametrize("form", ["prefill", "decode"])
def test_rows_whose_squares_pass_float32(form):
    """Normalizing such a row must not turn it into zeros: its outputs, and of k the state, are not finite."""
    from reax_engine_runtime_v3_b200 import gated_delta
    x = inputs(37, 3, 2, 2, D, D, 3)
    x[0][0, 0] *= 2.0 ** 70
    x[1][1, 1] *= 2.0 ** 70
    on = [t.cuda() for t in x]
    if form == "decode":
        out = gated_delta.decode(*on)
    else:
        out = gated_delta.prefill(*on, cu_seqlens=torch.arange(4, dtype=torch.int32).cuda())
    out, state = out.cpu().isfinite(), on[5].cpu().isfinite()
    for fine, row, head in ((out, 0, 0), (out, 1, 1), (state, 1, 1)):
        assert not fine[row, head].any()
        fine[row, head] = True
    assert out.all() and state.all()
