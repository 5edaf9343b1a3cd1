"""GPU checks of attention over the INT8 cache where a query row or a scale is not finite.

The rule, the same whichever form the hint picks: a row that holds a NaN or an infinity, or that sees a place of a page whose
scale of k or v is one, comes out as NaN, its log-sum-exp too; a row that sees nothing gives zeros and -inf whatever it holds;
every other row comes out as it does without them, bit for bit (rows share tiles, but no arithmetic).
"""
import math

import pytest
import torch

from tests import helpers as H
from tests.test_gpu_kv_int8 import filled, offsets

pytestmark = pytest.mark.gpu

FORMS = pytest.mark.parametrize("hint", [1, 1000])            # the form of a step, that of many rows
SIZES = pytest.mark.parametrize("dim,page,heads,group", [(64, 16, 2, 2), (128, 32, 1, 4), (256, 64, 2, 4)])


def attend(cache, tables, rows, lens, q, hint):
    out, lse = cache.attend(q.cuda(), tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                            cu_seqlens=offsets(rows).cuda(), max_rows=hint, return_lse=True)
    torch.cuda.synchronize()
    return out.cpu(), lse.cpu()


def check(clean, spoilt, bad):
    """`bad` [rows, heads]: NaN there, and elsewhere as without."""
    assert clean[0].isfinite().all()
    assert spoilt[0][bad].isnan().all() and spoilt[1][bad].isnan().all()
    assert torch.equal(spoilt[0][~bad], clean[0][~bad]) and torch.equal(spoilt[1][~bad], clean[1][~bad])


# few rows of short sequences; a context that many blocks share; many rows, of which the last of one sequence share a tile
SPANS = pytest.mark.parametrize("rows,lens", [([1, 1, 3], [1, 70, 333]), ([2], [9000]), ([70, 40], [70, 500])])


@FORMS
@SIZES
@SPANS
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_query_rows(hint, dim, page, heads, group, rows, lens, value):
    cache, tables = filled(dim + sum(lens), lens, heads, dim, page)
    q = torch.randn(sum(rows), heads * group, dim, generator=H.gen(1)).bfloat16()
    clean = attend(cache, tables, rows, lens, q, hint)
    bad = torch.zeros(sum(rows), heads * group, dtype=torch.bool)
    for row, head, at in ((0, heads * group - 1, 3), (sum(rows) - 1, 0, dim - 1), (sum(rows) // 2, 1, dim // 2)):
        q[row, head, at] = value
        bad[row, head] = True
    check(clean, attend(cache, tables, rows, lens, q, hint), bad)


@FORMS
@SIZES
@SPANS
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_scales_of_pages_that_are_seen(hint, dim, page, heads, group, rows, lens, which, value):
    """The last page of the longest sequence, one cached head: its rows from the first that sees the page on."""
    cache, tables = filled(dim + sum(lens), lens, heads, dim, page)
    q = torch.randn(sum(rows), heads * group, dim, generator=H.gen(2)).bfloat16()
    clean = attend(cache, tables, rows, lens, q, hint)
    b = max(range(len(lens)), key=lambda i: lens[i])
    last = (lens[b] - 1) // page
    getattr(cache, which)[tables[b, last].item(), heads - 1] = value
    bad = torch.zeros(sum(rows), heads * group, dtype=torch.bool)
    first = max(last * page - (lens[b] - rows[b]), 0)          # row i sees places up to lens - rows + i
    bad[sum(rows[:b]) + first:sum(rows[:b + 1]), (heads - 1) * group:] = True
    check(clean, attend(cache, tables, rows, lens, q, hint), bad)


@FORMS
def test_rows_that_see_nothing_and_all_rows(hint):
    """More rows than are cached: the first see none and stay zeros; then every row of a batch is NaN."""
    rows, lens = [9, 40], [5, 30]
    cache, tables = filled(3, lens, 2, 128, 16)
    q = torch.full((49, 8, 128), math.nan, dtype=torch.bfloat16)
    out, lse = attend(cache, tables, rows, lens, q, hint)
    none = torch.zeros(49, dtype=torch.bool)
    none[:4] = none[9:19] = True
    assert not out[none].any() and (lse[none] == -math.inf).all()
    assert out[~none].isnan().all() and lse[~none].isnan().all()
