"""GPU checks of the paged INT8 cache: append and read bit for bit against the rule, attention against its definition
in 64 bits over the cache's values.

Tolerance of the attention's output: half a bf16 unit (2^-9 of the value) for the last rounding, and for the weights,
which are rounded to 11 bits (relative 2^-12), 2^-10 of the same weights' sum of |v|: |error| <= 2^-8 |o| + 2^-10 A with
A = sum p |v|.  Log-sum-exp (float32): scores are float32 sums of up to 256 products, so 1e-5 (1 + |lse|).
"""
import math

import numpy as np
import pytest
import torch

from tests import helpers as H

pytestmark = pytest.mark.gpu


def filled(seed, lens, heads, dim, page, spare=3, width=0):
    """A cache whose pages hold random codes and scales, scattered tables for `lens` rows each."""
    from reax_engine_runtime_v3_b200.kv_int8 import Int8Cache
    gen = H.gen(seed)
    per = [-(-n // page) for n in lens]
    pages = sum(per) + spare
    ids = torch.randperm(pages, generator=gen, dtype=torch.int64)
    tables = torch.full((len(lens), max(max(per), width, 1)), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(per):
        tables[b, :m] = ids[at:at + m]
        at += m
    codes = [torch.randint(-127, 128, (pages, heads, page, dim), generator=gen, dtype=torch.int32).to(torch.int8) for _ in "kv"]
    scales = [(0.5 + torch.rand(pages, heads, generator=gen)) / 127 for _ in "kv"]
    return Int8Cache(*(t.cuda() for t in (*codes, *scales))), tables


def values(cache, tables, b, n):
    """Sequence b's first n rows as float64 [n, heads, dim] k and v."""
    pages = tables[b, :-(-n // cache.page)].long()
    out = []
    for codes, scales in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = codes.cpu()[pages].double() * scales.cpu()[pages].double()[..., None, None]
        out.append(x.transpose(1, 2).reshape(-1, cache.heads, cache.dim)[:n])
    return out


def offsets(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32)


def attention(q, cache, tables, rows, lens, scale):
    outs, sizes, lses, at = [], [], [], 0
    group = q.shape[1] // cache.heads
    for b, (n, length) in enumerate(zip(rows, lens)):
        k, v = values(cache, tables, b, length)
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        s = torch.einsum("nhd,lhd->hnl", q[at:at + n].double(), k) * scale
        seen = torch.arange(length)[None] <= length - n + torch.arange(n)[:, None]
        s = s.masked_fill(~seen, -math.inf)
        lse = torch.logsumexp(s, -1)
        p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None])
        outs.append(torch.einsum("hnl,lhd->nhd", p, v))
        sizes.append(torch.einsum("hnl,lhd->nhd", p, v.abs()))
        lses.append(lse.T)
        at += n
    return torch.cat(outs), torch.cat(sizes), torch.cat(lses)


def check_attend(cache, tables, rows, lens, group, seed=0, q_scale=1.0, scale=None, **kw):
    q = (torch.randn(sum(rows), cache.heads * group, cache.dim, generator=H.gen(seed)) * q_scale).bfloat16()
    scale_ = cache.dim ** -0.5 if scale is None else scale
    want, size, want_lse = attention(q, cache, tables, rows, lens, scale_)
    out, lse = cache.attend(q.cuda(), tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                            cu_seqlens=offsets(rows).cuda(), scale=scale, return_lse=True, **kw)
    torch.cuda.synchronize()
    err = (out.cpu().double() - want).abs()
    excess = err - (want.abs() * 2.0 ** -8 + size * 2.0 ** -10)
    assert torch.isfinite(out).all() and (excess <= 1e-30).all(), f"off by {err.max():.3g}, beyond by {excess.max():.3g}"
    empty = want_lse == -math.inf
    got = lse.cpu().double()
    assert torch.equal(got == -math.inf, empty)
    assert ((got - want_lse).abs()[~empty] <= 1e-5 * (1 + want_lse.abs()[~empty])).all()
    return out, lse


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("group", [1, 3, 4, 8, 16])
def test_attend_step(dim, page, group):
    lens = [1, 15, 16, 17, 64, 65, 333]
    cache, tables = filled(dim + page + group, lens, 2, dim, page)
    check_attend(cache, tables, [1] * len(lens), lens, group, max_rows=1)


@pytest.mark.parametrize("rows,lens", [([1], [5000]), ([1, 1], [1, 9000]), ([1] * 40, [(37 * i) % 700 + 1 for i in range(40)]),
                                       ([2, 0, 3, 1], [2, 10, 700, 0])])
def test_attend_few_rows(rows, lens):
    """One long context (split over many blocks), ragged batches, a sequence without rows, one without a cache."""
    cache, tables = filled(sum(lens), lens, 4, 128, 64)
    check_attend(cache, tables, rows, lens, 4, seed=1)


@pytest.mark.parametrize("dim,page,heads,group", [(64, 16, 3, 2), (128, 32, 2, 8), (256, 64, 2, 4), (256, 16, 1, 1), (128, 64, 1, 5)])
@pytest.mark.parametrize("rows,lens", [([70], [70]), ([33, 129, 1], [40, 500, 77]), ([200, 5], [1200, 5])])
def test_attend_many_rows(dim, page, heads, group, rows, lens):
    cache, tables = filled(dim + sum(rows), lens, heads, dim, page)
    check_attend(cache, tables, rows, lens, group, seed=2)


def test_attend_rows_that_see_nothing():
    """More query rows than cached rows: the first ones see none."""
    lens, rows = [5, 0, 100], [9, 4, 130]
    cache, tables = filled(5, lens, 2, 128, 16)
    out, lse = check_attend(cache, tables, rows, lens, 4, seed=3)
    assert not out[:4].any() and (lse[:4] == -math.inf).all() and not out[9:13].any()


@pytest.mark.parametrize("heads,group,rows,lens", [
    (1, 4, [(5 * i) % 9 + 1 for i in range(300)], [(37 * i) % 150 + 9 for i in range(300)]),    # more sequences than are counted at once
    (3, 1, [17] * 50, [17] * 50),                                                                # items of a tile each
    (2, 4, [0, 40, 0, 0, 25, 0], [10, 900, 0, 64, 25, 3]),                                       # sequences without rows
    (1, 2, [20], [30000]),                                                                       # one item for all blocks
    (2, 5, [131, 3], [2500, 4000]),
])
def test_attend_blocks_share_the_tiles(heads, group, rows, lens):
    cache, tables = filled(len(rows), lens, heads, 128, 32)
    check_attend(cache, tables, rows, lens, group, seed=8, max_rows=1000)


def test_attend_hint_does_not_change_results_beyond_rounding():
    """Every value of the hint has to be right, a wrong one too."""
    lens, rows = [300, 64, 1], [20, 3, 1]
    cache, tables = filled(6, lens, 2, 256, 64)
    for hint in (1, 3, 20, 1000):
        check_attend(cache, tables, rows, lens, 4, seed=4, max_rows=hint)


def test_attend_large_scores_and_scale():
    """Scores in the hundreds (one row takes nearly all the weight) and a scale of the caller's."""
    lens = [700, 31]
    cache, tables = filled(7, lens, 2, 128, 32)
    check_attend(cache, tables, [1, 1], lens, 8, seed=5, q_scale=30.0, max_rows=1)
    check_attend(cache, tables, [40, 20], lens, 8, seed=5, q_scale=30.0)
    check_attend(cache, tables, [40, 20], lens, 2, seed=6, scale=0.01)


def test_attend_pages_of_unlike_scales_and_zeros():
    """Pages whose scales differ by 2^20, and pages of zeros with the least scale."""
    lens = [640]
    for rows in ([1], [50]):
        cache, tables = filled(8, lens, 2, 128, 64)
        cache.v_scale[tables[0, 2].item()] *= 2.0 ** 10
        cache.v_scale[tables[0, 5].item()] *= 2.0 ** -10
        cache.v_scale[tables[0, 7].item()] = 1e-12 / 127
        cache.k_scale[tables[0, 3].item()] = 1e-12 / 127
        cache.v[tables[0, 7].item()] = 0
        cache.k[tables[0, 3].item()] = 0
        check_attend(cache, tables, rows, lens, 4, seed=9)


def test_attend_unused_places_do_not_matter():
    """What lies in a page behind the last row (NaN scales in unused pages among it) is not used."""
    lens = [70, 9]
    cache, tables = filled(9, lens, 2, 256, 16, width=12)
    q = torch.randn(5, 8, 256, generator=H.gen(1)).bfloat16().cuda()
    cu, ln = torch.tensor([0, 3, 5], dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    for hint in (3, 200):
        a = cache.attend(q, tables.cuda(), ln, cu_seqlens=cu, max_rows=hint)
        used = set(tables[0, :5].tolist() + tables[1, :1].tolist())
        for p in range(cache.pages):
            if p not in used:
                cache.k_scale[p], cache.v_scale[p] = math.nan, math.inf
                cache.k[p], cache.v[p] = 127, -128
        cache.k[tables[0, 4].item(), :, 6:], cache.v[tables[0, 4].item(), :, 6:] = 127, 127
        more = tables.clone()
        more[0, 5:], more[1, 1:] = 1 << 30, -7
        b = cache.attend(q, more.cuda(), ln, cu_seqlens=cu, max_rows=hint)
        torch.cuda.synchronize()
        assert torch.equal(a, b)


def test_attend_repeats_bit_for_bit_strided_in_a_graph_and_on_streams():
    lens = [3000, 40, 900]
    cache, tables = filled(10, lens, 2, 128, 64)
    gen = H.gen(2)
    row = torch.randn(3, 8 * 128 + 64, generator=gen).bfloat16().cuda()
    q = row[:, :8 * 128].view(3, 8, 128)
    t, ln = tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    first = cache.attend(q.contiguous(), t, ln)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for i in range(10):
        with torch.cuda.stream(streams[i % 2]):
            got.append(cache.attend(q, t, ln))
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for x in got)
    out = torch.empty_like(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(q, t, ln, out=out)
    ln.copy_(torch.tensor([100, 3, 1], dtype=torch.int32))             # replay with other lengths
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, cache.attend(q, t, ln))


# ------------------------------------------------------------------------------------------------ append, read
def append_rule(codes, scales, x, tables, lens, rows, page):
    """The rule in float32 numpy, on copies."""
    codes, scales = codes.cpu().numpy().copy(), scales.cpu().numpy().copy()
    x = x.float().numpy()
    f = np.float32
    at = 0
    for b, n in enumerate(rows):
        done = 0
        while done < n:
            pos = lens[b] + done
            take = min(n - done, page - pos % page)
            if pos // page < tables.shape[1]:
                pid, off = int(tables[b, pos // page]), pos % page
                for h in range(codes.shape[1]):
                    new = x[at + done:at + done + take, h]
                    finite = np.abs(new[np.isfinite(new)])
                    top = f(max(finite.max() if finite.size else f(0), f(1e-12)))
                    was = scales[pid, h] if off else f(0)
                    now = max(was, f(top / f(127)))
                    if off and now > was:
                        old = codes[pid, h, :off].astype(f) * f(was / now)
                        codes[pid, h, :off] = np.rint(old).astype(np.int8)
                    scales[pid, h] = now
                    with np.errstate(invalid="ignore"):
                        c = np.clip(np.rint(new / now), -127, 127)
                    codes[pid, h, off:off + take] = np.nan_to_num(c, nan=0.0).astype(np.int8)
            done += take
        at += n
    return codes, scales


@pytest.mark.parametrize("dim,page,heads", [(64, 16, 1), (128, 32, 3), (256, 64, 2)])
@pytest.mark.parametrize("lens,rows", [([0], [1]), ([5, 64, 63, 200], [1, 1, 1, 1]), ([0, 3, 16, 100, 7], [130, 0, 64, 61, 9]),
                                       ([31] * 70, [2] * 70)])
def test_append_and_read(dim, page, heads, lens, rows):
    total = [a + b for a, b in zip(lens, rows)]
    cache, tables = filled(dim + sum(lens), total, heads, dim, page)
    gen = H.gen(sum(rows))
    k, v = ((torch.randn(sum(rows), heads, dim, generator=gen) * torch.exp(torch.randn(sum(rows), heads, 1, generator=gen))
             ).bfloat16() for _ in "kv")
    if sum(rows) > 20:
        k[3, 0, 5], k[4, 0, 6], v[6, 0, 1], v[7] = math.inf, -math.inf, math.nan, 0
    want = [append_rule(c, s, x, tables, lens, rows, page) for c, s, x in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v))]
    cu = None if all(n == 1 for n in rows) else offsets(rows).cuda()
    cache.append(k.cuda(), v.cuda(), tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), cu_seqlens=cu)
    torch.cuda.synchronize()
    for (codes, scales), c, s in zip(want, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        assert np.array_equal(s.cpu().numpy(), scales) and np.array_equal(c.cpu().numpy(), codes)
    starts = [n // 2 for n in lens]
    counts = [t - s for t, s in zip(total, starts)]
    got = cache.read(tables.cuda(), torch.tensor(starts, dtype=torch.int32).cuda(), offsets(counts).cuda(), sum(counts))
    torch.cuda.synchronize()
    for x, (codes, scales) in zip(got, want):
        rows_ = []
        for b in range(len(lens)):
            i = np.arange(starts[b], total[b])
            pid = tables[b].numpy()[i // page]
            rows_.append(codes[pid, :, i % page].astype(np.float32) * scales[pid][..., None])
        assert torch.equal(x.cpu(), torch.from_numpy(np.concatenate(rows_)).bfloat16())


def test_append_past_the_table_and_unknown_pages_write_nothing_else():
    cache, tables = filled(20, [40], 2, 64, 16)
    tables[0, 1] = 1 << 20
    before = cache.k.clone(), cache.v.clone()
    k = torch.ones(40, 2, 64, dtype=torch.bfloat16, device="cuda")
    cache.append(k, k, tables.cuda(), torch.tensor([12], dtype=torch.int32).cuda(), cu_seqlens=offsets([40]).cuda())
    got = cache.read(tables.cuda(), torch.tensor([10], dtype=torch.int32).cuda(), offsets([100]).cuda(), 100)[0]
    torch.cuda.synchronize()
    touched = tables[0, [0, 2]].tolist()
    for p in range(cache.pages):
        if p not in touched:
            assert torch.equal(cache.k[p], before[0][p]) and torch.equal(cache.v[p], before[1][p])
    assert not got[6:22].any() and not got[38:].any()


def test_offsets_past_32_bits():
    """A pool of more than 2^32 codes: the pages at its end are written and read at their place."""
    from reax_engine_runtime_v3_b200.kv_int8 import Int8Cache
    heads, page, dim = 4, 64, 256
    pages = (1 << 32) // (heads * page * dim) + 3
    cache = Int8Cache.empty(pages, heads, dim, page)
    x = torch.randn(70, heads, dim, generator=H.gen(3)).bfloat16()
    tables = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32)
    cache.append(x.cuda(), x.cuda(), tables.cuda(), torch.zeros(1, dtype=torch.int32).cuda(), cu_seqlens=offsets([70]).cuda())
    assert not cache.k[:4].any()
    back = cache.read(tables.cuda(), torch.zeros(1, dtype=torch.int32).cuda(), offsets([70]).cuda(), 70)[0]
    assert (back.cpu().float() - x.float()).abs().max() < 0.04
    small = Int8Cache(*(t[pages - 2:].contiguous() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)))
    for rows in (1, 70):
        q = torch.randn(rows, heads * 4, dim, generator=H.gen(4)).bfloat16().cuda()
        arg = dict(cu_seqlens=offsets([rows]).cuda(), max_rows=rows)
        ln = torch.tensor([70], dtype=torch.int32).cuda()
        a = cache.attend(q, tables.cuda(), ln, **arg)
        b = small.attend(q, torch.tensor([[1, 0]], dtype=torch.int32).cuda(), ln, **arg)
        torch.cuda.synchronize()
        assert torch.equal(a, b)


def test_refusals():
    from reax_engine_runtime_v3_b200.kv_int8 import Int8Cache
    cache, tables = filled(30, [40, 40], 2, 64, 16)
    t, ln = tables.cuda(), torch.tensor([40, 40], dtype=torch.int32).cuda()
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(AssertionError, match="pages have"):
        Int8Cache.empty(4, 2, 64, page=48)
    with pytest.raises(AssertionError, match="heads"):
        Int8Cache.empty(4, 2, 80)
    with pytest.raises(AssertionError, match="multiple of the cached heads"):
        cache.attend(q[:, :3], t, ln)
    with pytest.raises(AssertionError, match="bf16"):
        cache.attend(q.float(), t, ln)
    with pytest.raises(AssertionError, match="lengths"):
        cache.attend(q, t, ln.long())
    with pytest.raises(AssertionError, match="one row"):
        cache.attend(q[:1], t, ln)
    with pytest.raises(AssertionError, match="the same rows"):
        cache.append(q[:, :2], q[:1, :2], t, ln)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        cache.attend(q.cpu(), t, ln)
    odd = torch.empty(2 * 256 + 4, dtype=torch.bfloat16, device="cuda")[4:].view(2, 4, 64)
    with pytest.raises(RuntimeError, match="status 2"):
        cache.attend(odd, t, ln)
