"""GPU check of the bounded waits in attention of many rows: an expired one is reported, and the call after it is right."""
import pytest
import torch

from tests import helpers as H
from tests.test_gpu_kv_int8 import filled, offsets

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,lens", [([40], [3000]), ([300, 200], [3000, 500])])
def test_expired_wait_is_reported_and_the_next_call_is_right(dim, rows, lens):
    """With waits bounded by a nanosecond blocks give up, end and say so, the join of what they left included."""
    from reax_engine_runtime_v3_b200 import _native
    cache, tables = filled(dim, lens, 2, dim, 64)
    q = torch.randn(sum(rows), 8, dim, generator=H.gen(1)).bfloat16().cuda()
    arg = q, tables.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    want = cache.attend(*arg, cu_seqlens=offsets(rows).cuda(), return_lse=True)
    assert _native.mixer_status(clear=True) == 0
    _native.load().reax_set_wait_timeout_ns(1)
    try:
        cache.attend(*arg, cu_seqlens=offsets(rows).cuda())
        assert _native.mixer_status(clear=True) != 0
    finally:
        _native.load().reax_set_wait_timeout_ns(0)
    got = cache.attend(*arg, cu_seqlens=offsets(rows).cuda(), return_lse=True)
    assert _native.mixer_status() == 0
    assert all(torch.equal(a, b) for a, b in zip(want, got))
