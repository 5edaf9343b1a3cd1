"""GPU check of a table so wide that its rows pass 32 bits: what it can hold must not wrap around."""
import pytest
import torch

from tests.test_gpu_kv_int8 import filled

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hint", [1, 100])
def test_attend(hint):
    cache, tables = filled(1, [300], 2, 128, 64)
    wide = torch.full((1, (1 << 31) // 64 + 8), -1, dtype=torch.int32, device="cuda")
    wide[:, :tables.shape[1]] = tables.cuda()
    q = torch.randn(3, 4, 128, device="cuda").bfloat16()
    arg = dict(cu_seqlens=torch.tensor([0, 3], dtype=torch.int32, device="cuda"), max_rows=hint, return_lse=True)
    ln = torch.tensor([300], dtype=torch.int32, device="cuda")
    want, got = cache.attend(q, tables.cuda(), ln, **arg), cache.attend(q, wide, ln, **arg)
    torch.cuda.synchronize()
    assert want[0].any() and torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
