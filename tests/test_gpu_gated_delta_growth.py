"""GPU check of the gated delta rule's prompt form where g is above 0: states may grow up to 2^8 fold within 64 rows (the
room that 16-bit operands leave); the tolerances are those of decays."""
import pytest
import torch

from tests.test_gpu_gated_delta import compare, definition, inputs, run_prefill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fold", [1.0, 100.0, 250.0])
def test_growth(fold):
    """Rows 0 to 63 grow the state evenly, one jump in the next chunk does it at once, decays follow."""
    lens = [200, 64]
    x = inputs(41, sum(lens), 2, 4, 128, 128, 2)
    x[3][:64] = torch.log(torch.tensor(fold)) / 64
    x[3][80], x[3][200:] = torch.log(torch.tensor(fold)), torch.log(torch.tensor(fold)) / 64
    out, state, spans = run_prefill(x, lens, [1, 0])
    compare(out, state, *definition(*x, spans, [1, 0]))
