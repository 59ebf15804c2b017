"""A decode step of more than 32 sequences: its products are a chunk's, everything around them the step's own, with the bounds of the narrower ones."""
import pytest

from test_gpu_decoder import LOGIT_REL_TOL, _run
from torq_b200.runtime import Executable
from torq_b200.workloads import gemma3

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch", [33, 70])
def test_a_decode_step_of_many_sequences(device, batch):
    ex = Executable(device, gemma3.build_decode_step(gemma3.SMALL, batch, gemma3.random_weights(gemma3.SMALL, 1, 0.3)).serialize())
    kernels = ex.op_kernels()
    ex.destroy()
    assert "linear_rows" in kernels and not any("linear_w8" in k for k in kernels)
    worst, exact, near_tie, wrong, _ = _run(device, gemma3.SMALL, batch, 6, 6, embed_gain=0.3)
    assert worst <= LOGIT_REL_TOL and wrong == 0 and exact > 0, (worst, exact, near_tie, wrong)
