"""The serving operators at the edges of what they take, on the GPU.  Tolerances as in
test_paged_gpu.py and test_logprobs_gpu.py."""
import pytest
import torch

import lucid_b200 as lb
from lucid_b200 import _lib
from test_paged_gpu import check_attention, check_step, make, run_attention, run_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", range(4, 128, 8))
@pytest.mark.parametrize("Hq", [2, 16])
def test_dense_rows_on_8_byte_boundaries(cuda_device, D, Hq):
    """Pages of dense rows of every odd multiple of 4, used up to the pool's last row; the
    values that follow a row in memory are the next one's."""
    s = make(cuda_device, [96, 31, 160], Hq, 2, D, 32, seed=D, spare=0, room=0)
    assert s["kp"].is_contiguous() and s["table"].max() == s["kp"].shape[0] - 1
    check_step(s, *run_step(s, append=False))
    check_attention(s, run_attention(s))
    _lib.check_status()
