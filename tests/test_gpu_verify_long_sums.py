"""Verification over a vocabulary of which a thread sums so many terms that the sum's roundings in 32 bits decide for a draft."""
import numpy as np
import pytest
import torch

from test_gpu_verify import call, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("off,count", [(-2.5e-4, 2), (2.5e-4, 1)])
@pytest.mark.parametrize("z", [-0.671875, -0.8515625])
def test_a_draft_near_its_border(z, off, count):
    """65,537 terms a thread where 600 sequences share the device (599 of them without rows), all but the first e^z: each addition is rounded to the same side, 5e-4 of the sum
    (upwards for the first z, downwards for the second), and the draft's number is 2.5e-4 from its probability."""
    run, n = 65537, 600
    vocab = 256 * run
    x = torch.full((2, vocab), z, dtype=torch.bfloat16, device="cuda")
    x[:, ::run] = 0.0
    p = 1.0 / (256 + (vocab - 256) * np.exp(z))
    u = torch.tensor([0.5, p * (1 + off)], dtype=torch.float32, device="cuda")
    assert (float(u[1]) < p) == (count == 2)
    path, got, following = call(x, ints([0, 0]), None, u, first=ints([0] + [2] * n), n_seqs=n)
    assert got[0] == count and (got[1:] == 0).all() and following[0] >= 0
