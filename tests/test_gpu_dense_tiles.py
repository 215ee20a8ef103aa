"""The linear operator's product kernel as CTA pairs."""
import pytest
import torch

import granulelayer_b200 as gl
from test_gpu_dense import BF16, data

pytestmark = pytest.mark.gpu


def test_many_pair_launches_in_a_row():
    """Launches back to back on one stream, each as the first: a CTA that left too early would leave its partner, or the
    next launch, with something unfinished."""
    x, w = data(512, 1024, dtype=BF16, seed=1), data(4096, 1024, dtype=BF16, seed=2, scale=0.03)
    with torch.no_grad():
        want = gl.linear_act(x, w)
        got = [gl.linear_act(x, w) for _ in range(200)]
    assert all(torch.equal(g, want) for g in got)
