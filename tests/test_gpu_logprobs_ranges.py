"""Log probabilities at the ends of the temperature's range."""
import math

import numpy as np
import pytest

from gpu_util import torch_cuda
from test_gpu_logprobs import SUM, _call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 700])
@pytest.mark.parametrize("inv_t", [1e30, 2.0 ** 127, 3.4e38])
def test_temperatures_near_zero(rows, inv_t):
    """All of the probability goes to the largest logits: two of them share it, any other token's is 0."""
    torch = torch_cuda()
    x = torch.linspace(-4, 3, 9001, device="cuda").repeat(rows, 1)
    x[:, 40], x[:, 7000] = 3.5, 3.5
    tokens = torch.tensor([[7000, 0]] * rows, dtype=torch.int32, device="cuda")
    got = _call(torch, x, "f32", tokens, 2, inv_t=inv_t)
    assert (got["ids"] == [40, 7000]).all()
    for a in (got["lp"][:, 0], got["top"][:, 0], got["top"][:, 1], -got["h"]):
        assert np.abs(a + math.log(2)).max() <= SUM
    # 7.5 * inv_t, past fp32 in the larger two
    assert (got["lp"][:, 1] == -np.inf).all() if inv_t > 1e38 else np.allclose(got["lp"][:, 1], -7.5 * inv_t, rtol=1e-6)


@pytest.mark.parametrize("inv_t", [1e-30, 1e-6])
def test_temperatures_near_infinity(inv_t):
    """All tokens are alike."""
    torch = torch_cuda()
    x = torch.linspace(-4, 3, 9001, device="cuda").view(1, -1)
    got = _call(torch, x, "f32", torch.tensor([[0, 9000]], dtype=torch.int32, device="cuda"), 1, inv_t=inv_t)
    assert np.abs(got["lp"] + math.log(9001)).max() <= SUM + 7 * inv_t and abs(got["h"][0] - math.log(9001)) <= 2 * SUM + 7 * inv_t
    assert got["ids"][0, 0] == 9000
