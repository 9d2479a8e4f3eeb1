"""8-bit KV rows of values near the smallest that fp32 and bf16 hold."""
import numpy as np
import pytest

from gpu_util import torch_cuda
from test_gpu_kv_quant import _append, _torch_type

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("d", [128, 33])
def test_rows_of_tiny_values(kind, name, d):
    """Codes are x * M / absmax to nearest, also where M / absmax is past fp32."""
    torch = torch_cuda()
    rng = np.random.default_rng(d)
    sizes = np.array([1e-34, 1.1e-35, 9e-36, 1e-36, 1e-37, 1e-38, 1e-39])
    x = torch.from_numpy((rng.uniform(-1, 1, (7, 2, d)) * sizes[:, None, None]).astype(np.float32))
    x = x.to(_torch_type(torch, name)).cuda()
    kc, ks, vc, vs = _append(torch, x, x.flip(0), None, 7, kind, name)
    most = 448.0 if kind == "fp8" else 127.0
    for y, codes, scales in ((x, kc, ks), (x.flip(0), vc, vs)):
        y = y.double()
        top = y.abs().amax(-1, keepdim=True)
        want = y * (most / top)
        got = codes.view(torch.float8_e4m3fn).double() if kind == "fp8" else codes.view(torch.int8).double()
        # half a step of the code, and what x, M / absmax and their product lose
        half = torch.clamp(want.abs() * 2.0 ** -4, min=2.0 ** -10) if kind == "fp8" else 0.5
        assert ((got - want).abs() <= half + want.abs() * 2.0 ** -22).all()
        # a quotient of tensors: torch multiplies by the reciprocal of a number
        assert torch.equal(scales, (top.float() / torch.full_like(top, most, dtype=torch.float32)).squeeze(-1))
