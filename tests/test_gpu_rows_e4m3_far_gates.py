"""Gates far from zero as 8-bit rows: the values, not the scales alone, against the formula in 64 bits, with the bound of test_gpu_rows_e4m3.py.

Between -87.3 and -88.7 exp(-g) is a 32-bit number whose reciprocal is below 2^-126; beside a large enough up the product counts all the same.
Below -88.7 exp(-g) leaves 32 bits and silu(g) counts as 0, as in any 32-bit form of it; the ups here make nothing of that visible."""
import pytest
import torch

from test_gpu_rows_e4m3 import D_GATE, DEV, _check, _places, ops  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]


def _gated(ops, gate, up, dtype, size):  # noqa: F811
    """Rows that repeat these pairs over `size` columns; their 8-bit rows and the exact ones."""
    times = -(-size // len(gate))
    x = torch.cat([torch.tensor(v).repeat(times)[:size] for v in (gate, up)]).to(dtype).to(DEV).repeat(3, 1)
    q, scales = _places(3, size)
    ops.swiglu_e4m3(x, q, scales)
    g, u = x.double().chunk(2, 1)
    # silu of far gates in a form that does not overflow; what is below 2^-1074 is zero
    h = g * torch.exp(torch.clamp(g, max=0.0)) / (1.0 + torch.exp(-g.abs())) * u
    return h, q, scales


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [2, 64, 1030, 4096, 10241])
@pytest.mark.parametrize("gate,up", [([-200.0, -1e30], [1e30, 0.0]), ([1e4, 1e4], [1e4, 1e4]), ([1e30, -1e30], [0.5, 3.0]), ([0.0, -0.0], [1e30, 5.0]),
                                     ([-87.0, -86.5], [1e20, 1e20]), ([-88.0, -88.5], [1e20, -2e20]), ([-87.5, -40.0], [1e30, 1e10]),
                                     ([-88.5, -89.5], [1e25, 1.0]), ([3e38, -20.0], [0.25, 1e30])])
def test_far_gates(ops, dtype, size, gate, up):  # noqa: F811
    h, q, scales = _gated(ops, gate, up, dtype, size)
    _check(h, q, scales, D_GATE)
