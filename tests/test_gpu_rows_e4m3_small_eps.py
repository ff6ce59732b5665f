"""The norm's 8-bit rows with an eps so small that 1 / sqrt(mean + eps) is large: rows near zero.

With eps = 1e-12 that root's reciprocal is 1e6 in a row of zeros, and over the least scale, 2^-100 / 448 = 1.76e-33, it would be above the
largest 32-bit number; with smaller eps it is so for rows whose scale is not the least, too.  The bounds are those of test_gpu_rows_e4m3.py, whose norm
takes a product less: the factor is taken in two parts here, one rounding more, 74 half steps."""
import pytest
import torch

from test_gpu_rows_e4m3 import DEV, F8, _check, _norm, _places, _rand, ops  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
D = 74 * 2.0 ** -24


@pytest.mark.parametrize("size", [1, 7, 64, 96, 1030, 4096, 10242, 10241, 30728, 31000])          # a warp a row, a block, pieces of two, the long kernel by two and one
@pytest.mark.parametrize("eps", [1e-6, 1e-12, 1e-13, 1e-15, 1e-20])
@pytest.mark.parametrize("with_delta", [False, True])
def test_rows_near_zero(ops, size, eps, with_delta):  # noqa: F811
    x = torch.zeros(8, size, device=DEV)
    x[1] = 1e-38
    x[2] = -1.2e-37
    x[3] = _rand(size, seed=1, scale=3e-37)
    x[4] = _rand(size, seed=2, scale=1e-30)
    x[5] = _rand(size, seed=3, scale=1e-9)
    x[6] = _rand(size, seed=4)
    x[7, size // 2] = 2.0 ** -110
    gain = 1 + 0.1 * _rand(size, seed=5)
    delta = torch.zeros_like(x) if with_delta else None
    q, scales = _places(8, size)
    before = x.clone()
    ops.rmsnorm_e4m3(x, gain, eps, q, scales, delta=delta)
    assert torch.equal(x, before)
    # (what the sum of squares loses below 2^-126 is far below every eps here)
    h = _norm(x, gain, torch.tensor(eps, dtype=torch.float32).double().item())
    _check(h, q, scales, D)
    assert torch.all(q[0].float() == 0) and torch.all(scales[0].double() == (torch.tensor(2.0 ** -100) / 448).double().item())
    # the same numbers as 8-bit rows of the norm's 32-bit output: nothing here is out of any range
    assert torch.isfinite(q.float()).all() and torch.isfinite(scales).all()
