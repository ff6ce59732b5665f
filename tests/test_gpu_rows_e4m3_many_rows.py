"""8-bit rows of so many rows that a thread holds several pieces of one (from two rows an SM on), every row against the formula in 64 bits, with the
bounds of test_gpu_rows_e4m3.py."""
import pytest
import torch

from test_gpu_rows_e4m3 import D_GATE, D_NORM, D_ROWS, DEV, F8, _check, _norm, _places, ops  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
ROWS = [295, 296, 1000]                         # 148 SMs: the last count before, the first one from which on, and several rounds
SIZES = [1016, 1024, 2048, 4096, 5504, 8200, 12288, 12296, 17408]
DTYPES = [torch.float32, torch.bfloat16]


def _rand(*shape, seed, scale):
    """Rows of different magnitudes."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g) * scale * torch.exp(torch.randn(shape[0], 1, device=DEV, generator=g))


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows(ops, rows, size, dtype):  # noqa: F811
    x = _rand(rows, size, seed=1, scale=3.0).to(dtype)
    q, scales = _places(rows, size)
    ops.rows_e4m3(x, q, scales)
    _check(x.double(), q, scales, D_ROWS)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_gate(ops, rows, size, dtype):  # noqa: F811
    x = _rand(rows, 2 * size, seed=2, scale=4.0).to(dtype)
    q, scales = _places(rows, size)
    ops.swiglu_e4m3(x, q, scales)
    g, u = x.double().chunk(2, 1)
    _check(g * torch.sigmoid(g) * u, q, scales, D_GATE)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("delta", [None, *DTYPES])
def test_norm(ops, rows, size, delta):  # noqa: F811
    x, gain = _rand(rows, size, seed=3, scale=2.0), 1 + 0.1 * torch.randn(size, device=DEV)
    d = None if delta is None else _rand(rows, size, seed=4, scale=1.0).to(delta)
    total = x.clone() if d is None else x + d.float()
    q, scales = _places(rows, size)
    ops.rmsnorm_e4m3(x, gain, 1e-6, q, scales, delta=d)
    assert torch.equal(x, total)
    _check(_norm(total, gain, 1e-6), q, scales, D_NORM)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", ["rows", "gate"])
def test_strides_and_what_lies_between(ops, dtype, what):  # noqa: F811
    """Rows apart from one another, in and out, by whole pieces and by odd numbers."""
    rows, size, halves = 600, 4096, 2 if what == "gate" else 1
    for extra in (8, 3):
        x = _rand(rows, halves * size + extra, seed=5, scale=2.0).to(dtype)[:, :halves * size]
        q, scales = _places(rows, size, size + extra)
        (ops.swiglu_e4m3 if what == "gate" else ops.rows_e4m3)(x, q, scales)
        h = x.double()
        if what == "gate":
            h = h[:, :size] * torch.sigmoid(h[:, :size]) * h[:, size:]
        _check(h, q, scales, D_GATE if what == "gate" else D_ROWS)
        assert torch.all(torch.as_strided(q, (rows - 1, extra), (size + extra, 1), size).float() == 3.0)
