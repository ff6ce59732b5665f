"""Rows of 8-bit numbers with a scale each (of a norm, of rows as they are, of a gate) against the formulas in 64 bits.

A value's place in 8 bits is held against both ends of what the 32-bit arithmetic may have made of it: rounding is monotone, so the
stored number lies between the roundings of y (1 - d) and y (1 + d), where y is the exact quotient and d bounds the relative error of the
32-bit steps.  A norm's sum of n squares is off by at most n / 2 half steps of 2^-24 in any order (each addition rounds once, and all
terms are positive), and half of that reaches the root; the scale, the factor and the two products add six roundings: d = (n / 2 + 8) 2^-24
at worst, 2^-24 (64 + 8) for the pieces of 32 values and less a thread, added by five and five steps, that these kernels add.  The gate's exponential
is the hardware's: 2 units in the last place of exp2 and the rounding of its argument, |x| 2^-24 for |x| < 90 where the result counts: 100 2^-24."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F8 = torch.float8_e4m3fn
D_NORM, D_ROWS, D_GATE = 72 * 2.0 ** -24, 4 * 2.0 ** -24, 110 * 2.0 ** -24
LEAST = 2.0 ** -100


@pytest.fixture(scope="module")
def ops():
    from llmengine_b200.kernels.ops import CudaOps
    return CudaOps(torch.device(DEV))


def _rand(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def _places(rows, size, stride=None):
    """(out, scales) full of other numbers, out with its rows `stride` apart."""
    out = torch.full((rows, stride or size), 3.0, device=DEV).to(F8)
    return out[:, :size], torch.full((rows,), -7.0, device=DEV)


def _check(h, q, scales, d):
    """q and scales against the exact rows h (64 bits)."""
    a = h.abs().amax(1).clamp(min=LEAST) / 448
    assert torch.all((scales.double() - a).abs() <= d * a)
    y = h / a[:, None]
    lo, hi = torch.minimum(y * (1 - d), y * (1 + d)), torch.maximum(y * (1 - d), y * (1 + d))
    # (a quotient above the largest number by its error rounds to it)
    lo, hi = (v.clamp(-448, 448).float().to(F8).float() for v in (lo, hi))
    assert torch.all((lo <= q.float()) & (q.float() <= hi))


def _norm(x, gain, eps):
    x = x.double()
    return x / torch.sqrt((x * x).mean(1, keepdim=True) + eps) * gain.double()


SIZES = [1, 2, 7, 8, 64, 256, 264, 1000, 1026, 4096, 5120, 8190, 8200, 10241, 17408, 20480, 25600]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("rows", [1, 5, 37])
@pytest.mark.parametrize("delta,gain", [(None, torch.bfloat16), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_norm(ops, rows, size, delta, gain):
    eps = 3e-6
    x, g = _rand(rows, size, seed=1, scale=2.0), (1 + 0.1 * _rand(size, seed=2)).to(gain)
    d = None if delta is None else _rand(rows, size, seed=3).to(delta)
    total = x if d is None else x + d.float()
    before = x.clone()
    for place in ([None] if d is None else [None, torch.empty_like(x)]):
        x.copy_(before)
        q, scales = _places(rows, size)
        assert ops.rmsnorm_e4m3(x, g, eps, q, scales, delta=d, total=place) == (q, scales)
        _check(_norm(total, g, eps), q, scales, D_NORM)
        if d is not None:
            assert torch.equal(x if place is None else place, total)
        if place is not None or d is None:
            assert torch.equal(x, before)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("rows", [1, 6, 33])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows(ops, rows, size, dtype):
    for extra in (0, 3, 8):                                        # row strides: none, odd, whole pieces
        x = _rand(rows, size + extra, dtype=dtype, seed=4, scale=3.0)[:, :size]
        q, scales = _places(rows, size, size + extra)
        ops.rows_e4m3(x, q, scales)
        _check(x.double(), q, scales, D_ROWS)
        if extra and rows > 1:                                     # what lies between the rows stays as it was
            assert torch.all(torch.as_strided(q, (rows - 1, extra), (size + extra, 1), size).float() == 3.0)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("rows", [1, 6, 33])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gate(ops, rows, size, dtype):
    x = _rand(rows, 2 * size, dtype=dtype, seed=5, scale=4.0)
    q, scales = _places(rows, size)
    ops.swiglu_e4m3(x, q, scales)
    g, u = x.double().chunk(2, 1)
    _check(g * torch.sigmoid(g) * u, q, scales, D_GATE)


def test_extremes(ops):
    """Rows of zeros, of numbers too small to be divided by, of the largest ones, and of one value alone."""
    x = torch.zeros(7, 96, device=DEV)
    x[1] = 1e-38
    x[2] = 2.0 ** -99
    x[3] = 3.0e38
    x[4, 17] = -5.0
    x[5] = torch.linspace(-1e-3, 1e-3, 96, device=DEV)
    x[6] = -0.0
    q, scales = _places(7, 96)
    ops.rows_e4m3(x, q, scales)
    _check(x.double(), q, scales, D_ROWS)
    assert torch.all(q[0].float() == 0) and q[4, 17].float() == -448 and torch.all(scales > 0)
    gain = torch.ones(96, device=DEV)
    ops.rmsnorm_e4m3(x[:3].contiguous(), gain, 1e-6, q[:3], scales[:3])
    _check(_norm(x[:3], gain, 1e-6), q[:3], scales[:3], D_NORM)
    g = torch.tensor([[-200.0, -1e30, 1e30, 0.0], [1e4, 1e4, 1e4, 1e4]], device=DEV)       # silu of far values is 0 and the value
    for dtype in (torch.float32, torch.bfloat16):
        x = g.to(dtype)
        ops.swiglu_e4m3(x, q[:2, :2].contiguous(), scales[:2])
        h = x.double()
        h = h[:, :2] * torch.sigmoid(h[:, :2]) * h[:, 2:]
        a = h.abs().amax(1).clamp(min=LEAST) / 448
        assert torch.all((scales[:2].double() - a).abs() <= D_GATE * a)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("size", [5, 64, 1030, 4096, 30000])
def test_rows_that_are_no_numbers(ops, size, bad):
    """A row with a NaN or an infinity has no finite scale, nothing in it counts as a number any more, and its neighbours are as ever."""
    x = _rand(4, size, seed=6)
    clean = x.clone()
    x[2, size - 1] = bad
    gain = torch.ones(size, device=DEV)
    for what in ("rows", "norm", "gate"):
        q, scales = _places(4, size)
        ref, ref_scales = _places(4, size)
        if what == "rows":
            ops.rows_e4m3(x, q, scales), ops.rows_e4m3(clean, ref, ref_scales)
        elif what == "norm":
            ops.rmsnorm_e4m3(x, gain, 1e-6, q, scales), ops.rmsnorm_e4m3(clean, gain, 1e-6, ref, ref_scales)
        else:
            up = torch.ones_like(x)
            ops.swiglu_e4m3(torch.cat([up, x], 1), q, scales), ops.swiglu_e4m3(torch.cat([up, clean], 1), ref, ref_scales)
        assert not torch.isfinite(scales[2]) and torch.isnan(q[2].float() * scales[2]).all()
        for r in (0, 1, 3):
            assert torch.equal(q[r].view(torch.uint8), ref[r].view(torch.uint8)) and scales[r] == ref_scales[r]


def test_a_row_does_not_depend_on_the_others(ops):
    x, gain = _rand(300, 4096, seed=7), 1 + 0.1 * _rand(4096, seed=8)
    q, scales = _places(300, 4096)
    ops.rmsnorm_e4m3(x, gain, 1e-6, q, scales)
    for n in (1, 16, 150):
        q1, s1 = _places(n, 4096)
        ops.rmsnorm_e4m3(x[:n].contiguous(), gain, 1e-6, q1, s1)
        assert torch.equal(q1.view(torch.uint8), q[:n].view(torch.uint8)) and torch.equal(s1, scales[:n])


def test_no_rows(ops):
    q, scales = _places(0, 64)
    n = ops.launches
    ops.rows_e4m3(torch.empty(0, 64, device=DEV), q, scales)
    ops.swiglu_e4m3(torch.empty(0, 128, device=DEV), q, scales)
    ops.rmsnorm_e4m3(torch.empty(0, 64, device=DEV), torch.ones(64, device=DEV), 1e-6, q, scales)
    assert ops.launches == n


def test_another_stream_and_a_captured_call(ops):
    x, gain, delta = _rand(9, 1000, seed=9), 1 + 0.1 * _rand(1000, seed=10), _rand(9, 1000, seed=11)
    q, scales = _places(9, 1000)
    total = torch.empty_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.rmsnorm_e4m3(x, gain, 1e-6, q, scales, delta=delta, total=total)
    torch.cuda.current_stream().wait_stream(s)
    want, want_scales = q.clone(), scales.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rmsnorm_e4m3(x, gain, 1e-6, q, scales, delta=delta, total=total)
    for _ in range(3):
        q.view(torch.uint8).zero_(), scales.zero_()
        graph.replay()
        assert torch.equal(q.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales, want_scales)


def test_refusals(ops):
    from llmengine_b200.kernels.ops import KernelError
    x, gain = _rand(4, 64, seed=12), torch.ones(64, device=DEV)
    q, scales = _places(4, 64)
    calls = [
        lambda: ops.rows_e4m3(x.cpu(), q, scales),
        lambda: ops.rows_e4m3(x.half(), q, scales),
        lambda: ops.rows_e4m3(x[0], q, scales),
        lambda: ops.rows_e4m3(x.t(), _places(64, 4)[0], _places(64, 4)[1]),
        lambda: ops.rows_e4m3(x, q[:, :32], scales),
        lambda: ops.rows_e4m3(x, q.view(torch.uint8), scales),
        lambda: ops.rows_e4m3(x, q, scales[:3]),
        lambda: ops.rows_e4m3(x, q, scales.double()),
        lambda: ops.rows_e4m3(x, q[:1].expand(4, 64), scales),
        lambda: ops.rows_e4m3(x[:1].expand(4, 64), q, scales),
        lambda: ops.rows_e4m3(x, x.view(F8)[:, :64], scales),
        lambda: ops.rows_e4m3(x, q, x.view(-1)[:4]),
        lambda: ops.rows_e4m3(torch.empty(4, 0, device=DEV), q[:, :0], scales),
        lambda: ops.swiglu_e4m3(x[:, :63], _places(4, 31)[0], scales),
        lambda: ops.swiglu_e4m3(x, q, scales),
        lambda: ops.rmsnorm_e4m3(x, gain[:32], 1e-6, q, scales),
        lambda: ops.rmsnorm_e4m3(x, gain, 0.0, q, scales),
        lambda: ops.rmsnorm_e4m3(x, gain, float("nan"), q, scales),
        lambda: ops.rmsnorm_e4m3(x.bfloat16(), gain, 1e-6, q, scales),
        lambda: ops.rmsnorm_e4m3(x[:, :32], gain[:32], 1e-6, _places(4, 32)[0], scales),
        lambda: ops.rmsnorm_e4m3(x, gain, 1e-6, _places(4, 64, 80)[0], scales),
        lambda: ops.rmsnorm_e4m3(x, gain, 1e-6, q, scales, total=torch.empty_like(x)),
        lambda: ops.rmsnorm_e4m3(x, gain, 1e-6, q, scales, delta=x),
        lambda: ops.rmsnorm_e4m3(x, gain, 1e-6, q, scales, delta=_rand(3, 64)),
        lambda: ops.rmsnorm_e4m3(x, gain, 1e-6, q, scales, delta=torch.zeros_like(x), total=torch.empty(4, 64, device=DEV).half()),
    ]
    n = ops.launches
    for i, call in enumerate(calls):
        with pytest.raises(KernelError):
            call()
            print("not refused:", i)
    assert ops.launches == n


def test_rows_behind_32_bits(ops):
    """More than 2^31 values: the last rows are read and written where they are."""
    rows, size = 540000, 4096
    x = torch.zeros(rows, size, dtype=torch.bfloat16, device=DEV)
    x[-3:] = _rand(3, size, dtype=torch.bfloat16, seed=13)
    q, scales = torch.empty(rows, size, dtype=F8, device=DEV), torch.empty(rows, device=DEV)
    ops.rows_e4m3(x, q, scales)
    _check(x[-3:].double(), q[-3:], scales[-3:], D_ROWS)
    assert torch.all(q[:-3].view(torch.uint8).amax(1) == 0)
    ops.swiglu_e4m3(x.view(rows // 2, 2 * size), q[:rows // 2], scales[:rows // 2])
    g, u = x[-2:].double()
    _check((g * torch.sigmoid(g) * u)[None], q[rows // 2 - 1][None], scales[rows // 2 - 1][None], D_GATE)
