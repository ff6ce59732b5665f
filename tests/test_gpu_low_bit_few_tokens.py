"""Products with weights of 8 and 4 bits: a token's result up to 16 tokens does not depend on the others, and 4-bit operands behind 32 bits."""
import pytest
import torch

from test_gpu_low_bit_products import DEV, F8, _weights64, _whole_int4, ops  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu
# weight rows and values for each way in which warps share the row groups, and a few that end anywhere
SHAPES = [(2048, 4096), (2050, 1000), (4096, 1536), (7168, 5120), (10000, 264), (17408, 1024)]


def _randn(*shape, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g)


@pytest.mark.parametrize("n,k", SHAPES)
def test_e4m3_tokens_by_themselves(ops, n, k):  # noqa: F811
    from llmengine_b200.weights.quantize import quantize_e4m3
    k = k // 16 * 16
    x, xs = quantize_e4m3(3 * _randn(16, k, seed=1))
    w, ws = quantize_e4m3(0.02 * _randn(n, k, seed=2))
    for dtype in (torch.float32, torch.bfloat16):
        alone = torch.stack([ops.linear_e4m3(x[i:i + 1], xs[i:i + 1], w, ws, torch.empty(1, n, dtype=dtype, device=DEV))[0] for i in range(16)])
        for m in (2, 7, 8, 9, 15, 16):
            for first in (0, 16 - m):
                out = ops.linear_e4m3(x[first:first + m], xs[first:first + m], w, ws, torch.empty(m, n, dtype=dtype, device=DEV))
                assert torch.equal(out, alone[first:first + m])


@pytest.mark.parametrize("n,k", SHAPES)
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, False)])
def test_int4_tokens_by_themselves(ops, n, k, group, zeros):  # noqa: F811
    from llmengine_b200.weights.quantize import quantize_int4
    x = (3 * _randn(16, k, seed=1)).to(torch.bfloat16)
    packed, scales, zero = quantize_int4(0.02 * _randn(n, k, seed=2), group, zeros)
    alone = torch.stack([ops.linear_int4(x[i:i + 1], packed, scales, torch.empty(1, n, dtype=torch.bfloat16, device=DEV), zeros=zero)[0] for i in range(16)])
    for m in (2, 7, 8, 9, 15, 16):
        for first in (0, 16 - m):
            out = ops.linear_int4(x[first:first + m], packed, scales, torch.empty(m, n, dtype=torch.bfloat16, device=DEV), zeros=zero)
            assert torch.equal(out, alone[first:first + m])


@pytest.mark.parametrize("form", ["wide", "pair"])
@pytest.mark.parametrize("m", [16, 40, 300])
def test_int4_rows_behind_32_bits(ops, m, form):  # noqa: F811
    """Rows of x and of codes so far apart that the last ones begin behind 2^31 values and bytes."""
    from llmengine_b200.weights.quantize import pack_int4
    n, k = 40, 136
    x, codes, scales, zero = _whole_int4(m, n, k, 32, True, seed=12)
    packed, want = pack_int4(codes), (x.double() @ _weights64(codes, scales, zero, 32).t()).to(torch.bfloat16)
    ops.low_bit_form(form)
    try:
        sx = (1 << 31) // (m - 2) // 8 * 8 + 8
        far = torch.zeros((m - 1) * sx + k, dtype=torch.bfloat16, device=DEV).as_strided((m, k), (sx, 1))
        far.copy_(x)
        out = torch.full((m, n), 5.0, dtype=torch.bfloat16, device=DEV)
        ops.linear_int4(far, packed, scales, out, zeros=zero)
        assert torch.equal(out, want)
        del far
        sw = (1 << 31) // (n - 2) // 16 * 16 + 16
        far = torch.zeros((n - 1) * sw + packed.shape[1], dtype=torch.uint8, device=DEV).as_strided(tuple(packed.shape), (sw, 1))
        far.copy_(packed)
        out.fill_(5.0)
        ops.linear_int4(x, far, scales, out, zeros=zero)
        assert torch.equal(out, want)
    finally:
        ops.low_bit_form("auto")


@pytest.mark.parametrize("m", [3, 20])
def test_int4_scales_behind_32_bits(ops, m):  # noqa: F811
    """More than 2^31 scales and zero points, a group of 32 each: the last weight rows are multiplied by theirs."""
    from llmengine_b200.weights.quantize import pack_int4
    k, last = 4096, 48
    n = (1 << 31) // (k // 32) + 16
    x, codes, scales, zero = _whole_int4(m, last, k, 32, True, seed=13)
    w = torch.zeros(n, k // 2, dtype=torch.uint8, device=DEV)
    s, z = torch.zeros(n, k // 32, dtype=torch.bfloat16, device=DEV), torch.zeros(n, k // 32, dtype=torch.uint8, device=DEV)
    w[-last:], s[-last:], z[-last:] = pack_int4(codes), scales, zero
    out = torch.full((m, n), 5.0, dtype=torch.bfloat16, device=DEV)
    ops.linear_int4(x, w, s, out, zeros=z)
    assert torch.equal(out[:, -last:], (x.double() @ _weights64(codes, scales, zero, 32).t()).to(torch.bfloat16))
    assert torch.all(out[:, :-last] == 0)
