"""How matrices are rounded to 8 and 4 bits, and how 4-bit codes lie."""
import pytest
import torch

from llmengine_b200.weights import quantize as qz


def _w(n, k, seed=0):
    return torch.randn(n, k, generator=torch.Generator().manual_seed(seed)) * 0.05


@pytest.mark.parametrize("k", [1, 8, 31, 32, 127, 128, 129, 200, 384])
def test_codes_come_back(k):
    codes = torch.randint(0, 16, (5, k), generator=torch.Generator().manual_seed(k)).to(torch.uint8)
    packed = qz.pack_int4(codes)
    assert packed.shape == (5, -(-k // 128) * 64) and packed.dtype == torch.uint8
    assert torch.equal(qz.unpack_int4(packed, k), codes)


def test_where_a_code_lies():
    """Value 32 j + 8 q + e of a block is in word 4 q + j, at bits 4 (e / 2) + 16 (e % 2)."""
    for k in range(256):
        codes = torch.zeros(1, 256, dtype=torch.uint8)
        codes[0, k] = 11
        words = qz.pack_int4(codes).view(torch.int32).tolist()[0]
        block, j, q, e = k // 128, k % 128 // 32, k % 32 // 8, k % 8
        want = [0] * 32
        want[16 * block + 4 * q + j] = 11 << (4 * (e // 2) + 16 * (e % 2))
        assert [w & 0xFFFFFFFF for w in words] == want


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("k", [8, 100, 512])
def test_4_bits_are_near(group, zeros, k):
    w = _w(9, k, seed=group + k)
    packed, scales, zero = qz.quantize_int4(w, group, zeros)
    assert scales.shape == (9, -(-k // group)) and scales.dtype == torch.bfloat16 and (zero is None) != zeros
    back = qz.dequantize_int4(packed, scales, zero, k, group)
    at = torch.arange(k) // group
    # half a step of the scale; the scale itself is rounded to bfloat16 (2^-8), which can move the ends of the range, 7 or 15 steps away,
    # and a zero point rounded by half a step cuts off as much at one end
    step = scales.float()[:, at]
    assert torch.all((back - w).abs() <= step * (0.5 + (0.5 if zeros else 0.0) + 15 * 2.0 ** -8) + 1e-12)


def test_8_bits_are_near():
    w = _w(7, 300)
    w[3] = 0
    q, scales = qz.quantize_e4m3(w)
    assert q.dtype == torch.float8_e4m3fn and scales.shape == (7,) and torch.all(q[3].float() == 0) and torch.all(scales > 0)
    y = w / scales[:, None]
    assert torch.all((q.float() - y).abs() <= torch.maximum(y.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10)) * (1 + 2.0 ** -20))
    assert torch.all(q.float().abs().amax(1)[[0, 1, 2, 4, 5, 6]] == 448)


def test_rows_of_zeros_in_4_bits():
    for zeros in (False, True):
        packed, scales, zero = qz.quantize_int4(torch.zeros(3, 64), 32, zeros)
        assert torch.all(qz.dequantize_int4(packed, scales, zero, 64, 32) == 0) and torch.all(scales.float() > 0)


def test_refusals():
    for call in (lambda: qz.quantize_int4(_w(4, 64), 48), lambda: qz.quantize_int4(torch.full((2, 64), float("nan")), 64),
                 lambda: qz.quantize_e4m3(torch.full((2, 64), float("inf"))), lambda: qz.quantize_e4m3(torch.ones(2, 3, 4)),
                 lambda: qz.pack_int4(torch.full((2, 64), 16)), lambda: qz.pack_int4(torch.full((2, 64), -1)),
                 lambda: qz.pack_int4(torch.zeros(2, 64)), lambda: qz.unpack_int4(torch.zeros(2, 64, dtype=torch.uint8), 129)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("zeros", [False, True])
def test_the_largest_numbers_in_4_bits(zeros):
    """A group whose largest and least values are farther apart than the largest 32-bit number."""
    w = torch.zeros(3, 64)
    w[0, 0], w[0, 1], w[1, 40] = 3e38, -3e38, -2.5e38
    packed, scales, zero = qz.quantize_int4(w, 32, zeros)
    back = qz.dequantize_int4(packed, scales, zero, 64, 32)
    # half a step, the scale's rounding over the whole span, and with a zero point its half step (test_4_bits_are_near)
    step = scales.float().repeat_interleave(32, 1)
    assert torch.isfinite(scales.float()).all() and torch.all((back / step - w / step).abs() <= 0.5 + (0.5 if zeros else 0.0) + 15 * 2.0 ** -8)


def test_spans_that_fit_are_rounded_as_they_were():
    w = torch.cat([_w(64, 256, seed=s) * scale for s, scale in ((1, 1.0), (2, 1e-6), (3, 1e30))])
    packed, scales, zero = qz.quantize_int4(w, 64, True)
    g = w.view(len(w), -1, 64)
    least, most = g.amin(2).clamp(max=0.0), g.amax(2).clamp(min=0.0)
    assert torch.equal(scales, ((most - least) / 15).to(torch.bfloat16))
    assert torch.equal(zero, (-least / scales.float()).round().clamp(0, 15).to(torch.uint8))


@pytest.mark.parametrize("n,k", [(0, 64), (0, 200), (3, 0)])
def test_matrices_without_values(n, k):
    packed = qz.pack_int4(torch.zeros(n, k, dtype=torch.uint8))
    assert packed.shape == (n, -(-k // 128) * 64) and qz.unpack_int4(packed, k).shape == (n, k)
    for zeros in (False, True):
        packed, scales, zero = qz.quantize_int4(torch.zeros(n, k), 64, zeros)
        assert scales.shape == (n, -(-k // 64)) and (zero is None or zero.shape == scales.shape)
        assert qz.dequantize_int4(packed, scales, zero, k, 64).shape == (n, k)
    q, scales = qz.quantize_e4m3(torch.zeros(n, k))
    assert q.shape == (n, k) and scales.shape == (n,)
