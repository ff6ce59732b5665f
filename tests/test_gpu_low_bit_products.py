"""Products with weights of 8 and 4 bits against the formulas in 64 bits.

Two kinds of inputs.  Small whole numbers with scales that are powers of two: every product and every sum of them is a 32-bit number
without rounding, so the output is the rounding of the exact value and nothing else, whichever kernel serves the shape and in whichever order
it adds; a value read from a wrong place, twice or not at all shows.  And numbers as layers have them, for the rounding itself: with S = sum
|x w| the 32-bit sums are off by at most one unit of 2^-22 of S for each of the K / 16 additions of a chain of matrix instructions
(which may cut off what they add: 2^-23, and once more inside an instruction) and the few of the sums' parts; the output by half a step of
its type, eps / 2.  Where more than 16 rows meet weights of 4 bits, the tensor cores take each weight as one bfloat16 number: another half step, 2^-8,
of every |x w|."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from llmengine_b200.kernels.ops import CudaOps
    return CudaOps(torch.device(DEV))


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _bound(out_dtype, exact, size, k, weight_rounding=0.0):
    return torch.finfo(out_dtype).eps / 2 * exact.abs() + ((k / 16 + 40) * 2.0 ** -22 + weight_rounding) * size + 1e-30


def _out(m, n, dtype, extra=0):
    """A place for the output whose rows are n + extra apart, full of other numbers."""
    whole = torch.full((m, n + extra), 5.0, dtype=dtype, device=DEV)
    return whole, whole[:, :n]


def _rest_untouched(whole, n):
    assert torch.all(whole[:, n:] == 5.0)


# ----------------------------------------------------------------------------- 8 bits
def _whole_e4m3(m, n, k, seed):
    """Whole numbers -4..4, scales 2^-3..2^3: |sum| <= 16 k, exact in 32 bits for k < 2^20."""
    g = _gen(seed)
    x, w = (torch.randint(-4, 5, (r, k), generator=g).float().to(F8).to(DEV) for r in (m, n))
    xs, ws = (2.0 ** torch.randint(-3, 4, (r,), generator=g).float() for r in (m, n))
    return x, xs.to(DEV), w, ws.to(DEV)


def _exact_e4m3(x, xs, w, ws):
    return (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()


@pytest.fixture(params=["wide", "pair", "auto"])
def forms(ops, request):
    """The products of more than 16 rows also by the kernel that their own choice would not take."""
    ops.low_bit_form(request.param)
    yield ops
    ops.low_bit_form("auto")


M_SIZES = [1, 2, 8, 9, 16, 17, 24, 33, 64, 77, 128, 129, 200, 256, 257, 513]


@pytest.mark.parametrize("m", M_SIZES)
@pytest.mark.parametrize("n,k", [(1, 16), (8, 128), (100, 144), (129, 4096), (1000, 272), (2048, 1040), (264, 12288)])
def test_e4m3_places(forms, m, n, k):
    x, xs, w, ws = _whole_e4m3(m, n, k, seed=m + n + k)
    want = _exact_e4m3(x, xs, w, ws)
    for dtype in (torch.float32, torch.bfloat16):
        for extra in (0, 5):
            whole, out = _out(m, n, dtype, extra)
            assert forms.linear_e4m3(x, xs, w, ws, out) is out
            assert torch.equal(out.double(), want.to(dtype).double())
            _rest_untouched(whole, n)


@pytest.mark.parametrize("m", [1, 8, 16, 40, 77, 128, 300, 1024])
@pytest.mark.parametrize("n,k", [(512, 4096), (264, 12288), (4096, 528)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_e4m3_rounding(forms, m, n, k, dtype):
    from llmengine_b200.weights.quantize import quantize_e4m3
    g = _gen(m + n)
    x, xs = quantize_e4m3((torch.randn(m, k, generator=g) * 3).to(DEV))
    w, ws = quantize_e4m3((torch.randn(n, k, generator=g) * 0.02).to(DEV))
    _, out = _out(m, n, dtype)
    forms.linear_e4m3(x, xs, w, ws, out)
    want, size = _exact_e4m3(x, xs, w, ws), _exact_e4m3(x.float().abs(), xs, w.float().abs(), ws)
    assert torch.all((out.double() - want).abs() <= _bound(dtype, want, size, k))


@pytest.mark.parametrize("m", [3, 16, 40, 130, 300])
def test_e4m3_strides(forms, m):
    """Operands that are columns and rows of larger matrices."""
    n, k = 200, 400
    x, xs, w, ws = _whole_e4m3(m, n, k, seed=m)
    big_x, big_w = torch.zeros(m, k + 48, device=DEV).to(F8), torch.zeros(n + 3, k + 16, device=DEV).to(F8)
    big_x[:, 32:32 + k], big_w[2:2 + n, :k] = x, w
    big_x.view(torch.uint8)[:, :32] = 0x7F                          # NaN around what is multiplied
    big_w.view(torch.uint8)[:, k:] = 0x7F
    big_w.view(torch.uint8)[:2] = 0x7F
    big_w.view(torch.uint8)[2 + n:] = 0x7F
    whole, out = _out(m, n, torch.bfloat16, 8)
    forms.linear_e4m3(big_x[:, 32:32 + k], xs, big_w[2:2 + n, :k], ws, out)
    assert torch.equal(out.double(), _exact_e4m3(x, xs, w, ws).to(torch.bfloat16).double())
    _rest_untouched(whole, n)


@pytest.mark.parametrize("m", [4, 16, 40, 200, 300])
def test_e4m3_rows_that_are_no_numbers(forms, m):
    n, k = 300, 512
    x, xs, w, ws = _whole_e4m3(m, n, k, seed=1)
    clean = _exact_e4m3(x, xs, w, ws)
    x.view(torch.uint8)[1, 77] = 0x7F
    xs[2] = float("inf")
    x.view(torch.uint8)[2, 5] = 0x7F
    w.view(torch.uint8)[250, 3] = 0xFF
    _, out = _out(m, n, torch.float32)
    forms.linear_e4m3(x, xs, w, ws, out)
    bad = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    bad[1:3] = True
    bad[:, 250] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad].double(), clean[~bad])


# ----------------------------------------------------------------------------- 4 bits
# Many tiles for every pair of SMs and few steps in each: the ends of tiles in every order that the steps can have.
MANY_TILES = [(1000, 9000), (777, 12289)]


@pytest.mark.parametrize("m,n", MANY_TILES)
@pytest.mark.parametrize("k", [16, 256, 272, 640])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_e4m3_many_tiles(forms, m, n, k, dtype):
    x, xs, w, ws = _whole_e4m3(m, n, k, seed=m + k)
    whole, out = _out(m, n, dtype, 0)
    forms.linear_e4m3(x, xs, w, ws, out)
    assert torch.equal(out, _exact_e4m3(x, xs, w, ws).to(dtype))


def _whole_int4(m, n, k, group, zeros, seed):
    """Whole numbers -4..4, any codes, scales 2^-3..2^3, zero points over the whole range: |sum| <= 4 * 15 * 2^3 k in steps of 2^-3: exact in 32
    bits for k < 2^15."""
    g = _gen(seed)
    groups = -(-k // group)
    x = torch.randint(-4, 5, (m, k), generator=g).to(torch.bfloat16).to(DEV)
    codes = torch.randint(0, 16, (n, k), generator=g).to(torch.uint8).to(DEV)
    scales = (2.0 ** torch.randint(-3, 4, (n, groups), generator=g).float()).to(torch.bfloat16).to(DEV)
    zero = torch.randint(0, 16, (n, groups), generator=g).to(torch.uint8).to(DEV) if zeros else None
    return x, codes, scales, zero


def _weights64(codes, scales, zero, group):
    at = torch.arange(codes.shape[1], device=codes.device) // group
    return (codes.double() - (8.0 if zero is None else zero.double()[:, at])) * scales.double()[:, at]


@pytest.mark.parametrize("m", M_SIZES)
@pytest.mark.parametrize("n,k", [(1, 8), (8, 128), (100, 136), (129, 4096), (1000, 264), (2048, 1000), (264, 12288)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True), (128, False)])
def test_int4_places(forms, m, n, k, group, zeros):
    from llmengine_b200.weights.quantize import pack_int4
    x, codes, scales, zero = _whole_int4(m, n, k, group, zeros, seed=m + n + k)
    want = (x.double() @ _weights64(codes, scales, zero, group).t()).to(torch.bfloat16)
    for extra in (0, 5):
        whole, out = _out(m, n, torch.bfloat16, extra)
        assert forms.linear_int4(x, pack_int4(codes), scales, out, zeros=zero) is out
        assert torch.equal(out, want)
        _rest_untouched(whole, n)


@pytest.mark.parametrize("m,n", MANY_TILES)
@pytest.mark.parametrize("k", [40, 200, 384, 520, 1032])
@pytest.mark.parametrize("group,zeros", [(32, True), (128, False)])
def test_int4_many_tiles(forms, m, n, k, group, zeros):
    from llmengine_b200.weights.quantize import pack_int4
    x, codes, scales, zero = _whole_int4(m, n, k, group, zeros, seed=m + k)
    whole, out = _out(m, n, torch.bfloat16, 0)
    forms.linear_int4(x, pack_int4(codes), scales, out, zeros=zero)
    assert torch.equal(out, (x.double() @ _weights64(codes, scales, zero, group).t()).to(torch.bfloat16))


@pytest.mark.parametrize("m", [1, 8, 16, 40, 77, 128, 300, 1024])
@pytest.mark.parametrize("n,k", [(512, 4096), (264, 12288), (4096, 520)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_int4_rounding(forms, m, n, k, group, zeros):
    from llmengine_b200.weights.quantize import dequantize_int4, quantize_int4
    g = _gen(m + n)
    x = (torch.randn(m, k, generator=g) * 3).to(torch.bfloat16).to(DEV)
    packed, scales, zero = quantize_int4((torch.randn(n, k, generator=g) * 0.02).to(DEV), group, zeros)
    _, out = _out(m, n, torch.bfloat16)
    forms.linear_int4(x, packed, scales, out, zeros=zero)
    w = dequantize_int4(packed, scales, zero, k, group).double()
    want, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    assert torch.all((out.double() - want).abs() <= _bound(torch.bfloat16, want, size, k, 2.0 ** -8 if m > 16 else 0.0))


@pytest.mark.parametrize("m", [3, 16, 40, 130, 300])
def test_int4_strides(forms, m):
    from llmengine_b200.weights.quantize import pack_int4
    n, k, group = 200, 400, 64
    x, codes, scales, zero = _whole_int4(m, n, k, group, True, seed=m)
    packed = pack_int4(codes)
    big_x = torch.full((m, k + 24), float("nan"), dtype=torch.bfloat16, device=DEV)
    big_x[:, 16:16 + k] = x
    big_w = torch.full((n + 3, packed.shape[1] + 16), 0xFF, dtype=torch.uint8, device=DEV)
    big_w[2:2 + n, :packed.shape[1]] = packed
    whole, out = _out(m, n, torch.bfloat16, 8)
    forms.linear_int4(big_x[:, 16:16 + k], big_w[2:2 + n, :packed.shape[1]], scales, out, zeros=zero)
    assert torch.equal(out, (x.double() @ _weights64(codes, scales, zero, group).t()).to(torch.bfloat16))
    _rest_untouched(whole, n)


@pytest.mark.parametrize("m", [4, 16, 40, 200, 300])
def test_int4_rows_that_are_no_numbers(forms, m):
    from llmengine_b200.weights.quantize import pack_int4
    n, k = 300, 520
    x, codes, scales, _ = _whole_int4(m, n, k, 128, False, seed=1)
    clean = (x.double() @ _weights64(codes, scales, None, 128).t()).to(torch.bfloat16)
    x[1, 77], x[2, 519] = float("nan"), float("inf")
    scales[250, 3] = float("nan")
    codes[:, 519], codes[7, 519] = 9, 8                             # infinity times 1, and once times 0
    _, out = _out(m, n, torch.bfloat16)
    before = x.clone()
    forms.linear_int4(x, pack_int4(codes), scales, out)
    before[1:3] = 0
    clean = (before.double() @ _weights64(codes, scales.nan_to_num(1.0), None, 128).t()).to(torch.bfloat16)
    assert torch.isnan(out[1]).all() and torch.isnan(out[:, 250]).all() and torch.isnan(out[2, 7])
    keep = [c for c in range(n) if c != 250]
    assert (out[2, [c for c in keep if c != 7]] == float("inf")).all()
    rows = [r for r in range(m) if r not in (1, 2)]
    assert torch.equal(out[rows][:, keep], clean[rows][:, keep])


# ----------------------------------------------------------------------------- both
@pytest.mark.parametrize("m", [8, 40, 300])
def test_another_stream_and_captured_calls(ops, m):
    from llmengine_b200.weights.quantize import pack_int4
    n, k = 264, 1024
    a, b = _whole_e4m3(m, n, k, seed=2), _whole_int4(m, n, k, 128, False, seed=3)
    packed = pack_int4(b[1])
    want8, want4 = _exact_e4m3(*a).float(), (b[0].double() @ _weights64(b[1], b[2], None, 128).t()).to(torch.bfloat16)
    out8, out4 = _out(m, n, torch.float32)[1], _out(m, n, torch.bfloat16)[1]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.linear_e4m3(*a, out8), ops.linear_int4(b[0], packed, b[2], out4)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out8, want8) and torch.equal(out4, want4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.linear_e4m3(*a, out8), ops.linear_int4(b[0], packed, b[2], out4)
    for _ in range(3):
        out8.zero_(), out4.zero_()
        graph.replay()
        assert torch.equal(out8, want8) and torch.equal(out4, want4)


def test_no_rows(ops):
    n = ops.launches
    x, xs, w, ws = _whole_e4m3(4, 8, 32, seed=4)
    ops.linear_e4m3(x[:0], xs[:0], w, ws, torch.empty(0, 8, device=DEV))
    ops.linear_e4m3(x, xs, w[:0], ws[:0], torch.empty(4, 0, device=DEV))
    x, codes, scales, _ = _whole_int4(4, 8, 32, 32, False, seed=4)
    ops.linear_int4(x[:0], torch.zeros(8, 64, dtype=torch.uint8, device=DEV), scales, torch.empty(0, 8, dtype=torch.bfloat16, device=DEV))
    assert ops.launches == n


def test_refusals(ops):
    from llmengine_b200.kernels.ops import KernelError
    from llmengine_b200.weights.quantize import pack_int4
    x, xs, w, ws = _whole_e4m3(4, 24, 64, seed=5)
    out = torch.empty(4, 24, device=DEV)
    y, codes, scales, zero = _whole_int4(4, 24, 64, 32, True, seed=5)
    p, o = pack_int4(codes), torch.empty(4, 24, dtype=torch.bfloat16, device=DEV)
    calls = [
        lambda: ops.linear_e4m3(x.cpu(), xs, w, ws, out),
        lambda: ops.linear_e4m3(x.float(), xs, w, ws, out),
        lambda: ops.linear_e4m3(x, xs, w[:, :48], ws, out),
        lambda: ops.linear_e4m3(x[:, :24], xs, w[:, :24], ws, out),                  # K is no multiple of 16
        lambda: ops.linear_e4m3(x[:, 8:56], xs, w[:, 8:56], ws, out),                # rows that do not begin on 16 bytes
        lambda: ops.linear_e4m3(x, xs[:3], w, ws, out),
        lambda: ops.linear_e4m3(x, xs, w, ws[:3], out),
        lambda: ops.linear_e4m3(x, xs, w, ws.double(), out),
        lambda: ops.linear_e4m3(x, xs, w, ws, out[:, :23]),
        lambda: ops.linear_e4m3(x, xs, w, ws, out.half()),
        lambda: ops.linear_e4m3(x, xs, w, ws, out[:1].expand(4, 24)),
        lambda: ops.linear_e4m3(x, xs, w, ws, w.view(-1).view(torch.float32)[:96].view(4, 24)),
        lambda: ops.linear_e4m3(x[:1].expand(4, 64), xs, w, ws, out),
        lambda: ops.linear_int4(y.float(), p, scales, o),
        lambda: ops.linear_int4(y[:, :60], p, scales, o),                            # K is no multiple of 8
        lambda: ops.linear_int4(y[:, 4:52], p, scales, o),                           # rows that do not begin on 16 bytes
        lambda: ops.linear_int4(y, p[:, :32], scales, o),
        lambda: ops.linear_int4(y, p.view(torch.int8), scales, o),
        lambda: ops.linear_int4(y, p, scales.float(), o),
        lambda: ops.linear_int4(y, p, scales[:20], o),
        lambda: ops.linear_int4(y, p, torch.ones(24, 3, dtype=torch.bfloat16, device=DEV), o),
        lambda: ops.linear_int4(y, p, scales, o, zeros=zero[:, :1]),
        lambda: ops.linear_int4(y, p, scales, o, zeros=zero.to(torch.bfloat16)),
        lambda: ops.linear_int4(y, p, scales, o.float()),
        lambda: ops.linear_int4(y, p, scales, o[:, :23]),
        lambda: ops.linear_int4(y, p, scales, y[:, :24]),
        lambda: ops.linear_int4(y, p[1:].view(-1)[8:8 + 20 * 64].view(20, 64), scales[:20], o[:, :20]),
    ]
    n = ops.launches
    for i, call in enumerate(calls):
        with pytest.raises(KernelError):
            call()
            print("not refused:", i)
    assert ops.launches == n


def test_operands_side_by_side(ops):
    """Rows and output in one buffer, column range beside column range."""
    x, xs, w, ws = _whole_e4m3(9, 32, 64, seed=6)
    both = torch.zeros(9, 64 + 32 * 4, dtype=torch.uint8, device=DEV)
    both[:, :64] = x.view(torch.uint8)
    out = both[:, 64:].view(torch.float32)
    ops.linear_e4m3(both[:, :64].view(F8), xs, w, ws, out)
    assert torch.equal(out.double(), _exact_e4m3(x, xs, w, ws)) and torch.equal(both[:, :64], x.view(torch.uint8))


@pytest.mark.parametrize("m", [8, 40, 700])
def test_two_streams_at_once(ops, m):
    """Calls on two streams, whose blocks may share SMs and their tensor memory, each give what one alone gives."""
    from llmengine_b200.weights.quantize import pack_int4
    n, k = 520, 2048
    a, b = _whole_e4m3(m, n, k, seed=7), _whole_int4(m, n, k, 64, True, seed=8)
    packed = pack_int4(b[1])
    want8, want4 = _exact_e4m3(*a).float(), (b[0].double() @ _weights64(b[1], b[2], b[3], 64).t()).to(torch.bfloat16)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[(torch.empty(m, n, device=DEV), torch.empty(m, n, dtype=torch.bfloat16, device=DEV)) for _ in range(20)] for _ in streams]
    torch.cuda.synchronize()
    for i in range(20):
        for s, mine in zip(streams, outs):
            with torch.cuda.stream(s):
                ops.linear_e4m3(*a, mine[i][0])
                ops.linear_int4(b[0], packed, b[2], mine[i][1], zeros=b[3])
    torch.cuda.synchronize()
    for mine in outs:
        for out8, out4 in mine:
            assert torch.equal(out8, want8) and torch.equal(out4, want4)


@pytest.mark.parametrize("m", [9, 40, 300])
def test_outputs_behind_32_bits(ops, m):
    """Output rows so far apart that the last ones begin behind 2^31 values."""
    from llmengine_b200.weights.quantize import pack_int4
    n, k, stride = 136, 256, (1 << 31) // (m - 2)
    stride += -stride % 8
    a, b = _whole_e4m3(m, n, k, seed=9), _whole_int4(m, n, k, 128, False, seed=10)
    whole = torch.empty(m * stride, dtype=torch.bfloat16, device=DEV)
    for extra in (0, 3):                                            # rows that begin on 16 bytes, and that do not
        out = whole[extra:].as_strided((m, n), (stride, 1))
        out.fill_(5.0)
        ops.linear_e4m3(*a, out)
        assert torch.equal(out, _exact_e4m3(*a).to(torch.bfloat16))
        out.fill_(5.0)
        ops.linear_int4(b[0], pack_int4(b[1]), b[2], out)
        assert torch.equal(out, (b[0].double() @ _weights64(b[1], b[2], None, 128).t()).to(torch.bfloat16))


def test_operands_behind_32_bits(ops):
    """Rows and weights whose last ones begin behind 2^31 bytes and values."""
    n, k = 40, 64
    for m in (16, 40, 300):
        x, xs, w, ws = _whole_e4m3(m, n, k, seed=11)
        big = torch.zeros(2200000000, dtype=torch.uint8, device=DEV)
        sx, sw = 2199990000 // m // 16 * 16, 2199990000 // n // 16 * 16
        out = torch.empty(m, n, device=DEV)
        far = big.as_strided((m, k), (sx, 1))
        far.copy_(x.view(torch.uint8))
        ops.linear_e4m3(far.view(F8), xs, w, ws, out)
        assert torch.equal(out.double(), _exact_e4m3(x, xs, w, ws))
        far = big.as_strided((n, k), (sw, 1))
        far.copy_(w.view(torch.uint8))
        ops.linear_e4m3(x, xs, far.view(F8), ws, out)
        assert torch.equal(out.double(), _exact_e4m3(x, xs, w, ws))
