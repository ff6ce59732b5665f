"""Products with 4-bit weights into 32 bits (the plan's record, for what goes into the residual stream), with the inputs and the bounds of
test_gpu_low_bit_products.py: whole numbers come out exactly, others within the sums' own error and no rounding to fewer bits."""
import pytest
import torch

from test_gpu_low_bit_products import DEV, MANY_TILES, _bound, _gen, _out, _rest_untouched, _weights64, _whole_int4, forms, ops  # noqa: F401  (the fixtures)

pytestmark = pytest.mark.gpu


def _run(ops, x, packed, scales, zero, group, out):  # noqa: F811
    ops._run_one(lambda plan: plan.linear_int4(x, packed, scales, zero, group, out))


@pytest.mark.parametrize("m", [17, 33, 77, 129, 200, 257, 513])
@pytest.mark.parametrize("n,k", [(1, 8), (100, 136), (129, 4096), (1000, 264), (264, 12288)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_places(forms, m, n, k, group, zeros):  # noqa: F811
    from llmengine_b200.weights.quantize import pack_int4
    x, codes, scales, zero = _whole_int4(m, n, k, group, zeros, seed=m + n + k)
    want = x.double() @ _weights64(codes, scales, zero, group).t()
    for extra in (0, 5):
        whole, out = _out(m, n, torch.float32, extra)
        _run(forms, x, pack_int4(codes), scales, zero, group, out)
        assert torch.equal(out.double(), want)
        _rest_untouched(whole, n)


@pytest.mark.parametrize("m", [1, 7, 8, 9, 16])
@pytest.mark.parametrize("n,k", [(1, 8), (100, 136), (2048, 1000), (4096, 1024), (17000, 264)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
def test_places_of_few_tokens(ops, m, n, k, group, zeros):  # noqa: F811
    from llmengine_b200.weights.quantize import pack_int4
    x, codes, scales, zero = _whole_int4(m, n, k, group, zeros, seed=m + n + k)
    whole, out = _out(m, n, torch.float32, 5)
    _run(ops, x, pack_int4(codes), scales, zero, group, out)
    assert torch.equal(out.double(), x.double() @ _weights64(codes, scales, zero, group).t())
    _rest_untouched(whole, n)


@pytest.mark.parametrize("m,n", MANY_TILES)
@pytest.mark.parametrize("k", [40, 384, 1032])
def test_many_tiles(forms, m, n, k):  # noqa: F811
    from llmengine_b200.weights.quantize import pack_int4
    x, codes, scales, zero = _whole_int4(m, n, k, 32, True, seed=m + k)
    out = _out(m, n, torch.float32)[1]
    _run(forms, x, pack_int4(codes), scales, zero, 32, out)
    assert torch.equal(out.double(), x.double() @ _weights64(codes, scales, zero, 32).t())


@pytest.mark.parametrize("m", [1, 16, 40, 128, 300, 1024])
@pytest.mark.parametrize("n,k", [(512, 4096), (264, 12288)])
def test_rounding(forms, m, n, k):  # noqa: F811
    from llmengine_b200.weights.quantize import dequantize_int4, quantize_int4
    g = _gen(m + n)
    x = (torch.randn(m, k, generator=g) * 3).to(torch.bfloat16).to(DEV)
    packed, scales, zero = quantize_int4((torch.randn(n, k, generator=g) * 0.02).to(DEV), 64, True)
    out = _out(m, n, torch.float32)[1]
    _run(forms, x, packed, scales, zero, 64, out)
    w = dequantize_int4(packed, scales, zero, k, 64).double()
    want, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    assert torch.all((out.double() - want).abs() <= _bound(torch.float32, want, size, k, 2.0 ** -8 if m > 16 else 0.0))


@pytest.mark.parametrize("m", [8, 40, 300])
def test_captured(ops, m):  # noqa: F811
    """A record that is replayed reads and writes where it did."""
    from llmengine_b200.engine.batch import StepBatch
    from llmengine_b200.engine.plan import Plan
    from llmengine_b200.weights.quantize import pack_int4
    x, codes, scales, _ = _whole_int4(m, 264, 1024, 128, False, seed=3)
    want, out, plan = (x.double() @ _weights64(codes, scales, None, 128).t()).float(), _out(m, 264, torch.float32)[1], Plan()
    plan.linear_int4(x, pack_int4(codes), scales, None, 128, out)
    compiled, batch = ops.compile(plan), StepBatch.bare(m, torch.device(DEV))
    compiled.run(batch)
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        compiled.run(batch)
    for _ in range(2):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
