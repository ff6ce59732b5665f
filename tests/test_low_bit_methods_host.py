"""What the methods of the low-bit operators refuse before anything is loaded or launched, on CPU tensors (whose device has the index -1)."""
import pytest
import torch

from llmengine_b200.kernels.ops import CudaOps, KernelError

F8, BF16 = torch.float8_e4m3fn, torch.bfloat16


@pytest.fixture
def ops():
    """The methods without a device: a call that is not refused fails for want of a library."""
    o = CudaOps.__new__(CudaOps)
    o._device_index, o._libs, o._typed, o._direct = -1, {}, {}, 0
    return o


def _given():
    x, q, s = torch.zeros(4, 64), torch.zeros(4, 64).to(F8), torch.zeros(4)
    w8, ws, out = torch.zeros(24, 64).to(F8), torch.zeros(24), torch.zeros(4, 24)
    w4, sc = torch.zeros(24, 64, dtype=torch.uint8), torch.zeros(24, 2, dtype=BF16)
    return {"rmsnorm_e4m3": (x, torch.ones(64), 1e-6, q, s), "rows_e4m3": (x, q, s), "swiglu_e4m3": (torch.zeros(4, 128), q, s),
            "linear_e4m3": (q, s, w8, ws, out), "linear_int4": (x.to(BF16), w4, sc, out.to(BF16))}


@pytest.mark.parametrize("wrong", [None, 3.0, [1.0, 2.0]])
def test_operands_that_are_no_tensors(ops, wrong):
    for name, args in _given().items():
        for i, a in enumerate(args):
            if isinstance(a, torch.Tensor):
                with pytest.raises(KernelError, match=name):
                    getattr(ops, name)(*args[:i], wrong, *args[i + 1:])


@pytest.mark.parametrize("many", [(1 << 31) - 8191, (1 << 31) + 64, (1 << 32) + 64])
def test_more_rows_or_values_than_an_index_holds(ops, many):
    """(A size is handed on as a 32-bit number: one above 2^32 would look like a small one.)"""
    tall = lambda dtype, cols: torch.zeros(1, cols).to(dtype).expand(many, cols)                     # noqa: E731
    long = lambda dtype, rows: torch.zeros(1, 1).to(dtype).expand(rows, many)                        # noqa: E731
    column = torch.zeros(1).expand(many)
    calls = {
        "rmsnorm_e4m3": [(torch.empty(many, 0), torch.ones(0), 1e-6, torch.empty(many, 0, dtype=F8), column), (long(torch.float32, 1), column, 1e-6, long(F8, 1), torch.zeros(1))],
        "rows_e4m3": [(tall(BF16, 4), tall(F8, 4), column), (long(BF16, 2), long(F8, 2), torch.zeros(2))],
        "swiglu_e4m3": [(tall(BF16, 4), tall(F8, 2), column), (torch.zeros(1, 1).expand(2, 2 * many), long(F8, 2), torch.zeros(2))],
        "linear_e4m3": [(tall(F8, 16), column, torch.zeros(1, 16).to(F8), torch.zeros(1), tall(torch.float32, 1)),
                        (torch.zeros(1, 16).to(F8), torch.zeros(1), tall(F8, 16), column, torch.zeros(1, 1).expand(1, many))],
        "linear_int4": [(tall(BF16, 8), torch.zeros(1, 64, dtype=torch.uint8), torch.zeros(1, 1, dtype=BF16), tall(BF16, 1)),
                        (torch.zeros(1, 8, dtype=BF16), tall(torch.uint8, 64), tall(BF16, 1), torch.zeros(1, 1, dtype=BF16).expand(1, many))]}
    for name, some in calls.items():
        for args in some:
            with pytest.raises(KernelError, match="too many|at most"):
                getattr(ops, name)(*args)


def test_the_usual_calls_get_through_to_the_library(ops, monkeypatch):
    from llmengine_b200.kernels import ops as module
    asked = []
    monkeypatch.setattr(module.CudaOps, "_lib", lambda self, key: asked.append(key) or (_ for _ in ()).throw(LookupError(key)))
    for name, args in _given().items():
        with pytest.raises(LookupError):
            getattr(ops, name)(*args)
    assert asked == ["rows_e4m3", "rows_e4m3", "rows_e4m3", "gemm_e4m3", "gemm_int4"]
