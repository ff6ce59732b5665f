"""What a sublayer of 4-bit weights adds to the residual stream is 32-bit, as with every other kind of weights."""
import pytest
import torch

from helpers import engine_for, make_model_dir, random_ids
from low_bit_cases import LowBitOps, PlainLowBit
from llmengine_b200.engine.engine import StepEntry
from tiny_configs import TINY_A, TINY_B, TINY_C


class Plain32(PlainLowBit):
    """The plain forward pass whose sublayers' results are not rounded on their way into the stream."""

    def product(self, layer, matrix, h):
        y = super().product(layer, matrix, h)
        return Kept(y) if matrix in ("self_attn.o_proj", "mlp.down_proj") else y


class Kept(torch.Tensor):
    """A 32-bit result that stays one where the formula asks for bfloat16."""

    @staticmethod
    def __new__(cls, data):
        return data.as_subclass(cls)

    def to(self, *args, **kwargs):
        return self.as_subclass(torch.Tensor)


@pytest.mark.parametrize("form", [dict(weights="int4"), dict(weights="int4", weight_group=32, weight_zero_points=True)], ids=["128", "32-with-zero-points"])
@pytest.mark.parametrize("cfg", [TINY_A, TINY_B, TINY_C], ids=["A", "B", "C"])
def test_the_stream_holds_32_bits(tmp_path, cfg, form):
    """The stand-in and the formula take the same steps: what is left between them is the order of 32-bit sums, and where such a sum lies on the
    edge of a rounding to bfloat16 (keys, values, rows of the next product) one step of that, some 2^-8 of single values."""
    folder = make_model_dir(str(tmp_path), cfg, seed=3)
    ids = random_ids(24, cfg["vocab_size"], 5)
    eng = engine_for(folder, "bfloat16", 64, ops=LowBitOps(), device="cpu", **form)
    plan = eng.model.plan(eng._caches)
    written = [op.a["out"].dtype for op in plan.ops if op.kind == "linear_int4"]
    assert written == [torch.bfloat16, torch.float32] * (len(written) // 2)             # q|k|v, output, gate|up, down
    assert all(op.a["delta"].dtype == torch.float32 for op in plan.ops if op.kind == "rmsnorm" and op.a["delta"] is not None)
    got = eng.step([StepEntry("r", ids, list(range(len(ids))))])
    more = (form.get("weight_group", 128), form.get("weight_zero_points", False))
    rounded, kept = PlainLowBit(folder, "int4", *more).logits(ids), Plain32(folder, "int4", *more).logits(ids)
    # a stream whose additions are rounded to bfloat16 is farther from the engine's than one whose additions are not
    assert (got - kept).norm() < 0.5 * (got - rounded).norm()
