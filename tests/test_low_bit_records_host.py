"""The records of low-bit weights one by one (low_bit_records.py) on the CPU stand-in, and that the checks see the mistakes they are for: each is planted
in the stand-in."""
from types import SimpleNamespace

import pytest
import torch

from helpers import engine_for, make_model_dir, random_ids
from low_bit_cases import LowBitOps, LowBitPlan, rows8
from low_bit_records import check_plan, watch
from llmengine_b200.engine.engine import StepEntry
from plain_model import PlainQwen3
from tiny_configs import TINY_A, TINY_B, TINY_C, TINY_D

E4M3, INT4, INT4_32 = dict(weights="e4m3"), dict(weights="int4"), dict(weights="int4", weight_group=32, weight_zero_points=True)
CONFIGS = [TINY_A, TINY_B, TINY_C, TINY_D]


class OneByOne:
    """The stand-in's plan, a part of it at a time."""

    def __init__(self, ops, plan):
        self.plan, self.one = plan, [LowBitPlan(ops, SimpleNamespace(ops=[op])) for op in plan.ops]

    def run(self, batch, first=0, count=-1):
        for one in self.one[first:None if count < 0 else first + count]:
            one.run(batch)


class Ops(LowBitOps):
    def compile(self, plan):
        return OneByOne(self, plan)


def _engine(tmp_path, cfg, form, ops):
    if form["weights"] == "e4m3":
        cfg = dict(cfg, intermediate_size=cfg["intermediate_size"] // 16 * 16)
    folder = make_model_dir(str(tmp_path), cfg, seed=3)
    return engine_for(folder, "bfloat16", 64, ops=ops, device="cpu", **form), folder, cfg


def _steps(eng, cfg):
    ids = random_ids(33, cfg["vocab_size"], 5)
    eng.step([StepEntry("r", ids[:20], [19])])
    for t in ids[20:22]:
        eng.step([StepEntry("r", [t], [0])])
    eng.step([StepEntry("r", ids[22:], [])])


@pytest.mark.parametrize("form", [E4M3, INT4, INT4_32], ids=["e4m3", "int4", "int4-groups-of-32"])
@pytest.mark.parametrize("cfg", CONFIGS, ids=["A", "B", "C", "D"])
def test_records(tmp_path, cfg, form):
    eng, folder, cfg = _engine(tmp_path, cfg, form, Ops())
    check_plan(eng, PlainQwen3(folder, torch.bfloat16), form["weights"], form.get("weight_group", 128), form.get("weight_zero_points", False))
    seen = watch(eng)
    _steps(eng, cfg)
    runs = len(eng.model.order)
    assert seen.count("linear_e4m3" if form["weights"] == "e4m3" else "linear_int4") == 4 * 4 * runs
    assert len(seen) == 4 * runs * (8 if form["weights"] == "e4m3" else 5)


class _Mistaken(OneByOne):
    """`at`: the kind of record the mistake is in; `mistake(record's operands, rows)`: it spoils what the record has written."""

    at = mistake = None

    def run(self, batch, first=0, count=-1):
        op, T = self.plan.ops[first], batch.num_tokens
        before = op.a["x"][:T].clone() if op.kind == "rows_e4m3" else None
        super().run(batch, first, 1)
        if op.kind == self.at:
            self.mistake(op.a, T, before)


def _unrounded(a, T, _):
    """The product of the rows before they were rounded to 8 bits, as nearly as it can be made: rows off by a quarter of a step."""
    x = a["x"][:T].float() * (1 + 2.0 ** -6 * torch.sin(torch.arange(a["x"].shape[1])))
    a["out"][:T] = ((x @ a["w"].float().t()) * a["x_scales"][:T, None] * a["w_scales"]).to(a["out"].dtype)


def _smaller_rows(a, T, _):
    a["scales"][:T] *= 1 - 2.0 ** -5


def _larger_scale(a, T, before):
    """Rows whose scale is twice what it may be: every value still half a step from the right one, of a row with a bit less."""
    q, s = rows8(before.float() if not a["gated"] else torch.nn.functional.silu(before.float().chunk(2, 1)[0]) * before.float().chunk(2, 1)[1])
    a["out"][:T], a["scales"][:T] = (q.float() / 2).to(torch.float8_e4m3fn), 2 * s


def _rounded_towards_zero(a, T, _):
    b = a["out"][:T].view(torch.uint8)
    b[:] = torch.where((b & 127) > 0, b - 1, b)


def _rounded_first(a, T, _):
    """The norm's output through bfloat16 before it goes to 8 bits."""
    h = a["x"][:T].float()
    h = (h / torch.sqrt((h * h).mean(1, keepdim=True) + a["eps"]) * a["gain"].float()).to(torch.bfloat16).float()
    a["out"][:T], a["scales"][:T] = rows8(h)


def _neighbours_scale(a, T, _):
    a["out"][:T] = (a["out"][:T].float() / a["w_scales"] * a["w_scales"].roll(1)).to(a["out"].dtype)


def _one_zero_point(a, T, _):
    """The last group's zero point taken for one more than it is."""
    last = a["x"][:T, (a["scales"].shape[1] - 1) * a["group"]:].float()
    a["out"][:T] = (a["out"][:T].float() - last.sum(1, keepdim=True) * a["scales"][:, -1].float()).to(a["out"].dtype)


def _stream_in_fewer_bits(a, T, _):
    a["x"][:T] = a["x"][:T].to(torch.bfloat16).float()


def _no_up(a, T, _):
    a["out"][:T] = torch.nn.functional.silu(a["gate_up"][:T].float().chunk(2, 1)[0]).to(a["out"].dtype)


@pytest.mark.parametrize("form,at,mistake,word", [
    (E4M3, "linear_e4m3", _unrounded, "product"), (E4M3, "rows_e4m3", _smaller_rows, "scales"), (E4M3, "rmsnorm_e4m3", _smaller_rows, "scales"),
    (E4M3, "rows_e4m3", _larger_scale, "scales"), (E4M3, "rows_e4m3", _rounded_towards_zero, "8-bit values"), (E4M3, "rmsnorm_e4m3", _rounded_towards_zero, "8-bit values"),
    (E4M3, "rmsnorm_e4m3", _rounded_first, "scales|8-bit values"), (E4M3, "linear_e4m3", _neighbours_scale, "product"), (E4M3, "rmsnorm_e4m3", _stream_in_fewer_bits, "residual"),
    (INT4_32, "linear_int4", _one_zero_point, "product"), (INT4, "swiglu", _no_up, "gate")])
@pytest.mark.parametrize("cfg", [TINY_A, TINY_C], ids=["A", "C"])
def test_mistakes_are_seen(tmp_path, cfg, form, at, mistake, word):
    plan = type("Mistaken", (_Mistaken,), dict(at=at, mistake=staticmethod(mistake)))
    ops = type("Ops", (Ops,), dict(compile=lambda self, p: plan(self, p)))()
    eng, _, cfg = _engine(tmp_path, cfg, form, ops)
    watch(eng)
    with pytest.raises(AssertionError, match=word):
        _steps(eng, cfg)


@pytest.mark.parametrize("form", [E4M3, INT4], ids=["e4m3", "int4"])
def test_a_wrong_plan_is_seen(tmp_path, form):
    eng, folder, cfg = _engine(tmp_path, TINY_A, form, Ops())
    plain = PlainQwen3(folder, torch.bfloat16)
    check_plan(eng, plain, form["weights"])
    for change in (lambda f: (f[0], f[1], f[3], f[2]), lambda f: (f[1], f[0], f[2], f[3])):              # gate|up and down's; the mixer's
        mixer, ffn = eng.model.blocks[1].mixer, eng.model.blocks[1].ffn
        kept = (mixer.w_qkv, mixer.w_o, ffn.w_gate_up, ffn.w_down)
        mixer.w_qkv, mixer.w_o, ffn.w_gate_up, ffn.w_down = change(kept)
        with pytest.raises((AssertionError, RuntimeError)):
            check_plan(eng, plain, form["weights"])
        mixer.w_qkv, mixer.w_o, ffn.w_gate_up, ffn.w_down = kept
    plain.w["model.layers.1.mlp.down_proj.weight"][0, 0] += 1
    with pytest.raises(AssertionError):
        check_plan(eng, plain, form["weights"])
