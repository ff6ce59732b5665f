"""The engine's records of low-bit weights one by one on the GPU (low_bit_records.py): prompt portions, decoded tokens and both in one step, every
8-bit row and every product against its formula on the operands that it had."""
import pytest
import torch

from helpers import engine_for, make_model_dir, random_ids
from low_bit_records import check_plan, watch
from llmengine_b200.engine.engine import StepEntry
from plain_model import PlainQwen3
from tiny_configs import TINY_A, TINY_B, TINY_C, TINY_D

pytestmark = pytest.mark.gpu
FORMS = [dict(weights="e4m3"), dict(weights="int4"), dict(weights="int4", weight_group=32, weight_zero_points=True)]


@pytest.mark.parametrize("form", FORMS, ids=["e4m3", "int4", "int4-groups-of-32"])
@pytest.mark.parametrize("cfg", [TINY_A, TINY_B, TINY_C, TINY_D], ids=["A", "B", "C", "D"])
def test_records(tmp_path, cfg, form):
    if form["weights"] == "e4m3":
        cfg = dict(cfg, intermediate_size=cfg["intermediate_size"] // 16 * 16)
    folder = make_model_dir(str(tmp_path), cfg, seed=3)
    eng = engine_for(folder, "bfloat16", 1024, **form)
    check_plan(eng, PlainQwen3(folder, torch.bfloat16), form["weights"], form.get("weight_group", 128), form.get("weight_zero_points", False))
    seen = watch(eng)
    ids = {n: random_ids(256, cfg["vocab_size"], seed) for n, seed in (("a", 5), ("b", 6), ("c", 7))}
    at, steps = dict.fromkeys(ids, 0), 0

    def step(**tokens):
        nonlocal steps
        eng.step([StepEntry(n, ids[n][at[n]:at[n] + t], [t - 1]) for n, t in tokens.items()])
        at.update({n: at[n] + t for n, t in tokens.items()})
        steps += 1
    for tokens in (dict(a=1), dict(a=15), dict(b=17), dict(a=1, b=1), dict(a=1, b=1, c=200), dict(a=128, b=1), dict(a=8, b=1), dict(a=1, b=1, c=1), dict(b=150)):
        step(**tokens)
    eng.check_kernels()
    assert len(seen) == steps * len(eng.model.order) * (8 if form["weights"] == "e4m3" else 5)


@pytest.mark.parametrize("form", FORMS, ids=["e4m3", "int4", "int4-groups-of-32"])
def test_records_beside_plain_kernels(tmp_path, form):
    """The other operations by their plain kernels: what the records of low-bit weights are, does not follow from that choice."""
    folder = make_model_dir(str(tmp_path), TINY_D, seed=3)
    eng = engine_for(folder, "bfloat16", 256, kernels="plain", **form)
    seen, ids = watch(eng), random_ids(60, TINY_D["vocab_size"], 5)
    eng.step([StepEntry("a", ids[:50], [49])])
    eng.step([StepEntry("a", ids[50:51], [0])])
    eng.check_kernels()
    assert len(seen) == 2 * len(eng.model.order) * (8 if form["weights"] == "e4m3" else 5)
