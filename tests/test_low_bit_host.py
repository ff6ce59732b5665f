"""The engine with weights of 8 and 4 bits on the CPU stand-in: the records its parts emit add up to the formula, and what it refuses.

The stand-in computes in 32 bits what the formula computes in 32 bits, with the sums of a product in another order here and there, so a value at
the edge of a rounding may fall to its other side.  How far that goes, against how far the low-bit formula is from the model as stored:
* 4 bits: what may differ is one step of a bfloat16 rounding, 2^-8 of a value, where the weights' rounding is a tenth of every product (half a
  step in 7 against values of 2 to 3): 2^-8 / 0.1 = 0.04, asked is 0.1;
* 8 bits: one value of a row of K that falls to its other side moves a product by a step of 2^-3 to 2^-4 over sqrt(K), for K = 64 to 128 some
  2^-7, and that takes a share p = 2^-7 / 2^-3.5 = 0.09 of the next row's values across an edge.  A crossing is a whole step, a rounding's error
  a step over sqrt(12) on average: sqrt(12 p) = 1.04 of the activations' error, and that is 1 / sqrt(2) of both operands': 0.74 if it happened to
  every row.  Asked is that.  (A record left out, a matrix or a scale taken for another, is off by the result itself.)
"""
import pytest
import torch

import plain_model as pm
from helpers import engine_for, make_model_dir, random_ids
from low_bit_cases import LowBitOps, PlainLowBit
from llmengine_b200.config import ConfigError, EngineConfig, config_from_dict
from llmengine_b200.engine.engine import Engine, StepEntry
from tiny_configs import TINY_A, TINY_B, TINY_C, TINY_E
from tiny_vifelix import TINY_A as OTHER_DESIGN

FORMS = [dict(weights="e4m3"), dict(weights="int4"), dict(weights="int4", weight_group=32, weight_zero_points=True)]
NAMES = ["e4m3", "int4", "int4-groups-of-32"]


def _plain(folder, form):
    return PlainLowBit(folder, form["weights"], form.get("weight_group", 128), form.get("weight_zero_points", False))


@pytest.mark.parametrize("form", FORMS, ids=NAMES)
@pytest.mark.parametrize("cfg", [TINY_A, TINY_B, TINY_C], ids=["A", "B", "C"])
def test_logits(tmp_path, cfg, form):
    if form["weights"] == "e4m3" and any(cfg[k] % 16 for k in ("hidden_size", "intermediate_size")):
        cfg = dict(cfg, intermediate_size=cfg["intermediate_size"] // 16 * 16)
    folder = make_model_dir(str(tmp_path), cfg, seed=3)
    ids = random_ids(33, cfg["vocab_size"], 5)
    eng = engine_for(folder, "bfloat16", 64, ops=LowBitOps(), device="cpu", **form)
    got = [eng.step([StepEntry("r", ids[:20], list(range(20)))]).clone()]
    got += [eng.step([StepEntry("r", [t], [0])]).clone() for t in ids[20:24]]
    got.append(eng.step([StepEntry("r", ids[24:], list(range(len(ids) - 24)))]).clone())
    got = torch.cat(got)
    want, stored = _plain(folder, form).logits(ids), pm.PlainQwen3(folder, torch.bfloat16).logits(ids)
    assert (got - want).norm() <= (0.1 if form["weights"] == "int4" else 0.74) * (stored - want).norm()


def test_what_is_refused(tmp_path):
    for bad in (dict(weights="int8"), dict(weights="e4m3", dtype="float32"), dict(weights="int4", weight_group=16), dict(weight_group=256)):
        with pytest.raises(ConfigError):
            EngineConfig(**bad)
    for cfg, form, word in ((TINY_E, dict(weights="e4m3"), "multiple of 16"), (TINY_E, dict(weights="int4"), "multiple of 8"),
                            (OTHER_DESIGN, dict(weights="e4m3"), "another kind"), (OTHER_DESIGN, dict(weights="int4"), "another kind")):
        with pytest.raises(ValueError, match=word):
            Engine(config=config_from_dict(cfg), random_seed=1, ops=LowBitOps(),
                   engine_config=EngineConfig(max_cached_tokens=64, page_size=16, max_num_seqs=2, max_num_batched_tokens=64, device="cpu", **form))


def test_stored_weights_emit_what_they_did(tmp_path):
    """Nothing of a model as stored goes through the new records."""
    folder = make_model_dir(str(tmp_path), TINY_A, seed=3)
    eng = engine_for(folder, "bfloat16", 64, ops=LowBitOps(), device="cpu")
    kinds = {op.kind for op in eng.model.plan(eng._caches).ops}
    assert kinds == {"embedding", "rmsnorm", "linear", "attention", "linear_swiglu"}
    assert isinstance(eng.model.blocks[0].mixer.w_qkv, torch.Tensor) and eng.model.blocks[0].ffn.w_down.dtype == torch.bfloat16
