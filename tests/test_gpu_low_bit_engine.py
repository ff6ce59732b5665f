"""The engine with weights of 8 and 4 bits on the GPU: prompts in portions beside decoded tokens against the plain formula with the same roundings
(bounds: test_low_bit_host.py), and generation with captured steps."""
import pytest
import torch

import plain_model as pm
from helpers import engine_for, make_model_dir, random_ids
from low_bit_cases import PlainLowBit
from llmengine_b200.engine.engine import StepEntry
from tiny_configs import TINY_A, TINY_B, TINY_C, TINY_D

pytestmark = pytest.mark.gpu
FORMS = [dict(weights="e4m3"), dict(weights="int4"), dict(weights="int4", weight_group=32, weight_zero_points=True)]
NAMES = ["e4m3", "int4", "int4-groups-of-32"]


def _config(cfg, form):
    """The configuration with a feed-forward whose rows 8-bit weights can have."""
    return dict(cfg, intermediate_size=cfg["intermediate_size"] // 16 * 16) if form["weights"] == "e4m3" else cfg


def _plain(folder, form):
    return PlainLowBit(folder, form["weights"], form.get("weight_group", 128), form.get("weight_zero_points", False))


def _near(got, want, stored, form):
    assert (got - want).norm() <= (0.1 if form["weights"] == "int4" else 0.74) * (stored - want).norm()


@pytest.mark.parametrize("form", FORMS, ids=NAMES)
@pytest.mark.parametrize("cfg", [TINY_A, TINY_B, TINY_C, TINY_D], ids=["A", "B", "C", "D"])
def test_logits(tmp_path, cfg, form):
    cfg = _config(cfg, form)
    folder = make_model_dir(str(tmp_path), cfg, seed=3)
    a, b = random_ids(150, cfg["vocab_size"], 5), random_ids(61, cfg["vocab_size"], 6)
    eng = engine_for(folder, "bfloat16", 512, **form)
    before = eng.ops.launches
    logits = {"a": [], "b": []}

    def step(**parts):                                           # name = tokens; all places wanted
        out = eng.step([StepEntry(n, t, list(range(len(t)))) for n, t in parts.items()]).cpu()
        for n, t in parts.items():
            logits[n].append(out[:len(t)])
            out = out[len(t):]
    step(a=a[:70])                                               # a portion alone, beside another request, single tokens, the rest
    step(a=a[70:130], b=b[:40])
    for i in range(4):
        step(a=[a[130 + i]], b=[b[40 + i]])
    step(a=a[134:140], b=[b[44]])
    step(a=a[140:], b=b[45:])
    eng.check_kernels()
    assert eng.ops.launches > before and ("gemm_e4m3" if form["weights"] == "e4m3" else "gemm_int4") in eng.ops._libs
    plain, stored = _plain(folder, form), pm.PlainQwen3(folder, torch.bfloat16)
    for n, ids in (("a", a), ("b", b)):
        _near(torch.cat(logits[n]), plain.logits(ids), stored.logits(ids), form)


@pytest.mark.parametrize("form", FORMS, ids=NAMES)
def test_generation_with_captured_steps(tmp_path, form):
    """The same tokens with and without captured decode steps, request beside request."""
    from llmengine_b200 import LLM, SamplingParams
    folder = make_model_dir(str(tmp_path), TINY_D, seed=4)
    prompts = [random_ids(n, TINY_D["vocab_size"], n) for n in (5, 37, 120)]
    outs = []
    for graphs in (False, True):
        llm = LLM(folder, max_cached_tokens=1024, page_size=16, max_num_seqs=4, max_num_batched_tokens=256, use_cuda_graphs=graphs, **form)
        outs.append([o.token_ids for o in llm.generate(prompts, SamplingParams(greedy=True), max_tokens=24)])
        del llm
    assert outs[0] == outs[1] and all(len(t) > 0 for t in outs[0])


@pytest.mark.parametrize("flags", [["--weights", "e4m3"], ["--weights", "int4", "--weight-group", "64", "--weight-zero-points"]])
def test_the_command(tmp_path, capsys, flags):
    from llmengine_b200.generate import main
    folder = make_model_dir(str(tmp_path), TINY_D, seed=4)
    assert main([folder, "5,17,3", "6", "--ignore-eos", "--greedy", "--max-cached-tokens", "512", *flags]) == 0
    out = capsys.readouterr().out.splitlines()
    assert len(out[0].split()) == 6 and "[Generated 6 tokens total]" in out
