"""A model's records of low-bit weights, each held against its formula in 64 bits on the operands that it really had.

A whole forward pass of 8-bit rows cannot be held closely: one value on the edge of a rounding that falls to its other side takes others with it.
A record by itself can: `Watch` runs a compiled plan one record at a time and asks of each of the low-bit ones what its formula makes of what lay in
its operands.  `check_plan` asks of the plan that the operands are the right ones: every product reads what the record before it wrote and the
weights of its place in the model.

Bounds, relative to the value (u = 2^-24, half a step of 32 bits): a norm's 8-bit rows 72 u and the gate's 110 u of the value before its rounding to 8
bits, plain rows 4 u; a product K / 16 + 40 units of 2^-22 of sum |x w| and half a step of its output; where more than 16 rows meet 4-bit weights 2^-8
of every |x w| (each weight is one bfloat16 number); the gate in bfloat16 110 u and half a step."""
import torch

from llmengine_b200.weights.quantize import dequantize_int4, quantize_e4m3, quantize_int4
from low_bit_cases import MATRICES

LEAST = 2.0 ** -100
U = 2.0 ** -24
F8 = torch.float8_e4m3fn
LOW = ("rmsnorm_e4m3", "rows_e4m3", "linear_e4m3", "linear_int4", "swiglu")


def check_rows8(h, q, scales, d):
    """8-bit rows and scales against the exact rows h: a stored number lies between the roundings of both ends of what 32 bits may make of it."""
    a = h.abs().amax(1).clamp(min=LEAST) / 448
    assert torch.all((scales.double() - a).abs() <= d * a), "scales"
    y = h / a[:, None]
    ends = torch.stack([y * (1 - d), y * (1 + d)]).clamp(-448, 448).float().to(F8).float()
    assert torch.all((ends.amin(0) <= q.float()) & (q.float() <= ends.amax(0))), "8-bit values"


def _gated(gate_up):
    g, u = gate_up.double().chunk(2, 1)
    return g * torch.sigmoid(g) * u


def _near(out, want, size, k, weight_rounding=0.0):
    half = torch.finfo(out.dtype).eps / 2
    assert torch.all((out.double() - want).abs() <= half * want.abs() + ((k / 16 + 40) * 2.0 ** -22 + weight_rounding) * size + 1e-30), "product"


def int4_weights(a):
    """The weights of a `linear_int4` record in 64 bits, from the codes as they lie: value 32 j + 8 q + e of a block in word 4 q + j, at bits 4 (e / 2)
    + 16 (e % 2)."""
    k = a["x"].shape[1]
    at = torch.arange(k, device=a["w"].device)
    block, j, q, e = at // 128, at % 128 // 32, at % 32 // 8, at % 8
    bit = 4 * (e // 2) + 16 * (e % 2)
    code = (a["w"][:, block * 64 + (4 * q + j) * 4 + bit // 8].long() >> (bit % 8)) & 15
    zero = 8.0 if a["zeros"] is None else a["zeros"].double()[:, at // a["group"]]
    return (code.double() - zero) * a["scales"].double()[:, at // a["group"]]


def check_record(op, before, T):
    """One record that has run on T rows; `before`: its x (and delta) as they were."""
    a, k = op.a, op.kind
    if k == "rmsnorm_e4m3":
        x = before["x"]
        if a["delta"] is not None:
            x = x + before["delta"].float()
        assert torch.equal(a["x"][:T], x), "residual stream"
        h = x.double()
        h = h / torch.sqrt((h * h).mean(1, keepdim=True) + a["eps"]) * a["gain"].double()
        check_rows8(h, a["out"][:T], a["scales"][:T], 72 * U)
    elif k == "rows_e4m3":
        x = before["x"]
        check_rows8(_gated(x) if a["gated"] else x.double(), a["out"][:T], a["scales"][:T], (110 if a["gated"] else 4) * U)
    elif k == "linear_e4m3":
        x, w = a["x"][:T].double() * a["x_scales"][:T].double()[:, None], a["w"].double() * a["w_scales"].double()[:, None]
        _near(a["out"][:T], x @ w.t(), x.abs() @ w.abs().t(), x.shape[1])
    elif k == "linear_int4":
        x, w = a["x"][:T].double(), int4_weights(a)
        _near(a["out"][:T], x @ w.t(), x.abs() @ w.abs().t(), x.shape[1], 2.0 ** -8 if T > 16 else 0.0)
    elif k == "swiglu":
        h = _gated(before["gate_up"])
        assert torch.all((a["out"][:T].double() - h).abs() <= (torch.finfo(a["out"].dtype).eps / 2 + 110 * U) * h.abs() + 1e-38), "gate"


class Watch:
    """A compiled plan that runs one record at a time, the low-bit ones checked."""

    def __init__(self, plan, compiled):
        self.plan, self.compiled, self.checked = plan, compiled, []

    def run(self, batch, first=0, count=-1):
        T = batch.num_tokens
        for i, op in enumerate(self.plan.ops):
            before = {n: op.a[n][:T].clone() for n in ("x", "delta", "gate_up") if op.kind in LOW and op.a.get(n) is not None}
            self.compiled.run(batch, i, 1)
            if op.kind in LOW:
                check_record(op, before, T)
                self.checked.append(op.kind)


def watch(eng):
    """The engine runs its plan so from now on; the list of what was checked."""
    compile_, seen = eng.ops.compile, []

    def watched(plan):
        w = Watch(plan, compile_(plan))
        w.checked = seen
        return w
    eng.ops.compile = watched
    return seen


def check_plan(eng, plain, kind, group=128, zeros=False):
    """The plan's products read what was written for them, and the weights of their place, rounded on the engine's device: q|k|v, output, gate|up, down
    of every run."""
    ops = [op for op in eng.model.plan(eng._caches).ops]
    same = lambda a, b: a.data_ptr() == b.data_ptr() and a.shape[1:] == b.shape[1:]                     # noqa: E731
    products = [i for i, op in enumerate(ops) if op.kind == ("linear_e4m3" if kind == "e4m3" else "linear_int4")]
    assert len(products) == 4 * len(plain.order)
    last = None

    def rounded(layer, m):
        w = plain.w[f"model.layers.{layer}.{m}.weight"].to(torch.bfloat16).to(eng.device)
        if kind == "e4m3":
            q, s = quantize_e4m3(w)
            return q.float() * s[:, None]
        packed, s, z = quantize_int4(w, group, zeros)
        return dequantize_int4(packed, s, z, w.shape[1], group)
    for n, i in enumerate(products):
        a, (layer, _), place = ops[i].a, plain.order[n // 4], n % 4
        made = next(op for op in reversed(ops[:i]) if op.kind in ("rmsnorm", "rmsnorm_e4m3", "rows_e4m3", "swiglu", "attention", "attend"))
        assert same(a["x"], made.a["out"])
        if kind == "e4m3":
            assert made.kind == ("rows_e4m3" if place in (1, 3) else "rmsnorm_e4m3") and same(a["x_scales"], made.a["scales"])
            if place == 1:
                source = next(op for op in reversed(ops[:i]) if op.kind in ("attention", "attend"))
                assert not made.a["gated"] and same(made.a["x"], source.a["out"])
            if place == 3:
                assert made.a["gated"] and same(made.a["x"], ops[products[n - 1]].a["out"])
        elif place == 3:
            assert made.kind == "swiglu" and same(made.a["gate_up"], ops[products[n - 1]].a["out"])
        if place in (0, 2):                                                                             # the norm adds the sublayer before
            assert (made.a["delta"] is None) == (last is None) and (last is None or same(made.a["delta"], last))
        if place in (1, 3):
            last = a["out"]
        names = (MATRICES[:3], MATRICES[3:4], MATRICES[4:6], MATRICES[6:])[place]
        want = torch.cat([rounded(layer, m) for m in names])[:a["w"].shape[0]]                   # (a run that reads another's cache: q alone)
        got = a["w"].float() * a["w_scales"][:, None] if kind == "e4m3" else int4_weights(a).float()
        assert torch.equal(got, want), (n, names)
