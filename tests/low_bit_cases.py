"""Models with weights of 8 and 4 bits: the plain forward pass in the order of roundings of the engine's, and the CPU stand-in's part of the
records."""
import torch

import plain_model as pm
from host_ops import HostOps, HostPlan
from llmengine_b200.weights.quantize import dequantize_int4, quantize_e4m3, quantize_int4

LEAST = 2.0 ** -100
BF16 = torch.bfloat16
MATRICES = ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj")


def rows8(h):
    """Rows as their 8-bit numbers and scales stand for, and the two apart."""
    a = h.abs().amax(1).clamp(min=LEAST) / 448
    q = (h / a[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q, a


class PlainLowBit(pm.PlainQwen3):
    """`weights` "e4m3" or "int4": every layer matrix rounded as the engine rounds it (the matrices that share a product are rounded row by
    row, so rounding them one by one is the same), every product's rows 8-bit where its weights are."""

    def __init__(self, model_dir, weights, group=128, zeros=False):
        super().__init__(model_dir, BF16)
        self.kind = weights
        self.rounded = {}
        for layer in range(self.L):
            for m in MATRICES:
                w = self.w[f"model.layers.{layer}.{m}.weight"]
                if weights == "e4m3":
                    q, s = quantize_e4m3(w)
                    self.rounded[layer, m] = q.float() * s[:, None]
                else:
                    packed, s, z = quantize_int4(w, group, zeros)
                    self.rounded[layer, m] = dequantize_int4(packed, s, z, w.shape[1], group)

    def product(self, layer, matrix, h):
        if self.kind == "e4m3":
            q, a = rows8(h)
            h = q.float() * a[:, None]
        return h @ self.rounded[layer, matrix].t()

    def logits(self, ids):
        r = lambda v: v.to(BF16).float()                                       # noqa: E731
        late = r if self.kind == "int4" else (lambda v: v)                     # a sublayer's result on its way into the stream
        first = r if self.kind == "int4" else (lambda v: v)                    # the norm's output: its 8-bit rows are made from 32 bits
        w, n, pos = self.w, len(ids), torch.arange(len(ids))
        x, kept = pm.embedding(w["model.embed_tokens.weight"], ids), []
        for layer, cache_from in self.order:
            p = f"model.layers.{layer}."
            h = first(pm.rms_norm(x, w[p + "input_layernorm.weight"], self.eps))

            def head(m, norm=None):
                y = r(self.product(layer, f"self_attn.{m}_proj", h)).view(n, -1, self.hd)
                return y if norm is None else r(pm.rope(pm.qk_norm(y, w[p + f"self_attn.{norm}.weight"], self.eps), pos, self.theta))
            q = head("q", "q_norm")
            if cache_from is None:
                kept.append((head("k", "k_norm"), head("v")))
                k, v = kept[-1]
            else:
                k, v = kept[cache_from]
                kept.append(None)
            a = r(pm.attention(q, k, v, self.windows[layer]).reshape(n, -1))
            x = x + late(self.product(layer, "self_attn.o_proj", a))
            h = first(pm.rms_norm(x, w[p + "post_attention_layernorm.weight"], self.eps))
            act = pm.swiglu(r(self.product(layer, "mlp.gate_proj", h)), r(self.product(layer, "mlp.up_proj", h)))
            x = x + late(self.product(layer, "mlp.down_proj", first(act)))
        return pm.linear(r(pm.rms_norm(x, w["model.norm.weight"], self.eps)), w["lm_head.weight"])


class LowBitOps(HostOps):
    def compile(self, plan):
        return LowBitPlan(self, plan)


class LowBitPlan(HostPlan):
    def run(self, batch, first=0, count=-1):
        T = batch.num_tokens
        for i, op in enumerate(self.plan.ops):
            a, k = op.a, op.kind
            if k == "rmsnorm_e4m3":
                if a["delta"] is not None:
                    a["x"][:T] += a["delta"][:T].float()
                self._place(a, pm.rms_norm(a["x"][:T], a["gain"], a["eps"]), T)
            elif k == "rows_e4m3":
                x = a["x"][:T].float()
                self._place(a, pm.swiglu(*x.chunk(2, 1)) if a["gated"] else x, T)
            elif k == "linear_e4m3":
                y = (a["x"][:T].float() @ a["w"].float().t()) * a["x_scales"][:T, None] * a["w_scales"]
                a["out"][:T] = y.to(a["out"].dtype)
            elif k == "linear_int4":
                x = a["x"][:T].float()
                a["out"][:T] = (x @ dequantize_int4(a["w"], a["scales"], a["zeros"], x.shape[1], a["group"]).t()).to(a["out"].dtype)
            elif k == "swiglu":
                self.ops.swiglu(a["gate_up"][:T], a["out"][:T])
            else:
                super().run(batch, i, 1)

    @staticmethod
    def _place(a, h, T):
        a["out"][:T], a["scales"][:T] = rows8(h)
