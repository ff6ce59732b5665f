"""What is timed of the operators that serve a dense model from weights of 8 or 4 bits.

`rmsnorm_e4m3`, `rows_e4m3` and `swiglu_e4m3` write rows of 8-bit floating-point numbers (e4m3: four bits of exponent, three of
mantissa, no infinity, 448 the largest) with one 32-bit scale a row; `linear_e4m3` multiplies such rows by weights of the same kind with
one scale an output; `linear_int4` multiplies bfloat16 rows by weights of 4 bits with a scale, and where given a zero point, for every
32, 64 or 128 neighbouring values of a weight row.  Sizes are those of the benchmark's shapes (8B: 4096 / 12288, 14B: 5120 / 17408, 32B:
5120 / 25600, and the small model of width 2,048) with token counts from one decoded token to a whole prompt portion.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-6
LARGEST = 448.0                 # the largest e4m3 number
LEAST = 2.0 ** -100             # a row's largest value counts as at least this
F8 = torch.float8_e4m3fn
_ops = None


# ----------------------------------------------------------------------------- the cases
def listed():
    return [
        # the norm in front of a layer's first product, one decoded token: the smallest call there is
        {"name": "norm_one_token", "op": "norm", "tokens": 1, "size": 4096, "delta": "float32"},
        # the same of the 14B shape for a prompt portion of no round length
        {"name": "norm_prompt", "op": "norm", "tokens": 1999, "size": 5120, "delta": "bfloat16"},
        # attention's output of eight decoded tokens on its way into the output product
        {"name": "rows_decode", "op": "rows", "tokens": 8, "size": 4096, "dtype": "bfloat16"},
        # the same for two prompt portions of the 8B shape
        {"name": "rows_prompt", "op": "rows", "tokens": 4096, "size": 4096, "dtype": "bfloat16"},
        # the gate of the 8B shape while 16 requests decode
        {"name": "swiglu_decode", "op": "swiglu", "tokens": 16, "size": 12288, "dtype": "bfloat16"},
        # the gate of the 14B shape for a prompt portion
        {"name": "swiglu_prompt", "op": "swiglu", "tokens": 2048, "size": 17408, "dtype": "bfloat16"},
        # the q|k|v product of the 8B shape while 8 requests decode: weights streamed once
        {"name": "e4m3_decode", "op": "e4m3", "tokens": 8, "n": 6144, "k": 4096, "out": "bfloat16"},
        # the down product of the 8B shape in a step that mixes a short prompt with decoded tokens, into the 32-bit stream
        {"name": "e4m3_mixed", "op": "e4m3", "tokens": 77, "n": 4096, "k": 12288, "out": "float32"},
        # gate and up of the 8B shape for a whole prompt portion: the largest pass
        {"name": "e4m3_prompt", "op": "e4m3", "tokens": 2048, "n": 24576, "k": 4096, "out": "bfloat16"},
        # gate and up of the 8B shape for one decoded token: the matrix-vector product
        {"name": "int4_one_token", "op": "int4", "tokens": 1, "n": 24576, "k": 4096, "group": 128, "zeros": False},
        # the down product of the small model while 13 requests decode, small groups with zero points
        {"name": "int4_few_tokens", "op": "int4", "tokens": 13, "n": 2048, "k": 5504, "group": 32, "zeros": True},
        # the q|k|v product of the 14B shape for a prompt portion of no round length
        {"name": "int4_prompt", "op": "int4", "tokens": 1900, "n": 7168, "k": 5120, "group": 128, "zeros": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rows", "swiglu", "e4m3", "e4m3", "int4", "int4"])
    tokens = _log(rng, 1, 4096)
    if op in ("norm", "rows", "swiglu"):
        # widths in whole pieces of eight values, a few of any even size
        size = 8 * _log(rng, 8, 2176) if rng.random() < 0.8 else 2 * _log(rng, 32, 8704)
        tokens = min(tokens, (2048 * 17408) // size)
        if op == "norm":
            return {"op": op, "tokens": tokens, "size": min(size, 8192), "delta": rng.choice(["float32", "bfloat16", "none"])}
        return {"op": op, "tokens": tokens, "size": size, "dtype": rng.choice(["bfloat16", "bfloat16", "float32"])}
    n, tokens = _log(rng, 64, 24576), min(tokens, 2048)
    if op == "e4m3":
        return {"op": op, "tokens": tokens, "n": n, "k": 16 * _log(rng, 8, 256 if n > 8192 else 768), "out": rng.choice(["bfloat16", "float32"])}
    # half the largest listed product at most: the weights are also unpacked in the plain form
    return {"op": op, "tokens": tokens if n <= 8192 else min(tokens, 512), "n": n, "k": 8 * _log(rng, 16, 512 if n > 8192 else 640),
            "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5}


# ----------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed * 7919 + 13)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, device=DEVICE, generator=g)


def _activations(g, tokens, size):
    """Rows as a layer has them: every row its own magnitude, a few channels far larger than the rest."""
    x = _randn(g, tokens, size) * torch.exp(0.5 * _randn(g, tokens, 1))
    loud = torch.randint(0, size, (max(1, size // 512),), device=DEVICE, generator=g)
    x[:, loud] *= 12.0
    return x


def _pack(w):
    """Values 0..15, [n, k], as the framework stores them: a row in blocks of 128 values (the last one filled up with zeros), 64 bytes
    each; word 4 q + j of a block's sixteen 32-bit words holds values 32 j + 8 q .. + 7, the even ones in its low half, the odd ones in
    its high half, four bits each, in order."""
    n, k = w.shape
    w = torch.nn.functional.pad(w, (0, -k % 128)).view(n, -1, 4, 4, 4, 2)             # block, j, q, pair, even or odd
    w = w.permute(0, 1, 3, 2, 5, 4).reshape(n, -1, 2)                                  # block, q, j, even then odd, pair
    return (w[..., 0] | (w[..., 1] << 4)).to(torch.uint8).contiguous()


def prepare(case, seed):
    g = _generator(seed)
    t, op = case["tokens"], case["op"]
    s = {"case": case}
    if op == "norm":
        d = case["size"]
        s["x"] = _activations(g, t, d)
        s["gain"] = (1.0 + 0.1 * _randn(g, d)).to(torch.bfloat16)
        s["delta"] = None if case["delta"] == "none" else (0.3 * _randn(g, t, d)).to(getattr(torch, case["delta"]))
        s["sum"] = torch.empty_like(s["x"])
    elif op in ("rows", "swiglu"):
        d = case["size"]
        s["x"] = _activations(g, t, d if op == "rows" else 2 * d).to(getattr(torch, case["dtype"]))
    else:
        n, k = case["n"], case["k"]
        if op == "e4m3":
            x, w = _activations(g, t, k), 0.02 * _randn(g, n, k)
            s["xs"], s["ws"] = x.abs().amax(1) / LARGEST, w.abs().amax(1) / LARGEST
            s["x"], s["w"] = (x / s["xs"][:, None]).to(F8), (w / s["ws"][:, None]).to(F8)
            s["out"] = torch.empty(t, n, dtype=getattr(torch, case["out"]), device=DEVICE)
        else:
            group = case["group"]
            groups = (k + group - 1) // group
            s["x"] = _activations(g, t, k).to(torch.bfloat16)
            s["scales"] = (0.02 * (0.2 + torch.rand(n, groups, device=DEVICE, generator=g)) / 4).to(torch.bfloat16)
            s["zeros"] = torch.randint(5, 11, (n, groups), device=DEVICE, generator=g).to(torch.uint8) if case["zeros"] else None
            s["w"] = _pack((3.0 * _randn(g, n, k) + 8.0).round().clamp(0, 15).to(torch.int32))
            s["out"] = torch.empty(t, n, dtype=torch.bfloat16, device=DEVICE)
        return s
    s["q"] = torch.empty(t, case["size"], dtype=F8, device=DEVICE)
    s["scales"] = torch.empty(t, device=DEVICE)
    return s


# ----------------------------------------------------------------------------- the plain forms and the framework's
def _quantised(h):
    scales = h.abs().amax(1).clamp(min=LEAST) / LARGEST
    return (h / scales[:, None]).to(F8), scales


def _unpacked(w, k):
    n = w.shape[0]
    w = torch.stack([w & 15, w >> 4], -1).view(n, -1, 4, 4, 2, 4)                      # block, q, j, even then odd, pair
    return w.permute(0, 1, 3, 2, 5, 4).reshape(n, -1)[:, :k]


def _framework():
    global _ops
    if _ops is None:
        from llmengine_b200.kernels.ops import CudaOps
        _ops = CudaOps(torch.device(DEVICE))
    return _ops


def run(s):
    case, op = s["case"], s["case"]["op"]
    if own:
        ops = _framework()
        if op == "norm":
            total = s["sum"] if s["delta"] is not None else None
            ops.rmsnorm_e4m3(s["x"], s["gain"], EPS, s["q"], s["scales"], delta=s["delta"], total=total)
            return (s["q"], s["scales"]) + ((total,) if total is not None else ())
        if op == "rows":
            return ops.rows_e4m3(s["x"], s["q"], s["scales"])
        if op == "swiglu":
            return ops.swiglu_e4m3(s["x"], s["q"], s["scales"])
        if op == "e4m3":
            return ops.linear_e4m3(s["x"], s["xs"], s["w"], s["ws"], s["out"])
        return ops.linear_int4(s["x"], s["w"], s["scales"], s["out"], zeros=s["zeros"])
    if op == "norm":
        x = s["x"] if s["delta"] is None else s["x"] + s["delta"].float()
        h = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * s["gain"].float()
        return _quantised(h) + ((x,) if s["delta"] is not None else ())
    if op == "rows":
        return _quantised(s["x"].float())
    if op == "swiglu":
        gate, up = s["x"].float().chunk(2, 1)
        return _quantised(gate / (1.0 + torch.exp(-gate)) * up)
    if op == "e4m3":
        return ((s["x"].float() @ s["w"].float().t()) * s["xs"][:, None] * s["ws"]).to(s["out"].dtype)
    k, group = case["k"], case["group"]
    zero = 8.0 if s["zeros"] is None else s["zeros"].float().repeat_interleave(group, 1)[:, :k]
    w = (_unpacked(s["w"], k).float() - zero) * s["scales"].float().repeat_interleave(group, 1)[:, :k]
    return (s["x"].float() @ w.t()).to(torch.bfloat16)


def work(case):
    t, op = case["tokens"], case["op"]
    if op == "norm":
        d, extra = case["size"], {"none": 0, "bfloat16": 2 + 4, "float32": 4 + 4}[case["delta"]]
        return {"bytes": t * d * (4 + extra + 1) + 2 * d + 4 * t, "flops": 8 * t * d}
    if op in ("rows", "swiglu"):
        d, e = case["size"], 4 if case["dtype"] == "float32" else 2
        return {"bytes": t * d * (e * (2 if op == "swiglu" else 1) + 1) + 4 * t, "flops": (9 if op == "swiglu" else 3) * t * d}
    n, k = case["n"], case["k"]
    if op == "e4m3":
        return {"bytes": t * k + n * k + 4 * (t + n) + t * n * (4 if case["out"] == "float32" else 2), "flops": 2 * t * n * k}
    groups = (k + case["group"] - 1) // case["group"]
    return {"bytes": 2 * t * k + n * ((k + 127) // 128 * 64) + n * groups * (3 if case["zeros"] else 2) + 2 * t * n, "flops": 2 * t * n * k}


# ----------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    """Quantised rows are given before their rounding to 8 bits, products from the stored 8- and 4-bit values."""
    s, op = prepare(case, seed), case["op"]
    x = s["x"].double()
    if op in ("norm", "rows", "swiglu"):
        total = None
        if op == "norm":
            if s["delta"] is not None:
                x = total = x + s["delta"].double()
            x = x / torch.sqrt((x ** 2).sum(1, keepdim=True) / x.shape[1] + EPS) * s["gain"].double()
        elif op == "swiglu":
            d = case["size"]
            x = x[:, :d] * torch.sigmoid(x[:, :d]) * x[:, d:]
        a = torch.clamp(torch.max(torch.abs(x), dim=1).values, min=LEAST) / LARGEST
        return (x / a.unsqueeze(1), a) + ((total,) if total is not None else ())
    if op == "e4m3":
        return (x * s["xs"].double().unsqueeze(1)) @ (s["w"].double() * s["ws"].double().unsqueeze(1)).T
    n, k, group = case["n"], case["k"], case["group"]
    column = torch.arange(k, device=DEVICE)
    within, block = column % 128, column // 128
    word = 4 * (within % 32 // 8) + within // 32
    place = within % 8 // 2 + 4 * (within % 2)                      # which four bits of the word
    stored = s["w"][:, block * 64 + word * 4 + place // 2].long()
    values = torch.where(place % 2 == 1, stored >> 4, stored & 15).double()
    at = column // group
    zero = s["zeros"].double()[:, at] if s["zeros"] is not None else 8.0
    return x @ ((values - zero) * s["scales"].double()[:, at]).T
