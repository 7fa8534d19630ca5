"""Cases for the feed-forward operators: the gated block, the product with activation and residual,
and 8-bit activation checkpoints.

Where ``own`` is false, ``run`` computes each operator with elementary torch operations in 32 bits and
rounds once at the end; where it is true, it calls ``tensorplay_mlu_b200.ops``.  ``exact`` gives the same
results in 64 bits.

Shapes: x is [m, k]; the gated block's weight is [2n, k] (n gate rows, then n up rows) and its result
[m, n]; the plain product's weight is [n, k].  Checkpoints hold blocks of 32 elements of a row as int8
multiples of a power of two.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 32  # elements of a row that share one checkpoint exponent
ACTS = ("relu", "gelu", "gelu_tanh", "silu")
OPS = ("gated", "gated_save", "gated_pack", "gated_grad", "gated_grad8", "linear", "linear_save",
       "linear_grad", "pack", "act_grad8")


def _case(op, dtype, m, k, n, act, bias=False, residual=False, name=None):
    c = {"op": op, "dtype": dtype, "m": m, "k": k, "n": n, "act": act, "bias": bias, "residual": residual}
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # Serving: one token through the gated block's two projections (weights read once, nothing else).
        _case("gated", "bf16", 1, 4096, 11008, "silu", name="gated, one token"),
        # Serving: an odd batch of running requests, a block with biases.
        _case("gated", "f16", 37, 4096, 16384, "gelu_tanh", bias=True, name="gated, 37 tokens"),
        # Training, or a long prompt: the forward pass, pre-activations kept for the backward pass.
        _case("gated_save", "bf16", 16384, 4096, 11008, "silu", name="gated forward, 16384 tokens"),
        # Training: the gradients of input and weight.
        _case("gated_grad", "bf16", 8192, 4096, 11008, "silu", name="gated backward, 8192 tokens"),
        # Training on a ragged batch, a width that leaves rows off 16-byte boundaries, biases.
        _case("gated_grad", "f16", 1001, 1000, 2729, "gelu", bias=True, name="gated backward, ragged"),
        # Training in less memory: the forward pass that keeps its pre-activations in 8 bits.
        _case("gated_pack", "bf16", 8192, 4096, 8192, "silu", name="gated forward to 8 bits"),
        # ... and its gradients from them.
        _case("gated_grad8", "f16", 2048, 2048, 5504, "gelu_tanh", bias=True, name="gated backward from 8 bits"),
        # Serving: one token through the block's second product, added to the residual stream.
        _case("linear", "bf16", 1, 11008, 4096, "none", residual=True, name="linear + residual, one token"),
        # Training: Linear 4096 -> 16384 with GELU, bias and residual, the pre-activation kept.
        _case("linear_save", "bf16", 8192, 4096, 16384, "gelu", bias=True, residual=True,
              name="linear + gelu + residual, 8192 tokens"),
        # Training in full precision at the data-parallel MLP's width.
        _case("linear_grad", "f32", 512, 1024, 4096, "relu", bias=True, name="linear backward, f32"),
        # Activations into 8 bits and back (1 GiB of traffic and a quarter, out of every cache).
        _case("pack", "bf16", 8192, 1, 16384, "none", name="checkpoint and back"),
        # The activation's gradient from a checkpoint whose rows end inside a block.
        _case("act_grad8", "f16", 333, 1, 4097, "gelu", name="gelu backward from 8 bits, ragged"),
    ]


def _spread(rng, low, high):
    """An integer of [low, high], even over its logarithm: half of them any, half on a multiple of 64."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and v >= 64:
        v = v // 64 * 64
    return min(max(v, low), high)


def draw(rng):
    op = rng.choice(OPS)
    # A fused checkpoint is drawn in 16 bits alone: where the last bit of a 32-bit sum puts a value on the
    # other side of a rounding border, its 8 bits move by a whole step, far more than f32 values may differ.
    dtype = rng.choice(("bf16", "bf16", "f16", "f16") + (("f32",) if op != "gated_pack" else ()))
    elementwise = op in ("pack", "act_grad8")
    m, n = _spread(rng, 1, 16384), _spread(rng, 32, 16384)
    k = 1 if elementwise else _spread(rng, 32, 11008)
    act = rng.choice(ACTS if op not in ("linear", "linear_save") else ACTS + ("none",))
    c = _case(op, dtype, m, k, n, act, bias=not elementwise and rng.random() < 0.5,
              residual=op.startswith("linear") and op != "linear_grad" and rng.random() < 0.5)
    most = [max(work(x)[key] for x in listed()) for key in ("bytes", "flops")]
    while c["m"] > 1 and (work(c)["bytes"] > most[0] or work(c)["flops"] > most[1]):
        c["m"] = c["m"] * 2 // 3
    return c


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, m, k, n, op = DTYPES[case["dtype"]], case["m"], case["k"], case["n"], case["op"]

    def normal(*shape, scale=1.0):
        t = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)
        return t.mul_(scale).to(dtype)

    s = {"op": op, "act": case["act"], "dtype": dtype, "bias": None, "residual": None}
    rows = 2 * n if op.startswith("gated") else n
    wide = (m, 2, n) if op.startswith("gated") else (m, n)
    if op in ("pack", "act_grad8"):
        # Pre-activations: near normal, a few columns an order of magnitude larger than the rest.
        x = torch.randn(m, n, generator=g, device="cuda", dtype=torch.float32)
        x[:, ::97] *= 10.0
        s["x"] = x.to(dtype)
        if op == "act_grad8":
            s["saved"] = _pack(s["x"].float())
            s["grad"] = normal(m, n, scale=0.05)
        return s
    s["x"] = normal(m, k)
    s["weight"] = normal(rows, k, scale=k ** -0.5)
    if case["bias"]:
        s["bias"] = normal(rows, scale=0.1)
    if case["residual"]:
        s["residual"] = normal(m, n)
    if op.endswith(("grad", "grad8")):
        saved = normal(*wide)
        s["saved"] = _pack(saved.float()) if op == "gated_grad8" else saved
        s["grad"] = normal(m, n, scale=0.05)
    return s


# ------------------------------------------------------------------ plain forms, in 32 bits

def _phi(z):
    return 0.5 * (1.0 + torch.erf(z * 0.7071067811865476))


def _act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return z * _phi(z)
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z)))
    return z / (1.0 + torch.exp(-z))


def _slope(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return torch.where(z > 0, torch.ones_like(z), torch.zeros_like(z))
    if act == "gelu":
        return _phi(z) + z * torch.exp(-0.5 * z * z) * 0.3989422804014327
    if act == "gelu_tanh":
        t = torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * 0.7978845608028654 * (1.0 + 0.134145 * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 + z * (1.0 - s))


def _two_to(e):
    """2^e for whole e of [-126, 127], by its bits: a power function may be off in the last one."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _pack(z):
    """Blocks of 32 along the last dimension: the least power of two 2^e with max|z| <= 127 * 2^e, and
    z / 2^e rounded to the nearest integer, ties to even.  (int8 values, uint8 e + 127)."""
    n = z.shape[-1]
    pad = -n % BLOCK
    b = torch.nn.functional.pad(z, (0, pad)).unflatten(-1, (-1, BLOCK))
    fraction, power = torch.frexp(b.abs().amax(-1))  # amax = fraction * 2^power, 0.5 <= fraction < 1
    e = torch.where(fraction > 127.0 / 128.0, power - 6, power - 7).clamp(-126, 122)
    e = torch.where(fraction == 0, torch.full_like(e, -126), e)
    q = torch.round(b * _two_to(-e.unsqueeze(-1)))
    return q.flatten(-2)[..., :n].to(torch.int8), (e + 127).to(torch.uint8)


def _unpack(values, exponents):
    n = values.shape[-1]
    step = _two_to(exponents.to(torch.int32) - 127)
    return values.float() * step.repeat_interleave(BLOCK, -1)[..., :n]


def _plain(s):
    op, act, dtype = s["op"], s["act"], s["dtype"]
    if op == "pack":
        return {"values": _unpack(*_pack(s["x"].float())).to(dtype)}
    if op == "act_grad8":
        return {"grad": (s["grad"].float() * _slope(_unpack(*s["saved"]), act)).to(dtype)}
    x, w = s["x"].float(), s["weight"].float()
    if not op.endswith(("grad", "grad8")):
        z = x @ w.t()
        if s["bias"] is not None:
            z = z + s["bias"].float()
        if op.startswith("linear"):
            y = _act(z, act)
            if s["residual"] is not None:
                y = y + s["residual"].float()
            return {"y": y.to(dtype), "pre": z.to(dtype)} if op == "linear_save" else {"y": y.to(dtype)}
        z = z.unflatten(-1, (2, -1))
        h = (_act(z[:, 0], act) * z[:, 1]).to(dtype)
        if op == "gated_save":
            return {"h": h, "gate_up": z.to(dtype)}
        if op == "gated_pack":
            return {"h": h, "gate_up": _unpack(*_pack(z)).to(dtype)}
        return {"h": h}
    grad = s["grad"].float()
    z = _unpack(*s["saved"]) if op == "gated_grad8" else s["saved"].float()
    if op == "linear_grad":
        dz = grad * _slope(z, act)
    else:
        dz = torch.cat([grad * z[:, 1] * _slope(z[:, 0], act), grad * _act(z[:, 0], act)], -1)
    out = {"dx": (dz @ w).to(dtype), "dw": (dz.t() @ x).to(dtype)}
    if s["bias"] is not None:
        out["db"] = dz.sum(0).to(dtype)
    return out


# ------------------------------------------------------------------ the framework's operators

def _own(s):
    from tensorplay_mlu_b200 import ops

    op, act = s["op"], s["act"]
    if op == "pack":
        return {"values": ops.checkpoint_unpack(*ops.checkpoint_pack(s["x"]), s["dtype"])}
    if op == "act_grad8":
        return {"grad": ops.checkpoint_activation_backward(s["grad"], *s["saved"], act)}
    x, w, b = s["x"], s["weight"], s["bias"]
    if op == "gated":
        return {"h": ops.gated_linear(x, w, b, act)}
    if op == "gated_save":
        h, gate_up = ops.native_gated_linear(x, w, b, act)
        return {"h": h, "gate_up": gate_up}
    if op == "gated_pack":
        h, saved = ops.native_gated_linear(x, w, b, act, checkpoint=True)
        return {"h": h, "gate_up": ops.checkpoint_unpack(*saved, s["dtype"])}
    if op == "linear":
        return {"y": ops.linear_act(x, w, b, s["residual"], act)}
    if op == "linear_save":
        y, pre = ops.native_linear_act(x, w, b, s["residual"], act)
        return {"y": y, "pre": pre}
    backward = ops.native_linear_act_backward if op == "linear_grad" else ops.native_gated_linear_backward
    dx, dw, db = backward(s["grad"], x, w, s["saved"], act, (True, True, b is not None))
    return {"dx": dx, "dw": dw} if b is None else {"dx": dx, "dw": dw, "db": db}


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    m, k, n, op = case["m"], case["k"], case["n"], case["op"]
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    wide = 2 * n if op.startswith("gated") else n
    packed = m * wide + m * (wide // n) * -(-n // BLOCK)
    if op == "pack":
        return {"bytes": 2 * m * n * size + 2 * packed, "flops": 4 * m * n}
    if op == "act_grad8":
        return {"bytes": 2 * m * n * size + packed, "flops": 20 * m * n}
    elements = m * k + wide * k + (wide if case["bias"] else 0)
    if op.endswith(("grad", "grad8")):
        # gradient in; dx, dw, db out; what the forward pass saved
        elements += m * n + m * k + wide * k + (wide if case["bias"] else 0)
        saved = packed if op == "gated_grad8" else m * wide * size
        return {"bytes": elements * size + saved, "flops": 4 * m * k * wide}
    elements += m * n * (2 if case["residual"] else 1)
    if op in ("gated_save", "linear_save"):
        elements += m * wide
    # the checkpoint written, read back, and the values written
    extra = 2 * packed + m * wide * size if op == "gated_pack" else 0
    return {"bytes": elements * size + extra, "flops": 2 * m * k * wide}


# ------------------------------------------------------------------ 64 bits

def _exact_act(z, act):
    f = torch.nn.functional
    return {"none": lambda: z, "relu": lambda: f.relu(z), "gelu": lambda: f.gelu(z),
            "gelu_tanh": lambda: f.gelu(z, approximate="tanh"), "silu": lambda: f.silu(z)}[act]()


def _exact_slope(z, act):
    with torch.enable_grad():
        v = z.detach().requires_grad_()
        y = _exact_act(v, act)
        return torch.ones_like(z) if act == "none" else torch.autograd.grad(y, v, torch.ones_like(y))[0]


def _powers(device):
    return torch.tensor([math.ldexp(1.0, i) for i in range(-127, 128)], dtype=torch.float64, device=device)


def _exact_values(values, exponents):
    step = _powers(values.device)[exponents.long()]
    return values.double() * torch.repeat_interleave(step, BLOCK, dim=-1)[..., :values.shape[-1]]


def _exact_rounded(z):
    """What a checkpoint of z stands for, by its definition: the first of the powers of two that fits."""
    powers = _powers(z.device)
    out = torch.empty_like(z)
    for a in range(0, z.shape[-1], BLOCK):
        part = z[..., a:a + BLOCK]
        step = powers[1:250]  # 2^-126 .. 2^122
        first = torch.searchsorted(127.0 * step, part.abs().amax(-1, keepdim=True).contiguous()).clamp_max(248)
        out[..., a:a + BLOCK] = torch.round(part / step[first]) * step[first]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op, act = s["op"], s["act"]
    if op == "pack":
        return {"values": _exact_rounded(s["x"].double())}
    if op == "act_grad8":
        return {"grad": s["grad"].double() * _exact_slope(_exact_values(*s["saved"]), act)}
    x, w = s["x"].double(), s["weight"].double()
    n = case["n"]
    if not op.endswith(("grad", "grad8")):
        b = s["bias"].double() if s["bias"] is not None else torch.zeros((), dtype=torch.float64, device=x.device)
        z = torch.einsum("mk,nk->mn", x, w) + b
        if op.startswith("linear"):
            y = _exact_act(z, act) + (0 if s["residual"] is None else s["residual"].double())
            return {"y": y, "pre": z} if op == "linear_save" else {"y": y}
        h = _exact_act(z[:, :n], act) * z[:, n:]
        if op == "gated":
            return {"h": h}
        z = z.reshape(case["m"], 2, n)
        # A checkpoint of the pre-activations has no value in 64 bits: a rounding border may fall either way.
        return {"h": h, "gate_up": z if op == "gated_save" else None}
    grad = s["grad"].double()
    z = _exact_values(*s["saved"]) if op == "gated_grad8" else s["saved"].double()
    if op == "linear_grad":
        parts = [(grad * _exact_slope(z, act), w)]
    else:
        gate, up = z[:, 0], z[:, 1]
        parts = [(grad * up * _exact_slope(gate, act), w[:n]), (grad * _exact_act(gate, act), w[n:])]
    dx = torch.zeros_like(x)
    for dz, part in parts:
        dx += torch.einsum("mn,nk->mk", dz, part)
    out = {"dx": dx, "dw": torch.cat([torch.einsum("mn,mk->nk", dz, x) for dz, _ in parts])}
    if s["bias"] is not None:
        out["db"] = torch.cat([dz.sum(0) for dz, _ in parts])
    return out
