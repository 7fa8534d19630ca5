"""The feed-forward operators to the accuracy their arithmetic allows.

The activations are tested on pre-activations that are exact: a weight of
zeros leaves the bias, and a weight of ones on the diagonal hands the
gradient through, so that nothing but the evaluation of the activation, its
roundings and the result's rounding remains.  With g the activation's gate (a
= z g), u half the dtype's eps, t the exponent of the sigmoid in octaves:

* 16-bit results.  silu and gelu_tanh evaluate g = 1 / (1 + 2^t) with ex2 and
  rcp instructions: 2^-22 and 2^-23 relative, and the exponent's own rounding,
  at most four half steps of |t| 2^-24 ln 2, of which the factor 1 - g reaches
  g.  gelu's Phi is good to 3e-7 absolutely (that is more than a step of
  float16 in the far negative tail, where the result is below 1e-4).
* float32 results.  expf is good to 2 units in the last place, normcdff to 5.
* none and relu are exact.

Products: a sum of K exact products accumulated in fp32 is off by at most
(K + 8) 2^-23 of the summed magnitudes (room for the split into TF32 parts
included)."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
BETA, KAPPA = math.sqrt(2 / math.pi), 0.044715


@pytest.fixture(scope="module")
def ops(backend):
    return backend.ops


def rand(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def half_eps(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half the spacing of the dtype's subnormals (and what flushing loses, where fp32 results underflow)."""
    return {torch.float16: 2.0 ** -25}.get(dtype, 1e-36)


def gate(z, act):
    """The gate and 2u (the sigmoid's argument), in 64 bits.  Phi by the
    complementary error function: (1 + erf) / 2 has nothing left in the tail."""
    if act == "gelu":
        return torch.special.erfc(-z * math.sqrt(0.5)) / 2, None
    v = z if act == "silu" else 2 * BETA * (z + KAPPA * z ** 3)
    return torch.sigmoid(v), v


def value(z, act):
    if act == "none":
        return z
    if act == "relu":
        return z.clamp_min(0)
    return z * gate(z, act)[0]


def slope(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    g, _ = gate(z, act)
    if act == "gelu":
        return g + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    s = 2 * BETA * (1 + 3 * KAPPA * z * z) if act == "gelu_tanh" else 1.0
    return g + z * g * (1 - g) * s


def gate_error(z, act, dtype):
    g, v = gate(z, act)
    if act == "gelu":
        return 5 * 2.0 ** -23 * g if dtype == torch.float32 else torch.full_like(z, 3e-7) + 2.0 ** -23 * g
    # exp: 2^-22; reciprocal or division and the sum: 2^-23; the argument: six half steps at most
    return g * (2.0 ** -22 + 2.0 ** -23 + (1 - g) * (2.0 ** -22 + 6 * 2.0 ** -24 * v.abs()))


def value_error(z, act, dtype):
    if act in ("none", "relu"):
        return torch.zeros_like(z)
    return z.abs() * gate_error(z, act, dtype) + 2.0 ** -23 * value(z, act).abs()


def slope_error(z, act, dtype):
    if act in ("none", "relu"):
        return torch.zeros_like(z)
    g, _ = gate(z, act)
    e = gate_error(z, act, dtype)
    if act == "gelu":
        # z phi(z): exp's 2^-22, the square's two half steps in its argument z^2 / 2, three products
        bell = (z * torch.exp(-z * z / 2)).abs() / math.sqrt(2 * math.pi)
        return e + bell * (2.0 ** -21 + z * z * 2.0 ** -23) + 2.0 ** -23 * (g + bell)
    s = 2 * BETA * (1 + 3 * KAPPA * z * z) if act == "gelu_tanh" else torch.ones_like(z)
    term = (z * g * (1 - g) * s).abs()
    return e * (1 + (z * s * (1 - 2 * g)).abs()) + (z * s * g).abs() * 2.0 ** -23 + 2.0 ** -21 * (g + term)


def check(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert bool(torch.isfinite(got).all()), what
    bad = (got - want).abs() > bound
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got - want).abs() / bound.clamp_min(1e-300)).max()))


def grid(n, dtype):
    """n values over (-12, 12), denser near zero, and a few beyond."""
    z = torch.linspace(-1, 1, n, dtype=torch.float64) ** 3 * 12
    z[:6] = torch.tensor([-60.0, 60.0, -30.0, 30.0, 0.0, -0.0])
    return z.to(dtype).cuda()


# ------------------------------------------------- activations by themselves

# Few rows (16 and 64 rows a tile), the CTA-pair kernel with one and several tiles.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [3, 40, 1030])
def test_activations_of_exact_pre_activations(ops, dtype, m):
    n, k, u = 1032, 8, half_eps(dtype)
    bias = grid(n, dtype)
    x, w, ones = rand(m, k, dtype=dtype), torch.zeros(n, k, dtype=dtype, device="cuda"), torch.ones_like(bias)
    z = bias.double().expand(m, n)
    for act in ACTS:
        want, e = value(z, act), value_error(z, act, dtype)
        bound = e + u * (want.abs() + e) + least(dtype)
        if act in ("none", "relu"):
            bound = torch.zeros_like(want)
        y, pre = ops.native_linear_act(x, w, bias, None, act)
        assert torch.equal(pre, bias.expand(m, n))
        check(y, want, bound, (act, "linear_act"))
        h, pre = ops.native_gated_linear(x, torch.cat([w, w]), torch.cat([bias, ones]), act)
        assert torch.equal(pre[:, 0], bias.expand(m, n)) and bool((pre[:, 1] == 1).all())
        check(h, want, bound, (act, "gated_linear"))
    # without input features: the elementwise kernel
    for act in ACTS:
        want, e = value(z, act), value_error(z, act, dtype)
        y = ops.linear_act(x[:, :0], w[:, :0], bias, None, act)
        check(y, want, e + u * (want.abs() + e) + least(dtype) * (act not in ("none", "relu")), (act, "no features"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [64, 65])
def test_slopes_of_exact_pre_activations(ops, dtype, n):
    """dx = dz I, so dx is dz after its rounding to the dtype (float32: but for the low part's last bits, 2^-21)."""
    m, u = 37, half_eps(dtype)
    saved = grid(m * n, dtype).view(m, n)
    dy = rand(m, n, dtype=dtype, seed=1)
    eye = torch.eye(n, dtype=dtype, device="cuda")
    x = rand(m, n, dtype=dtype, seed=2)
    z = saved.double()
    for act in ACTS:
        want = dy.double() * slope(z, act)
        e = dy.double().abs() * slope_error(z, act, dtype) + 2.0 ** -23 * want.abs()
        bound = e + (u + (2.0 ** -21 if dtype == torch.float32 else 0.0)) * (want.abs() + e) + least(dtype)
        dx, _, db = ops.native_linear_act_backward(dy, x, eye, saved, act)
        check(dx, want, bound, (act, "dx"))
        total = want.sum(0)
        eb = e.sum(0) + (m + 8) * 2.0 ** -23 * want.abs().sum(0)
        check(db, total, eb + u * (total.abs() + eb) + least(dtype), (act, "db"))
        gated = torch.stack([saved, torch.ones_like(saved)], 1)
        dx, _, _ = ops.native_gated_linear_backward(dy, x, torch.cat([eye, torch.zeros_like(eye)]), gated, act)
        check(dx, want, bound, (act, "gated dx"))
        up, ea = dy.double() * value(z, act), dy.double().abs() * value_error(z, act, dtype)
        ea = ea + 2.0 ** -23 * up.abs()
        dx, _, _ = ops.native_gated_linear_backward(dy, x, torch.cat([torch.zeros_like(eye), eye]), gated, act)
        bound = ea + (u + (2.0 ** -21 if dtype == torch.float32 else 0.0)) * (up.abs() + ea) + least(dtype)
        check(dx, up, bound, (act, "gated dx through the up part"))


# ------------------------------------------------ gradients and differences

def losses(x, w, b, r, dy, gated, act):
    z = x @ w.t() + b
    n = dy.shape[1]
    y = value(z[:, :n], act) * z[:, n:] if gated else value(z, act) + r
    return (y * dy).sum()


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gradients_against_differences_in_64_bits(ops, gated, act):
    """float32 gradients along a direction, against central differences of the
    loss in 64 bits.  With steps of 2^-16 the differences' own truncation is
    2^-32 of third derivatives (below 100 times the first here), their rounding
    2^-52 / 2^-16; what is left is the kernels' error, element by element: of
    the saved pre-activations (slopes change by at most 1.2 a unit), of the
    slope, and of the sums.  The direction follows the gradient's signs, so a
    gradient that is zero, halved or transposed is far outside."""
    m, k, n = 6, 24, 40
    parts = 2 if gated else 1
    x, w, b = rand(m, k, seed=1), rand(parts * n, k, seed=2, scale=k ** -0.5), rand(parts * n, seed=3)
    dy, r = rand(m, n, seed=4), rand(m, n, seed=5)
    if gated:
        _, saved = ops.native_gated_linear(x, w, b, act)
        grads = ops.native_gated_linear_backward(dy, x, w, saved, act)
    else:
        _, saved = ops.native_linear_act(x, w, b, r, act)
        grads = ops.native_linear_act_backward(dy, x, w, saved, act)
    xd, wd, bd, rd, gd = x.double(), w.double(), b.double(), r.double(), dy.double()
    z = xd @ wd.t() + bd
    ez = (k + 8) * 2.0 ** -23 * (xd.abs() @ wd.abs().t() + bd.abs()) + 2.0 ** -23 * z.abs()
    zg = z[:, :n]
    d, ed = slope(zg, act), slope_error(zg, act, torch.float32) + 1.2 * ez[:, :n]
    if gated:
        zu, eu = z[:, n:], ez[:, n:]
        a, ea = value(zg, act), value_error(zg, act, torch.float32) + 1.2 * ez[:, :n]
        dz = torch.cat([gd * zu * d, gd * a], 1)
        edz = torch.cat([gd.abs() * (zu.abs() * ed + d.abs() * eu + ed * eu), gd.abs() * ea], 1) + 2.0 ** -22 * dz.abs()
    else:
        dz, edz = gd * d, gd.abs() * ed + 2.0 ** -22 * (gd * d).abs()
    acc = 2.0 ** -23
    errors = (edz @ wd.abs() + (parts * n + 8) * acc * (dz.abs() @ wd.abs()),
              edz.t() @ xd.abs() + (m + 8) * acc * (dz.abs().t() @ xd.abs()),
              edz.sum(0) + (m + 8) * acc * dz.abs().sum(0))
    exact = (dz @ wd, dz.t() @ xd, dz.sum(0))
    for which, (grad, error, right) in enumerate(zip(grads, errors, exact)):
        g = torch.Generator().manual_seed(20 + which)
        step = (torch.rand(grad.shape, generator=g).double().cuda() + 0.5) * right.sign()
        h = 2.0 ** -16 / float(step.norm())

        def at(sign):
            args = [xd, wd, bd]
            args[which] = args[which] + sign * h * step
            return float(losses(*args, rd, gd, gated, act))

        want = (at(1) - at(-1)) / (2 * h)
        got = float((grad.double() * step).sum())
        bound = float((step.abs() * (error + half_eps(torch.float32) * right.abs())).sum())
        bound += 100 * 2.0 ** -32 * abs(want) + 2.0 ** -30 * float((step * right).abs().sum())
        assert bound < 2e-3 * abs(want), (which, bound, want)   # a bound that would notice
        assert abs(got - want) <= bound, (which, got, want, bound)


# ----------------------------------------- products in the kernels users run

def forward_bound(z, ez, act, dtype, residual):
    u, want = half_eps(dtype), value(z, act)
    e = value_error(z, act, dtype) + 1.13 * ez
    if residual is not None:
        want = want + residual.double()
    return want, e + u * (want.abs() + e) + least(dtype)


# More k-blocks than the CTA pair's ring holds, several tiles a cluster; saved
# rows and checkpoint bytes that TMA stores, and ones it does not.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [4112, 4104, 4099])
def test_linear_act_of_many_tiles(ops, dtype, n):
    m, k, u = 4000, 520, half_eps(dtype)
    x, w, b = rand(m, k, dtype=dtype, seed=1), rand(n, k, dtype=dtype, seed=2, scale=k ** -0.5), rand(n, dtype=dtype, seed=3)
    r = rand(m, n, dtype=dtype, seed=4)
    z = x.double() @ w.double().t() + b.double()
    ez = (k + 8) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t() + b.double().abs())
    want, bound = forward_bound(z, ez, "gelu_tanh", dtype, r)
    y, pre = ops.native_linear_act(x, w, b, r, "gelu_tanh")
    check(y, want, bound, "y")
    check(pre, z, ez + u * z.abs() + least(dtype), "pre")
    y2, (values, exponents) = ops.native_linear_act(x, w, b, r, "gelu_tanh", checkpoint=True)
    assert torch.equal(y, y2)
    got = ops.checkpoint_unpack(values, exponents, torch.float32)
    blocks = torch.nn.functional.pad(z.abs() + ez, (0, -n % 32)).unflatten(-1, (-1, 32))
    step = blocks.amax(-1, keepdim=True).expand_as(blocks).flatten(-2)[:, :n] * (2 / 127)
    check(got, z, ez + step / 2, "checkpoint")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [2064, 2049])
def test_gated_linear_of_many_tiles(ops, dtype, n):
    m, k, u = 4000, 520, half_eps(dtype)
    x, w = rand(m, k, dtype=dtype, seed=1), rand(2 * n, k, dtype=dtype, seed=2, scale=k ** -0.5)
    b = rand(2 * n, dtype=dtype, seed=3)
    z = x.double() @ w.double().t() + b.double()
    ez = (k + 8) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t() + b.double().abs())
    g, up, eg, eu = z[:, :n], z[:, n:], ez[:, :n], ez[:, n:]
    a, ea = value(g, "silu"), value_error(g, "silu", dtype) + 1.13 * eg
    e = ea * up.abs() + a.abs() * eu + ea * eu + 2.0 ** -23 * (a * up).abs()
    bound = e + u * ((a * up).abs() + e) + least(dtype)
    h, pre = ops.native_gated_linear(x, w, b, "silu")
    check(h, a * up, bound, "h")
    check(pre.flatten(1), z, ez + u * z.abs() + least(dtype), "gate and up")
    h2, (values, exponents) = ops.native_gated_linear(x, w, b, "silu", checkpoint=True)
    assert torch.equal(h, h2)
    got = ops.checkpoint_unpack(values, exponents, torch.float32).flatten(1)
    blocks = torch.nn.functional.pad((z.abs() + ez).unflatten(1, (2, n)), (0, -n % 32)).unflatten(-1, (-1, 32))
    step = blocks.amax(-1, keepdim=True).expand_as(blocks).flatten(-2)[..., :n].flatten(1) * (2 / 127)
    check(got, z, ez + step / 2, "checkpoint")


# Tiles of 128 rows in all three products of float32 (each with enough of them
# for every SM), sums of more than 500 terms, rows off 16-byte boundaries.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1024, 2432, 1100), (1031, 2433, 1101)])
@pytest.mark.parametrize("gated", [False, True])
def test_backward_of_many_tiles(ops, dtype, shape, gated):
    m, k, n = shape
    u, parts = half_eps(dtype), 2 if gated else 1
    x, w = rand(m, k, dtype=dtype, seed=1), rand(parts * n, k, dtype=dtype, seed=2, scale=k ** -0.5)
    saved = rand(*((m, 2, n) if gated else (m, n)), dtype=dtype, seed=3)
    dy = rand(m, n, dtype=dtype, seed=4, scale=0.1)
    z, g = saved.double(), dy.double()
    gz = z[:, 0] if gated else z
    d, ed = slope(gz, "silu"), slope_error(gz, "silu", dtype)
    if gated:
        a, ea = value(gz, "silu"), value_error(gz, "silu", dtype)
        dz = torch.cat([g * z[:, 1] * d, g * a], 1)
        e = torch.cat([(g * z[:, 1]).abs() * ed, g.abs() * ea], 1) + 2.0 ** -22 * dz.abs()
    else:
        dz = g * d
        e = g.abs() * ed + 2.0 ** -22 * dz.abs()
    edz = e + u * (dz.abs() + e) + least(dtype)
    backward = ops.native_gated_linear_backward if gated else ops.native_linear_act_backward
    dx, dw, db = backward(dy, x, w, saved, "silu")
    acc = 2.0 ** -23
    for got, left, right, el, length, what in ((dx, dz, w.double(), edz, parts * n, "dx"),
                                               (dw, dz.t(), x.double(), edz.t(), m, "dw")):
        want, terms = left @ right, left.abs() @ right.abs()
        bound = el @ right.abs() + (length + 8) * acc * terms
        check(got, want, bound + u * (want.abs() + bound) + least(dtype), what)
    bound = e.sum(0) + (m + 8) * acc * dz.abs().sum(0)
    check(db, dz.sum(0), bound + u * (dz.sum(0).abs() + bound) + least(dtype), "db")


def test_results_and_sums_past_32_bits(ops):
    """More than 2^31 pre-activations: rows at both ends of the result and of
    the input gradient, and every bias sum, in 64 bits."""
    m, k, n, u = 98304, 64, 11008, half_eps(torch.bfloat16)
    assert 2 * m * n > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(m, k, generator=g, device="cuda").bfloat16()
    w = rand(2 * n, k, dtype=torch.bfloat16, seed=2, scale=k ** -0.5)
    h, gate_up = ops.native_gated_linear(x, w)
    rows = torch.tensor([0, 1, 48777, 97999, 98302, 98303], device="cuda")
    z = x[rows].double() @ w.double().t()
    ez = (k + 8) * 2.0 ** -23 * (x[rows].double().abs() @ w.double().abs().t())
    zg, up, eg, eu = z[:, :n], z[:, n:], ez[:, :n], ez[:, n:]
    a, ea = value(zg, "silu"), value_error(zg, "silu", torch.bfloat16) + 1.13 * eg
    e = ea * up.abs() + a.abs() * eu + ea * eu + 2.0 ** -23 * (a * up).abs()
    check(h[rows], a * up, e + u * ((a * up).abs() + e) + 1e-36, "h")
    del h
    held = ops.checkpoint_pack(gate_up)
    del gate_up
    dy = torch.ones(m, n, device="cuda", dtype=torch.bfloat16)
    dx, _, db = ops.native_gated_linear_backward(dy, x, w, held, "none", (True, False, True))
    # dy is 1 and the activation none: dz is the up part beside the gate part, as the checkpoint holds them.
    sums = torch.zeros(2, n, dtype=torch.float64, device="cuda")
    terms = torch.zeros_like(sums)
    for at in range(0, m, 4096):
        part = ops.checkpoint_unpack(held[0][at:at + 4096], held[1][at:at + 4096], torch.float32)
        sums += part.sum(0, dtype=torch.float64)
        terms += part.abs().sum(0, dtype=torch.float64)
    sums, terms = sums.flip(0).reshape(-1), terms.flip(0).reshape(-1)
    # 128 groups of 768 rows, each added in order by 8 warps' threads at most, then joined: fewer than 1024 additions.
    bound = 1024 * 2.0 ** -24 * terms
    check(db, sums, bound + u * (sums.abs() + bound), "db")
    dz = ops.checkpoint_unpack(held[0][rows], held[1][rows], torch.float32).flip(1).reshape(6, -1).double()
    want, size = dz @ w.double(), dz.abs() @ w.double().abs()
    bound = (u + (2 * n + 8) * 2.0 ** -23) * size
    check(dx[rows], want, bound + u * (want.abs() + bound), "dx")
