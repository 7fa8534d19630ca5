"""The feed-forward operators against a plain implementation in 64 bits:
gated_linear, linear_act (activation and residual), their backward passes, and
8-bit activation checkpoints.

Tolerances count roundings.  With u the largest relative error of one rounding
to the dtype (half its eps), a pre-activation z = sum_k x w + b accumulated in
fp32 and possibly rounded to the dtype is off by

    e_z <= (K + 8) 2^-23 sum_k |x w| + u |z|

(fp32 sums of K exact products, with room for the products' split into TF32
parts: 4 * 2^-23).  The activations' slopes are at most 1.13 in magnitude
(gelu's maximum, 1.129), their evaluation is off by at most 2^-18 |z| (the
16-bit forms: 3e-7 in the normal CDF, 2^-21 in exp and reciprocal, times the
exponent's magnitude of at most 16 before the result is below the rounding
step).  Results are rounded once more: u |y|.  A 16-bit gradient dz is rounded
once before its products, so a product with it is off by u sum |dz w| (and for
float16's subnormals by 2^-25 sum |w|), plus the fp32 accumulation.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


@pytest.fixture(scope="module")
def ops(backend):
    return backend.ops


def rand(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def dev(t):
    return None if t is None else t.cuda()


def half_eps(dtype):
    return torch.finfo(dtype).eps / 2


def act64(z, act):
    if act == "none":
        return z
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return z * torch.special.ndtr(z)
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z * torch.sigmoid(z)


def slope64(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s))


def check(got, want, bound, what):
    got = got.cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = (got - want).abs() > bound
    assert torch.isfinite(got).all(), what
    assert not bad.any(), (what, int(bad.sum()), float(((got - want).abs() / bound.clamp_min(1e-300)).max()))


def pack_reference(x):
    """Checkpoints by their definition, in 64 bits: (values, exponents, the values they stand for)."""
    n = x.shape[-1]
    pad = -n % 32
    b = torch.nn.functional.pad(x.double(), (0, pad)).unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    steps = torch.tensor([math.ldexp(1.0, i) for i in range(-126, 123)], dtype=torch.float64)
    e = torch.searchsorted(127.0 * steps, top.nan_to_num(0, 0, 0).contiguous()).clamp_max(248)
    step = steps[e].unsqueeze(-1)
    q = torch.round(b / step)
    largest = torch.finfo(x.dtype).max
    q = torch.where((q * step).abs() > largest, q.sign() * 63, q)
    bad = ~torch.isfinite(top)
    q = torch.where(bad.unsqueeze(-1), torch.zeros_like(q), q)
    value = torch.where(bad.unsqueeze(-1), torch.full_like(q, math.nan), q * step)
    exponents = torch.where(bad, torch.full_like(e, 255), e + 1)
    return q.flatten(-2)[..., :n].to(torch.int8), exponents.to(torch.uint8), value.flatten(-2)[..., :n]


def pre_activation(x, w, b):
    """z in 64 bits and the bound of its error before any rounding to the dtype."""
    z = x.double() @ w.double().t()
    terms = x.double().abs() @ w.double().abs().t()
    if b is not None:
        z = z + b.double()
        terms = terms + b.double().abs()
    return z, (x.shape[-1] + 8) * 2.0 ** -23 * terms


def activation_bound(z, e):
    return 1.13 * e + 2.0 ** -18 * z.abs() + 1e-30


# ------------------------------------------------------------------ forward

# (M, K, N): one token; a few; below, at and above the tiles of 128 and 256
# rows; ragged in every dimension; rows off 16-byte boundaries (odd K, odd N).
SHAPES = [(1, 64, 32), (1, 4096, 1000), (3, 1027, 129), (17, 256, 96), (33, 512, 4099), (64, 96, 640),
          (129, 200, 264), (255, 72, 1000), (300, 520, 1032), (513, 1000, 777), (1030, 64, 1536), (2, 1, 1),
          (65, 8, 7)]
# A wide weight for one and a few rows (tiles of 128 + 128 columns), more rows
# than one tile of 64 or 128 with K split over a cluster.
WIDE = [(1, 768, 11008), (24, 256, 11008), (100, 2048, 520), (200, 4096, 96), (600, 512, 1032)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES + WIDE)
def test_gated_linear_forward(ops, dtype, shape):
    m, k, n = shape
    u = half_eps(dtype)
    x, w = rand(m, k, dtype=dtype, seed=1), rand(2 * n, k, dtype=dtype, seed=2, scale=k ** -0.5)
    for act, bias in (("silu", None), ("gelu", 1), ("gelu_tanh", None), ("relu", 1), ("none", None)):
        b = rand(2 * n, dtype=dtype, seed=3) if bias else None
        z, e = pre_activation(x, w, b)
        ez = e + u * z.abs()
        g, up, eg, eu = z[:, :n], z[:, n:], ez[:, :n], ez[:, n:]
        a, ea = act64(g, act), activation_bound(g, eg)
        want = a * up
        bound = ea * up.abs() + a.abs() * eu + ea * eu
        bound = bound + u * (want.abs() + bound) + torch.finfo(dtype).smallest_normal * u
        h = ops.gated_linear(dev(x), dev(w), dev(b), act)
        check(h, want, bound, (act, "h"))
        h2, gate_up = ops.native_gated_linear(dev(x), dev(w), dev(b), act)
        check(h2, want, bound, (act, "h, saving"))
        assert gate_up.shape == (m, 2, n) and gate_up.dtype == dtype
        zb = ez + torch.finfo(dtype).smallest_normal * u
        check(gate_up.flatten(1), z, zb, (act, "gate_up"))
        h3, (values, exponents) = ops.native_gated_linear(dev(x), dev(w), dev(b), act, checkpoint=True)
        check(h3, want, bound, (act, "h, checkpoint"))
        assert values.shape == (m, 2, n) and exponents.shape == (m, 2, -(-n // 32))
        # The checkpoint: half a step, where a step is at most 2/127 of the block's largest value.
        got = ops.checkpoint_unpack(values, exponents, torch.float32).flatten(1)
        zp = torch.nn.functional.pad((z.abs() + ez).unflatten(1, (2, n)), (0, -n % 32)).unflatten(-1, (-1, 32))
        step = zp.amax(-1, keepdim=True).expand_as(zp).flatten(-2)[..., :n].flatten(1) * (2 / 127)
        check(got, z, ez + step / 2, (act, "checkpoint"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES + WIDE)
def test_linear_act_forward(ops, dtype, shape):
    m, k, n = shape
    u = half_eps(dtype)
    x, w = rand(m, k, dtype=dtype, seed=1), rand(n, k, dtype=dtype, seed=2, scale=k ** -0.5)
    r0 = rand(m, n, dtype=dtype, seed=4)
    for act, bias, res in (("none", None, 1), ("silu", 1, 1), ("gelu", 1, None), ("gelu_tanh", None, 1),
                           ("relu", None, None)):
        b, r = (rand(n, dtype=dtype, seed=3) if bias else None), (r0 if res else None)
        z, e = pre_activation(x, w, b)
        ez = e + u * z.abs()
        a, ea = act64(z, act), activation_bound(z, ez)
        want = a + (r.double() if res else 0)
        tiny = torch.finfo(dtype).smallest_normal * u
        bound = ea + u * (want.abs() + ea) + tiny
        check(ops.linear_act(dev(x), dev(w), dev(b), dev(r), act), want, bound, (act, "y"))
        y, pre = ops.native_linear_act(dev(x), dev(w), dev(b), dev(r), act)
        check(y, want, bound, (act, "y, saving"))
        check(pre, z, ez + tiny, (act, "pre"))
        y, (values, exponents) = ops.native_linear_act(dev(x), dev(w), dev(b), dev(r), act, checkpoint=True)
        check(y, want, bound, (act, "y, checkpoint"))
        got = ops.checkpoint_unpack(values, exponents, torch.float32)
        zp = torch.nn.functional.pad(z.abs() + ez, (0, -n % 32)).unflatten(-1, (-1, 32))
        step = zp.amax(-1, keepdim=True).expand_as(zp).flatten(-2)[..., :n] * (2 / 127)
        check(got, z, ez + step / 2, (act, "checkpoint"))


# ----------------------------------------------------------------- backward

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 64, 32), (1, 1000, 129), (5, 130, 72), (40, 512, 257), (300, 264, 136),
                                   (257, 1000, 333), (2, 1, 1), (1025, 72, 96)])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("packed", [False, True])
def test_backward(ops, dtype, shape, gated, packed):
    m, k, n = shape
    u = half_eps(dtype)
    parts = 2 if gated else 1
    x, w = rand(m, k, dtype=dtype, seed=1), rand(parts * n, k, dtype=dtype, seed=2, scale=k ** -0.5)
    saved = rand(*((m, 2, n) if gated else (m, n)), dtype=dtype, seed=5)
    dy = rand(m, n, dtype=dtype, seed=6, scale=0.1)
    backward = ops.native_gated_linear_backward if gated else ops.native_linear_act_backward
    for act in ACTS:
        z, held = saved.double(), dev(saved)
        if packed:
            _, _, z = pack_reference(saved)
            held = ops.checkpoint_pack(dev(saved))
        g = dy.double()
        if gated:
            a, s = act64(z[:, 0], act), slope64(z[:, 0], act)
            dz = torch.cat([g * z[:, 1] * s, g * a], 1)
            e = torch.cat([(g * z[:, 1]).abs(), g.abs()], 1) * 2.0 ** -16 * (1 + z[:, 0].abs()).repeat(1, 2)
        else:
            dz = g * slope64(z, act)
            e = g.abs() * 2.0 ** -16 * (1 + z.abs())
        if act in ("none", "relu"):
            e = dz.abs() * 2.0 ** -22
        # dz as it enters the products: evaluated in fp32 (e), rounded to the dtype.
        sub = 2.0 ** -25 if dtype == torch.float16 else 0.0
        edz = e + u * (dz.abs() + e) + sub
        wd, xd = w.double(), x.double()
        dx, dw, db = backward(dev(dy), dev(x), dev(w), held, act)
        acc = 2.0 ** -23
        want, terms = dz @ wd, dz.abs() @ wd.abs()
        bx = edz @ wd.abs() + (parts * n + 8) * acc * terms
        check(dx, want, bx + u * (want.abs() + bx) + sub + 1e-30, (act, "dx"))
        want, terms = dz.t() @ xd, dz.abs().t() @ xd.abs()
        bw = edz.t() @ xd.abs() + (m + 8) * acc * terms
        check(dw, want, bw + u * (want.abs() + bw) + sub + 1e-30, (act, "dw"))
        want, terms = dz.sum(0), dz.abs().sum(0)
        bb = e.sum(0) + (m + 8) * acc * terms
        check(db, want, bb + u * (want.abs() + bb) + sub + 1e-30, (act, "db"))


def test_backward_output_mask(ops):
    m, k, n = 9, 40, 24
    x, w, dy = dev(rand(m, k, seed=1)), dev(rand(2 * n, k, seed=2)), dev(rand(m, n, seed=3))
    saved = dev(rand(m, 2, n, seed=4))
    full = ops.native_gated_linear_backward(dy, x, w, saved, "silu")
    for mask in ((True, False, False), (False, True, False), (False, False, True), (False, False, False)):
        got = ops.native_gated_linear_backward(dy, x, w, saved, "silu", mask)
        for a, b, want in zip(got, full, mask):
            assert (a is None) == (not want)
            if want:
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [40, 41])
def test_backward_without_an_activation_needs_nothing_saved(ops, dtype, n):
    """dz is dy, read where it lies (rows on 16-byte boundaries) or copied; a
    saved tensor changes nothing."""
    m, k = 70, 136
    x, w = dev(rand(m, k, dtype=dtype, seed=1)), dev(rand(n, k, dtype=dtype, seed=2))
    wide = dev(rand(m, n + 8, dtype=dtype, seed=3))
    nan = torch.full((m, n), math.nan, dtype=dtype, device="cuda")
    for dy in (wide[:, :n].contiguous(), wide[:, :n], wide[:, 5:5 + n], wide[:1, :n].expand(m, n)):
        for mask in ((True, True, True), (True, True, False)):
            a = ops.native_linear_act_backward(dy, x, w, None, "none", mask)
            b = ops.native_linear_act_backward(dy, x, w, nan, "none", mask)
            c = ops.native_linear_act_backward(dy.contiguous(), x, w, nan, "none", (True, True, True))
            for i in range(3):
                assert (a[i] is None) == (not mask[i])
                if mask[i]:
                    assert torch.equal(a[i], b[i]) and torch.equal(a[i], c[i])


def test_gradients_against_differences(ops):
    """The backward passes against central differences of the forward ones, in
    float32: with a step of 2^-6 the difference quotient of a loss of M N terms
    is off by its third derivative (below 2^-12 of the gradient's terms) and by
    the forward pass's own error over the step."""
    m, k, n = 4, 24, 40
    x, w, b = rand(m, k, seed=1), rand(2 * n, k, seed=2, scale=k ** -0.5), rand(2 * n, seed=3)
    dy = rand(m, n, seed=4)

    def loss(x_, w_, b_, gated, act):
        if gated:
            y = ops.gated_linear(dev(x_), dev(w_), dev(b_), act)
        else:
            y = ops.linear_act(dev(x_), dev(w_[:n].contiguous()), dev(b_[:n].contiguous()), None, act)
        return float((y.cpu().double() * dy.double()).sum())

    for gated in (True, False):
        for act in ("silu", "gelu", "gelu_tanh"):
            wf, bf = (w, b) if gated else (w[:n].contiguous(), b[:n].contiguous())
            if gated:
                _, saved = ops.native_gated_linear(dev(x), dev(wf), dev(bf), act)
                grads = ops.native_gated_linear_backward(dev(dy), dev(x), dev(wf), saved, act)
            else:
                _, saved = ops.native_linear_act(dev(x), dev(wf), dev(bf), None, act)
                grads = ops.native_linear_act_backward(dev(dy), dev(x), dev(wf), saved, act)
            for which, tensor, grad in zip(range(3), (x, w, b), grads):
                grad = grad.cpu().double()
                # one random direction over every element of the tensor
                d = rand(*tensor.shape, seed=10 + which)
                if not gated and which:
                    d[n:] = 0
                h = 2.0 ** -6 / float(d.double().norm())
                args = [x, w, b]

                def at(sign):
                    moved = list(args)
                    moved[which] = (tensor.double() + sign * h * d.double()).float()
                    return loss(*moved, gated, act), moved[which].double()

                up, plus = at(1)
                down, minus = at(-1)
                step = (plus - minus)[:grad.shape[0]] if grad.dim() else plus - minus
                want = up - down
                got = float((grad * step).sum())
                # forward error: (K + 8) 2^-23 of each of the M N terms (|y| of order 1), twice; curvature:
                # third derivatives below 8 |direction|^3 times the 2 h^3 / 6 of a central difference.
                terms = float(dy.abs().double().sum()) * 16
                bound = 2 * (k + 8) * 2.0 ** -23 * terms + terms * 8 * (2.0 ** -6) ** 3 / 3 \
                    + 2.0 ** -20 * float((grad * step).abs().sum())
                assert abs(got - want) <= bound, (gated, act, which, got, want, bound)


# -------------------------------------------------------------- checkpoints

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (1, 32), (7, 33), (5, 8), (3, 40), (129, 1000), (64, 4096),
                                   (2, 3, 65), (4097,), (1000, 24)])
def test_checkpoint_is_exact(ops, dtype, shape):
    x = rand(*shape, dtype=torch.float32, seed=7)
    if shape[-1] > 8 and len(shape) > 1:
        rows = x.view(-1, shape[-1])
        rows[:, 3] *= 1000.0
        rows[0, 5:9] = torch.tensor([127.0, 63.5, 0.5, 1.5])  # ties, and the largest value that fits
        if rows.shape[0] > 2:
            rows[1] = 0.0                                    # a block of zeros
            rows[2] *= 1e-30                                 # below float16's range
    x = x.to(dtype)
    values, exponents = ops.checkpoint_pack(dev(x))
    wv, we, wx = pack_reference(x)
    assert torch.equal(values.cpu(), wv)
    assert torch.equal(exponents.cpu(), we)
    for to in DTYPES:
        got = ops.checkpoint_unpack(values, exponents, to).cpu()
        assert got.dtype == to and torch.equal(got, wx.to(to))


@pytest.mark.parametrize("dtype", DTYPES)
def test_checkpoint_of_extreme_values(ops, dtype):
    top = torch.finfo(dtype)
    rows = [
        [top.max, -top.max, 1.0, top.max / 2], [top.smallest_normal, top.tiny, 0.0, -top.smallest_normal],
        [math.inf, 1.0, 2.0, 3.0], [1.0, -math.inf, 0.0, 0.0], [math.nan, 1.0, 0.0, math.inf], [-0.0, 0.0, 0.0, 0.0],
        [127.0, 126.5, 125.5, -0.5], [127.5, 1.0, -1.0, 0.75], [128.0, 2.0, 1.0, -3.0],
        [top.smallest_normal * top.eps, 0.0, 0.0, 0.0],
    ]
    x = torch.zeros(len(rows), 64, dtype=torch.float64)
    for i, r in enumerate(rows):
        x[i, :4] = torch.tensor(r, dtype=torch.float64)
        x[i, 36:40] = 1.0  # the second block of every row is ordinary
    x = x.to(dtype)
    values, exponents = ops.checkpoint_pack(dev(x))
    wv, we, wx = pack_reference(x)
    assert torch.equal(exponents.cpu(), we)
    assert torch.equal(values.cpu(), wv)
    got = ops.checkpoint_unpack(values, exponents, dtype).cpu()
    assert torch.equal(got.isnan(), wx.isnan())
    assert torch.equal(got.nan_to_num(), wx.to(dtype).nan_to_num())
    assert torch.isfinite(got[:2]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 33), (333, 4097), (64, 4096), (2, 5, 96)])
def test_activation_backward_from_a_checkpoint(ops, dtype, shape):
    x, dy = rand(*shape, dtype=dtype, seed=8), rand(*shape, dtype=dtype, seed=9)
    held = ops.checkpoint_pack(dev(x))
    _, _, z = pack_reference(x)
    u = half_eps(dtype)
    for act in ACTS:
        want = dy.double() * slope64(z, act)
        e = dy.double().abs() * 2.0 ** -16 * (1 + z.abs()) if act not in ("none", "relu") else torch.zeros_like(want)
        bound = e + u * (want.abs() + e) + (2.0 ** -25 if dtype == torch.float16 else 1e-38)
        check(ops.checkpoint_activation_backward(dev(dy), *held, act), want, bound, act)


# ------------------------------------------------------- layouts and corners

@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_operands_give_the_dense_results(ops, dtype):
    m, k, n = 70, 136, 200
    wide = dev(rand(m, k + 24, dtype=dtype, seed=1))
    tall = dev(rand(2 * n, 2 * k, dtype=dtype, seed=2, scale=k ** -0.5))
    x, w = wide[:, 8:8 + k], tall[:, k:]
    odd = dev(rand(m, k + 3, dtype=dtype, seed=1))[:, 3:]    # rows off 16-byte boundaries
    columns = dev(rand(k, m, dtype=dtype, seed=1)).t()       # unit stride on the rows
    repeated = dev(rand(1, k, dtype=dtype, seed=1)).expand(m, k)
    r = dev(rand(m, 2 * n, dtype=dtype, seed=4))[:, n:]
    dy = dev(rand(m, n + 8, dtype=dtype, seed=5))[:, :n]
    saved = dev(rand(m, 2, n, dtype=dtype, seed=6))
    for v in (x, odd, columns, repeated):
        assert torch.equal(ops.gated_linear(v, w), ops.gated_linear(v.contiguous(), w.contiguous()))
        assert torch.equal(ops.linear_act(v, w[:n], None, r, "gelu"),
                           ops.linear_act(v.contiguous(), w[:n].contiguous(), None, r.contiguous(), "gelu"))
        got = ops.native_gated_linear_backward(dy, v, w, saved)
        want = ops.native_gated_linear_backward(dy.contiguous(), v.contiguous(), w.contiguous(), saved)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        a, b = ops.checkpoint_pack(v), ops.checkpoint_pack(v.contiguous())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_leading_dimensions(ops):
    x, w = dev(rand(2, 3, 5, 64, seed=1)), dev(rand(96, 64, seed=2))
    h, gate_up = ops.native_gated_linear(x, w)
    assert h.shape == (2, 3, 5, 48) and gate_up.shape == (2, 3, 5, 2, 48)
    flat = ops.gated_linear(x.reshape(30, 64), w)
    assert torch.equal(h.reshape(30, 48), flat)
    h2, (v, e) = ops.native_gated_linear(x, w, checkpoint=True)
    assert v.shape == (2, 3, 5, 2, 48) and e.shape == (2, 3, 5, 2, 2) and torch.equal(h, h2)
    dx, dw, db = ops.native_gated_linear_backward(h, x, w, gate_up)
    assert dx.shape == x.shape and dw.shape == w.shape and db.shape == (96,)
    dx, dw, db = ops.native_gated_linear_backward(h, x, w, (v, e))
    assert dx.shape == x.shape
    y, pre = ops.native_linear_act(x[0, 0, 0], w, None, None, "relu")
    assert y.shape == (96,) and pre.shape == (96,)


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty_sizes(ops, dtype):
    e = lambda *s: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
    w = dev(rand(32, 16, dtype=dtype))
    h, saved = ops.native_gated_linear(e(0, 16), w)
    assert h.shape == (0, 16) and saved.shape == (0, 2, 16)
    dx, dw, db = ops.native_gated_linear_backward(h, e(0, 16), w, saved)
    assert dx.shape == (0, 16) and not dw.any() and not db.any() and dw.shape == (32, 16) and db.shape == (32,)
    h, (v, x) = ops.native_gated_linear(e(0, 16), w, checkpoint=True)
    assert v.shape == (0, 2, 16) and x.shape == (0, 2, 1)
    y, pre = ops.native_linear_act(e(3, 16), e(0, 16))
    assert y.shape == (3, 0) and pre.shape == (3, 0)
    # No input features: the bias alone.
    b = dev(rand(32, dtype=dtype, seed=2))
    y = ops.linear_act(e(3, 0), e(32, 0), b, None, "relu")
    assert torch.equal(y, b.clamp_min(0).expand(3, 32))
    h = ops.gated_linear(e(3, 0), e(32, 0), b, "none")
    assert torch.equal(h, (b[:16].float() * b[16:].float()).to(dtype).expand(3, 16))
    dx, dw, db = ops.native_linear_act_backward(dev(rand(3, 32, dtype=dtype)), e(3, 0), e(32, 0), y)
    assert dx.shape == (3, 0) and dw.shape == (32, 0) and db.shape == (32,)
    v, x = ops.checkpoint_pack(e(4, 0))
    assert ops.checkpoint_unpack(v, x, dtype).shape == (4, 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [3, 140])
def test_infinities_and_nan_go_where_arithmetic_puts_them(ops, dtype, m):
    """A row of x or of the weight with an infinity or a NaN gives the
    infinities and NaN of a plain sum, and leaves the other results alone; so
    do values near the type's largest, whose products overflow."""
    k, n = 200, 136
    x, w = rand(m, k, dtype=dtype, seed=1), rand(n, k, dtype=dtype, seed=2, scale=k ** -0.5)
    x[0, 3] = math.inf
    x[1, 150] = -math.inf
    x[2, 7], x[2, 8] = math.inf, -math.inf
    w[5, 3] = 0.0            # inf * 0
    w[9, 60] = math.nan
    w[17, 70] = math.inf
    z = x.float().double() @ w.float().double().t()
    y, pre = ops.native_linear_act(dev(x), dev(w), None, None, "relu")
    want = torch.where(torch.isnan(z), z, z.clamp_min(0))
    for got, ref in ((pre, z), (y, want)):
        got = got.cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert torch.equal(torch.isinf(got), torch.isinf(ref))
        assert torch.equal(got[torch.isinf(ref)], ref[torch.isinf(ref)])
        fine = torch.isfinite(ref)
        bound = (k + 8) * 2.0 ** -23 * 200 + half_eps(dtype) * (ref.abs() + 1) * 2
        assert bool(((got - ref).abs() <= bound)[fine].all())
    # gradients: dx rows of an infinite dy, dw columns of an infinite x
    dy = rand(m, n, dtype=dtype, seed=3, scale=0.1)
    dy[0, 0] = math.inf
    saved = torch.ones(m, n, dtype=dtype)
    dx, dw, db = ops.native_linear_act_backward(dev(dy), dev(x), dev(w), dev(saved), "none")
    for got, ref in ((dx, dy.double() @ w.double()), (dw, dy.double().t() @ x.double()), (db, dy.double().sum(0))):
        got = got.cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert torch.equal(torch.isinf(got), torch.isinf(ref))
    if dtype == torch.float32:
        big = torch.full((m, 4), torch.finfo(dtype).max, dtype=dtype)
        got = ops.linear_act(dev(big), dev(torch.eye(4, dtype=dtype)))
        assert torch.equal(got.cpu(), big)   # a value that rounds past the largest TF32
        # the checkpoint of a row with an infinity
    h, (v, e) = ops.native_linear_act(dev(x), dev(w), None, None, "none", checkpoint=True)
    back = ops.checkpoint_unpack(v, e, torch.float32).cpu()
    blocks = torch.nn.functional.pad(z, (0, -n % 32)).unflatten(1, (-1, 32))
    bad = (~torch.isfinite(blocks)).any(-1, keepdim=True).expand_as(blocks).flatten(1)[:, :n]
    assert torch.equal(torch.isnan(back), bad)


def test_offsets_past_32_bits(ops):
    """Results of more than 2^31 elements, checked on rows at both ends."""
    m, k, n = 98304, 64, 11008
    assert 2 * m * n > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(m, k, generator=g, device="cuda", dtype=torch.float32).bfloat16()
    w = dev(rand(2 * n, k, dtype=torch.bfloat16, seed=2, scale=k ** -0.5))
    h, gate_up = ops.native_gated_linear(x, w)
    rows = torch.tensor([0, 1, 48777, 97999, 98302, 98303], device="cuda")
    z = x[rows].double() @ w.double().t()
    u = half_eps(torch.bfloat16)
    bound = (k + 8) * 2.0 ** -23 * (x[rows].double().abs() @ w.double().abs().t()) + u * z.abs() + 1e-30
    assert bool(((gate_up[rows].flatten(1).double() - z).abs() <= bound).all())
    held = ops.checkpoint_pack(gate_up)
    for r in rows.tolist():
        v, e, _ = pack_reference(gate_up[r].cpu())
        assert torch.equal(held[0][r].cpu(), v) and torch.equal(held[1][r].cpu(), e)
    del h
    dy = torch.ones(m, n, device="cuda", dtype=torch.bfloat16)
    dx, _, db = ops.native_gated_linear_backward(dy, x, w, held, "none", (True, False, True))
    del held
    packed = ops.checkpoint_pack(gate_up[rows])
    part, _, _ = ops.native_gated_linear_backward(dy[:6], x[rows], w, packed, "none", (True, False, False))
    scale = part.double().abs().max()
    assert bool(((dx[rows].double() - part.double()).abs() <= 2.0 ** -6 * scale).all())


def test_first_call_in_a_recording(backend):
    """A process whose first feed-forward calls are recorded, without a warm-up."""
    import subprocess
    import sys

    script = """
import torch, tensorplay_mlu_b200 as tpb
tpb.load()
from tensorplay_mlu_b200.graph import Graph
ops = tpb.ops
torch.manual_seed(0)
for dt in (torch.bfloat16, torch.float32):
    for m in (2, 300):
        x, w = torch.randn(m, 136).to(dt).cuda(), torch.randn(160, 136).to(dt).cuda()
        def body():
            h, s = ops.native_gated_linear(x, w)
            return (h, *ops.native_gated_linear_backward(h, x, w, s))
        g = Graph()
        out = g.capture(body)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, body())), (dt, m)
        del out
        g.reset()
assert tpb._native.lib().tp_b200_take_device_error(0) == 0
print("recorded")
"""
    root = __import__("os").path.dirname(__import__("os").path.dirname(__import__("os").path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, cwd=root, timeout=300)
    assert done.returncode == 0 and "recorded" in done.stdout, done.stderr[-2000:]


def test_refusals(ops):
    x, w, b = dev(rand(4, 16)), dev(rand(8, 16)), dev(rand(8))
    cases = [
        (lambda: ops.gated_linear(x, w, None, "tanh"), "activation must be one of"),
        (lambda: ops.gated_linear(x, w, None, None), "activation must be one of"),
        (lambda: ops.gated_linear(x, w[:7]), "even number of rows"),
        (lambda: ops.gated_linear(x, w[:, :8]), "do not match the weight"),
        (lambda: ops.gated_linear(x.double(), w.double()), "bfloat16, float16 or float32"),
        (lambda: ops.gated_linear(x, w.half()), "one dtype"),
        (lambda: ops.gated_linear(x, w.cpu()), "device tensor"),
        (lambda: ops.gated_linear(x.cpu(), w), "device tensor"),
        (lambda: ops.gated_linear(x, w, b[:4]), "bias of 8"),
        (lambda: ops.linear_act(x, w, b, x), "residual of the result's shape"),
        (lambda: ops.linear_act(x, w, b, b), "residual of the result's shape"),
        (lambda: ops.linear_act(x, w.view(2, 4, 16)), "2-d weight"),
        (lambda: ops.native_linear_act_backward(x, x, w, x), "gradient of shape"),
        (lambda: ops.native_linear_act_backward(dev(rand(4, 8)), x, w, x), "pre-activations of shape"),
        (lambda: ops.native_linear_act_backward(dev(rand(4, 8)), x, w, None, "relu"), "pre-activations of shape"),
        (lambda: ops.native_gated_linear_backward(dev(rand(4, 4)), x, w, None, "none"), "pre-activations of shape"),
        (lambda: ops.native_linear_act_backward(dev(rand(4, 8)), x, w, (x,)), "values, exponents"),
        (lambda: ops.native_linear_act_backward(dev(rand(4, 8)), x, w, (x, x)), "int8 values"),
        (lambda: ops.checkpoint_pack(x.int()), "bfloat16, float16 or float32"),
        (lambda: ops.checkpoint_pack(x[0, 0]), "at least one dimension"),
        (lambda: ops.checkpoint_unpack(*ops.checkpoint_pack(x), torch.float64), "bfloat16, float16 or float32"),
        (lambda: ops.checkpoint_unpack(ops.checkpoint_pack(x)[0], ops.checkpoint_pack(x)[1][:2], torch.float32),
         "exponents"),
        (lambda: ops.checkpoint_activation_backward(x[:2], *ops.checkpoint_pack(x), "gelu"), "a checkpoint of shape"),
    ]
    for call, match in cases:
        with pytest.raises(RuntimeError, match=match):
            call()


# --------------------------------------------------- in use: streams, graphs

def test_on_another_stream(ops):
    x, w = dev(rand(200, 512, dtype=torch.bfloat16, seed=1)), dev(rand(1024, 512, dtype=torch.bfloat16, seed=2))
    want = ops.native_gated_linear(x, w)
    dw = ops.native_gated_linear_backward(want[0], x, w, want[1])[1]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = ops.native_gated_linear(x, w)
            gw = ops.native_gated_linear_backward(got[0], x, w, got[1])[1]
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(gw, dw)


def _block(ops, x, wg, bg, wd, bd, dy, checkpoint):
    """One feed-forward block with its residual, forward and backward."""
    h, saved = ops.native_gated_linear(x, wg, bg, "silu", checkpoint)
    y, _ = ops.native_linear_act(h, wd, bd, x, "none")
    dh, dwd, dbd = ops.native_linear_act_backward(dy, h, wd, y, "none")
    dx, dwg, dbg = ops.native_gated_linear_backward(dh, x, wg, saved, "silu")
    return y, ops.add_Tensor(dx, dy), dwg, dbg, dwd, dbd


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("m", [1, 48, 300])
def test_block_in_a_captured_step(backend, ops, checkpoint, m):
    from tensorplay_mlu_b200.graph import Graph

    d, f = 264, 520
    t = lambda *s, seed, scale=1.0: dev(rand(*s, dtype=torch.bfloat16, seed=seed, scale=scale))  # noqa: E731
    args = [t(m, d, seed=1), t(2 * f, d, seed=2, scale=d ** -0.5), t(2 * f, seed=3, scale=0.1),
            t(d, f, seed=4, scale=f ** -0.5), t(d, seed=5, scale=0.1), t(m, d, seed=6, scale=0.1)]
    first = _block(ops, *args, checkpoint)
    again = _block(ops, *args, checkpoint)
    assert all(torch.equal(a, b) for a, b in zip(first, again))  # no order of additions left to chance
    graph = Graph()
    try:
        out = graph.capture(lambda: _block(ops, *args, checkpoint))
        fresh = t(m, d, seed=9)
        ops.copy_(args[0], fresh)
        # eager calls between replays share no workspace with the recording
        want = _block(ops, *args, checkpoint)
        graph.replay()
        other = _block(ops, *args, checkpoint)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert all(torch.equal(a, b) for a, b in zip(other, want))
    finally:
        del out
        graph.reset()
    assert backend._native.lib().tp_b200_take_device_error(torch.cuda.current_device()) == 0


@pytest.mark.parametrize("checkpoint", [False, True])
def test_block_against_autograd(ops, checkpoint):
    """The whole block against PyTorch's autograd in 64 bits, relative to each
    result's norm: four roundings lie between the inputs and a gradient (the
    saved pre-activations, h or dh, dz, the result), each below u of its own
    norm, and each passes through one product, which amplifies a relative
    error of independent roundings by at most the ratio of sum |a b| norms,
    taken as 4; the checkpoint adds half a step, 1/127 of a block's largest
    value, at most 4 standard deviations of it: 4/127/sqrt(3)."""
    m, d, f = 96, 128, 192
    x, wg, bg = rand(m, d, seed=1), rand(2 * f, d, seed=2, scale=d ** -0.5), rand(2 * f, seed=3, scale=0.1)
    wd, bd, dy = rand(d, f, seed=4, scale=f ** -0.5), rand(d, seed=5, scale=0.1), rand(m, d, seed=6, scale=0.1)
    for dtype in DTYPES:
        ins = [t.to(dtype) for t in (x, wg, bg, wd, bd, dy)]
        got = _block(ops, *[dev(t) for t in ins], checkpoint)
        leaves = [t.double().requires_grad_() for t in ins[:5]]
        z = leaves[0] @ leaves[1].t() + leaves[2]
        h = torch.nn.functional.silu(z[:, :f]) * z[:, f:]
        y = h @ leaves[3].t() + leaves[4] + leaves[0]
        y.backward(ins[5].double())
        want = [y.detach()] + [t.grad for t in leaves]
        bound = 4 * 4 * half_eps(dtype) + 64 * 2.0 ** -23 + (4 / 127 / 3 ** 0.5 if checkpoint else 0.0)
        for i, (a, b) in enumerate(zip(got, want)):
            rel = float((a.cpu().double() - b).norm() / b.norm())
            assert rel <= bound, (dtype, i, rel, bound)
