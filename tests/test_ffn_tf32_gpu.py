"""float32 feed-forward layers when one TF32 product is allowed
(``torch.set_float32_matmul_precision("high")``).

Each operand is rounded to TF32, 11 significant bits: off by at most 2^-11 of
its value, so a product of two by at most 2^-10 + 2^-22; the sums add
(K + 8) 2^-23 of the summed magnitudes, as in full precision.  Infinities and
NaN come out where fp32 arithmetic puts them, whatever a NaN's payload."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TERM = 2.0 ** -10 + 2.0 ** -22


@pytest.fixture
def ops(backend):
    before = torch.get_float32_matmul_precision()
    torch.set_float32_matmul_precision("high")
    yield backend.ops
    torch.set_float32_matmul_precision(before)


def rand(*shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda") * scale


def nan_of(bits):
    return torch.tensor(bits - (1 << 32) if bits >= 1 << 31 else bits, dtype=torch.int32).view(torch.float32).item()


def set_bits(t, index, bits):
    """t[index] = the float with these bits (a Python float would lose a NaN's payload)."""
    t.view(torch.int32)[index] = bits - (1 << 32) if bits >= 1 << 31 else bits


def check(got, want, bound, what):
    got = got.double()
    assert bool(torch.isfinite(got).all()), what
    bad = (got - want).abs() > bound
    assert not bool(bad.any()), (what, int(bad.sum()), float(((got - want).abs() / bound.clamp_min(1e-300)).max()))


# Tiles of 32, 64 and 128 rows of x; ragged; enough tiles for 128 rows in each of
# the three products.
@pytest.mark.parametrize("shape", [(3, 520, 136), (50, 77, 33), (300, 264, 200), (1024, 520, 2432), (1030, 2432, 1100)])
@pytest.mark.parametrize("gated", [False, True])
def test_forward_and_backward(ops, shape, gated):
    m, k, n = shape
    parts = 2 if gated else 1
    x, w, b = rand(m, k, seed=1), rand(parts * n, k, seed=2, scale=k ** -0.5), rand(parts * n, seed=3)
    z = x.double() @ w.double().t() + b.double()
    ez = (TERM + (k + 8) * 2.0 ** -23) * (x.abs().double() @ w.abs().double().t()) + 2.0 ** -22 * z.abs()
    forward = ops.native_gated_linear if gated else ops.native_linear_act
    y, pre = forward(x, w, b, activation="relu")
    check(pre.reshape(m, parts * n), z, ez, "pre")
    a = z[:, :n].clamp_min(0)
    if gated:
        g, u, eg, eu = a, z[:, n:], ez[:, :n], ez[:, n:]
        check(y, g * u, eg * u.abs() + g * eu + eg * eu + 2.0 ** -22 * (g * u).abs(), "h")
    else:
        check(y, a, ez, "y")
    dy, saved = rand(m, n, seed=4, scale=0.1), rand(*((m, 2, n) if gated else (m, n)), seed=5)
    backward = ops.native_gated_linear_backward if gated else ops.native_linear_act_backward
    dx, dw, db = backward(dy, x, w, saved, "relu")
    s, g = saved.double(), dy.double()
    dz = torch.cat([g * s[:, 1] * (s[:, 0] > 0), g * s[:, 0].clamp_min(0)], 1) if gated else g * (s > 0)
    step = 2.0 ** -22
    for got, left, right, length in ((dx, dz, w.double(), parts * n), (dw, dz.t(), x.double(), m)):
        terms = left.abs() @ right.abs()
        check(got, left @ right, (TERM + step + (length + 8) * 2.0 ** -23) * terms + 1e-30, "product")
    check(db, dz.sum(0), (m + 8) * 2.0 ** -23 * dz.abs().sum(0) + 1e-30, "db")


NANS = [0x7FFFFFFF, 0xFFFFFFFF, 0x7FFFF000, 0xFFFFF000, 0x7FC00000, 0x7F800001, 0xFF800001, 0x7F801FFF]


@pytest.mark.parametrize("precision", ["high", "highest"])
@pytest.mark.parametrize("m", [5, 60, 700])
@pytest.mark.parametrize("bits", NANS)
def test_nan_of_any_payload(ops, precision, m, bits):
    """A NaN in x, in the weight or in the gradient reaches exactly the results that sum it."""
    torch.set_float32_matmul_precision(precision)
    k, n = 200, 136
    x, w, dy = rand(m, k, seed=1), rand(n, k, seed=2), rand(m, n, seed=3)
    w[:, 7] = 0.0                       # 0 * NaN is NaN as well
    set_bits(x, (2, 7), bits)
    set_bits(w, (9, 60), bits)
    set_bits(dy, (4, 11), bits)
    assert math.isnan(nan_of(bits)) and bool(x[2, 7].isnan()) and bool(dy[4, 11].isnan())
    y, pre = ops.native_linear_act(x, w)
    dx, dw, db = ops.native_linear_act_backward(dy, x, w, None)
    for got, want in ((y, x.double() @ w.double().t()), (pre, x.double() @ w.double().t()),
                      (dx, dy.double() @ w.double()), (dw, dy.double().t() @ x.double()), (db, dy.double().sum(0))):
        assert torch.equal(got.isnan(), want.isnan())
        assert bool(torch.isfinite(got[~want.isnan()]).all())


@pytest.mark.parametrize("m", [5, 60, 700])
def test_a_checkpoint_of_a_nan_reaches_every_gradient(ops, m):
    """Its block reads back as NaN: dx's row, dw's rows and db's elements of the block."""
    k, n = 200, 136
    x, w, dy, z = rand(m, k, seed=1), rand(n, k, seed=2), rand(m, n, seed=3), rand(m, n, seed=4)
    z[3, 40] = math.inf
    held = ops.checkpoint_pack(z)
    dx, dw, db = ops.native_linear_act_backward(dy, x, w, held, "silu")
    row, columns = torch.zeros(m, dtype=torch.bool), torch.zeros(n, dtype=torch.bool)
    row[3] = True
    columns[32:64] = True
    assert torch.equal(dx.isnan().cpu(), row[:, None].expand(m, k))
    assert torch.equal(dw.isnan().cpu(), columns[:, None].expand(n, k))
    assert torch.equal(db.isnan().cpu(), columns)


@pytest.mark.parametrize("m", [5, 60, 700])
def test_infinities_and_the_largest_values(ops, m):
    k, n = 200, 136
    x, w = rand(m, k, seed=1), rand(n, k, seed=2)
    x[0, 3] = math.inf
    x[1, 150] = -math.inf
    x[2, 7], x[2, 8] = math.inf, -math.inf
    w[5, 3] = 0.0
    w[17, 70] = math.inf
    y, pre = ops.native_linear_act(x, w)
    want = x.double() @ w.double().t()
    for got in (y, pre):
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.isinf(), want.isinf())
        assert torch.equal(got[want.isinf()].double(), want[want.isinf()])
    # The largest floats round past the range: their sums are computed again in fp32, or cut to 11 bits (2^-10).
    top = torch.finfo(torch.float32).max
    big = torch.full((m, 4), top, device="cuda")
    big[:, 1] = -top
    got = ops.linear_act(big, torch.eye(4, device="cuda"))
    assert bool(torch.isfinite(got).all())
    assert bool(((got.double() - big.double()).abs() <= 2.0 ** -10 * top).all())
