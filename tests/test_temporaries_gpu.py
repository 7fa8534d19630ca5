"""Operators that convert or copy more than one operand before their kernel:
the converted copies are temporaries of one size, and each has to keep its
memory until the kernel has been launched."""

from __future__ import annotations

import pytest
import torch

from conftest import assert_close, assert_equal

pytestmark = pytest.mark.gpu


def rand(*shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    if dtype.is_floating_point:
        return torch.randn(*shape, generator=g).to(dtype)
    return torch.randint(-100 if dtype.is_signed else 0, 100, shape, generator=g).to(dtype)


@pytest.mark.parametrize("da,db", [(torch.uint8, torch.int8), (torch.float16, torch.bfloat16)])
def test_binary_and_where_with_both_operands_converted(backend, da, db):
    ops = backend.ops
    a, b = rand(1000, 37, dtype=da, seed=1), rand(1000, 37, dtype=db, seed=2)
    to = torch.promote_types(da, db)
    for op, want in ((ops.add_Tensor, a.to(to) + b.to(to)), (ops.sub_Tensor, a.to(to) - b.to(to)),
                     (ops.mul_Tensor, a.to(to) * b.to(to))):
        got = ops.to_host(op(ops.to_device(a), ops.to_device(b)))
        assert got.dtype == to
        assert_close(got, want, to) if to.is_floating_point else assert_equal(got, want)
    cond = rand(1000, 37, dtype=torch.float32, seed=3) > 0
    got = ops.to_host(ops.where_self(ops.to_device(cond), ops.to_device(a), ops.to_device(b)))
    assert_equal(got, torch.where(cond, a.to(to), b.to(to)))


def test_layer_norm_backward_with_strided_operands(backend):
    ops = backend.ops
    x, dy = rand(64, 200, dtype=torch.float32, seed=4), rand(64, 200, dtype=torch.float32, seed=5)
    w = rand(200, dtype=torch.float32, seed=6)
    dx_, dy_ = ops.to_device(x.t().contiguous()).t(), ops.to_device(dy.t().contiguous()).t()
    _, mean, rstd = ops.native_layer_norm(ops.to_device(x), [200], ops.to_device(w))
    got = ops.native_layer_norm_backward(dy_, dx_, [200], mean, rstd, ops.to_device(w))
    want = ops.native_layer_norm_backward(ops.to_device(dy), ops.to_device(x), [200], mean, rstd, ops.to_device(w))
    for a, b in zip(got, want):
        assert_equal(ops.to_host(a), ops.to_host(b))
