"""Feed-forward layers under tp_b200_set_gemm_sm_limit: beyond 64 rows the
16-bit products are the persistent kernel's, which keeps to the limit."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sms", [2, 100])
def test_a_limit_selects_the_persistent_products(backend, dtype, sms):
    """Without an epilogue a layer is then the plain product bit for bit: one
    sum over K in order, where the kernel for few rows adds partial sums."""
    ops, lib = backend.ops, backend._native.lib()
    device = torch.cuda.current_device()
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    x, w, dy = rand(384, 4096), rand(2048, 4096), rand(384, 2048)
    tall, narrow, grad = rand(13898, 256), rand(304, 256), rand(13898, 304)
    assert lib.tp_b200_set_gemm_sm_limit(device, sms) == 0
    try:
        y = ops.linear_act(x, w)
        dx, _, _ = ops.native_linear_act_backward(dy, x, w, None, "none", (True, False, False))
        _, dw, _ = ops.native_linear_act_backward(grad, tall, narrow, None, "none", (False, True, False))
        assert torch.equal(y, ops.linear(x, w))
        assert torch.equal(dx, ops.mm(dy, w))
        assert torch.equal(dw, ops.mm(grad.t(), tall))
    finally:
        assert lib.tp_b200_set_gemm_sm_limit(device, 0) == 0
    assert lib.tp_b200_take_device_error(device) == 0
