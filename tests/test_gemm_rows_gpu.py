"""Products whose result rows lie off 16-byte boundaries (an odd number of
columns): the same bits as the product with columns added to the right
operand until the rows lie on them, in every kernel and with every addend."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def rand(*shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).cuda()


# One-SM kernel (128 and 256 columns a tile), CTA-pair kernel with one and
# several tiles a cluster; fp32 "high" is one TF32 product, "highest" the split one.
@pytest.mark.parametrize("dtype,precision", [(torch.bfloat16, None), (torch.float16, None), (torch.float32, "high"),
                                             (torch.float32, "highest")])
@pytest.mark.parametrize("shape", [(200, 301, 136), (129, 1357, 72), (520, 777, 1160), (2500, 4101, 64)])
def test_rows_off_16_byte_boundaries(backend, dtype, precision, shape):
    ops = backend.ops
    m, n, k = shape
    wide = -(-n // 8) * 8
    a, b = rand(m, k, dtype=dtype, seed=1), rand(wide, k, dtype=dtype, seed=2)
    full = rand(m, wide, dtype=dtype, seed=3)
    before = torch.get_float32_matmul_precision()
    torch.set_float32_matmul_precision(precision or before)
    try:
        for addend in (None, full[0], full, full[:, :1]):
            def product(cols):
                if addend is None:
                    return ops.mm(a, b[:cols].t())
                c = addend[..., :cols].contiguous() if addend.shape[-1] > 1 else addend
                return ops.addmm(c, a, b[:cols].t(), beta=2.0, alpha=0.5)

            assert torch.equal(product(n), product(wide)[:, :n])
        la, lb = rand(3, m, k, dtype=dtype, seed=4), rand(3, wide, k, dtype=dtype, seed=5)
        got = ops.bmm(la, lb[:, :n].transpose(1, 2))
        assert torch.equal(got, ops.bmm(la, lb.transpose(1, 2))[..., :n])
    finally:
        torch.set_float32_matmul_precision(before)
    assert backend._native.lib().tp_b200_take_device_error(torch.cuda.current_device()) == 0
