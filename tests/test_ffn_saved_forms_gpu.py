"""A feed-forward layer asked for its pre-activations in both forms at once,
through the C ABI (each output of tpb_layer is optional by itself): the same
bits as from two calls that ask for one form each, whichever kernel the row
count selects."""

from __future__ import annotations

import pytest
import torch

from tensorplay_mlu_b200 import _native as N

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def layer(x, w, bias, residual, act, parts, y, saved, values, exponents):
    """tp_b200_layer_forward on dense operands whose rows may lie off 16-byte boundaries."""
    (m, k), n = x.shape, w.shape[0] // parts
    es = x.element_size()
    pitch = -(-k * es // 128) * 128 // es
    work = torch.empty((m + parts * n) * pitch, dtype=x.dtype, device="cuda")
    at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    args = N.LAYER.pack(N.DTYPE_CODES[x.dtype], N.ACTIVATIONS[act], parts, 0, m, n, k, x.data_ptr(), k, w.data_ptr(), k,
                        at(bias), at(residual), n, y.data_ptr(), n, at(saved), at(values), at(exponents),
                        work.data_ptr(), work.data_ptr() + m * pitch * es)
    N.check(N.lib().tp_b200_layer_forward(args, N.stream_of(x.device)), "layer_forward")


# Few rows; the CTA-pair kernel with one and several tiles a cluster; results
# that TMA can store, and rows of saved values or bytes that it cannot.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3, 136, 96), (300, 520, 1032), (1030, 64, 1536), (1030, 72, 1001), (2048, 512, 1000),
                                   (2500, 136, 4104)])
@pytest.mark.parametrize("parts", [1, 2])
def test_both_forms_at_once(backend, dtype, shape, parts):
    m, k, n = shape
    g = torch.Generator(device="cuda").manual_seed(m + n)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda").to(dtype)  # noqa: E731
    x, w, b = rand(m, k), (rand(parts * n, k) * k ** -0.5).to(dtype), rand(parts * n)
    r = rand(m, n) if parts == 1 else None
    nb = -(-n // 32)

    def outputs():  # filled with what no result holds, so that an element left out shows
        return (torch.full((m, n), 1e4, dtype=dtype, device="cuda"),
                torch.full((m, parts, n), 1e4, dtype=dtype, device="cuda"),
                torch.full((m, parts, n), -128, dtype=torch.int8, device="cuda"),
                torch.full((m, parts, nb), 254, dtype=torch.uint8, device="cuda"))

    y, saved, values, exponents = outputs()
    layer(x, w, b, r, "silu", parts, y, saved, values, exponents)
    y1, saved1, _, _ = outputs()
    layer(x, w, b, r, "silu", parts, y1, saved1, None, None)
    y2, _, values2, exponents2 = outputs()
    layer(x, w, b, r, "silu", parts, y2, None, values2, exponents2)
    assert torch.equal(y, y1) and torch.equal(y, y2)
    assert torch.equal(saved, saved1)
    assert torch.equal(exponents, exponents2)
    assert torch.equal(values, values2)
    assert int(exponents.max()) < 254 and int(values.min()) > -128
    assert backend._native.lib().tp_b200_take_device_error(torch.cuda.current_device()) == 0
