"""The feed-forward entry points of the C ABI without a GPU: malformed calls
return a negative status with a message before any device is touched, and the
host-side shape checks refuse what the kernels do not take.  No kernel is
launched here; the pointers are never read."""

from __future__ import annotations

import os
import re
import subprocess

import pytest
import torch

from tensorplay_mlu_b200 import _native as N
from tensorplay_mlu_b200 import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F32, F64 = 7, 6, 8
P = 0x10000  # a pointer that is never followed

LAYER = dict(dtype=BF16, act=4, parts=2, flags=0, m=4, n=32, k=16, x=P, x_stride=16, w=P, w_stride=16, bias=0,
             residual=0, residual_stride=0, y=P, y_stride=32, saved=0, values=0, exponents=0, x_work=0, w_work=0)
GRAD = dict(dtype=BF16, act=4, parts=2, flags=0, m=4, n=32, k=16, groups=1, dy=P, dy_stride=32, x=P, x_stride=16, w=P,
            w_stride=16, saved=P, values=0, exponents=0, dx=P, dw=P, db=P, dz=P, dz_stride=64, partial=P, x_work=0,
            w_work=0)


def refused(entry, packer, base, **changes):
    lib = N.lib()
    args = {**base, **changes}
    assert getattr(lib, entry)(packer.pack(*args.values()), None) < 0
    return lib.tp_b200_last_error().decode()


@pytest.mark.parametrize("change,match", [
    (dict(dtype=F64), "float64"), (dict(dtype=3), "int32"), (dict(act=9), "unknown activation"), (dict(act=-1), "unknown activation"),
    (dict(parts=3), "one part"), (dict(m=-1), "out of range"), (dict(n=1 << 31), "out of range"),
    (dict(k=1 << 40), "out of range"), (dict(values=P), "values and exponents"), (dict(y=0), "null operand"),
    (dict(x=0), "null operand"), (dict(w=0), "null operand"), (dict(residual=P), "takes no residual"),
    (dict(k=0), "needs `saved`"),
])
def test_layer_forward_refusals(change, match):
    assert match in refused("tp_b200_layer_forward", N.LAYER, LAYER, **change)


@pytest.mark.parametrize("change,match", [
    (dict(dtype=F64), "float64"), (dict(act=5), "unknown activation"), (dict(parts=0), "one part"), (dict(m=-2), "out of range"),
    (dict(exponents=P), "values and exponents"), (dict(values=P, exponents=P), "in one form"),
    (dict(groups=0), "1 to 65535 groups"), (dict(groups=70000), "1 to 65535 groups"), (dict(partial=0), "1 to 65535 groups"),
    (dict(dy=0), "null operand"), (dict(dz=0), "null operand"), (dict(saved=0), "null operand"),
    (dict(dz_stride=63), "workspace's rows"), (dict(w=0), "null operand"), (dict(x=0), "null operand"),
])
def test_layer_backward_refusals(change, match):
    assert match in refused("tp_b200_layer_backward", N.LAYER_GRAD, GRAD, **change)


def test_null_arguments_are_refused():
    lib = N.lib()
    assert lib.tp_b200_layer_forward(None, None) < 0
    assert lib.tp_b200_layer_backward(None, None) < 0
    assert lib.tp_b200_checkpoint_pack(None, None) < 0
    assert lib.tp_b200_checkpoint_unpack(None, None) < 0
    assert lib.tp_b200_checkpoint_backward(None, None) < 0


def test_empty_calls_touch_no_device():
    lib = N.lib()
    assert lib.tp_b200_layer_forward(N.LAYER.pack(*{**LAYER, "m": 0}.values()), None) == 0
    assert lib.tp_b200_layer_forward(N.LAYER.pack(*{**LAYER, "n": 0, "y": 0}.values()), None) == 0
    empty = {**GRAD, "m": 0, "dx": 0, "dw": 0, "db": 0}
    assert lib.tp_b200_layer_backward(N.LAYER_GRAD.pack(*empty.values()), None) == 0


CHECKPOINT = dict(dtype=BF16, act=2, rows=4, n=40, x=P, x_stride=40, y=P, y_stride=40, values=P, exponents=P)


@pytest.mark.parametrize("entry", ["pack", "unpack", "backward"])
@pytest.mark.parametrize("change,match", [
    (dict(dtype=F64), "float64"), (dict(act=8), "unknown activation"), (dict(rows=-1), "out of range"), (dict(n=-3), "out of range"),
    (dict(n=1 << 50), "out of range"), (dict(values=0), "null operand"), (dict(exponents=0), "null operand"),
])
def test_checkpoint_refusals(entry, change, match):
    assert match in refused(f"tp_b200_checkpoint_{entry}", N.CHECKPOINT, CHECKPOINT, **change)


def test_checkpoint_operands():
    assert "null operand" in refused("tp_b200_checkpoint_pack", N.CHECKPOINT, CHECKPOINT, x=0)
    assert "null operand" in refused("tp_b200_checkpoint_unpack", N.CHECKPOINT, CHECKPOINT, y=0)
    assert "null operand" in refused("tp_b200_checkpoint_backward", N.CHECKPOINT, CHECKPOINT, x=0)
    assert "null operand" in refused("tp_b200_checkpoint_backward", N.CHECKPOINT, CHECKPOINT, y=0)
    for entry in ("pack", "unpack", "backward"):
        call = getattr(N.lib(), f"tp_b200_checkpoint_{entry}")
        assert call(N.CHECKPOINT.pack(*{**CHECKPOINT, "rows": 0}.values()), None) == 0
        assert call(N.CHECKPOINT.pack(*{**CHECKPOINT, "n": 0, "values": 0}.values()), None) == 0


def test_packed_arguments_match_the_header(tmp_path):
    """The structs Python packs have the sizes and offsets the C compiler gives them."""
    text = open(os.path.join(ROOT, "include", "tpb200.h")).read()
    lines = ['#include "tpb200.h"', "#include <stddef.h>", "#include <stdio.h>", "int main(void) {"]
    for name in ("tpb_layer", "tpb_layer_grad", "tpb_checkpoint"):
        lines.append(f'printf("%zu\\n", sizeof({name}));')
    last = {"tpb_layer": "w_work", "tpb_layer_grad": "w_work", "tpb_checkpoint": "exponents"}
    for name, field in last.items():
        lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
    source = tmp_path / "sizes.c"
    source.write_text("\n".join(lines + ["return 0;", "}"]))
    binary = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(source), "-o", str(binary)], check=True)
    got = [int(v) for v in subprocess.run([str(binary)], check=True, capture_output=True, text=True).stdout.split()]
    assert got[:3] == [N.LAYER.size, N.LAYER_GRAD.size, N.CHECKPOINT.size]
    assert got[3:] == [N.LAYER.size - 8, N.LAYER_GRAD.size - 8, N.CHECKPOINT.size - 8]
    # field order: as many fields as values packed
    for struct_name, packer in (("tpb_layer", N.LAYER), ("tpb_layer_grad", N.LAYER_GRAD),
                                ("tpb_checkpoint", N.CHECKPOINT)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % struct_name, text, re.S).group(1)
        fields = sum(len(line.split(",")) for line in body.split(";") if line.strip())
        assert fields == len(packer.unpack(bytes(packer.size)))


def test_operators_refuse_host_tensors():
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    for call in (lambda: ops.gated_linear(x, w), lambda: ops.linear_act(x, w), lambda: ops.checkpoint_pack(x),
                 lambda: ops.native_linear_act_backward(x, x, w, x),
                 lambda: ops.checkpoint_unpack(x.char(), x.byte(), torch.float32)):
        with pytest.raises(RuntimeError, match="device tensor"):
            call()
    with pytest.raises(RuntimeError, match="activation must be one of"):
        ops.gated_linear(x, w, None, "swish")


@pytest.mark.parametrize("n", [(1 << 30) - 1, (1 << 30) - 128])
def test_weight_rows_whose_tiles_pass_32_bits_are_refused(n):
    """Both parts together are a dimension of the gradients' products, which
    count it, and the last tile's rows, in 32-bit integers."""
    assert "out of range" in refused("tp_b200_layer_forward", N.LAYER, LAYER, n=n, y_stride=n)
    assert "out of range" in refused("tp_b200_layer_backward", N.LAYER_GRAD, GRAD, n=n, dy_stride=n, dz_stride=2 * n)
