"""The feed-forward operators in a profile: a row each, by their own names."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_profile_reports_the_feed_forward_operators(backend):
    from tensorplay_mlu_b200.profiler import profile

    ops = backend.ops
    x, w = torch.randn(5, 64, device="cuda"), torch.randn(96, 64, device="cuda")
    with profile() as prof:
        h, saved = ops.native_gated_linear(x, w)
        ops.native_gated_linear_backward(h, x, w, saved)
        for _ in range(2):
            ops.gated_linear(x, w)
        y, pre = ops.native_linear_act(x, w)
        ops.linear_act(x, w)
        ops.native_linear_act_backward(y, x, w, pre)
        held = ops.checkpoint_pack(y)
        ops.checkpoint_unpack(*held, torch.float32)
        ops.checkpoint_activation_backward(y, *held, "gelu")
    rows = {r.key: r for r in prof.key_averages()}
    assert {f.__name__ for f in ops.FEED_FORWARD} <= set(rows)
    for f in ops.FEED_FORWARD:
        row = rows[f.__name__]
        assert row.count == (2 if f.__name__ == "gated_linear" else 1)
        assert row.device_time_total > 0 and row.cpu_time_total > 0
    # Outside the block the operators are the plain functions again.
    assert ops.linear_act in ops.FEED_FORWARD
