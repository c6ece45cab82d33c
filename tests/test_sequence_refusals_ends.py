"""CPU: what the sequence operators refuse or take at the ends of their ranges."""
import importlib

import pytest
import torch

from segamd import sequence as seq

ffi = importlib.import_module("tf-1d-2d-segmentation-end2endpipelines_amd._ffi")
T = torch.zeros


# ------------------------------------------------------------------------------------------------------- extents past 32 bits
BIG = (1 << 32) + 8


@pytest.mark.parametrize("call", [
    lambda m: seq.layer_norm(m(2, BIG)),
    lambda m: seq.layer_norm_backward(m(2, BIG), m(2, BIG), m(2), m(2)),
    lambda m: seq.linear(m(2, BIG), m(4, BIG)),
    lambda m: seq.linear(m(2, 8), m(BIG, 8)),
    lambda m: seq.linear_backward(m(2, BIG), m(2, 8), m(BIG, 8)),
    lambda m: seq.linear_backward(m(2, 8), m(2, BIG), m(8, BIG)),
    lambda m: seq.activation_backward(m(2, BIG), m(2, BIG), "silu"),
    lambda m: seq.causal_conv(m(1, BIG, 8), m(4, 8)),
    lambda m: seq.causal_conv(m(BIG, 1, 8), m(4, 8)),
    lambda m: seq.causal_conv(m(1, 1, BIG), m(4, BIG)),
    lambda m: seq.causal_conv_backward(m(1, BIG, 8), m(1, BIG, 8), m(4, 8)),
    lambda m: seq.causal_conv_step(m(BIG, 8), m(BIG, 3, 8), m(4, 8)),
    lambda m: seq.selective_scan(m(1, BIG, 8), m(1, BIG, 8), m(8, 4), m(1, BIG, 4), m(1, BIG, 4)),
    lambda m: seq.selective_scan(m(BIG, 1, 8), m(BIG, 1, 8), m(8, 4), m(BIG, 1, 4), m(BIG, 1, 4)),
    lambda m: seq.selective_scan_backward(m(1, BIG, 8), m(1, BIG, 8), m(1, BIG, 8), m(8, 4), m(1, BIG, 4), m(1, BIG, 4), m(4)),
    lambda m: seq.selective_scan_step(m(1, BIG), m(1, BIG), m(BIG, 4), m(1, 4), m(1, 4), m(1, BIG, 4)),
])
def test_extents_that_an_int32_does_not_hold(call):
    """They would reach the C level as their low 32 bits, 8 here: refused in front of it (tensors without memory, on torch's meta device)."""
    with pytest.raises(ValueError, match="2147483647"):
        call(lambda *shape: T(*shape, device="meta"))


# ------------------------------------------------------------------------------------------------------------- empty extents
@pytest.mark.parametrize("shape", [(4, 0), (0, 4), (3, 0, 5), (2, 5, 0), (0, 0)])
def test_empty_leading_axes_are_calls_without_work(shape):
    """An extent of zero in any place in front of the channels passes the checks of strides (there are no rows to be spaced)."""
    x, y, w = T(*shape, 8), T(*shape, 6), T(6, 8)
    for f in (lambda: seq.layer_norm(x), lambda: seq.layer_norm_backward(x, x, T(*shape), T(*shape)), lambda: seq.linear(x, w, residual=y),
              lambda: seq.linear_backward(y, x, w, z=x, activation="gelu", residual=x), lambda: seq.activation_backward(x, x, "silu")):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f()
