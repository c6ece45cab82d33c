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


# --------------------------------------------------------------------------------------------------------------- C level
FAKE = 1 << 20            # a pointer that would fault if anything read it


def refused(rc, text):
    assert rc == -1
    assert text in ffi.lib().seg_last_error().decode(), ffi.lib().seg_last_error()


def test_causal_conv_length_limit():
    """Long sequences do not end at one grid axis of 65535 blocks of 64 rows; the workspace is counted in 64 bits."""
    lib = ffi.lib()

    def args(B, L, x=None):
        a = ffi.CausalConvArgs(B, L, 8, 4, 0, 0, x, 0, 8, FAKE)
        a.y, a.y_ld = FAKE, 8
        return a
    refused(lib.seg_causal_conv_fwd(args(1, (1 << 30) + 1, FAKE), None), "2^30")
    refused(lib.seg_causal_conv_fwd(args(32768, 65535 * 64 + 1, FAKE), None), "sequences of")
    refused(lib.seg_causal_conv_fwd(args(128, 1 << 30, FAKE), None), "sequences of")
    refused(lib.seg_causal_conv_fwd(args(127, 1 << 30), None), "NULL")
    refused(lib.seg_causal_conv_fwd(args(32767, 65535 * 64 + 1), None), "NULL")
    for L in (0, 1, 64, 65, 65535 * 64, 65535 * 64 + 1, 1 << 30):
        blocks = max(1, -(-L // 64))
        least, most = 3 * blocks * 5 * 8 * 4, 3 * (blocks + 512) * 5 * 8 * 4
        assert least <= lib.seg_causal_conv_bwd_workspace_bytes(args(3, L)) <= (least if blocks <= 65535 else most), L


def test_grids_that_would_wrap_are_refused():
    """An axis of a grid takes fewer than 2^32 threads and wraps without an error: refused in front of the launch."""
    lib = ffi.lib()
    a = ffi.CausalConvArgs(65535, 1, 1 << 20, 1, 0, 0, FAKE, 1 << 20, 1 << 20, FAKE)
    a.y, a.y_bs, a.y_ld = FAKE, 1 << 20, 1 << 20
    refused(lib.seg_causal_conv_step(a, None), "too many")
    for B, D, S, f in ((65535, 1 << 13, 64, lib.seg_selective_scan_step), (4, 1 << 28, 16, lib.seg_selective_scan_step), (1, 1 << 28, 64, lib.seg_selective_scan_fwd),
                       (1, 1 << 30, 16, lib.seg_selective_scan_fwd), (1, 1 << 28, 33, lib.seg_selective_scan_bwd)):
        a = ffi.ScanArgs(B, 1, D, S, 0, 1)
        for n, c in (("u", D), ("dt", D), ("Bm", S), ("Cm", S), ("y", D), ("dy", D)):
            setattr(a, n, FAKE)
            setattr(a, n + "_bs", c)
            setattr(a, n + "_ld", c)
        a.A = a.state = a.saved = a.workspace = FAKE
        refused(f(a, None), "too many")


# ------------------------------------------------------------------------------------------------------------- derivatives
def test_forward_mode_tangents_are_refused():
    """A dual tensor's tangent would be lost without a word; outside a dual level, and for operands without one, nothing changes."""
    from torch.autograd import forward_ad as fwd
    x, w = torch.ones(4, 8), torch.ones(6, 8)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for f in (lambda: seq.layer_norm(d), lambda: seq.linear(d, w), lambda: seq.linear(x, fwd.make_dual(w, torch.ones_like(w))),
                  lambda: seq.activation_backward(d, x, "silu"), lambda: seq.causal_conv(d[None], T(4, 8)), lambda: seq.causal_conv_step(d, T(4, 3, 8), T(4, 8)),
                  lambda: seq.selective_scan(d[None], T(1, 4, 8), T(8, 4), T(1, 4, 4), T(1, 4, 4)),
                  lambda: seq.selective_scan_step(d, T(4, 8), T(8, 4), T(4, 4), T(4, 4), T(4, 8, 4))):
            with pytest.raises(ValueError, match="tangent"):
                f()
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            seq.linear(x, w)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        seq.linear(x, w)


def test_a_new_state_that_requires_grad_is_refused():
    """It is written, so it gets the check that state gets; torch.no_grad() lifts both."""
    for f in (lambda n: seq.causal_conv_step(T(2, 8), T(2, 3, 8), T(4, 8), new_state=n(2, 3, 8)),
              lambda n: seq.selective_scan_step(T(2, 8), T(2, 8), T(8, 4), T(2, 4), T(2, 4), T(2, 8, 4), new_state=n(2, 8, 4))):
        with pytest.raises(ValueError, match="requires grad"):
            f(lambda *s: T(*s, requires_grad=True))
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
            f(lambda *s: T(*s, requires_grad=True))
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f(T)


def test_saved_states_that_require_grad_are_refused():
    t = T(2, 5, 8)
    args = (t, t, t, T(8, 4), T(2, 5, 4), T(2, 5, 4))
    n = 2 * 1 * 8 * 4
    with pytest.raises(ValueError, match="requires grad"):
        seq.selective_scan_backward(*args, T(n, requires_grad=True))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        seq.selective_scan_backward(*args, T(n))


def test_many_rows_and_large_tensors_are_no_large_extents():
    """Rows of layer_norm and linear count in 64 bits; a tensor of more than 2^31 elements has no large extent by that alone."""
    def m(*shape):
        return T(*shape, device="meta")
    for f in (lambda: seq.layer_norm(m(BIG, 8)), lambda: seq.linear(m(BIG, 8), m(4, 8)), lambda: seq.linear(m(2, 1 << 17), m(1 << 17, 1 << 17)),
              lambda: seq.causal_conv(m(1 << 10, 1 << 11, 1 << 12), m(4, 1 << 12)),
              lambda: seq.selective_scan(m(1 << 10, 1 << 11, 1 << 12), m(1 << 10, 1 << 11, 1 << 12), m(1 << 12, 4), m(1 << 10, 1 << 11, 4), m(1 << 10, 1 << 11, 4))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f()
    with pytest.raises(ValueError, match="2147483647"):
        seq.causal_conv(m(BIG, 0, 8), m(1, 8))


def test_channel_limit():
    """Channel indices of a last block reach 256 behind the last channel: they hold in 32 bits up to 2^30 channels."""
    lib = ffi.lib()
    D = (1 << 30) + 1
    a = ffi.CausalConvArgs(1, 1, D, 2, 0, 0, FAKE, D, D, FAKE)
    a.y, a.y_bs, a.y_ld, a.dy, a.dy_bs, a.dy_ld, a.workspace = FAKE, D, D, FAKE, D, D, FAKE
    for f in (lib.seg_causal_conv_fwd, lib.seg_causal_conv_bwd, lib.seg_causal_conv_step):
        refused(f(a, None), "D 1073741825")
    a = ffi.ScanArgs(1, 1, D, 1, 0, 1)
    for n, c in (("u", D), ("dt", D), ("Bm", 1), ("Cm", 1), ("y", D), ("dy", D)):
        setattr(a, n, FAKE)
        setattr(a, n + "_bs", c)
        setattr(a, n + "_ld", c)
    a.A = a.state = a.saved = a.workspace = FAKE
    for f in (lib.seg_selective_scan_fwd, lib.seg_selective_scan_bwd, lib.seg_selective_scan_step):
        refused(f(a, None), "D 1073741825")
