"""CPU: what the sequence operators refuse - the Python functions on host tensors (shapes, types, strides, then the device) and the C
entry points on argument blocks that no launch may follow.  No pointer given here is ever read."""
import ctypes as C
import importlib

import pytest
import torch

from segamd import sequence as seq

ffi = importlib.import_module("tf-1d-2d-segmentation-end2endpipelines_amd._ffi")
T = torch.zeros


@pytest.fixture(scope="module")
def lib():
    return ffi.lib()


# ---------------------------------------------------------------------------------------------------------------- Python level
def test_valid_calls_end_at_the_missing_gpu():
    x, w = T(4, 8), T(6, 8)
    for f in (lambda: seq.layer_norm(x), lambda: seq.layer_norm_backward(x, x, T(4), T(4)), lambda: seq.linear(x, w), lambda: seq.linear_backward(T(4, 6), x, w),
              lambda: seq.activation_backward(x, x, "silu"), lambda: seq.causal_conv(T(2, 5, 8), T(4, 8)),
              lambda: seq.causal_conv_backward(T(2, 5, 8), T(2, 5, 8), T(4, 8)), lambda: seq.causal_conv_step(T(2, 8), T(2, 3, 8), T(4, 8)),
              lambda: seq.selective_scan(T(2, 5, 8), T(2, 5, 8), T(8, 16), T(2, 5, 16), T(2, 5, 16)),
              lambda: seq.selective_scan_step(T(2, 8), T(2, 8), T(8, 16), T(2, 16), T(2, 16), T(2, 8, 16))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f()


@pytest.mark.parametrize("call,match", [
    (lambda: seq.layer_norm([1.0]), "torch tensor"),
    (lambda: seq.layer_norm(T(4, 8, dtype=torch.float64)), "float16, bfloat16 or float32"),
    (lambda: seq.layer_norm(T(4, 0)), "no channels"),
    (lambda: seq.layer_norm(T(4, 8), T(7)), "gamma has shape"),
    (lambda: seq.layer_norm(T(4, 8), T(8, dtype=torch.float16)), "gamma is"),
    (lambda: seq.layer_norm(T(8, 4).t()), "channel axis must be contiguous"),
    (lambda: seq.layer_norm(T(1, 8).expand(4, 8)), "rows overlap"),
    (lambda: seq.layer_norm(T(3, 4, 8)[:, :2]), "not evenly spaced"),
    (lambda: seq.layer_norm(T(4, 8), eps=-1.0), "eps"),
    (lambda: seq.layer_norm(T(4, 8, requires_grad=True)), "requires grad"),
    (lambda: seq.layer_norm_backward(T(4, 8), T(4, 8), None, T(4)), "mean is needed"),
    (lambda: seq.layer_norm_backward(T(4, 7), T(4, 8), T(4), T(4)), "dy has shape"),
    (lambda: seq.layer_norm_backward(T(4, 8), T(4, 8), T(5), T(4)), "mean has shape"),
    (lambda: seq.linear(T(4, 8), T(6, 7)), "inputs"),
    (lambda: seq.linear(T(4, 8), T(8)), "units, inputs"),
    (lambda: seq.linear(T(4, 8), T(6, 8, dtype=torch.float16)), "w is"),
    (lambda: seq.linear(T(4, 8), T(6, 8), T(5)), "bias has shape"),
    (lambda: seq.linear(T(4, 8), T(6, 8), activation="tanh"), "unknown activation"),
    (lambda: seq.linear(T(4, 8), T(6, 8), activation="softmax"), "unknown activation"),
    (lambda: seq.linear(T(4, 8), T(6, 8), residual=T(4, 8)), "residual has shape"),
    (lambda: seq.linear(T(4, 8), T(8, 6).t()), "w: the channel axis"),
    (lambda: seq.linear_backward(T(4, 6), T(4, 8), T(6, 8), activation="gelu"), "needs its input z"),
    (lambda: seq.linear_backward(T(4, 5), T(4, 8), T(6, 8)), "dy has shape"),
    (lambda: seq.linear_backward(T(4, 6), T(4, 8), T(6, 8), z=T(4, 6), activation="gelu"), "z has shape"),
    (lambda: seq.activation_backward(T(4, 8), T(4, 8), "tanh"), "unknown activation"),
    (lambda: seq.causal_conv(T(2, 8), T(4, 8)), "expected \\[B, L, D\\]"),
    (lambda: seq.causal_conv(T(2, 5, 8), T(9, 8)), "taps"),
    (lambda: seq.causal_conv(T(2, 5, 8), T(0, 8)), "taps"),
    (lambda: seq.causal_conv(T(2, 5, 8), T(4, 7)), "w has shape"),
    (lambda: seq.causal_conv(T(2, 5, 8), T(4, 8), activation="relu"), "activation"),
    (lambda: seq.causal_conv(T(2, 5, 8), T(4, 8), state=T(2, 4, 8)), "state has shape"),
    (lambda: seq.causal_conv(T(2, 5, 8), T(4, 8), lengths=T(2)), "lengths is"),
    (lambda: seq.causal_conv(T(2, 5, 8), T(4, 8), lengths=T(3, dtype=torch.int32)), "lengths has shape"),
    (lambda: seq.causal_conv(T(2, 1, 8).expand(2, 5, 8), T(4, 8)), "rows overlap"),
    (lambda: seq.causal_conv_step(T(2, 8), None, T(4, 8)), "state is needed"),
    (lambda: seq.causal_conv_step(T(2, 8), T(9, 3, 8)[:2], T(4, 8), new_state=T(2, 3, 7)), "new_state has shape"),
    (lambda: seq.selective_scan(T(2, 5, 8), T(2, 5, 8), T(8, 65), T(2, 5, 65), T(2, 5, 65)), "65 states"),
    (lambda: seq.selective_scan(T(2, 5, 8), T(2, 5, 8), T(7, 16), T(2, 5, 16), T(2, 5, 16)), "A has shape"),
    (lambda: seq.selective_scan(T(2, 5, 8), T(2, 4, 8), T(8, 16), T(2, 5, 16), T(2, 5, 16)), "dt has shape"),
    (lambda: seq.selective_scan(T(2, 5, 8), T(2, 5, 8), T(8, 16), T(2, 5, 16), T(2, 5, 15)), "C has shape"),
    (lambda: seq.selective_scan(T(2, 5, 8), T(2, 5, 8), T(8, 16), T(2, 5, 16), T(2, 5, 16), state=T(2, 8, 16).half()), "state is"),
    (lambda: seq.selective_scan(T(2, 5, 8), T(2, 5, 8), T(8, 16), T(2, 5, 16), T(2, 5, 16), z=T(2, 5, 8).half()), "z is"),
    (lambda: seq.selective_scan(T(2, 5, 8), T(2, 5, 8), T(8 * 16 + 1)[1:].view(8, 16), T(2, 5, 16), T(2, 5, 16)), "aligned"),
    (lambda: seq.selective_scan_backward(T(2, 5, 8), T(2, 5, 8), T(2, 5, 8), T(8, 16), T(2, 5, 16), T(2, 5, 16), None), "saved is needed"),
    (lambda: seq.selective_scan_backward(T(2, 5, 8), T(2, 5, 8), T(2, 5, 8), T(8, 16), T(2, 5, 16), T(2, 5, 16), T(3)), "saved has shape"),
    (lambda: seq.selective_scan_step(T(2, 8), T(2, 8), T(8, 16), T(2, 16), T(2, 16), None), "state is needed"),
])
def test_python_refusals(call, match):
    with pytest.raises((ValueError, TypeError), match=match):
        call()


def test_overlapping_state_buffers_are_refused():
    buf = T(5, 8, 16)
    with pytest.raises(ValueError, match="overlaps"):
        seq.selective_scan_step(T(3, 8), T(3, 8), T(8, 16), T(3, 16), T(3, 16), buf[:3], new_state=buf[1:4])


def test_graph_construction_needs_no_torch():
    import subprocess
    import sys
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = "import sys, segamd; assert 'torch' not in sys.modules; segamd.sequence; assert 'torch' in sys.modules"
    subprocess.run([sys.executable, "-c", code], cwd=root, check=True)


# --------------------------------------------------------------------------------------------------------------------- C level
FAKE = 1 << 20            # a pointer that would fault if anything read it


def refused(lib, rc, text):
    assert rc == -1
    assert text in lib.seg_last_error().decode(), lib.seg_last_error()


def test_struct_fields_match_the_header():
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    hdr = re.sub(r"/\*.*?\*/", "", open(os.path.join(root, "include", "seg_hip.h")).read(), flags=re.S)
    for struct, cls in (("seg_linear_args", ffi.LinearArgs), ("seg_causal_conv_args", ffi.CausalConvArgs), ("seg_scan_args", ffi.ScanArgs)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct, struct), hdr, re.S).group(1)
        names, kinds = [], []
        for decl in filter(None, (d.strip() for d in body.split(";"))):
            m = re.match(r"(const\s+)?(void|float|int64_t|int32_t)\s*(\*?)\s*(.*)", decl, re.S)
            for part in m.group(4).split(","):
                names.append(part.strip().lstrip("*").strip())
                kinds.append(C.c_void_p if m.group(3) or "*" in part else {"int64_t": C.c_int64, "int32_t": C.c_int32, "float": C.c_float}[m.group(2)])
        assert names == [f[0] for f in cls._fields_]
        assert kinds == [f[1] for f in cls._fields_]


def test_layernorm_arguments(lib):
    f = lib.seg_layernorm_fwd
    refused(lib, f(FAKE, 8, FAKE, 8, 4, 8, 3, None, None, 1e-3, None, None, None), "dtype")
    refused(lib, f(FAKE, 8, FAKE, 8, -1, 8, 0, None, None, 1e-3, None, None, None), "rows")
    refused(lib, f(FAKE, 7, FAKE, 8, 4, 8, 0, None, None, 1e-3, None, None, None), "strides")
    refused(lib, f(None, 8, FAKE, 8, 4, 8, 0, None, None, 1e-3, None, None, None), "NULL")
    b = lib.seg_layernorm_bwd
    refused(lib, b(FAKE, 8, FAKE, 8, FAKE, 8, 4, 8, 0, None, FAKE, None, FAKE, FAKE, FAKE, None), "NULL")
    refused(lib, b(FAKE, 8, FAKE, 8, FAKE, 8, 4, 8, 0, FAKE, FAKE, None, FAKE, FAKE, None, None), "workspace")
    assert f(None, 8, None, 8, 0, 8, 0, None, None, 1e-3, None, None, None) == 0
    assert lib.seg_layernorm_bwd_workspace_bytes(0, 8, 0) == 0 < lib.seg_layernorm_bwd_workspace_bytes(1, 8, 0)


def linear_args(**k):
    a = ffi.LinearArgs(64, 32, 16, 0, 0, 0.0, FAKE, 16, FAKE, 16)
    a.y, a.y_ld = FAKE, 32
    for n, v in k.items():
        setattr(a, n, v)
    return a


def test_linear_arguments(lib):
    for k, text in ((dict(dtype=5), "dtype"), (dict(N=0), "N 0"), (dict(K=0), "K 0"), (dict(M=-1), "M -1"), (dict(act=4), "activation"), (dict(x=None), "NULL"),
                    (dict(w=None), "NULL"), (dict(y=None), "NULL"), (dict(x_ld=15), "strides"), (dict(w_ld=15), "strides"), (dict(y_ld=31), "strides"),
                    (dict(z=FAKE, z_ld=31), "strides"), (dict(M=1 << 40), "too large")):
        refused(lib, lib.seg_linear_fwd(linear_args(**k), None), text)
    refused(lib, lib.seg_linear_bwd_data(linear_args(bias=FAKE), None), "bias")
    refused(lib, lib.seg_linear_bwd_data(linear_args(w_ld=31), None), "strides")
    long = linear_args(M=128, N=8, K=1 << 16, x_ld=1 << 16, w_ld=1 << 16)
    assert lib.seg_linear_workspace_bytes(long, ffi.LINEAR_FWD) > 0
    refused(lib, lib.seg_linear_fwd(long, None), "workspace")
    refused(lib, lib.seg_linear_bwd_weight(linear_args(dy=None), None), "NULL")
    refused(lib, lib.seg_linear_bwd_weight(linear_args(dy=FAKE, dy_ld=31, dw=FAKE, dw_ld=16), None), "strides")
    refused(lib, lib.seg_linear_bwd_weight(linear_args(dy=FAKE, dy_ld=32, dw=FAKE, dw_ld=15), None), "dw_ld")
    refused(lib, lib.seg_linear_bwd_weight(linear_args(dy=FAKE, dy_ld=32, db=FAKE), None), "workspace")
    # no rows: nothing to launch, nothing needed (a division by the number of tiles once ended the process here)
    assert lib.seg_linear_fwd(linear_args(M=0, x=None, y=None), None) == 0
    assert all(lib.seg_linear_workspace_bytes(linear_args(M=0), p) == 0 for p in (0, 1, 2))
    refused(lib, lib.seg_linear_act_bwd(FAKE, 8, FAKE, 8, FAKE, 7, 4, 8, 0, 1, 0.0, None), "strides")
    refused(lib, lib.seg_linear_act_bwd(FAKE, 8, FAKE, 8, FAKE, 8, 4, 8, 0, 4, 0.0, None), "activation")


def conv_args(**k):
    a = ffi.CausalConvArgs(2, 16, 8, 4, 0, 0, FAKE, 128, 8, FAKE)
    a.y, a.y_bs, a.y_ld = FAKE, 128, 8
    for n, v in k.items():
        setattr(a, n, v)
    return a


def test_causal_conv_arguments(lib):
    for k, text in ((dict(K=9), "K = 9"), (dict(K=0), "K = 0"), (dict(act=1), "activation"), (dict(dtype=-1), "dtype"), (dict(B=65536), "65535"), (dict(x=None), "NULL"),
                    (dict(w=None), "w is NULL"), (dict(x_ld=7), "strides"), (dict(y_ld=7), "strides"), (dict(state=FAKE, state_out=FAKE), "state_out")):
        refused(lib, lib.seg_causal_conv_fwd(conv_args(**k), None), text)
    refused(lib, lib.seg_causal_conv_bwd(conv_args(), None), "NULL")
    refused(lib, lib.seg_causal_conv_bwd(conv_args(dy=FAKE, dy_ld=8, dw=FAKE), None), "workspace")
    refused(lib, lib.seg_causal_conv_bwd(conv_args(dy=FAKE, dy_ld=8, dx=FAKE, dx_ld=8), None), "dx may not")
    refused(lib, lib.seg_causal_conv_step(conv_args(x_bs=7), None), "strides")
    assert lib.seg_causal_conv_fwd(conv_args(B=0, x=None), None) == 0


def scan_args(**k):
    a = ffi.ScanArgs(2, 16, 8, 16, 0, 1)
    for n, c in (("u", 8), ("dt", 8), ("Bm", 16), ("Cm", 16), ("y", 8), ("dy", 8)):
        setattr(a, n, FAKE)
        setattr(a, n + "_bs", 16 * c)
        setattr(a, n + "_ld", c)
    a.A = FAKE
    for n, v in k.items():
        setattr(a, n, v)
    return a


def test_selective_scan_arguments(lib):
    for k, text in ((dict(S=0), "states"), (dict(S=65), "states"), (dict(dtype=3), "dtype"), (dict(A=None), "A is NULL"), (dict(A=FAKE + 4), "alignment"),
                    (dict(state=FAKE + 8), "alignment"), (dict(u=None), "NULL"), (dict(Bm_ld=15), "strides"), (dict(y_ld=7), "strides"), (dict(B=65536), "65535"),
                    (dict(state=FAKE, state_out=FAKE), "state_out"), (dict(L=4096), "workspace")):
        refused(lib, lib.seg_selective_scan_fwd(scan_args(**k), None), text)
    refused(lib, lib.seg_selective_scan_bwd(scan_args(), None), "NULL")
    refused(lib, lib.seg_selective_scan_bwd(scan_args(saved=FAKE), None), "workspace")
    refused(lib, lib.seg_selective_scan_bwd(scan_args(saved=FAKE, workspace=FAKE, dz=FAKE, dz_ld=8), None), "dz without z")
    refused(lib, lib.seg_selective_scan_bwd(scan_args(saved=FAKE, workspace=FAKE + 4), None), "workspace needs")
    refused(lib, lib.seg_selective_scan_step(scan_args(u_bs=7), None), "strides")
    assert lib.seg_selective_scan_fwd(scan_args(B=0), None) == 0
    assert lib.seg_selective_scan_saved_bytes(scan_args()) == 2 * 1 * 8 * 16 * 4


def test_results_in_place_keep_the_row_stride(lib):
    """Where a result may take its operand's memory, rows of another stride would be written while other rows are still read."""
    refused(lib, lib.seg_layernorm_fwd(FAKE, 8, FAKE, 16, 4, 8, 0, None, None, 1e-3, None, None, None), "stride")
    b = lib.seg_layernorm_bwd
    refused(lib, b(FAKE, 8, 2 * FAKE, 8, FAKE, 16, 4, 8, 0, FAKE, FAKE, None, FAKE, FAKE, FAKE, None), "in place")
    refused(lib, b(FAKE, 8, 2 * FAKE, 8, 2 * FAKE, 16, 4, 8, 0, FAKE, FAKE, None, FAKE, FAKE, FAKE, None), "in place")
    refused(lib, lib.seg_linear_act_bwd(FAKE, 8, 2 * FAKE, 8, FAKE, 16, 4, 8, 0, 1, 0.0, None), "in place")
    refused(lib, lib.seg_linear_fwd(linear_args(residual=FAKE, residual_ld=40), None), "in place")
    refused(lib, lib.seg_linear_bwd_data(linear_args(w_ld=32, residual=FAKE, residual_ld=40), None), "in place")


def test_layernorm_row_length_limit(lib):
    refused(lib, lib.seg_layernorm_fwd(FAKE, 1 << 31, 2 * FAKE, 1 << 31, 4, (1 << 30) + 1, 0, None, None, 1e-3, None, None, None), "2^30")
    refused(lib, lib.seg_layernorm_bwd(FAKE, 1 << 31, 2 * FAKE, 1 << 31, None, 0, 4, (1 << 30) + 1, 0, FAKE, FAKE, None, FAKE, FAKE, FAKE, None), "2^30")
