"""Sequence operators: layer normalisation, the matrix product with its epilogue, the short causal convolution and the selective state
space scan - the pieces of a sequence mixer for 1D signals and flattened bottlenecks - on torch tensors of a GPU.

Every function enqueues kernels of libseg_hip.so on the current stream of its tensors' device and returns without synchronising; what
it allocates (outputs, workspaces) comes from torch's allocator on that stream, so calls can be captured into a graph.  Rows are
channels-last ([..., C], [B, L, D]) in fp16, bf16 or fp32; they may be slices of wider tensors as long as the channel axis is
contiguous.  Parameters, statistics, scan states and gradients of parameters are fp32.  Gradients are explicit functions, as everywhere
in this package: nothing is recorded by torch.autograd, and a call on tensors that ask for it - or carry a forward-mode tangent - raises.

Weights are stored the way the matrix cores read them: `linear` takes [units, inputs] (a Keras Dense kernel transposed), `causal_conv`
[K, D] (a Keras depthwise kernel without its last axis), tap K - 1 on the current row.

Parity-mode tensors of a SegModel (split pairs) are another storage: decode them first (DevTensor.values(), splitfmt.py)."""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _ffi
from ._ffi import SEQ_ACT, CausalConvArgs, LinearArgs, ScanArgs
from .ops import KernelProfile, _DryRun, call

__all__ = ["layer_norm", "layer_norm_backward", "linear", "linear_backward", "activation_backward", "causal_conv", "causal_conv_backward",
           "causal_conv_step", "selective_scan", "selective_scan_backward", "selective_scan_step", "ScanGrads"]

_DT = {torch.float16: _ffi.DT_F16, torch.bfloat16: _ffi.DT_BF16, torch.float32: _ffi.DT_F32}
MAX_TAPS, MAX_STATES = 8, 64
MAX_EXTENT = (1 << 31) - 1                   # of channels, units, rows of a sequence and sequences: the C level's int32 (rows of layer_norm and linear: int64)


# ----------------------------------------------------------------------------------------------------------------- checks
# Small calls are bound by the host: the checks look at what is right first (a few attribute reads) and find out what is wrong after.
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None
_fns = {}


def _fail(what, msg):
    raise ValueError(f"{what}: {msg}")


def _dtype(what, x):
    try:
        return _DT[x.dtype]
    except (AttributeError, KeyError):
        pass
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what}: a torch tensor is needed, got {type(x).__name__}")
    _fail(what, f"elements must be float16, bfloat16 or float32, got {x.dtype}")


def _wrong(what, name, t, ref, dtype, shape):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: {name} must be a torch tensor, got {type(t).__name__}")
    if t.dtype != dtype or t.device != ref.device:
        _fail(what, f"{name} is {t.dtype} on {t.device}, expected {dtype} on {ref.device}")
    if t.shape != shape:
        _fail(what, f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _like(what, name, t, ref, shape):
    """t: elements like ref's, of this shape, channels contiguous."""
    try:
        if t.dtype is ref.dtype and t.shape == shape and t.get_device() == ref.get_device() and (t.stride(-1) == 1 or shape[-1] == 1):
            return t
    except AttributeError:
        pass
    _wrong(what, name, t, ref, ref.dtype, shape)
    _fail(what, f"{name}: the channel axis must be contiguous (strides {t.stride()})")


def _param(what, name, t, ref, shape, dtype=torch.float32):
    """t: a dense tensor of parameters or states (None passes)."""
    if t is None:
        return None
    try:
        if t.dtype is dtype and t.shape == shape and t.get_device() == ref.get_device() and t.is_contiguous():
            return t
    except AttributeError:
        pass
    _wrong(what, name, t, ref, dtype, shape)
    _fail(what, f"{name} must be contiguous (strides {t.stride()})")


def _extents(what, t):
    """ctypes would hand on the low 32 bits of a larger extent.  (No extent of a tensor of few elements is large, unless it has none.)"""
    if not 0 < t.numel() <= MAX_EXTENT and max(t.shape) > MAX_EXTENT:
        _fail(what, f"an extent of {max(t.shape)} (at most {MAX_EXTENT} channels, units, rows of a sequence or sequences)")


def _rows(what, name, t):
    """(rows, row stride) of [..., C] whose leading axes collapse into one."""
    shape, strides = t.shape, t.stride()
    c = shape[-1]
    if c > MAX_EXTENT:                                           # (rows: int64)
        _extents(what, t)
    if c > 1 and strides[-1] != 1:
        _fail(what, f"{name}: the channel axis must be contiguous (strides {strides})")
    if len(shape) == 2:
        rows, ld = shape[0], strides[0]
    elif 0 in shape[:-1]:
        return 0, c
    else:
        rows, ld, first = 1, c, True
        for size, stride in zip(reversed(shape[:-1]), reversed(strides[:-1])):
            if size != 1:
                if first:
                    ld, first = stride, False
                elif stride != ld * rows:
                    _fail(what, f"{name}: leading axes of strides {strides} and sizes {tuple(shape)} are not evenly spaced rows; call .contiguous()")
                rows *= size
    if rows > 1:
        if ld < c:
            _fail(what, f"{name}: rows overlap (strides {strides}); call .contiguous()")
    else:
        ld = c
    return rows, ld


def _spaced(what, name, t):
    if t.shape[1] > 1 and t.stride(1) < t.shape[2]:
        _fail(what, f"{name}: rows overlap (strides {t.stride()}); call .contiguous()")


def _no_grad(what, *ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                _fail(what, "a tensor requires grad, but nothing here is recorded by torch.autograd: detach it and call the *_backward function")
    if getattr(forward_ad, "_current_level", 0) >= 0:           # (inside a dual level; torch without that name: always looked at)
        for t in ts:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                _fail(what, "a tensor carries a forward-mode tangent, which would be lost")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _gpu(what, t):
    """The index of t's device."""
    i = t.get_device()
    if i < 0:
        raise RuntimeError(f"{what}: the tensors are on {t.device}; the operators run on an MI355X only - there is no CPU fallback")
    return i


def _launch(i, name, *args):
    """Enqueue on device i's current stream."""
    if _DryRun.on or KernelProfile.on or _raw_stream is None or i != torch.cuda.current_device():
        with torch.cuda.device(i):
            call(name, *args, C.c_void_p(torch.cuda.current_stream().cuda_stream))
        return
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = getattr(_ffi.lib(), name)
    rc = fn(*args, _raw_stream(i))
    if rc != 0:
        _ffi.check(rc, name)


def _bytes(n, dev):
    return torch.empty(n, dtype=torch.uint8, device=dev) if n > 0 else None


def _act(what, name):
    a = SEQ_ACT.get(name)
    if a is None:
        _fail(what, f"unknown activation {name!r} (one of {sorted(k for k in SEQ_ACT if k)})")
    return a


# ------------------------------------------------------------------------------------------------------- layer normalisation
def layer_norm(x, gamma=None, beta=None, eps: float = 1e-3, stats: bool = False):
    """y = (x - mean) / sqrt(var + eps) * gamma + beta over the last axis (biased variance; gamma / beta None: 1 / 0).
    Returns y, or (y, mean, rstd) with stats=True - what layer_norm_backward takes."""
    what = "layer_norm"
    dt = _dtype(what, x)
    if x.dim() < 1 or x.shape[-1] < 1:
        _fail(what, f"x of shape {tuple(x.shape)} has no channels")
    if not eps >= 0:
        _fail(what, f"eps = {eps}")
    c = x.shape[-1]
    _param(what, "gamma", gamma, x, (c,))
    _param(what, "beta", beta, x, (c,))
    rows, ld = _rows(what, "x", x)
    _no_grad(what, x, gamma, beta)
    di = _gpu(what, x)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    mean = rstd = None
    if stats:
        mean, rstd = torch.empty((2,) + tuple(x.shape[:-1]), dtype=torch.float32, device=x.device).unbind(0)
    _launch(di, "seg_layernorm_fwd", _ptr(x), ld, _ptr(y), c, rows, c, dt, _ptr(gamma), _ptr(beta), eps, _ptr(mean), _ptr(rstd))
    return (y, mean, rstd) if stats else y


def layer_norm_backward(dy, x, mean, rstd, gamma=None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dgamma, dbeta) of layer_norm(x, gamma, beta, stats=True)."""
    what = "layer_norm_backward"
    dt = _dtype(what, x)
    if x.dim() < 1 or x.shape[-1] < 1:
        _fail(what, f"x of shape {tuple(x.shape)} has no channels")
    c = x.shape[-1]
    _like(what, "dy", dy, x, x.shape)
    for n, t in (("mean", mean), ("rstd", rstd)):
        if t is None:
            _fail(what, f"{n} is needed (layer_norm(..., stats=True) returns it)")
        _param(what, n, t, x, x.shape[:-1])
    _param(what, "gamma", gamma, x, (c,))
    rows, ld = _rows(what, "x", x)
    _r, dy_ld = _rows(what, "dy", dy)
    _no_grad(what, dy, x, mean, rstd, gamma)
    di = _gpu(what, x)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    par = torch.empty((2, c), dtype=torch.float32, device=x.device)
    ws = _bytes(_ffi.lib().seg_layernorm_bwd_workspace_bytes(rows, c, dt), x.device)
    p = par.data_ptr()
    _launch(di, "seg_layernorm_bwd", _ptr(dy), dy_ld, _ptr(x), ld, _ptr(dx), c, rows, c, dt, _ptr(mean), _ptr(rstd), _ptr(gamma), p, p + 4 * c, _ptr(ws))
    return dx, par[0], par[1]


# --------------------------------------------------------------------------------------------------------------------- linear
def _linear_args(what, x, w, activation, alpha):
    dt = _dtype(what, x)
    if x.dim() < 1 or not isinstance(w, torch.Tensor) or w.dim() != 2:
        _fail(what, "x must be [..., inputs] and w [units, inputs]")
    if min(w.shape) < 1:
        _fail(what, f"w has shape {tuple(w.shape)}")
    _extents(what, w)
    if w.dtype != x.dtype or w.device != x.device:
        _fail(what, f"w is {w.dtype} on {w.device}, expected {x.dtype} on {x.device}")
    _n, w_ld = _rows(what, "w", w)
    return dt, _act(what, activation), w_ld


def linear(x, w, bias=None, activation: Optional[str] = None, alpha: float = 0.3, residual=None, preactivation: bool = False):
    """act(x w^T + bias) + residual in one launch (plus one that joins split sums where the result is small).  x [..., inputs],
    w [units, inputs] of the same type, bias fp32 [units], residual [..., units]; activation None / "linear", "relu", "leaky_relu"
    (slope alpha), "sigmoid", "silu", "gelu" (the error-function form).  Returns y, or (y, z) with preactivation=True: z = x w^T + bias."""
    what = "linear"
    dt, act, w_ld = _linear_args(what, x, w, activation, alpha)
    n, k = w.shape
    if x.shape[-1] != k:
        _fail(what, f"x has {x.shape[-1]} inputs, w {k}")
    _param(what, "bias", bias, x, (n,))
    m, x_ld = _rows(what, "x", x)
    shape = x.shape[:-1] + (n,)
    r_ld = 0
    if residual is not None:
        _like(what, "residual", residual, x, shape)
        _r, r_ld = _rows(what, "residual", residual)
    _no_grad(what, x, w, bias, residual)
    di = _gpu(what, x)
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    z = torch.empty(shape, dtype=x.dtype, device=x.device) if preactivation else None
    a = LinearArgs(m, n, k, dt, act, alpha, _ptr(x), x_ld, _ptr(w), w_ld, _ptr(bias), _ptr(residual), r_ld, _ptr(z), n, _ptr(y), n)
    ws = _bytes(_ffi.lib().seg_linear_workspace_bytes(a, _ffi.LINEAR_FWD), x.device)
    a.workspace = _ptr(ws)
    _launch(di, "seg_linear_fwd", a)
    return (y, z) if preactivation else y


def linear_backward(dy, x, w, z=None, activation: Optional[str] = None, alpha: float = 0.3, residual=None, need_dx: bool = True,
                    need_dw: bool = True, need_db: bool = True):
    """Gradients of linear(x, w, bias) from dy, the gradient in front of the layer's own activation:
        dx = (dy w) * act'(z) + residual,   dw = dy^T x (fp32),   db = sum of dy's rows (fp32)
    z / activation belong to the layer in FRONT, whose output is x = act(z) - dx is then the gradient of its pre-activation and the next
    call's dy; None: dx is the gradient of x.  residual [..., inputs]: another gradient of the same tensor (a skip connection's).
    Returns (dx, dw, db), None for what is not wanted.  An activation with no product behind it: activation_backward."""
    what = "linear_backward"
    dt, act, w_ld = _linear_args(what, x, w, activation, alpha)
    n, k = w.shape
    if x.shape[-1] != k:
        _fail(what, f"x has {x.shape[-1]} inputs, w {k}")
    _like(what, "dy", dy, x, x.shape[:-1] + (n,))
    m, x_ld = _rows(what, "x", x)
    _m, dy_ld = _rows(what, "dy", dy)
    if act != 0 and z is None and need_dx:
        _fail(what, f"activation {activation!r} needs its input z")
    z_ld = r_ld = 0
    if z is not None:
        _like(what, "z", z, x, x.shape)
        _m, z_ld = _rows(what, "z", z)
    if residual is not None:
        _like(what, "residual", residual, x, x.shape)
        _m, r_ld = _rows(what, "residual", residual)
    _no_grad(what, dy, x, w, z, residual)
    di = _gpu(what, x)
    dev, lib = x.device, _ffi.lib()
    dx = dw = db = None
    if need_dx:
        dx = torch.empty_like(x, memory_format=torch.contiguous_format)
        a = LinearArgs(m, k, n, dt, act, alpha, _ptr(dy), dy_ld, _ptr(w), w_ld, None, _ptr(residual), r_ld, _ptr(z) if act != 0 else None, z_ld, _ptr(dx), k)
        ws = _bytes(lib.seg_linear_workspace_bytes(a, _ffi.LINEAR_BWD_DATA), dev)
        a.workspace = _ptr(ws)
        _launch(di, "seg_linear_bwd_data", a)
    if need_dw or need_db:
        dw = torch.empty((n, k), dtype=torch.float32, device=dev) if need_dw else None
        db = torch.empty((n,), dtype=torch.float32, device=dev) if need_db else None
        a = LinearArgs(m, n, k, dt, 0, 0.0, _ptr(x), x_ld, None, 0, None, None, 0, None, 0, None, 0, _ptr(dy), dy_ld, _ptr(dw), k, _ptr(db))
        ws = _bytes(lib.seg_linear_workspace_bytes(a, _ffi.LINEAR_BWD_WEIGHT), dev)
        a.workspace = _ptr(ws)
        _launch(di, "seg_linear_bwd_weight", a)
    return dx, dw, db


def activation_backward(dy, z, activation: str, alpha: float = 0.3):
    """dy * act'(z), z the activation's input."""
    what = "activation_backward"
    dt, act = _dtype(what, z), _act(what, activation)
    if z.dim() < 1 or z.shape[-1] < 1:
        _fail(what, f"z of shape {tuple(z.shape)} has no channels")
    _like(what, "dy", dy, z, z.shape)
    rows, z_ld = _rows(what, "z", z)
    _r, dy_ld = _rows(what, "dy", dy)
    _no_grad(what, dy, z)
    di = _gpu(what, z)
    c = z.shape[-1]
    dx = torch.empty_like(z, memory_format=torch.contiguous_format)
    _launch(di, "seg_linear_act_bwd", _ptr(dy), dy_ld, _ptr(z), z_ld, _ptr(dx), c, rows, c, dt, act, alpha)
    return dx


# --------------------------------------------------------------------------------------------------------- causal convolution
def _lengths(what, lengths, ref, B):
    return _param(what, "lengths", lengths, ref, (B,), torch.int32)


def _conv_common(what, x, w, bias, activation, state, rank):
    dt = _dtype(what, x)
    if x.dim() != rank or x.shape[-1] < 1:
        _fail(what, f"x has shape {tuple(x.shape)}, expected " + ("[B, L, D]" if rank == 3 else "[B, D]"))
    if not isinstance(w, torch.Tensor) or w.dim() != 2:
        _fail(what, "w must be [K, D]")
    K, d, B = w.shape[0], x.shape[-1], x.shape[0]
    _extents(what, x)
    if not 1 <= K <= MAX_TAPS:
        _fail(what, f"{K} taps (1 .. {MAX_TAPS})")
    if activation not in (None, "none", "linear", "silu"):
        _fail(what, f"activation {activation!r} (None or 'silu')")
    if d > 1 and x.stride(-1) != 1:
        _fail(what, f"x: the channel axis must be contiguous (strides {x.stride()})")
    _param(what, "w", w, x, (K, d))
    _param(what, "bias", bias, x, (d,))
    _param(what, "state", state, x, (B, K - 1, d), x.dtype)
    return dt, SEQ_ACT[activation], B, d, K


def causal_conv(x, w, bias=None, activation: Optional[str] = None, state=None, lengths=None):
    """Per channel: v[t] = bias + sum_k w[k] xx[t + k] over xx = [state; x], y = act(v).  x [B, L, D], w fp32 [K, D] (K <= 8), bias fp32
    [D], activation None or "silu", state [B, K - 1, D] (None: zeros), lengths int32 [B]: rows behind a length are not read, their y is 0.
    At most 65535 sequences (fewer by a power of two from 2^22 rows each on) of 2^30 rows and 2^30 channels in one call.
    Returns (y, the state that goes on: the last K - 1 rows in front of each length)."""
    what = "causal_conv"
    dt, act, B, d, K = _conv_common(what, x, w, bias, activation, state, 3)
    L = x.shape[1]
    _spaced(what, "x", x)
    _lengths(what, lengths, x, B)
    _no_grad(what, x, w, bias, state)
    di = _gpu(what, x)
    y = torch.empty((B, L, d), dtype=x.dtype, device=x.device)
    new = torch.empty((B, K - 1, d), dtype=x.dtype, device=x.device)
    a = CausalConvArgs(B, L, d, K, dt, act, _ptr(x), x.stride(0), x.stride(1), _ptr(w), _ptr(bias), _ptr(state), _ptr(lengths), _ptr(y), L * d, d, _ptr(new))
    _launch(di, "seg_causal_conv_fwd", a)
    return y, new


def causal_conv_backward(dy, x, w, bias=None, activation: Optional[str] = None, state=None, lengths=None, dstate=None):
    """(dx, dw, db, gradient of state) of causal_conv from dy and dstate, the gradient of the state that went on (None: zeros).  db is
    None without a bias, the last one None without a state.  Rows behind a length: dy is not read, dx is 0."""
    what = "causal_conv_backward"
    dt, act, B, d, K = _conv_common(what, x, w, bias, activation, state, 3)
    L = x.shape[1]
    _like(what, "dy", dy, x, x.shape)
    _spaced(what, "x", x)
    _spaced(what, "dy", dy)
    _lengths(what, lengths, x, B)
    _param(what, "dstate", dstate, x, (B, K - 1, d), x.dtype)
    _no_grad(what, dy, x, w, bias, state, dstate)
    di = _gpu(what, x)
    dev = x.device
    dx = torch.empty((B, L, d), dtype=x.dtype, device=dev)
    par = torch.empty((K + 1, d), dtype=torch.float32, device=dev)          # (one buffer: the sums over the blocks take one launch)
    dw, db = par[:K], par[K] if bias is not None else None
    dst = torch.empty((B, K - 1, d), dtype=x.dtype, device=dev) if state is not None else None
    a = CausalConvArgs(B, L, d, K, dt, act, _ptr(x), x.stride(0), x.stride(1), _ptr(w), _ptr(bias), _ptr(state), _ptr(lengths), None, 0, 0, None,
                       _ptr(dy), dy.stride(0), dy.stride(1), _ptr(dstate), _ptr(dx), L * d, d, _ptr(dw), _ptr(db), _ptr(dst))
    ws = _bytes(_ffi.lib().seg_causal_conv_bwd_workspace_bytes(a), dev)
    a.workspace = _ptr(ws)
    _launch(di, "seg_causal_conv_bwd", a)
    return dx, dw, db, dst


def _new_state(what, state, new_state):
    if new_state is None:
        return state
    _param(what, "new_state", new_state, state, state.shape, state.dtype)
    a, b = state.data_ptr(), new_state.data_ptr()
    if a != b and abs(a - b) < state.numel() * state.element_size():
        _fail(what, "new_state overlaps state: give the same tensor or another one")
    return new_state


def causal_conv_step(x, state, w, bias=None, activation: Optional[str] = None, new_state=None):
    """One more row per sequence: x [B, D] -> y [B, D].  state [B, K - 1, D] is updated in place, or written to new_state."""
    what = "causal_conv_step"
    if state is None:
        _fail(what, "state is needed")
    dt, act, B, d, K = _conv_common(what, x, w, bias, activation, state, 2)
    new = _new_state(what, state, new_state)
    if B > 1 and x.stride(0) < d:
        _fail(what, f"x: rows overlap (strides {x.stride()}); call .contiguous()")
    _no_grad(what, x, w, bias, state, new_state)
    di = _gpu(what, x)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    a = CausalConvArgs(B, 1, d, K, dt, act, _ptr(x), x.stride(0), d, _ptr(w), _ptr(bias), _ptr(state), None, _ptr(y), d, d, _ptr(new))
    _launch(di, "seg_causal_conv_step", a)
    return y


# ------------------------------------------------------------------------------------------------------- selective state space
class ScanGrads(NamedTuple):
    """Gradients of selective_scan (None for an operand that was not given); dstate: of the state in front of the first row."""
    du: torch.Tensor
    ddt: torch.Tensor
    dA: torch.Tensor
    dB: torch.Tensor
    dC: torch.Tensor
    dD: Optional[torch.Tensor]
    dz: Optional[torch.Tensor]
    ddt_bias: Optional[torch.Tensor]
    dstate: torch.Tensor


def _scan_common(what, u, dt, A, B, C_, D, z, dt_bias, rank):
    """Checks what every scan call has; (type code, batch, channels, states, [strides of u, dt, z, B, C])."""
    dtc = _dtype(what, u)
    shape = u.shape
    if len(shape) != rank or shape[-1] < 1:
        _fail(what, f"u has shape {tuple(shape)}, expected " + ("[B, L, D]" if rank == 3 else "[B, D]"))
    if not isinstance(A, torch.Tensor) or A.dim() != 2:
        _fail(what, "A must be [D, S]")
    d, S, nb = shape[-1], A.shape[1], shape[0]
    _extents(what, u)
    if not 1 <= S <= MAX_STATES:
        _fail(what, f"{S} states per channel (1 .. {MAX_STATES})")
    _param(what, "A", A, u, (d, S))
    bc = (nb, shape[1], S) if rank == 3 else (nb, S)
    strides = []
    for n, t, sh in (("u", u, shape), ("dt", dt, shape), ("z", z, shape), ("B", B, bc), ("C", C_, bc)):
        if t is None and n == "z":
            strides.append((0,) * rank)
            continue
        if t is not u:
            _like(what, n, t, u, sh)
        st = t.stride()
        if t is u and st[-1] != 1 and d > 1:
            _fail(what, f"u: the channel axis must be contiguous (strides {st})")
        if sh[-2] > 1 and st[-2] < sh[-1]:
            _fail(what, f"{n}: rows overlap (strides {st}); call .contiguous()")
        strides.append(st)
    _param(what, "D", D, u, (d,))
    _param(what, "dt_bias", dt_bias, u, (d,))
    if A.data_ptr() % 16:
        _fail(what, "A must be 16-byte aligned")
    return dtc, nb, d, S, strides


def _aligned(what, **ts):
    for n, t in ts.items():
        if t is not None and t.data_ptr() % 16:
            _fail(what, f"{n} must be 16-byte aligned")


def _scan_args(B, L, d, S, dtc, softplus, u, dt, z, Bm, Cm, A, D, dt_bias, state, lengths, st):
    (ub, ul, _), (tb, tl, _), (zb, zl, _), (bb, bl, _), (cb, cl, _) = st
    return ScanArgs(B, L, d, S, dtc, 1 if softplus else 0, u.data_ptr(), ub, ul, dt.data_ptr(), tb, tl, _ptr(z), zb, zl, Bm.data_ptr(), bb, bl,
                    Cm.data_ptr(), cb, cl, A.data_ptr(), _ptr(D), _ptr(dt_bias), _ptr(state), _ptr(lengths))


def selective_scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus: bool = True, state=None, lengths=None, training: bool = False):
    """h[t] = exp(delta[t] A) h[t-1] + delta[t] B[t] u[t],  y[t] = (C[t] . h[t] + D u[t]) * silu(z[t]),  delta = softplus(dt + dt_bias).

    u, dt, z [B, L, D], B, C [B, L, S] of one type; A fp32 [D, S] (negative rates), D, dt_bias fp32 [D]; state fp32 [B, D, S] in front of
    the first row (None: zeros); lengths int32 [B]: rows behind a length are not read, their y is 0 and the state stays what it was.
    At most 65535 sequences of 2^30 rows and 2^30 channels in one call.
    Returns (y, last state), with training=True (y, last state, saved) - `saved` is what selective_scan_backward needs."""
    what = "selective_scan"
    dtc, nb, d, S, st = _scan_common(what, u, dt, A, B, C, D, z, dt_bias, 3)
    L = u.shape[1]
    _param(what, "state", state, u, (nb, d, S))
    _aligned(what, state=state)
    _lengths(what, lengths, u, nb)
    _no_grad(what, u, dt, A, B, C, D, z, dt_bias, state)
    di = _gpu(what, u)
    dev, lib = u.device, _ffi.lib()
    y = torch.empty((nb, L, d), dtype=u.dtype, device=dev)
    last = torch.empty((nb, d, S), dtype=torch.float32, device=dev)
    a = _scan_args(nb, L, d, S, dtc, softplus, u, dt, z, B, C, A, D, dt_bias, state, lengths, st)
    a.y, a.y_bs, a.y_ld, a.state_out = _ptr(y), L * d, d, _ptr(last)
    saved = None
    if training:
        saved = torch.empty(lib.seg_selective_scan_saved_bytes(a) // 4, dtype=torch.float32, device=dev)
        a.saved = _ptr(saved)
    ws = _bytes(lib.seg_selective_scan_fwd_workspace_bytes(a), dev)
    a.workspace = _ptr(ws)
    _launch(di, "seg_selective_scan_fwd", a)
    return (y, last, saved) if training else (y, last)


def selective_scan_backward(dy, u, dt, A, B, C, saved, D=None, z=None, dt_bias=None, softplus: bool = True, lengths=None, dstate=None) -> ScanGrads:
    """All gradients of selective_scan(..., training=True) from dy and dstate, the gradient of the last state (None: zeros); the other
    operands as in the forward call.  Rows behind a length: dy is not read, their gradients are 0."""
    what = "selective_scan_backward"
    dtc, nb, d, S, st = _scan_common(what, u, dt, A, B, C, D, z, dt_bias, 3)
    L = u.shape[1]
    _like(what, "dy", dy, u, u.shape)
    _spaced(what, "dy", dy)
    _param(what, "dstate", dstate, u, (nb, d, S))
    _aligned(what, dstate=dstate)
    _lengths(what, lengths, u, nb)
    if saved is None:
        _fail(what, "saved is needed (selective_scan(..., training=True) returns it)")
    lib = _ffi.lib()
    a = _scan_args(nb, L, d, S, dtc, softplus, u, dt, z, B, C, A, D, dt_bias, None, lengths, st)
    _param(what, "saved", saved, u, (lib.seg_selective_scan_saved_bytes(a) // 4,))
    _no_grad(what, dy, u, dt, A, B, C, D, z, dt_bias, dstate, saved)
    di = _gpu(what, u)
    dev = u.device

    def rows(c):
        return torch.empty((nb, L, c), dtype=u.dtype, device=dev)

    def flat(*shape):
        return torch.empty(shape, dtype=torch.float32, device=dev)

    par = flat(2, d)
    g = ScanGrads(rows(d), rows(d), flat(d, S), rows(S), rows(S), None if D is None else par[0], None if z is None else rows(d),
                  None if dt_bias is None else par[1], flat(nb, d, S))
    a.saved, a.dy, a.dy_bs, a.dy_ld, a.dstate_out = _ptr(saved), _ptr(dy), dy.stride(0), dy.stride(1), _ptr(dstate)
    for n, t, c in (("du", g.du, d), ("ddt", g.ddt, d), ("dz", g.dz, d), ("dBm", g.dB, S), ("dCm", g.dC, S)):
        if t is not None:
            setattr(a, n, t.data_ptr())
            setattr(a, n + "_bs", L * c)
            setattr(a, n + "_ld", c)
    a.dA, a.dD, a.ddt_bias, a.dstate = _ptr(g.dA), _ptr(g.dD), _ptr(g.ddt_bias), _ptr(g.dstate)
    ws = _bytes(lib.seg_selective_scan_bwd_workspace_bytes(a), dev)
    a.workspace = _ptr(ws)
    _launch(di, "seg_selective_scan_bwd", a)
    return g


def selective_scan_step(u, dt, A, B, C, state, D=None, z=None, dt_bias=None, softplus: bool = True, new_state=None):
    """One more row per sequence: u, dt, z [B, D], B, C [B, S] -> y [B, D].  state fp32 [B, D, S] is updated in place, or written to
    new_state."""
    what = "selective_scan_step"
    dtc, nb, d, S, st = _scan_common(what, u, dt, A, B, C, D, z, dt_bias, 2)
    if state is None:
        _fail(what, "state is needed")
    _param(what, "state", state, u, (nb, d, S))
    new = _new_state(what, state, new_state)
    if state.data_ptr() % 16 or new.data_ptr() % 16:
        _fail(what, "state must be 16-byte aligned")
    _no_grad(what, u, dt, A, B, C, D, z, dt_bias, state, new_state)
    di = _gpu(what, u)
    y = torch.empty_like(u, memory_format=torch.contiguous_format)
    a = ScanArgs(nb, 1, d, S, dtc, 1 if softplus else 0, u.data_ptr(), st[0][0], 0, dt.data_ptr(), st[1][0], 0, _ptr(z), st[2][0], 0, B.data_ptr(), st[3][0], 0,
                 C.data_ptr(), st[4][0], 0, A.data_ptr(), _ptr(D), _ptr(dt_bias), state.data_ptr(), None, y.data_ptr(), d, d, new.data_ptr())
    _launch(di, "seg_selective_scan_step", a)
    return y
