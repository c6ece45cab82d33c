"""The sequence operators' definitions in 64 bits (torch on the CPU), with the error bound of a 32-bit evaluation beside each value.

Bounds.  One rounding is off by at most U32 = 2^-24 of the value, half a step; an output element rounds once more to its type (half a
step: finfo.eps / 2).  A sum of n terms evaluated in any order in 32 bits is off by at most n U32 sum|terms|; `scale` below is the sum
of the terms' absolute values (for a recurrence: the recurrence of the absolute values) and `n` counts the roundings on the longest
chain, generously.  Hardware exponentials and reciprocals count 4 roundings each."""
import torch
import torch.nn.functional as F

U32 = 2.0 ** -24
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
# half of the smallest step: what a value next to zero may lose when it is stored
FLOOR = {torch.float16: 2.0 ** -25, torch.bfloat16: 0.0, torch.float32: 0.0}


def assert_close(got, ref, scale, n, what=""):
    t = got.dtype
    got, ref = got.detach().double().cpu(), ref.detach().double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    tol = HALF[t] * (ref.abs() + n * U32 * scale) + n * U32 * scale + FLOOR[t] + 1e-37
    bad = (got - ref).abs() - tol
    assert not torch.isnan(got).any(), (what, "NaN")
    assert float(bad.max() if bad.numel() else -1.0) <= 0, (what, float(((got - ref).abs() / tol).max()), "times the bound")


def act(v, name, alpha=0.3):
    return {"relu": torch.relu, "leaky_relu": lambda t: F.leaky_relu(t, alpha), "sigmoid": torch.sigmoid, "silu": F.silu, "gelu": F.gelu,
            None: lambda t: t, "linear": lambda t: t}[name](v)


def act_slope(v, name, alpha=0.3):
    v = v.detach().clone().requires_grad_()
    with torch.enable_grad():
        y = act(v, name, alpha)
        return torch.autograd.grad(y.sum(), v)[0] if y.requires_grad else torch.ones_like(v)


def conv(x, w, bias, state, lengths, silu):
    """(y, state out) of the causal convolution, loops over the batch; every operand float64."""
    K, L = w.shape[0], x.shape[1]
    ys, states = [], []
    for b in range(x.shape[0]):
        m = L if lengths is None else min(max(int(lengths[b]), 0), L)
        st = torch.zeros(K - 1, x.shape[2], dtype=torch.float64) if state is None else state[b]
        xx = torch.cat([st, x[b, :m]])
        v = sum((xx[k:k + m] * w[k] for k in range(K)), torch.zeros(m, x.shape[2], dtype=torch.float64))
        if bias is not None:
            v = v + bias
        ys.append(torch.cat([F.silu(v) if silu else v, torch.zeros(L - m, x.shape[2], dtype=torch.float64)]))
        states.append(xx[m:])
    return torch.stack(ys), torch.stack(states)


def scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, state=None, lengths=None):
    """(y, last state) of the selective scan, one row after the other; every operand float64."""
    nb, L, d = u.shape
    h = torch.zeros(nb, d, A.shape[1], dtype=torch.float64) if state is None else state
    ys = []
    for t in range(L):
        v = dt[:, t] if dt_bias is None else dt[:, t] + dt_bias
        delta = torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs())) if softplus else v
        nxt = torch.exp(delta[..., None] * A) * h + (delta * u[:, t])[..., None] * B[:, t, None]
        y = (nxt * C[:, t, None]).sum(-1)
        if D is not None:
            y = y + D * u[:, t]
        if z is not None:
            y = y * F.silu(z[:, t])
        if lengths is not None:
            on = (lengths > t)[:, None]
            y, nxt = torch.where(on, y, torch.zeros_like(y)), torch.where(on[..., None], nxt, h)
        h = nxt
        ys.append(y)
    return (torch.stack(ys, 1) if ys else torch.zeros_like(u)), h


def scan_scales(u, dt, A, B, C, D, z, dt_bias, softplus, state, lengths, dy, dstate):
    """The scan's outputs and gradients with every term replaced by its absolute value: the scales of the error bounds.  dt_bias etc. may be
    None; lengths must be given (int tensor)."""
    nb, L, d = u.shape
    S = A.shape[1]
    on = (torch.arange(L)[None] < lengths[:, None])[..., None].double()
    v = dt if dt_bias is None else dt + dt_bias
    delta = (torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs())) if softplus else v) * on
    dm = delta.abs()
    um, Bm, Cm = (u.abs() * on), (B.abs() * on), (C.abs() * on)
    gate = (F.silu(z).abs() + z.abs() * 0.25 if z is not None else torch.ones_like(u)) * on
    gate_slope = (1.2 * torch.ones_like(u)) * on
    a = torch.exp(delta[..., None] * A)
    h = torch.zeros(nb, d, S, dtype=torch.float64) if state is None else state.abs()
    hs, prev = [], []
    for t in range(L):
        prev.append(h)
        h = a[:, t] * h + (dm * um)[:, t, :, None] * Bm[:, t, None]
        hs.append(h)
    hs, prev = torch.stack(hs, 1), torch.stack(prev, 1)
    pre = (hs * Cm[:, :, None]).sum(-1) + (0 if D is None else D.abs() * um)
    dp = dy.abs() * gate
    q = torch.zeros_like(h) if dstate is None else dstate.abs()
    out = {"state": h, "y": pre * gate, "dz": dy.abs() * on * pre * gate_slope}
    gs, ga = [None] * L, [None] * L
    for t in reversed(range(L)):
        gs[t] = q + dp[:, t, :, None] * Cm[:, t, None]
        ga[t] = q = gs[t] * a[:, t]
    gs, ga = torch.stack(gs, 1), torch.stack(ga, 1)
    out["dstate"] = q
    dec = ga * prev
    out["dA"] = (dec * dm[..., None]).sum((0, 1))
    out["dB"] = (gs * (dm * um)[..., None]).sum(2)
    out["dC"] = (dp[..., None] * hs).sum(2)
    sB = (gs * Bm[:, :, None]).sum(-1)
    out["du"] = (0 if D is None else D.abs() * dp) + sB * dm
    out["ddt"] = ((dec * A.abs()).sum(-1) + sB * um) * on
    out["ddt_bias"] = out["ddt"].sum((0, 1))
    out["dD"] = (dp * um).sum((0, 1))
    # roundings of one row's step: the exponent's own (its argument's error times the argument), two operations, the addition
    out["arg"] = float((dm[..., None] * A.abs()).max()) if L else 0.0
    return out
