"""The sequence operators of the framework - layer normalisation, the matrix product with its epilogue, the short causal convolution
and the selective state space scan - as cases that can be timed and compared.

`own` chooses what `run` calls: False - the operators' plain forms, elementary torch operations in 32 bits, rounded once at the end;
True - the framework's entry points, as a user's program calls them.  Both take the same state from `prepare`.  `exact` computes the
same outputs from the definitions in 64 bits (gradients by differentiating the definition)."""
import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the bottleneck of the depth-5 2D encoders (16 x 16 pixels, 16 images) as 4096 tokens of 1024 channels, inference
        dict(name="layer_norm/bottleneck", op="layer_norm", rows=4096, C=1024, stats=False, dtype="f16"),
        # the full-resolution level of the same models (16 images of 256 x 256, 64 channels), training: few channels, very many rows
        dict(name="layer_norm/full_resolution", op="layer_norm_backward", rows=1048576, C=64, dtype="f16"),
        # odd sizes in 32 bits, training: rows that no vector access fits
        dict(name="layer_norm/odd", op="layer_norm_backward", rows=5003, C=1111, dtype="f32"),
        # the up projection of four signals that are processed sample by sample: latency and the weights' bytes count
        dict(name="linear/token", op="linear", M=4, N=4096, K=1024, act="silu", bias=True, residual=False, keep=False, dtype="bf16"),
        # the first product of a two-layer perceptron over 16384 tokens in training: GELU, the pre-activation kept
        dict(name="linear/expand", op="linear", M=16384, N=4096, K=1024, act="gelu", bias=True, residual=False, keep=True, dtype="f16"),
        # the backward pass of its second product: data gradient through the GELU in front, weight and bias gradient
        dict(name="linear/contract_backward", op="linear_backward", M=16384, N=1024, K=4096, act="gelu", residual=False, dtype="bf16"),
        # sizes that no tile and no 16-byte access fits, with a residual
        dict(name="linear/ragged", op="linear", M=1111, N=333, K=700, act="relu", bias=True, residual=True, keep=False, dtype="f16"),
        # the causal convolution in front of a scan: eight prompts of up to 4096 samples, half a batch of them shorter
        dict(name="causal_conv/prompt", op="causal_conv", B=8, L=4096, D=2048, K=4, ragged=True, dtype="bf16"),
        # its backward pass in training on the 1D models' 1024-sample windows
        dict(name="causal_conv/train", op="causal_conv_backward", B=16, L=1024, D=512, K=4, ragged=False, dtype="f16"),
        # the scan over eight prompts of up to 2048 samples, shorter ones among them: outputs and the states that go on
        dict(name="selective_scan/prompt", op="selective_scan", B=8, L=2048, D=2048, S=16, ragged=True, dtype="bf16"),
        # a training step of the scan (forward with what the backward pass needs, and all gradients) on 1024-sample windows
        dict(name="selective_scan/train", op="selective_scan_train", B=8, L=1024, D=1024, S=16, ragged=False, dtype="f16"),
        # one more sample for each of 64 running signals
        dict(name="selective_scan/token", op="selective_scan_step", B=64, D=2048, S=16, dtype="f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer_norm", "layer_norm_backward", "linear", "linear", "linear_backward", "causal_conv", "causal_conv_backward", "causal_conv_step",
                     "selective_scan", "selective_scan_train", "selective_scan_step"])
    c = dict(op=op, dtype=rng.choice(["f16", "f16", "bf16", "bf16", "f32"]))
    if op.startswith("layer_norm"):
        c["C"] = _log(rng, 8, 8192)
        if rng.random() < 0.6:
            c["C"] = max(8, c["C"] // 8 * 8)
        c["rows"] = _log(rng, 1, min(1048576, (1 << 26) // c["C"]))
        if op == "layer_norm":
            c["stats"] = rng.random() < 0.5
    elif op.startswith("linear"):
        c["M"], c["N"], c["K"] = _log(rng, 1, 16384), _log(rng, 8, 4096), _log(rng, 8, 4096)
        if rng.random() < 0.6:
            c["N"], c["K"] = max(8, c["N"] // 8 * 8), max(8, c["K"] // 8 * 8)
        if c["dtype"] == "f32":
            c["M"] = max(1, min(c["M"], (1 << 31) // (c["N"] * c["K"])))
        c["act"] = rng.choice(["linear", "relu", "leaky_relu", "sigmoid", "silu", "gelu"])
        c["residual"] = rng.random() < 0.5
        if op == "linear":
            c["bias"], c["keep"] = rng.random() < 0.8, rng.random() < 0.4
    elif op.endswith("_step"):
        c["B"], c["D"] = _log(rng, 1, 512), _log(rng, 8, 4096)
        if op == "causal_conv_step":
            c["K"] = rng.randint(2, 5)
        else:
            c["S"] = rng.choice([4, 8, 12, 16, 16, 32, 64])
    else:
        c["B"], c["D"], c["ragged"] = _log(rng, 1, 16), _log(rng, 8, 4096), rng.random() < 0.5
        if rng.random() < 0.7:
            c["D"] = max(8, c["D"] // 8 * 8)
        if op.startswith("causal_conv"):
            c["K"] = rng.randint(2, 5)
            c["L"] = _log(rng, 1, min(16384, (1 << 26) // (c["B"] * c["D"])))
        else:
            c["S"] = rng.choice([4, 8, 12, 16, 16, 32, 64])
            most = (1 << 27 if op == "selective_scan_train" else 1 << 29) // (c["B"] * c["D"] * c["S"])
            c["L"] = _log(rng, 1, max(1, min(8192, most)))
    return c


def work(case):
    op, e = case["op"], SIZE[case["dtype"]]
    if op.startswith("layer_norm"):
        n, C = case["rows"] * case["C"], case["C"]
        if op == "layer_norm":
            return {"bytes": 2 * n * e + 8 * C + 8 * case["rows"] * bool(case["stats"]), "flops": 8 * n}
        return {"bytes": 3 * n * e + 12 * C + 8 * case["rows"], "flops": 14 * n}
    if op.startswith("linear"):
        M, N, K = case["M"], case["N"], case["K"]
        if op == "linear":
            outs = 1 + bool(case["residual"]) + bool(case["keep"])
            return {"bytes": (M * K + N * K + outs * M * N) * e + 4 * N * bool(case["bias"]), "flops": 2 * M * N * K}
        ios = 2 + (case["act"] != "linear") + bool(case["residual"])
        return {"bytes": (M * N + N * K + ios * M * K) * e + 4 * N * K + 4 * N, "flops": 4 * M * N * K}
    B, D = case["B"], case["D"]
    if op.startswith("causal_conv"):
        K = case["K"]
        if op == "causal_conv_step":
            return {"bytes": (2 * B * D + 2 * B * (K - 1) * D) * e + 4 * (K + 1) * D, "flops": 2 * B * D * (K + 2)}
        n, st = B * case["L"] * D, B * (K - 1) * D
        if op == "causal_conv":
            return {"bytes": (2 * n + 2 * st) * e + 4 * (K + 1) * D, "flops": 2 * n * (K + 2)}
        return {"bytes": (3 * n + 3 * st) * e + 8 * (K + 1) * D, "flops": 2 * n * (3 * K + 6)}
    S = case["S"]
    if op == "selective_scan_step":
        return {"bytes": 8 * B * D * S + (4 * B * D + 2 * B * S) * e + 4 * D * (S + 2), "flops": 6 * B * D * S}
    L = case["L"]
    n, bc, par, st = B * L * D, B * L * S, D * (S + 2), B * D * S
    if op == "selective_scan":
        return {"bytes": (4 * n + 2 * bc) * e + 4 * par + 8 * st, "flops": 6 * n * S}
    # training: u, dt, z, B, C and dy once, y and the gradients once
    return {"bytes": (8 * n + 4 * bc) * e + 8 * par + 16 * st, "flops": 24 * n * S}


# ----------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t, op = DTYPES[case["dtype"]], case["op"]

    def normal(*shape, scale=1.0, dtype=t):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def uniform(lo, hi, *shape):
        return torch.rand(*shape, generator=g, device="cuda") * (hi - lo) + lo

    s = {"op": op}
    if op.startswith("layer_norm"):
        rows, C = case["rows"], case["C"]
        # features with an offset of their own per row, the way they leave a ReLU or a residual stream
        s["x"] = (torch.randn(rows, C, generator=g, device="cuda") * uniform(0.3, 3.0, rows, 1) + uniform(-1.0, 1.0, rows, 1)).to(t)
        s["gamma"], s["beta"], s["eps"], s["stats"] = uniform(0.5, 1.5, C), uniform(-0.5, 0.5, C), 1e-3, case.get("stats", False)
        if op == "layer_norm_backward":
            s["dy"] = normal(rows, C)
            x = s["x"].double()
            s["mean"] = x.mean(1).float()
            s["rstd"] = (x.var(1, unbiased=False) + s["eps"]).rsqrt().float()
        return s
    if op.startswith("linear"):
        M, N, K = case["M"], case["N"], case["K"]
        s["act"], s["alpha"] = case["act"], 0.3
        s["x"], s["w"] = normal(M, K), normal(N, K, scale=K ** -0.5)
        if op == "linear":
            s["bias"] = normal(N, scale=0.1, dtype=torch.float32) if case["bias"] else None
            s["residual"] = normal(M, N) if case["residual"] else None
            s["keep"] = case["keep"]
        else:
            s["dy"] = normal(M, N)
            s["z"] = normal(M, K) if case["act"] != "linear" else None
            s["residual"] = normal(M, K) if case["residual"] else None
        return s
    B, D = case["B"], case["D"]
    if case.get("ragged"):
        # half of the batch whole, the others of any length, an empty one now and then
        r = np.random.default_rng(int(seed))
        n = [case["L"] if r.random() < 0.5 else int(r.integers(0, case["L"] + 1)) for _ in range(B)]
        s["lengths"] = torch.tensor(n, dtype=torch.int32, device="cuda")
    else:
        s["lengths"] = None
    if op.startswith("causal_conv"):
        K = case["K"]
        s["w"], s["bias"] = uniform(-0.6, 0.6, K, D), uniform(-0.3, 0.3, D)
        s["state"] = normal(B, K - 1, D)
        if op == "causal_conv_step":
            s["x"] = normal(B, D)
            return s
        s["x"] = normal(B, case["L"], D)
        if op == "causal_conv_backward":
            s["dy"], s["dstate"] = normal(B, case["L"], D), normal(B, K - 1, D)
        return s
    S = case["S"]
    # the usual start of such layers: rates 1 .. S with a spread per channel, steps between 1e-3 and 1e-1
    s["A"] = -(torch.arange(1, S + 1, device="cuda", dtype=torch.float32)[None, :] * uniform(0.7, 1.4, D, 1))
    step = torch.exp(uniform(math.log(1e-3), math.log(1e-1), D))
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))
    s["D"] = uniform(0.5, 1.5, D)
    s["state"] = normal(B, D, S, scale=0.5, dtype=torch.float32)
    lead = (B,) if op == "selective_scan_step" else (B, case["L"])
    s["u"], s["z"], s["dt"] = normal(*lead, D), normal(*lead, D), normal(*lead, D, scale=0.5)
    # B and C are columns of one projection's output, next to what the step is made from
    low = max(8, D // 16 // 8 * 8)
    s["proj"] = normal(*lead, low + 2 * S)
    s["Bm"], s["Cm"] = s["proj"][..., low:low + S], s["proj"][..., low + S:]
    if op == "selective_scan_train":
        s["dy"], s["dstate"] = normal(B, case["L"], D), normal(B, D, S, scale=0.1, dtype=torch.float32)
    return s


# -------------------------------------------------------------------------------------------------------------- plain forms
def _act(v, name, alpha):
    if name == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if name == "leaky_relu":
        return torch.where(v > 0, v, v * alpha)
    if name == "sigmoid":
        return 1 / (1 + torch.exp(-v))
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))
    return v


def _act_slope(v, name, alpha):
    if name == "relu":
        return (v > 0).to(v.dtype)
    if name == "leaky_relu":
        return torch.where(v > 0, torch.ones_like(v), torch.full_like(v, alpha))
    if name == "sigmoid":
        p = 1 / (1 + torch.exp(-v))
        return p * (1 - p)
    if name == "silu":
        p = 1 / (1 + torch.exp(-v))
        return p * (1 + v * (1 - p))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(v * 0.5 ** 0.5)) + v * torch.exp(-0.5 * v * v) * (2 * math.pi) ** -0.5
    return torch.ones_like(v)


def _live(s, L):
    """[B, L, 1] truth values: the positions in front of each sequence's length (None: all of them)."""
    if s["lengths"] is None:
        return None
    return (torch.arange(L, device="cuda")[None, :] < s["lengths"].clamp(0, L)[:, None])[:, :, None]


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def _recurrence(a, b):
    """h[t] = a[t] h[t-1] + b[t] along dimension 1 with h[-1] = 0, by doubling: after round n every h[t] holds its last 2^n terms."""
    n = 1
    while n < a.shape[1]:
        b = torch.cat([b[:, :n], b[:, n:] + a[:, n:] * b[:, :-n]], 1)
        a = torch.cat([a[:, :n], a[:, n:] * a[:, :-n]], 1)
        n *= 2
    return b


def _plain_layer_norm(s):
    t, x = s["x"].dtype, s["x"].float()
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + s["eps"])
    y = (d * rstd * s["gamma"] + s["beta"]).to(t)
    return {"y": y, "mean": mean[:, 0], "rstd": rstd[:, 0]} if s["stats"] else {"y": y}


def _plain_layer_norm_backward(s):
    t, x, dy = s["x"].dtype, s["x"].float(), s["dy"].float()
    xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * s["gamma"]
    dx = (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True)) * s["rstd"][:, None]
    return {"dx": dx.to(t), "dgamma": (dy * xhat).sum(0), "dbeta": dy.sum(0)}


def _plain_linear(s):
    t = s["x"].dtype
    z = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"]
    y = _act(z, s["act"], s["alpha"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(t), "z": z.to(t)} if s["keep"] else {"y": y.to(t)}


def _plain_linear_backward(s):
    t, dy = s["x"].dtype, s["dy"].float()
    dx = dy @ s["w"].float()
    if s["z"] is not None:
        dx = dx * _act_slope(s["z"].float(), s["act"], s["alpha"])
    if s["residual"] is not None:
        dx = dx + s["residual"].float()
    return {"dx": dx.to(t), "dw": dy.t() @ s["x"].float(), "db": dy.sum(0)}


def _shifted(x, K):
    """[K, B, L, D] views' stack of x with K - 1 earlier rows in front: row k holds the inputs that tap k sees."""
    L = x.shape[1] - (K - 1)
    return torch.stack([x[:, k:k + L] for k in range(K)])


def _tail(x, lengths, K):
    """The last K - 1 rows in front of each sequence's end, x being [state; inputs]."""
    L = x.shape[1] - (K - 1)
    n = torch.full((x.shape[0],), L, device="cuda") if lengths is None else lengths.clamp(0, L).long()
    at = n[:, None] + torch.arange(K - 1, device="cuda")[None, :]
    return torch.gather(x, 1, at[:, :, None].expand(-1, -1, x.shape[2]))


def _plain_causal_conv(s):
    t, K = s["x"].dtype, s["w"].shape[0]
    x = torch.cat([s["state"], s["x"]], 1)
    v = (_shifted(x.float(), K) * s["w"][:, None, None, :]).sum(0) + s["bias"]
    y, live = _act(v, "silu", 0.0), _live(s, s["x"].shape[1])
    if live is not None:
        y = torch.where(live, y, torch.zeros_like(y))
    return {"y": y.to(t), "state": _tail(x, s["lengths"], K)}


def _plain_causal_conv_backward(s):
    t, (K, D), (B, L) = s["x"].dtype, s["w"].shape, s["x"].shape[:2]
    taps = _shifted(torch.cat([s["state"], s["x"]], 1).float(), K)
    v = (taps * s["w"][:, None, None, :]).sum(0) + s["bias"]
    dv = s["dy"].float() * _act_slope(v, "silu", 0.0)
    live = _live(s, L)
    if live is not None:
        dv = torch.where(live, dv, torch.zeros_like(dv))
    # the gradient of [state; inputs]: tap k of output t read row t + k; the carried state read the last K - 1 rows
    after = _shifted(torch.cat([torch.zeros(B, K - 1, D, device="cuda"), dv, torch.zeros(B, K - 1, D, device="cuda")], 1), K)
    dxx = (after * s["w"].flip(0)[:, None, None, :]).sum(0)
    n = torch.full((B,), L, device="cuda") if s["lengths"] is None else s["lengths"].clamp(0, L).long()
    at = n[:, None] + torch.arange(K - 1, device="cuda")[None, :]
    dxx = dxx.scatter_add(1, at[:, :, None].expand(-1, -1, D), s["dstate"].float())
    return {"dx": dxx[:, K - 1:].to(t), "dw": (taps * dv[None]).sum((1, 2)), "db": dv.sum((0, 1)), "dstate": dxx[:, :K - 1].to(t)}


def _plain_causal_conv_step(s):
    t = s["x"].dtype
    x = torch.cat([s["state"], s["x"][:, None]], 1)
    y = _act((x.float() * s["w"]).sum(1) + s["bias"], "silu", 0.0)
    return {"y": y.to(t), "state": x[:, 1:]}


def _scan_states(s):
    """delta [B, L, D], a and h [B, L, D, S] of the recurrence h[t] = a[t] h[t-1] + delta[t] B[t] u[t]."""
    delta = _softplus(s["dt"].float() + s["dt_bias"])
    live = _live(s, delta.shape[1])
    if live is not None:
        delta = torch.where(live, delta, torch.zeros_like(delta))
    a = torch.exp(delta[..., None] * s["A"])
    b = (delta * s["u"].float())[..., None] * s["Bm"].float()[:, :, None, :]
    b[:, 0] += a[:, 0] * s["state"]
    return delta, a, _recurrence(a, b)


def _plain_selective_scan(s):
    t = s["u"].dtype
    _delta, _a, h = _scan_states(s)
    y = (h * s["Cm"].float()[:, :, None, :]).sum(-1) + s["D"] * s["u"].float()
    y, live = y * _act(s["z"].float(), "silu", 0.0), _live(s, y.shape[1])
    if live is not None:
        y = torch.where(live, y, torch.zeros_like(y))
    return {"y": y.to(t), "state": h[:, -1].contiguous()}


def _plain_selective_scan_train(s):
    t, u, z, A = s["u"].dtype, s["u"].float(), s["z"].float(), s["A"]
    Bm, Cm, live = s["Bm"].float()[:, :, None, :], s["Cm"].float()[:, :, None, :], _live(s, s["u"].shape[1])
    delta, a, h = _scan_states(s)
    before = torch.cat([s["state"][:, None], h[:, :-1]], 1)
    dout = s["dy"].float() if live is None else torch.where(live, s["dy"].float(), torch.zeros_like(u))
    ypre = (h * Cm).sum(-1) + s["D"] * u
    y = ypre * _act(z, "silu", 0.0)
    if live is not None:
        y = torch.where(live, y, torch.zeros_like(y))
    dp = dout * _act(z, "silu", 0.0)
    # g[t] = dp[t] C[t] + a[t+1] g[t+1]: the same recurrence from the end, the last state's gradient added at the last step
    g = dp[..., None] * Cm
    g[:, -1] += s["dstate"]
    g = _recurrence(torch.cat([torch.ones_like(a[:, :1]), a[:, 1:].flip(1)], 1), g.flip(1)).flip(1)
    ga = g * a
    decay = ga * before
    ddt = ((decay * A).sum(-1) + (g * Bm).sum(-1) * u) / (1 + torch.exp(-(s["dt"].float() + s["dt_bias"])))
    if live is not None:
        ddt = torch.where(live, ddt, torch.zeros_like(ddt))
    return {"y": y.to(t), "state": h[:, -1].contiguous(), "du": (s["D"] * dp + (g * Bm).sum(-1) * delta).to(t), "ddt": ddt.to(t),
            "dA": (decay * delta[..., None]).sum((0, 1)), "dB": (g * (delta * u)[..., None]).sum(2).to(t), "dC": (dp[..., None] * h).sum(2).to(t),
            "dD": (dp * u).sum((0, 1)), "dz": (dout * ypre * _act_slope(z, "silu", 0.0)).to(t), "ddt_bias": ddt.sum((0, 1)), "dstate": ga[:, 0].contiguous()}


def _plain_selective_scan_step(s):
    t, u = s["u"].dtype, s["u"].float()
    delta = _softplus(s["dt"].float() + s["dt_bias"])
    h = torch.exp(delta[..., None] * s["A"]) * s["state"] + (delta * u)[..., None] * s["Bm"].float()[:, None, :]
    y = (h * s["Cm"].float()[:, None, :]).sum(-1) + s["D"] * u
    return {"y": (y * _act(s["z"].float(), "silu", 0.0)).to(t), "state": h}


PLAIN = {"layer_norm": _plain_layer_norm, "layer_norm_backward": _plain_layer_norm_backward, "linear": _plain_linear,
         "linear_backward": _plain_linear_backward, "causal_conv": _plain_causal_conv, "causal_conv_backward": _plain_causal_conv_backward,
         "causal_conv_step": _plain_causal_conv_step, "selective_scan": _plain_selective_scan, "selective_scan_train": _plain_selective_scan_train,
         "selective_scan_step": _plain_selective_scan_step}


# --------------------------------------------------------------------------------------------------- the framework's own calls
def _own(s):
    from segamd import sequence as seq
    op = s["op"]
    if op == "layer_norm":
        if s["stats"]:
            y, mean, rstd = seq.layer_norm(s["x"], s["gamma"], s["beta"], eps=s["eps"], stats=True)
            return {"y": y, "mean": mean, "rstd": rstd}
        return {"y": seq.layer_norm(s["x"], s["gamma"], s["beta"], eps=s["eps"])}
    if op == "layer_norm_backward":
        dx, dgamma, dbeta = seq.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["gamma"])
        return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if op == "linear":
        if s["keep"]:
            y, z = seq.linear(s["x"], s["w"], s["bias"], activation=s["act"], alpha=s["alpha"], residual=s["residual"], preactivation=True)
            return {"y": y, "z": z}
        return {"y": seq.linear(s["x"], s["w"], s["bias"], activation=s["act"], alpha=s["alpha"], residual=s["residual"])}
    if op == "linear_backward":
        dx, dw, db = seq.linear_backward(s["dy"], s["x"], s["w"], z=s["z"], activation=s["act"], alpha=s["alpha"], residual=s["residual"])
        return {"dx": dx, "dw": dw, "db": db}
    if op == "causal_conv":
        y, state = seq.causal_conv(s["x"], s["w"], s["bias"], activation="silu", state=s["state"], lengths=s["lengths"])
        return {"y": y, "state": state}
    if op == "causal_conv_backward":
        dx, dw, db, dstate = seq.causal_conv_backward(s["dy"], s["x"], s["w"], s["bias"], activation="silu", state=s["state"], lengths=s["lengths"],
                                                      dstate=s["dstate"])
        return {"dx": dx, "dw": dw, "db": db, "dstate": dstate}
    if op == "causal_conv_step":
        # the new state goes to another buffer (a running program alternates between two, or updates one in place): the pass stays repeatable
        new = torch.empty_like(s["state"])
        return {"y": seq.causal_conv_step(s["x"], s["state"], s["w"], s["bias"], activation="silu", new_state=new), "state": new}
    given = dict(D=s["D"], z=s["z"], dt_bias=s["dt_bias"], softplus=True)
    if op == "selective_scan":
        y, state = seq.selective_scan(s["u"], s["dt"], s["A"], s["Bm"], s["Cm"], state=s["state"], lengths=s["lengths"], **given)
        return {"y": y, "state": state}
    if op == "selective_scan_train":
        y, state, saved = seq.selective_scan(s["u"], s["dt"], s["A"], s["Bm"], s["Cm"], state=s["state"], lengths=s["lengths"], training=True, **given)
        d = seq.selective_scan_backward(s["dy"], s["u"], s["dt"], s["A"], s["Bm"], s["Cm"], saved, lengths=s["lengths"], dstate=s["dstate"], **given)
        return {"y": y, "state": state, "du": d.du, "ddt": d.ddt, "dA": d.dA, "dB": d.dB, "dC": d.dC, "dD": d.dD, "dz": d.dz,
                "ddt_bias": d.ddt_bias, "dstate": d.dstate}
    new = torch.empty_like(s["state"])
    return {"y": seq.selective_scan_step(s["u"], s["dt"], s["A"], s["Bm"], s["Cm"], s["state"], new_state=new, **given), "state": new}


def run(state):
    return _own(state) if own else PLAIN[state["op"]](state)


# --------------------------------------------------------------------------------------------------------- 64-bit definitions
def exact(case, seed):
    s = prepare(case, seed)
    op = s["op"]
    d = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    F = torch.nn.functional
    acts = {"linear": lambda v: v, "relu": torch.relu, "leaky_relu": lambda v: F.leaky_relu(v, 0.3), "sigmoid": torch.sigmoid, "silu": F.silu,
            "gelu": F.gelu}
    with torch.enable_grad():
        if op.startswith("layer_norm"):
            x, gamma, beta = (d[k].requires_grad_() for k in ("x", "gamma", "beta"))
            y = F.layer_norm(x, x.shape[1:], gamma, beta, s["eps"])
            if op == "layer_norm":
                y, v = y.detach(), x.detach()
                return {"y": y, "mean": v.mean(1), "rstd": (v.var(1, unbiased=False) + s["eps"]).rsqrt()} if s["stats"] else {"y": y}
            dx, dgamma, dbeta = torch.autograd.grad(y, (x, gamma, beta), d["dy"])
            return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
        if op == "linear":
            z = F.linear(d["x"], d["w"], d["bias"])
            y = acts[s["act"]](z) + (0 if d["residual"] is None else d["residual"])
            return {"y": y, "z": z} if s["keep"] else {"y": y}
        if op == "linear_backward":
            # y = linear(act(z)) with the activation's output given as x: its gradient through z, the weights' from x
            dx = d["dy"] @ d["w"]
            if d["z"] is not None:
                z = d["z"].requires_grad_()
                dx, = torch.autograd.grad(acts[s["act"]](z), z, dx)
            return {"dx": dx + (0 if d["residual"] is None else d["residual"]), "dw": d["dy"].t() @ d["x"], "db": d["dy"].sum(0)}
        if op == "causal_conv_step":
            x = torch.cat([d["state"], d["x"][:, None]], 1)
            return {"y": F.silu(torch.einsum("bkd,kd->bd", x, d["w"]) + d["bias"]), "state": x[:, 1:]}
        if op.startswith("causal_conv"):
            x, w, bias, st = (d[k].requires_grad_() for k in ("x", "w", "bias", "state"))
            K, L = w.shape[0], x.shape[1]
            n = [L] * x.shape[0] if s["lengths"] is None else [min(max(int(v), 0), L) for v in s["lengths"].tolist()]
            ys, states = [], []
            for b, m in enumerate(n):
                xx = torch.cat([st[b], x[b, :m]])
                y = bias.expand(m, -1)
                for k in range(K):
                    y = y + xx[k:k + m] * w[k]
                ys.append(torch.cat([F.silu(y), torch.zeros(L - m, x.shape[2], dtype=torch.float64, device="cuda")]))
                states.append(xx[m:])
            y, state = torch.stack(ys), torch.stack(states)
            if op == "causal_conv":
                return {"y": y.detach(), "state": state.detach()}
            dx, dw, db, dst = torch.autograd.grad((y, state), (x, w, bias, st), (d["dy"], d["dstate"]))
            return {"dx": dx, "dw": dw, "db": db, "dstate": dst}
        if op == "selective_scan_step":
            delta = F.softplus(d["dt"] + d["dt_bias"], threshold=50)
            h = torch.exp(delta[..., None] * d["A"]) * d["state"] + (delta * d["u"])[..., None] * d["Bm"][:, None]
            return {"y": (torch.einsum("bds,bs->bd", h, d["Cm"]) + d["D"] * d["u"]) * F.silu(d["z"]), "state": h}
        train = op == "selective_scan_train"
        names = ("u", "dt", "A", "Bm", "Cm", "D", "z", "dt_bias", "state")
        v = {k: d[k].detach().requires_grad_(train) for k in names}
        h, L = v["state"], s["u"].shape[1]
        ys = []
        for t in range(L):
            delta = F.softplus(v["dt"][:, t] + v["dt_bias"], threshold=50)
            nxt = torch.exp(delta[..., None] * v["A"]) * h + (delta * v["u"][:, t])[..., None] * v["Bm"][:, t, None]
            y = (torch.einsum("bds,bs->bd", nxt, v["Cm"][:, t]) + v["D"] * v["u"][:, t]) * F.silu(v["z"][:, t])
            if s["lengths"] is not None:
                on = (s["lengths"] > t)[:, None]
                y, nxt = torch.where(on, y, torch.zeros_like(y)), torch.where(on[..., None], nxt, h)
            h = nxt
            ys.append(y)
        y = torch.stack(ys, 1)
        if not train:
            return {"y": y, "state": h}
        gr = dict(zip(names, torch.autograd.grad((y, h), [v[k] for k in names], (d["dy"], d["dstate"]))))
        return {"y": y.detach(), "state": h.detach(), "du": gr["u"], "ddt": gr["dt"], "dA": gr["A"], "dB": gr["Bm"], "dC": gr["Cm"], "dD": gr["D"],
                "dz": gr["z"], "ddt_bias": gr["dt_bias"], "dstate": gr["state"]}
