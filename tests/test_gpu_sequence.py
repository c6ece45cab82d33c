"""GPU: the sequence operators (sequence.py) against their definitions in 64 bits (tests/sequence_ref.py), with bounds that count
roundings; strides, lengths, empty and single rows, graphs, streams, and a whole mixer block forward, backward and row by row."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

import sequence_ref as R
from segamd import sequence as seq

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
IDS = ["f16", "bf16", "f32"]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def dev(t):
    return None if t is None else t.cuda()


def wide(t, left, right):
    """t's values as a slice of a wider device tensor whose other columns are NaN."""
    o = torch.full(t.shape[:-1] + (left + t.shape[-1] + right,), float("nan"), dtype=t.dtype, device="cuda")
    o[..., left:left + t.shape[-1]] = t.cuda()
    return o[..., left:left + t.shape[-1]]


# ------------------------------------------------------------------------------------------------------- layer normalisation
LN_SHAPES = [(1, 1), (3, 7), (5, 8), (70, 64), (9, 120), (33, 200), (7, 512), (6, 1000), (2, 2048), (5, 2056), (3, 4100), (2, 8192), (2, 16384), (2, 16390)]


def ln_ref(x, gamma, beta, eps, dy):
    x64 = x.double().requires_grad_()
    g64 = (torch.ones(x.shape[1]) if gamma is None else gamma).double().requires_grad_()
    b64 = (torch.zeros(x.shape[1]) if beta is None else beta).double().requires_grad_()
    mean = x64.mean(1, keepdim=True)
    rstd = (((x64 - mean) ** 2).mean(1, keepdim=True) + eps) ** -0.5
    y = (x64 - mean) * rstd * g64 + b64
    dx, dg, db = torch.autograd.grad(y, (x64, g64, b64), dy.double())
    return y.detach(), mean.detach()[:, 0], rstd.detach()[:, 0], dx, dg, db


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,C", LN_SHAPES)
def test_layer_norm(rows, C, dtype):
    g = gen(rows * 7 + C)
    x = (rnd(g, rows, C) * (torch.rand(rows, 1, generator=g) + 0.3) + rnd(g, rows, 1)).to(dtype)
    dy, gamma, beta = rnd(g, rows, C, dtype=dtype), torch.rand(C, generator=g) + 0.5, rnd(g, C)
    y, mean, rstd, dx, dgamma, dbeta = ln_ref(x, gamma, beta, 1e-3, dy)
    # longest chain of a sum over the row: a lane's own channels (64 at most; C / 256 where rows are walked), 8 to combine them
    n = max(64, C // 256 + 1) + 8
    x64, r = x.double(), rstd[:, None]
    xm = x64.abs().mean(1, keepdim=True)
    xh = ((x64 - mean[:, None]) * r).abs()
    xs = xh + xm * r                                         # xhat with the cancelled mean's terms
    # rstd: half of the variance's relative error, whose terms are (x - mean)^2 with a cancelled mean
    cond = (xs * xs).mean(1, keepdim=True)
    gy, gm, gr = seq.layer_norm(x.cuda(), gamma.cuda(), beta.cuda(), eps=1e-3, stats=True)
    R.assert_close(gm, mean, xm[:, 0], n, "mean")
    R.assert_close(gr, rstd, rstd * (1 + cond[:, 0]), n + 4, "rstd")
    R.assert_close(gy, y, (xs + xh * (1 + cond)) * gamma.double() + beta.double().abs(), n + 8, "y")
    assert torch.equal(gy, seq.layer_norm(x.cuda(), gamma.cuda(), beta.cuda(), eps=1e-3))
    gdx, gdg, gdb = seq.layer_norm_backward(dy.cuda(), x.cuda(), gm, gr, gamma.cuda())
    d64 = dy.double().abs()
    # the backward pass takes mean / rstd as they are in 32 bits: their errors (bounded above) enter xhat
    xe = xs + xh * (1 + cond)
    s = d64 * gamma.double()
    R.assert_close(gdx, dx, r * (s + s.mean(1, keepdim=True) + xe * (s * xe).mean(1, keepdim=True) * 2), 2 * n + 16, "dx")
    R.assert_close(gdb, dbeta, d64.sum(0), rows + 16, "dbeta")
    R.assert_close(gdg, dgamma, (d64 * xe).sum(0), rows + n + 16, "dgamma")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_layer_norm_many_rows_reduce_in_order(dtype):
    """Enough rows for every block to walk several of them: two runs give the same bits, gradients of the parameters hold."""
    g = gen(5)
    rows, C = 40001, 24
    x, dy = rnd(g, rows, C, dtype=dtype), rnd(g, rows, C, dtype=dtype)
    _y, mean, rstd, dx, dgamma, dbeta = ln_ref(x, None, None, 1e-3, dy)
    args = (dy.cuda(), x.cuda(), mean.float().cuda(), rstd.float().cuda())
    a, b = seq.layer_norm_backward(*args), seq.layer_norm_backward(*args)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    xh = ((x.double() - mean[:, None]) * rstd[:, None]).abs() + 1
    d64 = dy.double().abs()
    # a thread adds at most rows / (32 rows per block x 313 blocks) + the block's and the blocks' sums, far below the count used here
    R.assert_close(a[1], dgamma, (d64 * xh).sum(0), 400, "dgamma")
    R.assert_close(a[2], dbeta, d64.sum(0), 400, "dbeta")
    R.assert_close(a[0], dx, rstd[:, None] * (d64 + 2 * xh * (d64 * xh).mean(1, keepdim=True) + d64.mean(1, keepdim=True)), 64, "dx")


def test_layer_norm_slices_and_offsets():
    """Slices of wider tensors (aligned or not), NaN beside them; no gamma / beta; leading axes; nothing outside is written."""
    g = gen(6)
    for left, right, C in ((8, 8, 64), (3, 2, 64), (1, 0, 37)):
        x = rnd(g, 2, 9, C, dtype=torch.float16)
        y, mean, rstd = seq.layer_norm(wide(x, left, right), stats=True)
        assert y.shape == x.shape and mean.shape == (2, 9)
        w = seq.layer_norm(x.cuda())
        R.assert_close(y, w.double().cpu(), torch.ones(2, 9, C, dtype=torch.float64), 64, "slice")      # (another lane order: 32-bit error only)
        dy = rnd(g, 2, 9, C, dtype=torch.float16)
        for p, q in zip(seq.layer_norm_backward(wide(dy, left, right), wide(x, left, right), mean, rstd), seq.layer_norm_backward(dy.cuda(), x.cuda(), mean, rstd)):
            R.assert_close(p, q.double().cpu(), 64 * torch.ones(q.shape, dtype=torch.float64), 64, "slice backward")


def test_layer_norm_no_rows_and_constant_rows():
    y, mean, rstd = seq.layer_norm(torch.empty(0, 40, device="cuda"), stats=True)
    assert y.shape == (0, 40) and mean.shape == (0,)
    dx, dg, db = seq.layer_norm_backward(y, y, mean, rstd)
    assert dx.shape == (0, 40) and not dg.any() and not db.any() and dg.shape == (40,)
    x = torch.full((3, 72), 1.25, device="cuda", dtype=torch.bfloat16)
    y, mean, rstd = seq.layer_norm(x, eps=1e-3, stats=True)
    assert not y.any() and torch.equal(mean, torch.full_like(mean, 1.25))


def test_layer_norm_non_finite_rows_stay_in_their_row():
    x = torch.randn(4, 256, generator=gen(8)).cuda()
    want = seq.layer_norm(x)
    x[1, 3], x[2, 5] = float("inf"), float("nan")
    y = seq.layer_norm(x)
    assert torch.equal(y[0], want[0]) and torch.equal(y[3], want[3]) and torch.isnan(y[1:3]).any(1).all()


# --------------------------------------------------------------------------------------------------------------------- linear
LIN = [(1, 8, 8), (1, 1, 1), (3, 5, 7), (16, 64, 64), (64, 64, 32), (65, 130, 100), (17, 33, 257), (129, 256, 512), (300, 200, 1000), (2, 1000, 4096),
       (256, 256, 64), (257, 264, 72), (512, 384, 640), (300, 64, 64), (200, 40, 128), (70, 56, 48)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", LIN)
def test_linear_epilogue(M, N, K, dtype):
    g = gen(M + 3 * N + 5 * K)
    x, w, b, r = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype, scale=K ** -0.5), rnd(g, N), rnd(g, M, N, dtype=dtype)
    x64, w64 = x.double(), w.double()
    z = x64 @ w64.t() + b.double()
    s = x64.abs() @ w64.abs().t() + b.double().abs()
    for k, name in enumerate([None, "relu", "leaky_relu", "sigmoid", "silu", "gelu"]):
        if k % 3 != (M + N + K) % 3 and (M, N, K) != (65, 130, 100):
            continue
        y, gz = seq.linear(x.cuda(), w.cuda(), b.cuda(), activation=name, residual=r.cuda(), preactivation=True)
        R.assert_close(gz, z, s, K + 4, "z")
        # every activation here has a slope of at most 1.13; its own evaluation: 16 roundings of a value of at most |z| + 1
        R.assert_close(y, R.act(z, name) + r.double(), 1.13 * s + r.double().abs() + z.abs() + 1, K + 24, f"y {name}")
    y = seq.linear(x.cuda(), w.cuda())
    R.assert_close(y, x64 @ w64.t(), s, K + 4, "plain")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", LIN + [(4096, 24, 40), (5000, 136, 72)])
def test_linear_backward(M, N, K, dtype):
    g = gen(M + 3 * N + 7 * K)
    x, w, dy, z, r = (rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype, scale=N ** -0.5), rnd(g, M, N, dtype=dtype), rnd(g, M, K, dtype=dtype),
                      rnd(g, M, K, dtype=dtype))
    d64, w64, x64 = dy.double(), w.double(), x.double()
    name = ["relu", "gelu", "silu", "leaky_relu", "sigmoid"][(M + N + K) % 5]
    dx, dw, db = seq.linear_backward(dy.cuda(), x.cuda(), w.cuda(), z=z.cuda(), activation=name, residual=r.cuda())
    slope = R.act_slope(z.double(), name)
    s = d64.abs() @ w64.abs()
    R.assert_close(dx, (d64 @ w64) * slope + r.double(), 1.13 * s + (d64 @ w64).abs() * (1 + z.double().abs()) + r.double().abs(), N + 24, "dx")
    R.assert_close(dw, d64.t() @ x64, d64.abs().t() @ x64.abs(), M + 4, "dw")
    R.assert_close(db, d64.sum(0), d64.abs().sum(0), M + 4, "db")
    dx, none, db2 = seq.linear_backward(dy.cuda(), x.cuda(), w.cuda(), need_dw=False)
    assert none is None
    R.assert_close(db2, d64.sum(0), d64.abs().sum(0), M + 4, "db alone (another order of the same sum)")
    R.assert_close(dx, d64 @ w64, s, N + 4, "dx plain")


def test_linear_backward_is_the_difference_quotient():
    """f32: a two-layer perceptron's loss moved along every gradient agrees with the central difference (error of the quotient: step^2 of
    the third derivative, plus the loss' own rounding over the step)."""
    g = gen(11)
    x, w1, b1, w2 = rnd(g, 20, 24), rnd(g, 40, 24, scale=0.2), rnd(g, 40), rnd(g, 16, 40, scale=0.2)
    dy = rnd(g, 20, 16)

    def loss(x, w1, b1, w2):
        h = R.act(x.double() @ w1.double().t() + b1.double(), "gelu")
        return float(((h @ w2.double().t()) * dy.double()).sum())
    h, z = seq.linear(x.cuda(), w1.cuda(), b1.cuda(), activation="gelu", preactivation=True)
    dz, dw2, _ = seq.linear_backward(dy.cuda(), h, w2.cuda(), z=z, activation="gelu", need_db=False)
    dx, dw1, db1 = seq.linear_backward(dz, x.cuda(), w1.cuda())
    for i, grad in enumerate((dx, dw1, db1, dw2)):
        args = [x, w1, b1, w2]
        v = rnd(g, *args[i].shape).double()
        up, down = list(args), list(args)
        up[i], down[i] = args[i].double() + 1e-4 * v, args[i].double() - 1e-4 * v
        quotient = (loss(*up) - loss(*down)) / 2e-4
        got = float((grad.double().cpu() * v).sum())
        assert abs(got - quotient) <= 1e-4 * float((grad.double().cpu() * v).abs().sum()), (i, got, quotient)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_linear_slices(dtype):
    """Operands as slices of wider tensors, aligned or not, NaN beside them - also behind the last input of a row, where a tile ends."""
    g = gen(12)
    for left, right, (M, N, K) in ((8, 8, (70, 72, 40)), (8, 24, (130, 256, 136)), (3, 1, (33, 40, 48)), (4, 4, (33, 40, 44))):
        x, w, dy, z = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype), rnd(g, M, N, dtype=dtype), rnd(g, M, K, dtype=dtype)
        X, W, DY, Z = (wide(t, left, right) for t in (x, w, dy, z))
        s = x.double().abs() @ w.double().abs().t()
        R.assert_close(seq.linear(X, W), x.double() @ w.double().t(), s, K + 4, "fwd")
        dx, dw, db = seq.linear_backward(DY, X, W, z=Z, activation="relu")
        R.assert_close(dx, (dy.double() @ w.double()) * (z.double() > 0), dy.double().abs() @ w.double().abs(), N + 4, "dx")
        R.assert_close(dw, dy.double().t() @ x.double(), dy.double().abs().t() @ x.double().abs(), M + 4, "dw")
        R.assert_close(db, dy.double().sum(0), dy.double().abs().sum(0), M + 4, "db")


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=IDS[:2])
def test_linear_large_tiles(dtype):
    """Results that fill the card with the largest tiles, ragged against them in every direction (reference: 64-bit products on the device)."""
    g = gen(14)
    M, N, K = 12360, 1032, 136
    x, w, b, r, z, dy = (rnd(g, *s, dtype=t).cuda() for s, t in (((M, K), dtype), ((N, K), dtype), ((N,), torch.float32), ((M, N), dtype), ((M, N), dtype), ((M, N), dtype)))
    y, pre = seq.linear(x, w, b, activation="gelu", residual=r, preactivation=True)
    z64, s = x.double() @ w.double().t() + b.double(), x.double().abs() @ w.double().abs().t() + b.double().abs()
    R.assert_close(pre, z64.cpu(), s.cpu(), K + 4, "z")
    R.assert_close(y, (R.act(z64, "gelu") + r.double()).cpu(), (1.13 * s + r.double().abs() + z64.abs() + 1).cpu(), K + 24, "y")
    # as the second layer of a perceptron: inputs N, units K
    wb = rnd(g, K, N, dtype=dtype).cuda()
    dx, none, _db = seq.linear_backward(x, y, wb, z=z, activation="gelu", residual=r, need_dw=False)
    p, s = x.double() @ wb.double(), x.double().abs() @ wb.double().abs()
    R.assert_close(dx, (p * R.act_slope(z.double(), "gelu") + r.double()).cpu(), (1.13 * s + p.abs() * (1 + z.double().abs()) + r.double().abs()).cpu(), K + 24, "dx")
    M, N, K = 131080, 520, 264
    x, dy = rnd(g, M, K, dtype=dtype).cuda(), rnd(g, M, N, dtype=dtype).cuda()
    _dx, dw, db = seq.linear_backward(dy, x, torch.zeros(N, K, dtype=dtype, device="cuda"), need_dx=False)
    R.assert_close(dw, (dy.double().t() @ x.double()).cpu(), (dy.double().abs().t() @ x.double().abs()).cpu(), M, "dw")
    R.assert_close(db, dy.double().sum(0).cpu(), dy.double().abs().sum(0).cpu(), M, "db")
    assert torch.equal(dw, seq.linear_backward(dy, x, torch.zeros(N, K, dtype=dtype, device="cuda"), need_dx=False, need_db=False)[1])


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=IDS[:2])
def test_linear_large_and_odd(dtype):
    """Large products of operands that no 16-byte access fits - odd sizes, slices at odd columns with NaN beside them."""
    g = gen(15)
    M, N, K = 8200, 519, 523
    x, w, b, r, z = (rnd(g, *s, dtype=t).cuda() for s, t in (((M, K), dtype), ((N, K), dtype), ((N,), torch.float32), ((M, N), dtype), ((M, K), dtype)))
    dy = r
    for X, W, DY in ((x, w, dy), (wide(x, 3, 2), wide(w, 1, 4), wide(dy, 5, 0))):
        y, pre = seq.linear(X, W, b, activation="silu", residual=r, preactivation=True)
        z64, s = x.double() @ w.double().t() + b.double(), x.double().abs() @ w.double().abs().t() + b.double().abs()
        R.assert_close(pre, z64.cpu(), s.cpu(), K + 4, "z")
        R.assert_close(y, (R.act(z64, "silu") + r.double()).cpu(), (1.13 * s + r.double().abs() + z64.abs() + 1).cpu(), K + 24, "y")
        dx, dw, db = seq.linear_backward(DY, X, W, z=z, activation="silu")
        p, s = dy.double() @ w.double(), dy.double().abs() @ w.double().abs()
        R.assert_close(dx, (p * R.act_slope(z.double(), "silu")).cpu(), (1.13 * s + p.abs() * (1 + z.double().abs())).cpu(), N + 24, "dx")
        R.assert_close(dw, (dy.double().t() @ x.double()).cpu(), (dy.double().abs().t() @ x.double().abs()).cpu(), M, "dw")
        R.assert_close(db, dy.double().sum(0).cpu(), dy.double().abs().sum(0).cpu(), M, "db")


def test_linear_no_rows_and_leading_axes():
    w = torch.randn(6, 10, generator=gen(1)).cuda()
    y = seq.linear(torch.empty(0, 10, device="cuda"), w)
    assert y.shape == (0, 6)
    dx, dw, db = seq.linear_backward(y, torch.empty(0, 10, device="cuda"), w)
    assert dx.shape == (0, 10) and not dw.any() and not db.any()
    x = torch.randn(2, 3, 10, generator=gen(2)).cuda()
    assert torch.equal(seq.linear(x, w).reshape(6, 6), seq.linear(x.reshape(6, 10), w))
    assert torch.equal(seq.linear(x[0, 0], w), seq.linear(x[0, :1], w)[0])


@pytest.mark.parametrize("name", ["relu", "leaky_relu", "sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_activation_backward(name, dtype):
    g = gen(13)
    for shape in ((5, 33), (3, 7, 64)):
        z, dy = rnd(g, *shape, dtype=dtype, scale=3.0), rnd(g, *shape, dtype=dtype)
        R.assert_close(seq.activation_backward(dy.cuda(), z.cuda(), name), dy.double() * R.act_slope(z.double(), name), dy.double().abs() * (1 + z.double().abs()), 24, name)


@pytest.mark.parametrize("name", ["silu", "gelu", "sigmoid"])
def test_activations_at_the_ends(name):
    """Large arguments of either sign: finite, and the limits."""
    z = torch.tensor([[-3e38, -1e5, -200.0, -88.0, 0.0, 88.0, 200.0, 1e5]]).cuda()
    one = torch.eye(8).cuda()
    y = seq.linear(z, one, activation=name)
    want = R.act(z.double().cpu(), name)
    assert torch.isfinite(y).all() and torch.allclose(y.double().cpu(), want, rtol=1e-5, atol=1e-30)


# --------------------------------------------------------------------------------------------------------- causal convolution
CONV = [(1, 1, 1, 1), (2, 1, 8, 4), (3, 5, 16, 3), (2, 17, 40, 4), (2, 33, 7, 2), (1, 130, 264, 4), (2, 300, 24, 8), (3, 16, 12, 5), (1, 3, 8, 6), (2, 2, 16, 7)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("silu", [False, True], ids=["none", "silu"])
@pytest.mark.parametrize("B,L,D,K", CONV)
def test_causal_conv(B, L, D, K, silu, dtype):
    g = gen(B + 3 * L + 5 * D + 7 * K)
    x, dy, st, dst = rnd(g, B, L, D, dtype=dtype), rnd(g, B, L, D, dtype=dtype), rnd(g, B, K - 1, D, dtype=dtype), rnd(g, B, K - 1, D, dtype=dtype)
    w, bias = rnd(g, K, D), rnd(g, D)
    for ragged in (False, True):
        lengths = torch.randint(-1, L + 2, (B,), generator=g, dtype=torch.int32) if ragged else None
        if ragged:
            lengths[0] = 0
        args = [t.double().requires_grad_() for t in (x, w, bias, st)]
        y, so = R.conv(*args, lengths, silu)
        gx, gw, gb, gst = torch.autograd.grad((y, so), args, (dy.double(), dst.double()), allow_unused=True)
        act = "silu" if silu else None
        xd, dyd = x.cuda(), dy.cuda()
        if ragged:                                            # what stands behind a length is not read
            for b in range(B):
                xd[b, max(int(lengths[b]), 0):] = float("nan")
                dyd[b, max(int(lengths[b]), 0):] = float("inf")
        ln = dev(lengths)
        gy, gso = seq.causal_conv(xd, w.cuda(), bias.cuda(), activation=act, state=st.cuda(), lengths=ln)
        assert torch.equal(gso.cpu(), so.detach().to(dtype))
        ya, _ = R.conv(x.double().abs(), w.double().abs(), bias.double().abs(), st.double().abs(), lengths, False)
        R.assert_close(gy, y, 1.13 * ya + y.detach().abs(), K + 16, "y")
        dx, dw, db, dst_in = seq.causal_conv_backward(dyd, xd, w.cuda(), bias.cuda(), activation=act, state=st.cuda(), lengths=ln, dstate=dst.cuda())
        # gradients: dv = dy act'(v), |act'| <= 1.13 with a slope of at most 0.5 towards v's error
        dv = (1.2 * dy.double().abs() * (1 + ya))
        if ragged:
            for b in range(B):
                dv[b, max(int(lengths[b]), 0):] = 0
        sx = torch.zeros(B, L + K - 1, D, dtype=torch.float64)
        sw = torch.zeros(K, D, dtype=torch.float64)
        xx = torch.cat([st.double().abs(), x.double().abs()], 1)
        for k in range(K):
            sx[:, k:k + L] += dv * w[k].double().abs()
            sw[k] = (dv * xx[:, k:k + L]).sum((0, 1))
        for b in range(B):
            m = L if lengths is None else min(max(int(lengths[b]), 0), L)
            sx[b, m:m + K - 1] += dst[b].double().abs()
        R.assert_close(dx, gx, sx[:, K - 1:], 4 * K + 24, "dx")
        R.assert_close(dst_in, gst if gst is not None else torch.zeros_like(st).double(), sx[:, :K - 1], 4 * K + 24, "dstate")
        R.assert_close(dw, gw, sw, B * L + 2 * K + 24, "dw")
        R.assert_close(db, gb, dv.sum((0, 1)), B * L + 2 * K + 24, "db")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_causal_conv_steps_are_the_prompt(dtype):
    """A prompt, then row by row from its state: the same outputs as the whole prompt; in place and through a second buffer."""
    g = gen(21)
    B, L, D, K = 3, 9, 40, 4
    x, w, bias = rnd(g, B, L, D, dtype=dtype).cuda(), rnd(g, K, D).cuda(), rnd(g, D).cuda()
    y, last = seq.causal_conv(x, w, bias, activation="silu")
    first, state = seq.causal_conv(x[:, :4], w, bias, activation="silu")
    assert torch.equal(first, y[:, :4])
    other = torch.empty_like(state)
    for t in range(4, L):
        keep = state.clone()
        yt = seq.causal_conv_step(x[:, t], state, w, bias, activation="silu", new_state=other)
        assert torch.equal(state, keep)
        assert torch.equal(yt, seq.causal_conv_step(x[:, t], state, w, bias, activation="silu"))
        assert torch.equal(state, other)
        assert torch.equal(yt, y[:, t])
    assert torch.equal(state, last)


# ------------------------------------------------------------------------------------------------------- selective state space
SCAN = [(1, 1, 1, 1), (2, 3, 8, 4), (1, 31, 5, 3), (2, 33, 24, 16), (1, 64, 64, 16), (2, 70, 72, 8), (2, 100, 16, 32), (1, 65, 20, 64), (2, 40, 9, 61), (1, 260, 8, 16),
        (3, 50, 130, 6)]


def scan_inputs(seed, B, L, D, S, dtype):
    g = gen(seed)
    i = dict(u=rnd(g, B, L, D, dtype=dtype), dt=rnd(g, B, L, D, dtype=dtype, scale=0.7), A=-(torch.rand(D, S, generator=g) * 4 + 0.05),
             B=rnd(g, B, L, S, dtype=dtype), C=rnd(g, B, L, S, dtype=dtype), D=rnd(g, D), z=rnd(g, B, L, D, dtype=dtype), dt_bias=rnd(g, D) - 2.0,
             state=rnd(g, B, D, S))
    return i, rnd(g, B, L, D, dtype=dtype), rnd(g, B, D, S), g


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("B,L,D,S", SCAN)
def test_selective_scan(B, L, D, S, dtype):
    i, dy, dstate, g = scan_inputs(B + 3 * L + 5 * D + 7 * S, B, L, D, S, dtype)
    for ragged, bare, sp in ((False, False, True), (True, False, True), (False, True, True), (True, True, False)):
        k = dict(i)
        if not sp:
            k["dt"] = k["dt"].abs()                            # the step itself, as a caller's own softplus leaves it
        if bare:
            k["D"] = k["z"] = k["dt_bias"] = k["state"] = None
        lengths = torch.randint(-1, L + 2, (B,), generator=g, dtype=torch.int32) if ragged else torch.full((B,), L, dtype=torch.int32)
        if ragged and B > 1:
            lengths[0] = 0
        ds = None if bare else dstate
        v = {n: None if t is None else t.double().requires_grad_() for n, t in k.items()}
        y, last = R.scan(**v, softplus=sp, lengths=lengths)
        names = [n for n in v if v[n] is not None]
        gr = torch.autograd.grad((y, last), [v[n] for n in names], (dy.double(), torch.zeros_like(last) if ds is None else ds.double()), allow_unused=True)
        gr = {n: torch.zeros_like(v[n]) if t is None else t for n, t in zip(names, gr)}
        d64 = {n: None if t is None else t.double() for n, t in k.items()}
        sc = R.scan_scales(*(d64[n] for n in ("u", "dt", "A", "B", "C", "D", "z", "dt_bias")), sp, d64["state"], lengths.clamp(0, L), dy.double(),
                           None if ds is None else ds.double())
        # a row's step: 8 roundings, the exponent's argument (known to 12 roundings) times its error; every term passes at most L rows, forward
        # and again backward
        n = int((8 + 12 * (1 + sc["arg"])) * (L + 8)) + 64
        c = {m: dev(t) for m, t in k.items()}
        dyd = dy.cuda()
        if ragged:
            for b in range(B):
                for m in ("u", "dt", "B", "C", "z"):
                    if c[m] is not None:
                        c[m][b, max(int(lengths[b]), 0):] = float("nan")
                dyd[b, max(int(lengths[b]), 0):] = float("nan")
        ln = dev(lengths) if ragged else None
        state = c.pop("state")
        gy, gl, saved = seq.selective_scan(**c, softplus=sp, state=state, lengths=ln, training=True)
        R.assert_close(gy, y, sc["y"], n, "y")
        R.assert_close(gl, last, sc["state"], n, "state")
        y2, l2 = seq.selective_scan(**c, softplus=sp, state=state, lengths=ln)
        assert torch.equal(gy, y2) and torch.equal(gl, l2)
        d = seq.selective_scan_backward(dyd, c["u"], c["dt"], c["A"], c["B"], c["C"], saved, D=c["D"], z=c["z"], dt_bias=c["dt_bias"], softplus=sp,
                                        lengths=ln, dstate=dev(ds))
        nb = n + D + B * L
        for name, got in (("u", d.du), ("dt", d.ddt), ("A", d.dA), ("B", d.dB), ("C", d.dC), ("D", d.dD), ("z", d.dz), ("dt_bias", d.ddt_bias)):
            if k[name] is None:
                assert got is None
                continue
            R.assert_close(got, gr[name], sc["d" + name], nb, "d" + name)
        if state is not None:
            R.assert_close(d.dstate, gr["state"], sc["dstate"], n, "dstate")
        again = seq.selective_scan_backward(dyd, c["u"], c["dt"], c["A"], c["B"], c["C"], saved, D=c["D"], z=c["z"], dt_bias=c["dt_bias"], softplus=sp,
                                            lengths=ln, dstate=dev(ds))
        assert all(p is q or torch.equal(p, q) for p, q in zip(d, again))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_selective_scan_slices(dtype):
    """B, C next to each other in one projection's output, u and z halves of another, at aligned and odd columns."""
    B, L, D, S = 2, 45, 40, 16
    i, dy, dstate, g = scan_inputs(77, B, L, D, S, dtype)
    c = {m: dev(t) for m, t in i.items()}
    want = seq.selective_scan(**c, training=True)
    dw = seq.selective_scan_backward(dy.cuda(), c["u"], c["dt"], c["A"], c["B"], c["C"], want[2], D=c["D"], z=c["z"], dt_bias=c["dt_bias"])
    for left, right in ((8, 8), (5, 3)):
        s = dict(c)
        for m in ("u", "dt", "B", "C", "z"):
            s[m] = wide(i[m], left, right)
        got = seq.selective_scan(**s, training=True)
        assert all(torch.equal(p, q) for p, q in zip(want, got))
        dg = seq.selective_scan_backward(wide(dy, left, right), s["u"], s["dt"], s["A"], s["B"], s["C"], got[2], D=s["D"], z=s["z"], dt_bias=s["dt_bias"])
        assert all(torch.equal(p, q) for p, q in zip(dw, dg))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("S", [3, 16, 40])
def test_selective_scan_steps_are_the_prompt(S, dtype):
    B, L, D = 3, 8, 24
    i, _dy, _ds, _g = scan_inputs(31 + S, B, L, D, S, dtype)
    c = {m: dev(t) for m, t in i.items()}
    y, last = seq.selective_scan(**c)
    state = c["state"].clone()
    other = torch.empty_like(state)
    v = {m: None if t is None else t.double() for m, t in i.items()}
    sc = R.scan_scales(*(v[n] for n in ("u", "dt", "A", "B", "C", "D", "z", "dt_bias")), True, v["state"], torch.full((B,), L), torch.zeros(B, L, D).double(), None)
    n = int((8 + 12 * (1 + sc["arg"])) * (L + 8)) + 64
    want, _ = R.scan(**v)
    for t in range(L):
        at = dict(u=c["u"][:, t], dt=c["dt"][:, t], A=c["A"], B=c["B"][:, t], C=c["C"][:, t], D=c["D"], z=c["z"][:, t], dt_bias=c["dt_bias"])
        keep = state.clone()
        yt = seq.selective_scan_step(state=state, new_state=other, **at)
        assert torch.equal(state, keep)
        assert torch.equal(yt, seq.selective_scan_step(state=state, **at)) and torch.equal(state, other)
        R.assert_close(yt, want[:, t], sc["y"][:, t], n, f"row {t}")
    R.assert_close(state, last.double().cpu(), sc["state"], 2 * n, "state")


def test_selective_scan_no_rows():
    B, L, D, S = 2, 0, 8, 16
    i, _dy, _ds, g = scan_inputs(3, B, L, D, S, torch.float32)
    c = {m: dev(t) for m, t in i.items()}
    y, last, saved = seq.selective_scan(**c, training=True)
    assert y.shape == (2, 0, 8) and torch.equal(last, c["state"]) and saved.numel() == 0
    ds = rnd(g, B, D, S).cuda()
    d = seq.selective_scan_backward(y, c["u"], c["dt"], c["A"], c["B"], c["C"], saved, D=c["D"], z=c["z"], dt_bias=c["dt_bias"], dstate=ds)
    assert torch.equal(d.dstate, ds) and not d.dA.any() and not d.dD.any() and not d.ddt_bias.any()
    e = torch.empty(0, 5, 8, device="cuda")
    y, last = seq.selective_scan(e, e, c["A"], torch.empty(0, 5, 16, device="cuda"), torch.empty(0, 5, 16, device="cuda"))
    assert y.shape == (0, 5, 8) and last.shape == (0, 8, 16)


# ------------------------------------------------------------------------------------------------------------- a run together
class Mixer:
    """norm -> two projections -> causal convolution -> step / B / C projection -> gated scan -> projection + residual."""

    def __init__(self, g, D, H, S, Rk, K, dtype):
        def p(*s):
            return rnd(g, *s, scale=s[-1] ** -0.5).to(dtype)
        self.gamma, self.beta = torch.rand(D, generator=g) + 0.5, rnd(g, D, scale=0.1)
        self.w_in, self.w_x, self.w_dt, self.w_out = p(2 * H, D), p(Rk + 2 * S, H), p(H, Rk), p(D, H)
        self.cw, self.cb = rnd(g, K, H, scale=0.5), rnd(g, H, scale=0.1)
        self.A, self.D, self.bias = -(torch.rand(H, S, generator=g) * 3 + 0.1), rnd(g, H), rnd(g, H) - 2.0
        self.H, self.S, self.R = H, S, Rk

    def names(self):
        return ("gamma", "beta", "w_in", "w_x", "w_dt", "w_out", "cw", "cb", "A", "D", "bias")

    def to(self, f):
        m = object.__new__(Mixer)
        m.__dict__.update({k: f(v) if torch.is_tensor(v) else v for k, v in self.__dict__.items()})
        return m

    def reference(self, x):
        B, L, D = x.shape
        mean = x.mean(-1, keepdim=True)
        n = (x - mean) * (((x - mean) ** 2).mean(-1, keepdim=True) + 1e-3) ** -0.5 * self.gamma + self.beta
        xz = n @ self.w_in.t()
        c, _ = R.conv(xz[..., :self.H], self.cw, self.cb, None, None, True)
        q = c @ self.w_x.t()
        dt = q[..., :self.R] @ self.w_dt.t()
        y, last = R.scan(c, dt, self.A, q[..., self.R:self.R + self.S], q[..., self.R + self.S:], self.D, xz[..., self.H:], self.bias)
        return y @ self.w_out.t() + x, last

    def prompt(self, x):
        s = {}
        s["x"] = x
        s["n"], s["mean"], s["rstd"] = seq.layer_norm(x, self.gamma, self.beta, stats=True)
        s["xz"] = seq.linear(s["n"], self.w_in)
        s["c"], s["conv"] = seq.causal_conv(s["xz"][..., :self.H], self.cw, self.cb, activation="silu")
        s["q"] = seq.linear(s["c"], self.w_x)
        s["dt"] = seq.linear(s["q"][..., :self.R], self.w_dt)
        s["y"], s["h"], s["saved"] = seq.selective_scan(s["c"], s["dt"], self.A, s["q"][..., self.R:self.R + self.S], s["q"][..., self.R + self.S:], D=self.D,
                                                        z=s["xz"][..., self.H:], dt_bias=self.bias, training=True)
        return seq.linear(s["y"], self.w_out, residual=x), s

    def backward(self, dout, s):
        H, Rk, S = self.H, self.R, self.S
        g = {}
        dy, g["w_out"], _ = seq.linear_backward(dout, s["y"], self.w_out, need_db=False)
        q, z = s["q"], s["xz"][..., H:]
        d = seq.selective_scan_backward(dy, s["c"], s["dt"], self.A, q[..., Rk:Rk + S], q[..., Rk + S:], s["saved"], D=self.D, z=z, dt_bias=self.bias)
        g["A"], g["D"], g["bias"] = d.dA, d.dD, d.ddt_bias
        dlow, g["w_dt"], _ = seq.linear_backward(d.ddt, q[..., :Rk], self.w_dt, need_db=False)
        dc, g["w_x"], _ = seq.linear_backward(torch.cat([dlow, d.dB, d.dC], -1), s["c"], self.w_x, residual=d.du, need_db=False)
        dx, g["cw"], g["cb"], _ = seq.causal_conv_backward(dc, s["xz"][..., :H], self.cw, self.cb, activation="silu")
        dn, g["w_in"], _ = seq.linear_backward(torch.cat([dx, d.dz], -1), s["n"], self.w_in, need_db=False)
        dx, g["gamma"], g["beta"] = seq.layer_norm_backward(dn, s["x"], s["mean"], s["rstd"], self.gamma)
        return dx + dout, g

    def step(self, x, conv, h):
        xz = seq.linear(seq.layer_norm(x, self.gamma, self.beta), self.w_in)
        c = seq.causal_conv_step(xz[:, :self.H], conv, self.cw, self.cb, activation="silu")
        q = seq.linear(c, self.w_x)
        dt = seq.linear(q[:, :self.R], self.w_dt)
        y = seq.selective_scan_step(c, dt, self.A, q[:, self.R:self.R + self.S], q[:, self.R + self.S:], h, D=self.D, z=xz[:, self.H:], dt_bias=self.bias)
        return seq.linear(y, self.w_out, residual=x)


def test_mixer_block_forward_backward_and_row_by_row():
    """The operators in a row, in 32 bits: outputs, all gradients, and a prompt continued row by row."""
    g = gen(41)
    B, L, D = 2, 37, 24
    m = Mixer(g, D, 48, 16, 8, 4, torch.float32)
    x, dout = rnd(g, B, L, D), rnd(g, B, L, D)
    m64 = m.to(lambda t: t.double().requires_grad_())
    x64 = x.double().requires_grad_()
    out, last = m64.reference(x64)
    want = torch.autograd.grad(out, [x64] + [getattr(m64, n) for n in m.names()], dout.double())
    mc = m.to(lambda t: t.cuda())
    got, s = mc.prompt(x.cuda())
    # about 400 roundings stand on the longest path (the sums of 24 .. 64 terms of six products, 37 rows of 20 each), each carried on by
    # factors of order one between stages: 2^-24 x 400 x 8 = 2e-4 of the largest value
    def near(a, b, what):
        a, b = a.detach().double().cpu(), b.detach()
        assert float((a - b).abs().max()) <= 2e-4 * float(b.abs().max()), (what, float((a - b).abs().max()), float(b.abs().max()))
    near(got, out, "out")
    near(s["h"], last, "state")
    dx, gr = mc.backward(dout.cuda(), s)
    near(dx, want[0], "dx")
    for n, w in zip(m.names(), want[1:]):
        near(gr[n], w, n)
    head, s2 = mc.prompt(x[:, :20].contiguous().cuda())
    near(head, out[:, :20], "prompt")
    conv, h = s2["conv"], s2["h"]
    for t in range(20, L):
        near(mc.step(x[:, t].cuda(), conv, h), out[:, t], f"row {t}")
    near(h, last, "state row by row")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_mixer_block_in_a_graph(dtype):
    """Forward and backward captured once and replayed on changing inputs, eager work of the same kind between the replays; and two graphs
    of the same operators that replay in turn (their workspaces are their own)."""
    g = gen(43)
    B, L, D = 2, 130, 64
    m = Mixer(g, D, 128, 16, 8, 4, dtype).to(lambda t: t.cuda())
    xs = [rnd(g, B, L, D, dtype=dtype).cuda() for _ in range(4)]
    douts = [rnd(g, B, L, D, dtype=dtype).cuda() for _ in range(4)]

    def work(x, dout):
        out, s = m.prompt(x)
        dx, gr = m.backward(dout, s)
        return [out, s["h"], dx] + [gr[n] for n in m.names()]
    want = [[t.clone() for t in work(x, d)] for x, d in zip(xs, douts)]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        x, d = xs[0].clone(), douts[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            work(x, d)
        torch.cuda.current_stream().wait_stream(side)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = work(x, d)
        graphs.append((gr, x, d, res))
    for k in range(8):
        gr, x, d, res = graphs[k % 2]
        x.copy_(xs[k % 4])
        d.copy_(douts[k % 4])
        gr.replay()
        if k % 3 == 0:
            work(xs[(k + 1) % 4], douts[(k + 1) % 4])
            torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(res, want[k % 4])), k


def test_two_streams_at_once():
    g = gen(44)
    m = Mixer(g, 64, 128, 16, 8, 4, torch.float16).to(lambda t: t.cuda())
    xs = [rnd(g, 2, 200, 64, dtype=torch.float16).cuda() for _ in range(2)]
    want = [m.prompt(x)[0].clone() for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(m.prompt(xs[k])[0])
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[k]) for k in range(2) for y in got[k])


# ------------------------------------------------------------------------------------------------------- offsets past 32 bits
def test_offsets_past_32_bits():
    """Tensors of more than 2^31 elements: the last rows come out as they do from a call on those rows alone (products and sums of another
    launch shape: equal to two steps of the stored type)."""
    def near(a, b, what):
        a, b = a.float(), b.float()
        assert float((a - b).abs().max()) <= 2.0 ** -9 * float(b.abs().max()), what
    D = 1032
    rows = (1 << 31) // D + 77
    x = torch.randn(rows, D, device="cuda", dtype=torch.float16, generator=torch.Generator("cuda").manual_seed(1))
    tail = x[-100:].contiguous()
    y, mean, rstd = seq.layer_norm(x, stats=True)
    assert torch.equal(y[-100:], seq.layer_norm(tail))
    dx, _dg, _db = seq.layer_norm_backward(y, x, mean, rstd)
    assert torch.equal(dx[-100:], seq.layer_norm_backward(y[-100:].contiguous(), tail, mean[-100:].contiguous(), rstd[-100:].contiguous())[0])
    del dx
    for n in (64, 20):                                          # the tile kernels and the one for every size
        w = torch.randn(n, D, device="cuda", dtype=torch.float16, generator=torch.Generator("cuda").manual_seed(2)) * D ** -0.5
        z = seq.linear(x, w)
        near(z[-100:], seq.linear(tail, w), "linear")
        near(seq.linear_backward(z, x, w, need_dw=False, need_db=False)[0][-100:], seq.linear_backward(z[-100:].contiguous(), tail, w, need_dw=False, need_db=False)[0], "dx")
        _none, dw, db = seq.linear_backward(z, x, w, need_dx=False)
        head, rest = rows - 100, slice(rows - 100, rows)
        a = seq.linear_backward(z[:head], x[:head], w, need_dx=False)
        b = seq.linear_backward(z[rest].contiguous(), tail, w, need_dx=False)
        near(dw, a[1] + b[1], "dw")
        assert float((db - a[2] - b[2]).abs().max()) <= 2.0 ** -9 * float(z.float().abs().sum(0).max()) * 2.0 ** -8, "db"
    del z, y
    cw = torch.randn(4, D, device="cuda")
    xs = x[None]
    yc, st = seq.causal_conv(xs, cw, activation="silu")
    yt, st2 = seq.causal_conv(xs[:, -50:].contiguous(), cw, activation="silu", state=xs[:, -53:-50].contiguous())
    assert torch.equal(yc[:, -50:], yt) and torch.equal(st, st2)
    dxc = seq.causal_conv_backward(yc, xs, cw, activation="silu")[0]
    dxt = seq.causal_conv_backward(yt, xs[:, -50:].contiguous(), cw, activation="silu", state=xs[:, -53:-50].contiguous())[0]
    assert torch.equal(dxc[:, -50:], dxt)
    del dxc, dxt


def test_scan_offsets_past_32_bits():
    D, S = 1032, 4
    L = (1 << 31) // D + 77
    g = torch.Generator("cuda").manual_seed(3)
    u = torch.randn(1, L, D, device="cuda", dtype=torch.float16, generator=g)
    bc = torch.randn(1, L, 2 * S, device="cuda", dtype=torch.float16, generator=g)
    A = -(torch.rand(D, S, device="cuda", generator=g) + 0.1)
    args = (u, u, A, bc[..., :S], bc[..., S:])
    n = 96
    y, last, saved = seq.selective_scan(*args, training=True)
    front = seq.selective_scan(*(t if t is A else t[:, :-n] for t in args))[1]
    cut = [t if t is A else t[:, -n:] for t in args]
    yt, lt, st = seq.selective_scan(*cut, state=front, training=True)
    # the chunks' borders lie elsewhere: a state may differ by the roundings of the rows since one (a few hundred, 2^-24 each)
    assert float((last - lt).abs().max()) <= 1e-4 * float(lt.abs().max())
    assert float((y[:, -n:].float() - yt.float()).abs().max()) <= 2.0 ** -9 * float(yt.float().abs().max())
    d, dt_ = seq.selective_scan_backward(u, *args, saved), seq.selective_scan_backward(u[:, -n:], *cut, st)
    for a, b in ((d.du, dt_.du), (d.ddt, dt_.ddt), (d.dB, dt_.dB), (d.dC, dt_.dC)):
        assert float((a[:, -n:].float() - b.float()).abs().max()) <= 2.0 ** -9 * float(b.float().abs().max())


def test_a_stream_that_is_not_the_operands_own():
    """Operands made on one stream, the call on another that waits for it: what every operator promises is its tensors' device's current
    stream."""
    g = gen(51)
    x, w = rnd(g, 300, 256, dtype=torch.float16).cuda(), rnd(g, 320, 256, dtype=torch.float16).cuda()
    want = seq.linear(x, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = seq.linear(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_profiled_launches_are_the_same_launches():
    KernelProfile = importlib.import_module("tf-1d-2d-segmentation-end2endpipelines_amd.ops").KernelProfile
    x = torch.randn(40, 64, generator=gen(52)).cuda()
    want = seq.layer_norm(x)
    KernelProfile.on, KernelProfile.records = True, []
    try:
        got = seq.layer_norm(x)
        assert [r[0] for r in KernelProfile.records] == ["seg_layernorm_fwd"]
    finally:
        KernelProfile.on, KernelProfile.records = False, []
    assert torch.equal(got, want)


# ---------------------------------------------------------------------------------------------------------- difference quotients
def directional(loss, args, grads, g, names):
    """Every gradient along a random direction against the central difference of the 64-bit loss: the quotient is off by step^2 of a third
    derivative of order one (1e-8) and by the loss' rounding over the step (1e-16 / 1e-4); the gradient by its 32-bit sums - 1e-4 of the
    sum of its terms' absolute values covers both."""
    for n in names:
        v = torch.randn(args[n].shape, generator=g).double()
        up, down = dict(args), dict(args)
        up[n], down[n] = args[n] + 1e-4 * v, args[n] - 1e-4 * v
        quotient = (float(loss(up)) - float(loss(down))) / 2e-4
        got = grads[n].double().cpu()
        assert abs(float((got * v).sum()) - quotient) <= 1e-4 * float((got * v).abs().sum()), (n, float((got * v).sum()), quotient)


def test_gradients_are_difference_quotients():
    g = gen(61)
    # layer normalisation
    x, dy, gamma, beta = rnd(g, 9, 40), rnd(g, 9, 40), torch.rand(40, generator=g) + 0.5, rnd(g, 40)
    _y, mean, rstd = seq.layer_norm(x.cuda(), gamma.cuda(), beta.cuda(), stats=True)
    dx, dg, db = seq.layer_norm_backward(dy.cuda(), x.cuda(), mean, rstd, gamma.cuda())

    def ln(a):
        m = a["x"].mean(1, keepdim=True)
        return (((a["x"] - m) * (((a["x"] - m) ** 2).mean(1, keepdim=True) + 1e-3) ** -0.5 * a["gamma"] + a["beta"]) * dy.double()).sum()
    directional(ln, dict(x=x.double(), gamma=gamma.double(), beta=beta.double()), dict(x=dx, gamma=dg, beta=db), g, ("x", "gamma", "beta"))
    # causal convolution, the state that goes on among the outputs
    B, L, D, K = 2, 21, 12, 4
    a = dict(x=rnd(g, B, L, D), w=rnd(g, K, D), bias=rnd(g, D), state=rnd(g, B, K - 1, D))
    dy, dst, lengths = rnd(g, B, L, D), rnd(g, B, K - 1, D), torch.tensor([L, 13], dtype=torch.int32)
    c = {k: t.cuda() for k, t in a.items()}
    got = seq.causal_conv_backward(dy.cuda(), c["x"], c["w"], c["bias"], activation="silu", state=c["state"], lengths=lengths.cuda(), dstate=dst.cuda())

    def conv(a):
        y, st = R.conv(a["x"], a["w"], a["bias"], a["state"], lengths, True)
        return (y * dy.double()).sum() + (st * dst.double()).sum()
    directional(conv, {k: t.double() for k, t in a.items()}, dict(zip(("x", "w", "bias", "state"), got)), g, ("x", "w", "bias", "state"))
    # scan, the last state among the outputs
    B, L, D, S = 2, 70, 12, 8
    i, dy, dst, g = scan_inputs(62, B, L, D, S, torch.float32)
    lengths = torch.tensor([L, 41], dtype=torch.int32)
    c = {k: t.cuda() for k, t in i.items()}
    state = c.pop("state")
    _y, _l, saved = seq.selective_scan(**c, state=state, lengths=lengths.cuda(), training=True)
    d = seq.selective_scan_backward(dy.cuda(), c["u"], c["dt"], c["A"], c["B"], c["C"], saved, D=c["D"], z=c["z"], dt_bias=c["dt_bias"], lengths=lengths.cuda(),
                                    dstate=dst.cuda())

    def scan(a):
        y, last = R.scan(**a, lengths=lengths)
        return (y * dy.double()).sum() + (last * dst.double()).sum()
    directional(scan, {k: t.double() for k, t in i.items()},
                dict(u=d.du, dt=d.ddt, A=d.dA, B=d.dB, C=d.dC, D=d.dD, z=d.dz, dt_bias=d.ddt_bias, state=d.dstate), g,
                ("u", "dt", "A", "B", "C", "D", "z", "dt_bias", "state"))


# --------------------------------------------------------------------------------------------------- the C level's documented overlaps
def test_documented_overlaps():
    """What include/seg_hip.h allows to be the same memory: layer norm's y = x, dx = dy and dx = x (rows in registers and longer ones), linear's
    y = residual (every kernel, split sums too), the activation gradient's dx = dy.  The Python functions never alias; these are C calls."""
    ffi = importlib.import_module("tf-1d-2d-segmentation-end2endpipelines_amd._ffi")
    lib, st = ffi.lib(), torch.cuda.current_stream().cuda_stream
    g = gen(71)
    for rows, C in ((5, 64), (3, 2056), (2, 16400)):
        x, dy, gamma = rnd(g, rows, C).cuda(), rnd(g, rows, C).cuda(), (torch.rand(C, generator=g) + 0.5).cuda()
        y, mean, rstd = seq.layer_norm(x, gamma, stats=True)
        dx, dg, db = seq.layer_norm_backward(dy, x, mean, rstd, gamma)
        t = x.clone()
        assert lib.seg_layernorm_fwd(t.data_ptr(), C, t.data_ptr(), C, rows, C, 2, gamma.data_ptr(), None, 1e-3, None, None, st) == 0
        assert torch.equal(t, y)
        ws = torch.empty(lib.seg_layernorm_bwd_workspace_bytes(rows, C, 2), dtype=torch.uint8, device="cuda")
        for which in (0, 1):
            a, b, pg, pb = dy.clone(), x.clone(), torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
            out = (a, b)[which]
            assert lib.seg_layernorm_bwd(a.data_ptr(), C, b.data_ptr(), C, out.data_ptr(), C, rows, C, 2, mean.data_ptr(), rstd.data_ptr(), gamma.data_ptr(),
                                         pg.data_ptr(), pb.data_ptr(), ws.data_ptr(), st) == 0
            assert torch.equal(out, dx) and torch.equal(pg, dg) and torch.equal(pb, db)
    for M, N, K, dtype in ((4, 40, 64, torch.float16), (100, 37, 41, torch.float16), (300, 256, 128, torch.bfloat16), (100, 72, 4096, torch.float32), (130, 128, 4096, torch.float16),
                           (12360, 1032, 136, torch.float16)):
        x, w, r = rnd(g, M, K, dtype=dtype).cuda(), rnd(g, N, K, dtype=dtype).cuda(), rnd(g, M, N, dtype=dtype).cuda()
        want = seq.linear(x, w, activation="silu", residual=r)
        t = r.clone()
        a = ffi.LinearArgs(M, N, K, seq._DT[dtype], ffi.SEQ_ACT["silu"], 0.0, x.data_ptr(), K, w.data_ptr(), K, None, t.data_ptr(), N, None, 0, t.data_ptr(), N)
        ws = torch.empty(max(lib.seg_linear_workspace_bytes(a, 0), 16), dtype=torch.uint8, device="cuda")
        a.workspace = ws.data_ptr()
        assert lib.seg_linear_fwd(a, st) == 0
        assert torch.equal(t, want), (M, N, K)
        dy, r = rnd(g, M, N, dtype=dtype).cuda(), rnd(g, M, K, dtype=dtype).cuda()
        want = seq.linear_backward(dy, x, w, residual=r, need_dw=False, need_db=False)[0]
        t = r.clone()
        a = ffi.LinearArgs(M, K, N, seq._DT[dtype], 0, 0.0, dy.data_ptr(), N, w.data_ptr(), K, None, t.data_ptr(), K, None, 0, t.data_ptr(), K)
        ws = torch.empty(max(lib.seg_linear_workspace_bytes(a, 1), 16), dtype=torch.uint8, device="cuda")
        a.workspace = ws.data_ptr()
        assert lib.seg_linear_bwd_data(a, st) == 0
        assert torch.equal(t, want), (M, N, K)
    z, dy = rnd(g, 9, 50).cuda(), rnd(g, 9, 50).cuda()
    want, t = seq.activation_backward(dy, z, "gelu"), dy.clone()
    assert lib.seg_linear_act_bwd(t.data_ptr(), 50, z.data_ptr(), 50, t.data_ptr(), 50, 9, 50, 2, ffi.SEQ_ACT["gelu"], 0.0, st) == 0
    assert torch.equal(t, want)
    torch.cuda.synchronize()


def test_partial_gradients_at_the_c_level():
    """Gradients that are NULL are not wanted: the others come out as they do together."""
    ffi = importlib.import_module("tf-1d-2d-segmentation-end2endpipelines_amd._ffi")
    lib, st = ffi.lib(), torch.cuda.current_stream().cuda_stream
    B, L, D, S = 2, 70, 24, 16
    i, dy, dst, g = scan_inputs(72, B, L, D, S, torch.float32)
    c = {k: t.cuda() for k, t in i.items()}
    state = c.pop("state")
    _y, _l, saved = seq.selective_scan(**c, state=state, training=True)
    dy = dy.cuda()
    want = seq.selective_scan_backward(dy, c["u"], c["dt"], c["A"], c["B"], c["C"], saved, D=c["D"], z=c["z"], dt_bias=c["dt_bias"])
    shapes = dict(du=(B, L, D), ddt=(B, L, D), dz=(B, L, D), dBm=(B, L, S), dCm=(B, L, S), dA=(D, S), dD=(D,), ddt_bias=(D,), dstate=(B, D, S))
    both = dict(zip(shapes, (want.du, want.ddt, want.dz, want.dB, want.dC, want.dA, want.dD, want.ddt_bias, want.dstate)))
    for name, shape in shapes.items():
        a = ffi.ScanArgs(B, L, D, S, 2, 1)
        for n, t in (("u", c["u"]), ("dt", c["dt"]), ("z", c["z"]), ("Bm", c["B"]), ("Cm", c["C"]), ("dy", dy)):
            setattr(a, n, t.data_ptr())
            setattr(a, n + "_bs", t.stride(0))
            setattr(a, n + "_ld", t.stride(1))
        a.A, a.Dskip, a.dt_bias, a.saved = c["A"].data_ptr(), c["D"].data_ptr(), c["dt_bias"].data_ptr(), saved.data_ptr()
        out = torch.full(shape, float("nan"), device="cuda")
        setattr(a, name, out.data_ptr())
        if len(shape) == 3 and name != "dstate":
            setattr(a, name + "_bs", shape[1] * shape[2])
            setattr(a, name + "_ld", shape[2])
        ws = torch.empty(lib.seg_selective_scan_bwd_workspace_bytes(a), dtype=torch.uint8, device="cuda")
        a.workspace = ws.data_ptr()
        assert lib.seg_selective_scan_bwd(a, st) == 0, lib.seg_last_error()
        torch.cuda.synchronize()
        assert torch.equal(out, both[name]), name


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("wide_side", [136, 56])
def test_linear_every_number_of_steps(wide_side, dtype):
    """Contractions of one step of the tile kernels' ring to several rounds of it, whole and ragged, in the three passes."""
    g = gen(81)
    for L in (1, 8, 64, 72, 128, 192, 200, 256, 264, 320, 512, 576, 1030):
        a, b = rnd(g, 136, L, dtype=dtype), rnd(g, wide_side, L, dtype=dtype)
        want, s = a.double() @ b.double().t(), a.double().abs() @ b.double().abs().t()
        R.assert_close(seq.linear(a.cuda(), b.cuda()), want, s, L + 4, f"fwd {L}")
        bt, at = b.t().contiguous(), a.t().contiguous()
        none = torch.zeros(136, wide_side, dtype=dtype, device="cuda")
        R.assert_close(seq.linear_backward(a.cuda(), none, bt.cuda(), need_dw=False, need_db=False)[0], want, s, L + 4, f"dx {L}")
        none = torch.zeros(136, wide_side, dtype=dtype, device="cuda")
        dw, db = seq.linear_backward(at.cuda(), bt.cuda(), none, need_dx=False)[1:]
        R.assert_close(dw, want, s, L + 4, f"dw {L}")
        R.assert_close(db, at.double().sum(0), at.double().abs().sum(0), L + 4, f"db {L}")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", [(3, 40, 30008), (64, 64, 24576), (33, 16, 9000), (40, 4104, 520), (16, 40, 4096), (5, 2048, 5000), (17, 24, 4100)])
def test_linear_few_rows_and_long_contractions(M, N, K, dtype):
    """Both sides of the limits of the kernel for few rows, and sums split over many ranges (joined by several threads per element)."""
    g = gen(82)
    x, w, b, r = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype, scale=K ** -0.5), rnd(g, N), rnd(g, M, N, dtype=dtype)
    y, pre = seq.linear(x.cuda(), w.cuda(), b.cuda(), activation="relu", residual=r.cuda(), preactivation=True)
    z64, s = x.double() @ w.double().t() + b.double(), x.double().abs() @ w.double().abs().t() + b.double().abs()
    R.assert_close(pre, z64, s, K + 4, "z")
    R.assert_close(y, z64.clamp(min=0) + r.double(), s + r.double().abs(), K + 6, "y")
    # the same contraction as a weight gradient: K rows
    dy, xt = x.t().contiguous(), w.t().contiguous()
    dw, db = seq.linear_backward(dy.cuda(), xt.cuda(), torch.zeros(M, N, dtype=dtype, device="cuda"), need_dx=False)[1:]
    R.assert_close(dw, x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t(), K + 4, "dw")
    R.assert_close(db, x.double().sum(1), x.double().abs().sum(1), K + 4, "db")
    assert torch.equal(dw, seq.linear_backward(dy.cuda(), xt.cuda(), torch.zeros(M, N, dtype=dtype, device="cuda"), need_dx=False)[1])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rows_at_any_address(dtype):
    """Channels that are no whole eights, at every column offset: whole eights and the rows' ends, with NaN on either side, read and
    written next to what must stay."""
    g = gen(91)
    B, L, D, S = 2, 37, 27, 5
    i, dy, dst, g = scan_inputs(92, B, L, D, S, dtype)
    w = rnd(g, 4, D)
    ref = seq.selective_scan(**{k: t.cuda() for k, t in i.items()}, training=True)
    y0, s0 = seq.causal_conv(i["u"].cuda(), w.cuda(), activation="silu")
    c0 = seq.causal_conv_backward(dy.cuda(), i["u"].cuda(), w.cuda(), activation="silu")
    x64, w64 = i["u"].double(), w.double()
    R.assert_close(y0, R.conv(x64, w64, None, None, None, True)[0], 1.13 * R.conv(x64.abs(), w64.abs(), None, None, None, False)[0] + 1, 24, "conv")
    for left in range(8):
        s = {k: wide(t, left, 1) if k in ("u", "dt", "B", "C", "z") else t.cuda() for k, t in i.items()}
        assert all(torch.equal(p, q) for p, q in zip(ref, seq.selective_scan(**s, training=True)))
        y, st = seq.causal_conv(wide(i["u"], left, 1), w.cuda(), activation="silu")
        assert torch.equal(y, y0) and torch.equal(st, s0)
        c = seq.causal_conv_backward(wide(dy, left, 1), wide(i["u"], left, 1), w.cuda(), activation="silu")
        assert all(torch.equal(p, q) for p, q in zip(c[:2], c0[:2]))
    # results inside a wider tensor: nothing beside them changes
    ffi = importlib.import_module("tf-1d-2d-segmentation-end2endpipelines_amd._ffi")
    for left in (0, 1, 3):
        out = torch.full((B, L, left + D + 2), 7.0, dtype=dtype, device="cuda")
        x = i["u"].cuda()
        a = ffi.CausalConvArgs(B, L, D, 4, seq._DT[dtype], ffi.SEQ_ACT["silu"], x.data_ptr(), L * D, D, w.cuda().data_ptr(), None, None, None,
                               out[..., left:].data_ptr(), out.stride(0), out.stride(1), None)
        wd = w.cuda()
        a.w = wd.data_ptr()
        assert ffi.lib().seg_causal_conv_fwd(a, torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(out[..., left:left + D], y0)
        assert bool((out[..., :left] == 7).all()) and bool((out[..., left + D:] == 7).all())


@pytest.mark.parametrize("rows,C", [(1, 65537), (3, 20001), (40, 16391), (300, 4104), (64, 9000)])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_layer_norm_long_rows_and_few_blocks(rows, C, dtype):
    g = gen(93)
    x, dy, gamma, beta = rnd(g, rows, C, dtype=dtype), rnd(g, rows, C, dtype=dtype), torch.rand(C, generator=g) + 0.5, rnd(g, C)
    X = wide(x, 3, 2)
    y, mean, rstd = seq.layer_norm(X, gamma.cuda(), beta.cuda(), stats=True)
    dx, dg, db = seq.layer_norm_backward(wide(dy, 1, 4), X, mean, rstd, gamma.cuda())
    if C > 16384:                                              # (longer than the registers hold: one order of sums at every address)
        assert torch.equal(y, seq.layer_norm(x.cuda(), gamma.cuda(), beta.cuda()))
    x64, d64, g64 = x.double(), dy.double(), gamma.double()
    m, var = x64.mean(1, keepdim=True), x64.var(1, unbiased=False, keepdim=True)
    rs = 1 / torch.sqrt(var + 1e-3)
    xh = (x64 - m) * rs
    gd = d64 * g64
    # a sum of C terms of either sign, by a thread's share in turn and then in halves: at most C / 256 + 16 roundings of its partial sums
    n = C / 256 + 40
    R.assert_close(y, xh * g64 + beta.double(), xh.abs() * g64 + beta.double().abs() + g64, n, "y")
    R.assert_close(dx, rs * (gd - gd.mean(1, keepdim=True) - xh * (gd * xh).mean(1, keepdim=True)), rs * (gd.abs() + 2 * gd.abs().mean(1, keepdim=True) * (1 + xh.abs())), n, "dx")
    R.assert_close(dg, (d64 * xh).sum(0), (d64.abs() * (xh.abs() + 1)).sum(0), n + rows, "dgamma")
    R.assert_close(db, d64.sum(0), d64.abs().sum(0), n + rows, "dbeta")


@pytest.mark.parametrize("dtype", DTYPES[:2], ids=IDS[:2])
def test_linear_forward_from_packed_copies(dtype):
    """A forward product large enough for copies of operands that no 16-byte access fits (2^32 products), NaN beside them."""
    g = gen(95)
    M, N, K = 16392, 523, 519
    x, w, b = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype), rnd(g, N).cuda()
    X, W = wide(x, 3, 2), wide(w, 1, 4)
    x, w = x.cuda(), w.cuda()
    z64, s = x.double() @ w.double().t() + b.double(), x.double().abs() @ w.double().abs().t() + b.double().abs()
    for args in ((x, w), (X, W), (x, W)):
        R.assert_close(seq.linear(*args, b, activation="relu"), z64.clamp(min=0).cpu(), s.cpu(), K + 6, "y")
