"""GPU: the sequence operators at the ends of their ranges - infinities and NaN in activations, constant rows, empty and very long
extents, gradients of weights whose every row counts."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

from segamd import sequence as seq

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
IDS = ["f16", "bf16", "f32"]
INF = float("inf")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


# rows, units and inputs that every kernel of the product meets: few rows, any size, 128 x 64, 128 x 128 and 256 x 256 tiles
KERNELS = [(4, 64, 64), (100, 40, 33), (200, 64, 64), (130, 136, 64), (12360, 1032, 136)]
ACTIVATIONS = ["relu", "leaky_relu", "sigmoid", "silu", "gelu"]


# ---------------------------------------------------------------------------------------------------- activations at infinity
@pytest.mark.parametrize("name", ACTIVATIONS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_activations_of_infinity_are_their_limits(name, dtype):
    """z = bias here (x is zero).  At +-inf an activation takes its limit; a finite value next to them keeps its own.  1e-5: an exponential's
    argument of up to 40 carries 40 half steps of 2^-24 each way, a few times over; one step of the type where it is stored."""
    for M, N, K in KERNELS:
        v = torch.tensor([INF, -INF, 3e38, -3e38, 1e4, -1e4, 40.0, -40.0]).repeat(N // 8)
        want = {"relu": torch.relu, "leaky_relu": lambda t: torch.where(t > 0, t, t * 0.3), "sigmoid": torch.sigmoid,
                "silu": lambda t: torch.where(t < -1e3, 0.0, t * torch.sigmoid(t)),
                "gelu": lambda t: torch.where(t < -1e3, 0.0, 0.5 * t * torch.special.erfc(-t * 0.5 ** 0.5))}[name](v.double()).to(dtype).float()
        y, z = seq.linear(torch.zeros(M, K, dtype=dtype, device="cuda"), torch.ones(N, K, dtype=dtype, device="cuda"), v.cuda(), activation=name,
                          preactivation=True)
        assert torch.equal(z.cpu(), v.to(dtype).expand(M, N))
        assert torch.allclose(y.float().cpu(), want.expand(M, N), rtol=max(1e-5, torch.finfo(dtype).eps), atol=2.0 ** -24), (M, N, K)


@pytest.mark.parametrize("name", ACTIVATIONS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_slopes_at_infinity_are_their_limits(name, dtype):
    """A kept pre-activation that overflowed its type: the gradient through it is the one through any large value of that sign."""
    g = gen(61)
    for M, K, N in KERNELS:
        dy, w, x = rnd(g, M, N, dtype=dtype), rnd(g, N, K, dtype=dtype), rnd(g, M, K, dtype=dtype)
        z = rnd(g, M, K, dtype=dtype)
        far = torch.rand(M, K, generator=g).cuda()
        big, z = (torch.where(far < 0.2, v, torch.where(far > 0.8, -v, z.float())).to(dtype) for v in (1e4, INF))
        assert torch.isinf(z).any()
        got, want = (seq.linear_backward(dy, x, w, z=t, activation=name, need_dw=False, need_db=False)[0] for t in (z, big))
        assert torch.isfinite(got).all() and torch.equal(got, want), (M, N, K)
        d = torch.ones_like(z)
        got = seq.activation_backward(d, z, name)
        assert torch.equal(got, seq.activation_backward(d, big, name))
        up, down = {"relu": (1, 0), "leaky_relu": (1, 0.3), "sigmoid": (0, 0), "silu": (1, 0), "gelu": (1, 0)}[name]
        assert torch.equal(got[z == INF], torch.full_like(got[z == INF], up)) and torch.equal(got[z == -INF], torch.full_like(got[z == -INF], down))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("D", [24, 13])
def test_causal_conv_at_infinity(D, dtype):
    """The convolution's silu at +-inf (by way of the bias): limits forward, finite gradients backward."""
    g = gen(62)
    B, L, K = 2, 37, 4
    x, dy, w, st = rnd(g, B, L, D, dtype=dtype), rnd(g, B, L, D, dtype=dtype), rnd(g, K, D), rnd(g, B, K - 1, D, dtype=dtype)
    far = torch.arange(D).cuda() % 3
    big, bias = (torch.where(far == 0, v, torch.where(far == 1, -v, 0.1)).cuda() for v in (torch.tensor(1e4).cuda(), torch.tensor(INF).cuda()))
    y, _ = seq.causal_conv(x, w, bias, activation="silu", state=st)
    want, _ = seq.causal_conv(x, w, big, activation="silu", state=st)
    assert torch.equal(y[..., far != 0], want[..., far != 0]) and torch.isposinf(y[..., far == 0]).all() and not y[..., far == 1].any()
    for p, q in zip(seq.causal_conv_backward(dy, x, w, bias, activation="silu", state=st), seq.causal_conv_backward(dy, x, w, big, activation="silu", state=st)):
        assert torch.isfinite(p).all() and torch.equal(p, q)
    ys = seq.causal_conv_step(x[:, 0], st.clone(), w, bias, activation="silu")
    assert torch.equal(ys, y[:, 0])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("B,L,D,S", [(2, 40, 24, 5), (1, 300, 13, 16), (1, 150, 20, 40)])
def test_selective_scan_gates_at_infinity(B, L, D, S, dtype):
    """A gate of -inf shuts (outputs and gradients as with any gate far below zero); one of +inf leaves dz finite."""
    g = gen(63)
    u, dt, z, dy = (rnd(g, B, L, D, dtype=dtype) for _ in range(4))
    Bm, Cm = rnd(g, B, L, S, dtype=dtype), rnd(g, B, L, S, dtype=dtype)
    A, skip = -(torch.rand(D, S, generator=g) + 0.2).cuda(), rnd(g, D)
    far = torch.rand(B, L, D, generator=g).cuda()
    shut = far < 0.2
    big, low = (torch.where(shut, v, z.float()).to(dtype) for v in (-1e4, -INF))
    y, last, saved = seq.selective_scan(u, dt, A, Bm, Cm, D=skip, z=low, training=True)
    want, _, _ = seq.selective_scan(u, dt, A, Bm, Cm, D=skip, z=big, training=True)
    assert torch.equal(y, want) and not y[shut].any()
    for p, q in zip(*(seq.selective_scan_backward(dy, u, dt, A, Bm, Cm, saved, D=skip, z=t) for t in (low, big))):
        assert p is None or (torch.isfinite(p).all() and torch.equal(p, q))
    big, high = (torch.where(shut, v, z.float()).to(dtype) for v in (1e4, INF))
    p, q = (seq.selective_scan_backward(dy, u, dt, A, Bm, Cm, saved, D=skip, z=t).dz for t in (high, big))
    assert torch.isfinite(p).all() and torch.equal(p, q)
    st = rnd(g, B, D, S)
    p, q = (seq.selective_scan_step(u[:, 0], dt[:, 0], A, Bm[:, 0], Cm[:, 0], st, D=skip, z=t, new_state=torch.empty_like(st))
            for t in (torch.full_like(z[:, 0], -INF), torch.full_like(z[:, 0], -1e4)))
    assert torch.equal(p, q) and not p.any()


# ------------------------------------------------------------------------------------------------------------ NaN through relu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_relu_keeps_nan(dtype):
    """max(NaN, 0) is NaN, as for every other activation: a row that went wrong shows.  Its slope there is torch's (the gradient passes)."""
    g = gen(64)
    for M, N, K in KERNELS:
        x, w, b = rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype), rnd(g, N)
        want = seq.linear(x, w, b, activation="relu")
        x[M // 2, K // 2] = float("nan")
        y = seq.linear(x, w, b, activation="relu")
        on = torch.arange(M, device="cuda") == M // 2
        assert torch.isnan(y[on]).all() and torch.equal(y[~on], want[~on]), (M, N, K)
    z, dy = rnd(g, 9, 21, dtype=dtype), rnd(g, 9, 21, dtype=dtype)
    z[4, 3], z[5, 6], z[5, 7] = float("nan"), 0.0, -0.0
    v = z.float().cpu().requires_grad_()
    with torch.enable_grad():
        slope, = torch.autograd.grad(torch.relu(v).sum(), v)
    assert torch.equal(seq.activation_backward(dy, z, "relu").float().cpu(), dy.float().cpu() * slope)


# ------------------------------------------------------------------------------------------------------------- constant rows
@pytest.mark.parametrize("C", [1, 3, 37, 64, 200, 512, 1111, 2048, 2056, 5000, 16384, 20001, 100003])
def test_layer_norm_of_constant_rows_is_beta(C):
    """Rows without variance, of values whose sums round: the mean is the value, y is beta, rstd 1 / sqrt(eps) (three roundings)."""
    g = gen(C)
    v = torch.cat([torch.tensor([0.1, 1000.1, -3.3e-5, 7.7e7, 0.0]), torch.randn(20, generator=g) * 10.0 ** torch.randint(-3, 4, (20,), generator=g)])
    x = v[:, None].expand(-1, C).contiguous().cuda()
    gamma, beta = rnd(g, C), rnd(g, C)
    for off in (0, 1):                                          # rows that 16-byte accesses fit, and rows at any address
        rows = torch.empty(25, C + off, device="cuda")[:, off:].copy_(x) if off else x
        y, mean, rstd = seq.layer_norm(rows, gamma, beta, eps=1e-3, stats=True)
        assert torch.equal(mean.cpu(), v)
        assert torch.equal(y, beta.expand_as(y))
        assert torch.allclose(rstd.cpu(), torch.full((25,), 1e-3 ** -0.5), rtol=3 * 2.0 ** -23, atol=0)
    dx, dg, _ = seq.layer_norm_backward(x, x, mean, rstd, gamma)
    assert not dg.any()


# ------------------------------------------------------------------------------------------------------------- empty extents
@pytest.mark.parametrize("shape", [(4, 0), (0, 4), (2, 0, 3), (1, 0)])
def test_empty_leading_axes(shape):
    """Extents of zero anywhere in front of the channels are calls without work; gradients of parameters are zero."""
    x = torch.empty(shape + (8,), dtype=torch.float16, device="cuda")
    y, mean, rstd = seq.layer_norm(x, stats=True)
    assert y.shape == x.shape and mean.shape == shape == rstd.shape
    dx, dg, db = seq.layer_norm_backward(x, x, mean, rstd)
    assert dx.shape == x.shape and dg.shape == (8,) and not dg.any() and not db.any()
    w = torch.ones(6, 8, dtype=torch.float16, device="cuda")
    y, z = seq.linear(x, w, activation="gelu", preactivation=True, residual=torch.empty(shape + (6,), dtype=torch.float16, device="cuda"))
    assert y.shape == z.shape == shape + (6,)
    dx, dw, db = seq.linear_backward(y, x, w, z=x, activation="gelu", residual=x)
    assert dx.shape == x.shape and dw.shape == (6, 8) and not dw.any() and not db.any()
    assert seq.activation_backward(x, x, "silu").shape == x.shape


# ------------------------------------------------------------------------------------------------------------ long sequences
def test_causal_conv_of_millions_of_rows():
    """More rows than one axis of a grid of row blocks takes (65535 blocks of 128 or, backward, 64): whole numbers, so every sum is exact."""
    g = torch.Generator("cuda").manual_seed(65)
    L, D, K = 65535 * 128 + 4099, 8, 3
    x, dy = (torch.randint(-2, 3, (1, L, D), device="cuda", generator=g).half() for _ in range(2))
    w = torch.tensor([[1.0], [-2.0], [3.0]], device="cuda").expand(K, D).contiguous()
    y, st = seq.causal_conv(x, w)
    xx = torch.cat([torch.zeros(1, K - 1, D, dtype=torch.float16, device="cuda"), x], 1)
    assert torch.equal(y, sum(xx[:, k:k + L] * w[k, 0].half() for k in range(K))) and torch.equal(st, x[:, -(K - 1):])
    dx, dw, db, _ = seq.causal_conv_backward(dy, x, w, torch.zeros(D, device="cuda"))
    dd = torch.cat([dy, torch.zeros(1, K - 1, D, dtype=torch.float16, device="cuda")], 1)
    assert torch.equal(dx, sum(dd[:, K - 1 - k:K - 1 - k + L] * w[k, 0].half() for k in range(K)))
    assert torch.equal(dw.long(), torch.stack([(xx[0, k:k + L].long() * dy[0].long()).sum(0) for k in range(K)]))
    assert torch.equal(db.long(), dy[0].long().sum(0))


def test_layer_norm_backward_of_very_long_rows():
    """More columns than one grid of column sums takes (2^32 threads in a row of blocks)."""
    C = (1 << 27) + 5
    g = torch.Generator("cuda").manual_seed(66)
    x, dy = (torch.randint(-2, 3, (2, C), device="cuda", generator=g, dtype=torch.int8).half() for _ in range(2))
    mean, rstd = torch.tensor([0.5, -0.25], device="cuda"), torch.tensor([2.0, 0.5], device="cuda")
    _dx, dgamma, dbeta = seq.layer_norm_backward(dy, x, mean, rstd)
    for lo in range(0, C, 1 << 25):                             # every value is a whole number of 1/8: exact
        s = slice(lo, min(C, lo + (1 << 25)))
        assert torch.equal(dbeta[s], dy[:, s].float().sum(0)), lo
        assert torch.equal(dgamma[s], (dy[:, s].float() * ((x[:, s].float() - mean[:, None]) * rstd[:, None])).sum(0)), lo


@pytest.mark.parametrize("M", [1, 16])
def test_linear_with_very_many_units(M):
    """More units than a grid of the few-rows kernel takes (2^32 threads in a row of blocks of 512, 16 units each): whole numbers, exact."""
    N, K = (1 << 27) + 48, 4
    g = torch.Generator("cuda").manual_seed(68)
    x = torch.randint(-2, 3, (M, K), device="cuda", generator=g).float()
    w = torch.randint(-2, 3, (N, K), device="cuda", generator=g, dtype=torch.int8).float()
    y = seq.linear(x, w, activation="relu")
    for lo in range(0, N, 1 << 25):
        s = slice(lo, min(N, lo + (1 << 25)))
        assert torch.equal(y[:, s], torch.relu(x @ w[s].t())), lo


# ------------------------------------------------------------------------------------- gradients of weights: every row counts
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", [(131080, 520, 264), (131075, 520, 264), (20011, 136, 264), (100003, 64, 72), (8201, 519, 523), (5003, 24, 40), (65, 300, 1000)])
def test_weight_gradients_of_whole_numbers(M, N, K, dtype):
    """Products and sums of whole numbers up to 4 M < 2^24 are exact in 32 bits: a lost, doubled or misplaced row, range of rows or partial
    sum shows.  Every tile kernel, split ranges that end inside a step, operands that are copied, and the kernel for every size."""
    g = torch.Generator("cuda").manual_seed(M + N)
    x, dy = (torch.randint(-2, 3, (M, c), device="cuda", generator=g).to(dtype) for c in (K, N))
    w = torch.zeros(N, K, dtype=dtype, device="cuda")
    _none, dw, db = seq.linear_backward(dy, x, w, need_dx=False)
    want, sums = dy.double().t().contiguous() @ x.double(), dy.double().sum(0)
    assert torch.equal(dw.double(), want) and torch.equal(db.double(), sums)
    assert torch.equal(seq.linear_backward(dy, x, w, need_dx=False, need_db=False)[1], dw)
    assert torch.equal(seq.linear_backward(dy, x, w, need_dx=False, need_dw=False)[2], db)


@pytest.mark.parametrize("n", [64, 20])
def test_weight_gradients_of_rows_past_32_bits(n):
    """Only the last rows of an operand of more than 2^31 elements count (the others' gradient is zero): the same bits as those rows alone."""
    D = 1032
    rows = (1 << 31) // D + 77
    g = torch.Generator("cuda").manual_seed(67)
    x = torch.randint(-2, 3, (rows, D), device="cuda", generator=g, dtype=torch.int8).half()
    dy = torch.zeros(rows, n, dtype=torch.float16, device="cuda")
    dy[-70:] = torch.randint(-2, 3, (70, n), device="cuda", generator=g).half()
    w = torch.zeros(n, D, dtype=torch.float16, device="cuda")
    _none, dw, db = seq.linear_backward(dy, x, w, need_dx=False)
    want = dy[-70:].double().t().contiguous() @ x[-70:].double()
    assert torch.equal(dw.double(), want) and torch.equal(db.double(), dy[-70:].double().sum(0))


def test_activation_backward_of_the_longest_row():
    """2^31 - 3 channels: their pieces of eight are counted in 64 bits."""
    C = (1 << 31) - 3
    g = torch.Generator("cuda").manual_seed(69)
    z = torch.randint(-2, 3, (1, C), device="cuda", generator=g, dtype=torch.int8).half()
    dx = seq.activation_backward(z, z, "relu")
    for lo in range(0, C, 1 << 29):
        s = slice(lo, min(C, lo + (1 << 29)))
        assert torch.equal(dx[:, s], torch.relu(z[:, s])), lo


# ------------------------------------------------------------------------------------------------------------ growing states
@pytest.mark.parametrize("S", [4, 16])
def test_selective_scan_of_growing_states(S):
    """Steps of the wrong sign make states grow by e^1.5 a row (softplus=False, dt = -1): what is still zero stays zero however far a whole
    chunk's factor lies past 32 bits, and so do gradients that have not begun.  Inputs in the last 20 rows, dy in the first 20."""
    g = gen(70)
    B, L, D = 2, 600, 24
    u, dt, dy = torch.zeros(B, L, D), -torch.ones(B, L, D), torch.zeros(B, L, D)
    u[:, -20:], dy[:, :20] = torch.randn(B, 20, D, generator=g), torch.randn(B, 20, D, generator=g)
    A = -1.5 * torch.ones(D, S)
    Bm, Cm = torch.randn(B, L, S, generator=g), torch.randn(B, L, S, generator=g)
    ref = [t.double().requires_grad_() for t in (u, dt, A, Bm, Cm)]
    args = [t.cuda() for t in (u, dt, A, Bm, Cm)]
    y, last, saved = seq.selective_scan(*args, softplus=False, training=True)
    d = seq.selective_scan_backward(dy.cuda(), *args, saved, softplus=False)
    h, ys = torch.zeros(B, D, S, dtype=torch.float64), []
    with torch.enable_grad():
        for t in range(L):
            h = torch.exp(ref[1][:, t, :, None] * ref[2]) * h + (ref[1][:, t] * ref[0][:, t])[..., None] * ref[3][:, t, None]
            ys.append((h * ref[4][:, t, None]).sum(-1))
        want = torch.autograd.grad(torch.stack(ys, 1), ref, dy.double())
    # one sign of every factor e^1.5 and random signs of the terms: relative to the largest value, 20 rows x 8 roundings
    for name, got, exact in (("y", y, torch.stack(ys, 1)), ("state", last, h)) + tuple(zip(("du", "ddt", "dA", "dB", "dC"), (d.du, d.ddt, d.dA, d.dB, d.dC), want)):
        got, exact = got.double().cpu(), exact.detach()
        assert torch.isfinite(got).all(), name
        assert float((got - exact).abs().max()) <= 160 * 2.0 ** -24 * float(exact.abs().max()), name
    assert torch.isfinite(d.dstate).all()


@pytest.mark.parametrize("C", [64, 1111, 4096, 20001])
def test_layer_norm_of_rows_far_from_zero(C):
    """Offsets far above the spread: the mean is off by its own rounding alone (half a step, 2^-24 of it), beside the roundings of sums of the
    spread (a lane's channels and 8 to combine them, twice; xhat, rstd and the result 8)."""
    g = gen(71 + C)
    x = (torch.randn(9, C, generator=g) * torch.tensor([0.1, 1.0, 3.0])[:, None].repeat(3, 1) + torch.tensor([1000.0, -300.0, 70.0])[:, None].repeat_interleave(3, 0)).float()
    gamma, beta = torch.rand(C, generator=g) + 0.5, torch.randn(C, generator=g)
    y, mean, rstd = seq.layer_norm(x.cuda(), gamma.cuda(), beta.cuda(), stats=True)
    d = x.double()
    m = d.mean(1, keepdim=True)
    r = (((d - m) ** 2).mean(1, keepdim=True) + 1e-3) ** -0.5
    n, u = 2 * (max(64, C // 256 + 1) + 8) + 8, 2.0 ** -24
    off = m.abs() * u + n * u * (d - m).abs().mean(1, keepdim=True)                      # of the mean
    xh = ((d - m) * r).abs()
    assert float(((mean.double().cpu() - m[:, 0]).abs() / off[:, 0]).max()) <= 1
    assert float(((rstd.double().cpu()[:, None] / r - 1).abs() / (n * u + (off * r) ** 2)).max()) <= 1
    want = (d - m) * r * gamma.double() + beta.double()
    bound = (off * r + xh * (n * u + (off * r) ** 2)) * gamma.double() + 4 * u * (want.abs() + beta.double().abs() + xh * gamma.double())
    assert float(((y.double().cpu() - want).abs() / bound).max()) <= 1


def test_causal_conv_of_several_long_sequences():
    """Row blocks past one axis share the third with the sequences: every sequence's rows, lengths and states are its own."""
    g = torch.Generator("cuda").manual_seed(72)
    B, L, D, K = 3, 65535 * 64 + 130, 8, 4
    x, dy = (torch.randint(-2, 3, (B, L, D), device="cuda", generator=g).half() for _ in range(2))
    st, dst = (torch.randint(-2, 3, (B, K - 1, D), device="cuda", generator=g).half() for _ in range(2))
    w = torch.tensor([1.0, -2.0, 3.0, -1.0], device="cuda")[:, None].expand(K, D).contiguous()
    lengths = torch.tensor([L, 70, L - 65], dtype=torch.int32, device="cuda")
    y, new = seq.causal_conv(x, w, state=st, lengths=lengths)
    dx, dw, _db, dstate = seq.causal_conv_backward(dy, x, w, state=st, lengths=lengths, dstate=dst)
    sums = torch.zeros(K, D, dtype=torch.long, device="cuda")
    for b, n in enumerate(lengths.tolist()):
        xx, dd = torch.cat([st[b], x[b, :n]]), torch.cat([torch.zeros(K - 1, D, dtype=torch.float16, device="cuda"), dy[b, :n], torch.zeros(K - 1, D, dtype=torch.float16, device="cuda")])
        assert torch.equal(y[b, :n], sum(xx[k:k + n] * w[k, 0].half() for k in range(K))) and not y[b, n:].any() and torch.equal(new[b], xx[n:])
        dxx = sum(dd[K - 1 - k:K - 1 - k + n + K - 1] * w[k, 0].half() for k in range(K))
        dxx[n:] += dst[b]
        assert torch.equal(dx[b, :n], dxx[K - 1:]) and not dx[b, n:].any() and torch.equal(dstate[b], dxx[:K - 1])
        sums += torch.stack([(xx[k:k + n].long() * dy[b, :n].long()).sum(0) for k in range(K)])
    assert torch.equal(dw.long(), sums)


@pytest.mark.parametrize("name", ACTIVATIONS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_nan_goes_through_every_activation(name, dtype):
    g = gen(73)
    for M, N, K in KERNELS:
        b = rnd(g, N)
        b[N // 3] = float("nan")
        y = seq.linear(rnd(g, M, K, dtype=dtype), rnd(g, N, K, dtype=dtype), b, activation=name)
        on = torch.arange(N, device="cuda") == N // 3
        assert torch.isnan(y[:, on]).all() and not torch.isnan(y[:, ~on]).any(), (M, N, K)
    z, dy = rnd(g, 9, 21, dtype=dtype), rnd(g, 9, 21, dtype=dtype)
    z[4, 3] = float("nan")
    d = seq.activation_backward(dy, z, name)
    assert not torch.isnan(d[z == z]).any() and (name in ("relu", "leaky_relu") or torch.isnan(d[4, 3]))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_nan_goes_through_the_convolution_and_the_gate(dtype):
    """A NaN stays in its channel (and, in the convolution, in the rows whose window holds it)."""
    g = gen(74)
    x, w = rnd(g, 2, 40, 24, dtype=dtype), rnd(g, 4, 24)
    x[1, 10, 5] = float("nan")
    y, _ = seq.causal_conv(x, w, activation="silu")
    want = torch.zeros_like(y, dtype=torch.bool)
    want[1, 10:14, 5] = True
    assert torch.equal(torch.isnan(y), want)
    u, dt, z = (rnd(g, 2, 40, 24, dtype=dtype) for _ in range(3))
    Bm, Cm, A = rnd(g, 2, 40, 16, dtype=dtype), rnd(g, 2, 40, 16, dtype=dtype), -torch.rand(24, 16, generator=g).cuda()
    z[0, 7, 3] = float("nan")
    y, last = seq.selective_scan(u, dt, A, Bm, Cm, z=z)
    assert torch.equal(torch.isnan(y), torch.isnan(z)) and torch.isfinite(last).all()
