"""Layer norm and its gradients against the formulas in 64 bits.

Bounds, with u = 2^-24, D = d / 32 + 40 (more than the additions on the way of any term into a sum over a row) and h half a
step of the output's type:
  mean        D u mean|x|
  var         its terms (x - mean)^2 carry 3 u, the sum D u; an error e of the mean adds e^2
  rstd        half of var's relative error (e^2 against var + eps included) and 4 u for root, quotient and eps
  y           |gamma| (rstd e + |h| (rstd's relative error + 3 u)) + 2 u (|h gamma| + |y|), and h |y|
The backward pass takes mean and rstd as given; H = |h| + rstd u |mean| covers x - mean from rounded numbers:
  sums        means of g and g h are off by (D + 4) u of the means of their terms' magnitudes
  dx          rstd (both means' errors, the second times |h|, + 8 u (|g| + |mean g| + |h mean gh|)), and half a step
  dgamma      (T / 8 + 80) u of the sum over the rows of |dy| H; dbeta the same of |dy|."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
BF, F32 = torch.bfloat16, torch.float32


def rows(T, d, dtype, layout, seed, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    left, right = {"packed": (0, 0), "aligned": (8, 16), "odd": (3, 2)}[layout]
    whole = (torch.randn(T, left + d + right, generator=g, device="cuda") * scale + shift).to(dtype)
    return whole[:, left:left + d], whole


def forward_bounds(x, gamma, beta, eps, out):
    x = x.double()
    d = x.shape[1]
    D = d / 32 + 40
    g = torch.ones(d, dtype=torch.float64, device="cuda") if gamma is None else gamma.double()
    b = torch.zeros_like(g) if beta is None else beta.double()
    mean = x.mean(1, keepdim=True)
    var = (x - mean).square().mean(1, keepdim=True)
    rstd = (var + eps).rsqrt()
    h = (x - mean) * rstd
    y = h * g + b
    e = D * U * x.abs().mean(1, keepdim=True)
    r = ((D + 3) * U * var + e * e) / (2 * (var + eps)) + 4 * U
    y_off = g.abs() * (rstd * e + h.abs() * (r + 3 * U)) + 2 * U * ((h * g).abs() + y.abs())
    return mean, e, rstd, r * rstd * 1.01, y, y_off * 1.01 + HALF[out] * (y.abs() + y_off)


CASES = [
    # T, d, type of x, type of y, layout, parameters, scale, shift
    (1, 1, F32, F32, "packed", "both", 1.0, 0.0),
    (3, 7, F32, BF, "packed", "none", 1.0, 0.0),
    (5, 8, BF, BF, "packed", "both", 1.0, 0.0),
    (2, 64, BF, F32, "packed", "gamma", 1.0, 0.0),
    (130, 250, BF, BF, "packed", "both", 1.0, 0.0),
    (131, 256, F32, F32, "aligned", "beta", 1.0, 0.0),
    (77, 1001, F32, BF, "odd", "both", 1.0, 0.0),
    (77, 1024, BF, BF, "odd", "both", 1.0, 0.0),
    (400, 1032, BF, BF, "packed", "both", 1.0, 3.0),
    (33, 2048, F32, F32, "packed", "both", 1e-3, 10.0),   # spread small against the offset
    (700, 4096, BF, BF, "packed", "both", 1.0, 0.0),
    (9, 4104, F32, BF, "aligned", "both", 1e4, 0.0),
    (5, 8192, BF, BF, "packed", "both", 1.0, 0.0),
    (311, 8193, BF, BF, "packed", "gamma", 1.0, 0.0),
    (3, 16384, F32, F32, "packed", "both", 1.0, 0.0),
    (2, 16392, BF, BF, "aligned", "both", 1.0, 0.0),
    (2, 40000, BF, F32, "packed", "both", 1.0, 0.0),
    (1, 70001, F32, BF, "packed", "none", 1.0, 0.0),
    (300, 20000, BF, BF, "packed", "both", 1.0, 0.0),
    (150, 9001, F32, BF, "packed", "both", 1.0, 0.0),
    (70, 201, BF, F32, "odd", "both", 1.0, 0.0),
    (301, 401, BF, BF, "packed", "both", 1.0, 0.0),
    (9, 2047, F32, F32, "packed", "both", 1.0, 0.0),
    (600, 4095, BF, BF, "packed", "both", 1.0, 0.0),
    (33, 8191, F32, BF, "packed", "both", 1.0, 0.0),
    (5000, 24, F32, F32, "packed", "both", 1.0, 0.0),
    (1200, 520, F32, BF, "packed", "both", 1.0, 0.0),
]


@pytest.mark.parametrize("T,d,xt,yt,layout,params,scale,shift", CASES)
def test_forward_and_backward(T, d, xt, yt, layout, params, scale, shift):
    from omega_ai_b200 import layer_norm, layer_norm_backward

    eps = 1e-5
    x, _ = rows(T, d, xt, layout, 1, scale, shift)
    gamma = 1 + 0.3 * torch.randn(d, device="cuda") if params in ("both", "gamma") else None
    beta = 0.3 * torch.randn(d, device="cuda") if params in ("both", "beta") else None
    y, whole = rows(T, d, yt, layout, 2)
    margin, before = rows(T, d, yt, layout, 2)
    got, mean, rstd = layer_norm(x, gamma, beta, eps, out=y, stats=True)
    assert got is y
    m, m_off, r, r_off, ref, off = forward_bounds(x, gamma, beta, eps, yt)
    assert ((mean.double() - m[:, 0]).abs() <= m_off[:, 0] * 1.01 + U * m[:, 0].abs()).all()
    assert ((rstd.double() - r[:, 0]).abs() <= r_off[:, 0]).all()
    assert ((y.double() - ref).abs() <= off).all()
    assert torch.equal(layer_norm(x, gamma, beta, eps, dtype=yt), y)
    margin.copy_(y)
    assert torch.equal(whole, before)  # nothing outside the window

    dy, _ = rows(T, d, yt, layout, 3)
    dx, whole = rows(T, d, xt, layout, 4)
    margin, before = rows(T, d, xt, layout, 4)
    _, dgamma, dbeta = layer_norm_backward(dy, x, gamma, mean, rstd, out=dx)
    margin.copy_(dx)
    assert torch.equal(whole, before)
    D = d / 32 + 40
    m, r = mean.double().unsqueeze(1), rstd.double().unsqueeze(1)
    g = dy.double() * (1.0 if gamma is None else gamma.double())
    h = (x.double() - m) * r
    H = h.abs() + r * U * m.abs()
    mg, mh = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    mg_off, mh_off = ((D + 4) * U * t.abs().mean(1, keepdim=True) for t in (g, g.abs() * H))
    ref = r * (g - mg - h * mh)
    off = r * (mg_off + H * mh_off + 8 * U * (g.abs() + mg.abs() + H * mh.abs()))
    assert ((dx.double() - ref).abs() <= off * 1.01 + HALF[xt] * (ref.abs() + off)).all()
    n = (T / 8 + 80) * U
    assert ((dgamma.double() - (dy.double() * h).sum(0)).abs() <= n * (dy.double().abs() * H).sum(0)).all()
    assert ((dbeta.double() - dy.double().sum(0)).abs() <= n * dy.double().abs().sum(0)).all()
    # the same bits again, and without the parameters' gradients
    dx2, dgamma2, dbeta2 = layer_norm_backward(dy, x, gamma, mean, rstd)
    assert torch.equal(dx2, dx) and torch.equal(dgamma2, dgamma) and torch.equal(dbeta2, dbeta)
    dx3, none, none2 = layer_norm_backward(dy, x, gamma, mean, rstd, param_grads=False)
    assert torch.equal(dx3, dx) and none is None and none2 is None


def test_rows_without_spread_and_rows_with_infinities():
    """A row of equal numbers gives beta; an infinity or NaN stays in its own row."""
    from omega_ai_b200 import layer_norm

    for d in (8, 100, 1024, 4096, 20000):
        x = torch.randn(6, d, device="cuda")
        x[1] = 0.0
        x[2] = 1024.0
        x[3, 0] = float("inf")
        x[4, d - 1] = float("nan")
        gamma, beta = torch.randn(d, device="cuda"), torch.randn(d, device="cuda")
        y = layer_norm(x, gamma, beta)
        assert torch.equal(y[1], beta) and torch.equal(y[2], beta)
        assert y[3:5].isnan().any(1).all()
        alone = layer_norm(x[[0, 5]].contiguous(), gamma, beta)
        assert torch.equal(y[[0, 5]], alone)


def test_no_rows():
    from omega_ai_b200 import layer_norm, layer_norm_backward

    x = torch.empty(0, 64, device="cuda")
    y, mean, rstd = layer_norm(x, stats=True)
    assert y.shape == (0, 64)
    dx, dgamma, dbeta = layer_norm_backward(y, x, None, mean, rstd)
    assert dx.shape == (0, 64) and (dgamma == 0).all() and (dbeta == 0).all()


@pytest.mark.parametrize("xt,yt", [(BF, BF), (F32, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("T,d", [(1, 520), (4001, 520), (13, 768), (4001, 1032), (3, 1536), (3001, 1528), (2, 2056), (2500, 2560), (1, 4104),
                                 (901, 4352), (77, 7000), (8100, 648), (8001, 896), (400, 8184)])
def test_rows_between_powers_of_two(T, d, xt, yt):
    """Rows that leave whole warps of the next power of two idle: fewer threads share a row, several rows a block."""
    test_forward_and_backward(T, d, xt, yt, "packed", "both", 1.0, 0.5)


@pytest.mark.parametrize("d", [24, 57, 1040])
def test_gradients_against_differences(d):
    """<c, layer_norm(x)> along random directions: central differences of the plain formula in 64 bits with step 1e-5 (their
    own error is 1e-10 times third derivatives of order rstd^3)."""
    from omega_ai_b200 import layer_norm, layer_norm_backward

    T = 5
    gen = torch.Generator().manual_seed(d)
    rn = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64).float().double()
    x, c, gamma, beta = rn(T, d), rn(T, d), 1 + 0.2 * rn(d), rn(d)
    gamma = gamma.float().double()

    def L(x, gamma, beta):
        m = x.mean(1, keepdim=True)
        v = (x - m).square().mean(1, keepdim=True)
        return float((c * ((x - m) / (v + 1e-5).sqrt() * gamma + beta)).sum())

    f = lambda t: t.float().cuda()
    _, mean, rstd = layer_norm(f(x), f(gamma), f(beta), stats=True)
    dx, dg, db = (t.double().cpu() for t in layer_norm_backward(f(c), f(x), f(gamma), mean, rstd))
    h = 1e-5
    for _ in range(3):
        vx, vg, vb = rn(T, d), rn(d), rn(d)
        for num, got, terms in (
                (L(x + h * vx, gamma, beta) - L(x - h * vx, gamma, beta), (dx * vx).sum(), (dx * vx).abs().sum()),
                (L(x, gamma + h * vg, beta) - L(x, gamma - h * vg, beta), (dg * vg).sum(), (dg * vg).abs().sum()),
                (L(x, gamma, beta + h * vb) - L(x, gamma, beta - h * vb), (db * vb).sum(), (db * vb).abs().sum())):
            assert abs(num / (2 * h) - float(got)) <= 1e-5 * (float(terms) + 1.0)


def test_layer_surface():
    from omega_ai_b200 import LNLayer, Tensor, layer_norm, layer_norm_backward

    x, dy = torch.randn(17, 96, device="cuda"), torch.randn(17, 96, device="cuda")
    layer = LNLayer(96)
    layer.gamma.copy_(torch.randn(96))
    layer.beta.copy_(torch.randn(96))
    y = layer.forward(Tensor.from_device(x)).view2d()
    want, mean, rstd = layer_norm(x, layer.gamma, layer.beta, stats=True)
    assert torch.equal(y, want)
    dx = layer.diff(Tensor.from_device(dy)).view2d()
    wdx, wg, wb = layer_norm_backward(dy, x, layer.gamma, mean, rstd)
    assert torch.equal(dx, wdx) and torch.equal(layer.diffGamma, wg) and torch.equal(layer.diffBeta, wb)


def test_forward_and_backward_replay_from_two_graphs():
    """Two captured steps share no workspace: replayed at the same time on two streams they give what each gives alone."""
    from omega_ai_b200 import layer_norm, layer_norm_backward

    def build(T, d):
        x, dy = torch.randn(T, d, device="cuda").to(BF), torch.randn(T, d, device="cuda").to(BF)
        gamma, beta = torch.randn(d, device="cuda"), torch.randn(d, device="cuda")

        def step():
            y, mean, rstd = layer_norm(x, gamma, beta, stats=True)
            return (y,) + layer_norm_backward(dy, x, gamma, mean, rstd)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        x.copy_(torch.randn(T, d, device="cuda"))
        dy.copy_(torch.randn(T, d, device="cuda"))
        want = step()
        torch.cuda.synchronize()
        return graph, out, want, (x, dy, gamma, beta)  # the graph reads its inputs where they lie: they have to live

    a, b = build(3000, 1024), build(2500, 1024)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        for (graph, *_), s in zip((a, b), streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, want, _ in (a, b):
        assert all(torch.equal(o, w) for o, w in zip(out, want))


def test_more_than_32_bits_of_elements():
    from omega_ai_b200 import layer_norm, layer_norm_backward

    T, d = 530001, 4096
    x = torch.empty(T, d, dtype=BF, device="cuda")
    x[:T // 2].normal_()
    x[T // 2:].normal_()
    assert x.numel() > 2**31
    y, mean, rstd = layer_norm(x, stats=True)
    dx, _, dbeta = layer_norm_backward(y, x, None, mean, rstd)
    at = [0, T // 2, T - 1]
    one, m, r = layer_norm(x[at].contiguous(), stats=True)
    assert torch.equal(y[at], one)
    part, _, _ = layer_norm_backward(one, x[at].contiguous(), None, m, r)
    assert torch.equal(dx[at], part)
    total, size = torch.zeros(d, dtype=torch.float64, device="cuda"), torch.zeros(d, dtype=torch.float64, device="cuda")
    for part in y.split(1 << 16):
        total += part.sum(0, dtype=torch.float64)
        size += part.abs().sum(0, dtype=torch.float64)
    assert ((dbeta.double() - total).abs() <= (T / 8 + 80) * U * size).all()
