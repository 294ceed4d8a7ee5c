"""Layer norm where single rows or columns can go wrong, against the formulas in 64 bits.

Bounds of the backward pass as in test_layer_norm_gpu.py, with u = 2^-24 and D = d / 32 + 40.  Here mean is a number of x's type, so
x - mean carries one rounding and h two: with H = |h| (1 + 2 u)
  sums        means of g and g h are off by (D + 4) u of the means of their terms' magnitudes, the second with h's two roundings
  dx          rstd (both means' errors, the second times H, + 8 u (|g| + |mean g| + |h mean gh|)), and half a step of its type
  dgamma      (T / 8 + 80) u of the sum over the rows of |dy| H."""
import pytest
import torch
from test_layer_norm_gpu import BF, F32, HALF, U, forward_bounds, rows

pytestmark = pytest.mark.gpu

# widths that fill the threads of a row and widths that leave some without a column: one vector per thread, the forms for few
# threads (520 .. 7000), several vectors, rows of any width; then single elements
WIDTHS = [(d, "packed") for d in (8, 64, 256, 264, 512, 520, 1024, 1032, 1536, 2048, 2056, 4096, 4104, 7000, 8192, 8200, 16384, 16392)]
WIDTHS += [(d, "odd") for d in (1, 7, 57, 201, 401, 1001, 1024, 2047, 4095, 8191, 9001)]


@pytest.mark.parametrize("xt,yt", [(BF, BF), (F32, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("d,layout", WIDTHS)
def test_backward_of_rows_whose_mean_times_rstd_overflows(d, layout, xt, yt):
    """A row of equal numbers v has h = 0 and a finite gradient, also where v * rstd leaves fp32."""
    from omega_ai_b200 import layer_norm_backward

    T = 37
    x, _ = rows(T, d, xt, layout, 1)
    dy, _ = rows(T, d, yt, layout, 2)
    gamma = 1 + 0.3 * torch.randn(d, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    mean, rstd = torch.zeros(T, device="cuda"), torch.ones(T, device="cuda")
    for t, v in ((0, 2.0 ** 100), (5, -(2.0 ** 100)), (20, 2.0 ** 110), (T - 1, 2.0 ** 100)):
        x[t], mean[t], rstd[t] = v, v, 1e15  # of eps = 1e-30
    dx, dgamma, dbeta = layer_norm_backward(dy, x, gamma, mean, rstd)
    D = d / 32 + 40
    m, r = mean.double().unsqueeze(1), rstd.double().unsqueeze(1)
    g, h = dy.double() * gamma.double(), (x.double() - m) * r
    H = h.abs() * (1 + 2 * U)
    mg, mh = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    mg_off, mh_off = (D + 4) * U * g.abs().mean(1, keepdim=True), (D + 6) * U * (g.abs() * H).mean(1, keepdim=True)
    ref = r * (g - mg - h * mh)
    off = r * (mg_off + H * mh_off + 8 * U * (g.abs() + mg.abs() + H * mh.abs()))
    assert ((dx.double() - ref).abs() <= off * 1.01 + HALF[xt] * (ref.abs() + off)).all()
    n = (T / 8 + 80) * U
    assert ((dgamma.double() - (dy.double() * h).sum(0)).abs() <= n * (dy.double().abs() * H).sum(0)).all()
    assert ((dbeta.double() - dy.double().sum(0)).abs() <= n * dy.double().abs().sum(0)).all()

    # rows with an infinity or a NaN: none of it leaves the row but for the column sums of dy * h
    bad = x.clone()
    bad[3, 0], bad[T - 2, d - 1] = float("inf"), float("nan")
    mean[3], rstd[3], mean[T - 2], rstd[T - 2] = float("inf"), float("nan"), float("nan"), float("nan")
    dx2, _, dbeta2 = layer_norm_backward(dy, bad, gamma, mean, rstd)
    others = [t for t in range(T) if t not in (3, T - 2)]
    assert torch.equal(dx2[others], dx[others]) and torch.equal(dbeta2, dbeta)
    assert dx2[3].isnan().all() and dx2[T - 2].isnan().all()


@pytest.mark.parametrize("xt,yt", [(BF, BF), (F32, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("T,d,layout", [
    (9, 41, "packed"), (9, 328, "packed"), (9, 328, "odd"), (40, 656, "packed"), (8000, 656, "packed"), (8000, 776, "packed"), (40, 664, "aligned"),
    (40, 1312, "packed"), (9, 2624, "odd"), (5, 2624, "packed"), (5, 5248, "packed"), (5, 6560, "packed"), (5, 6560, "odd"), (3, 10496, "packed"),
    (3, 20992, "packed")])
def test_rows_of_equal_numbers_where_the_width_has_no_exact_inverse(T, d, layout, xt, yt):
    """The sum of d times v is exact for v of few bits, so the mean is v and every element is beta, rounded to its type."""
    from omega_ai_b200 import layer_norm

    values = torch.tensor([1.0, 3.0, -7.5, 255.0, 1024.0, 65536.0, -0.125, 0.0], device="cuda")
    x, _ = rows(T, d, xt, layout, 1)
    v = values[torch.arange(T, device="cuda") % len(values)]
    x.copy_(v.unsqueeze(1).expand(T, d))
    gen = torch.Generator(device="cuda").manual_seed(2)
    gamma, beta = torch.randn(d, generator=gen, device="cuda"), torch.randn(d, generator=gen, device="cuda")
    y, mean, _ = layer_norm(x, gamma, beta, dtype=yt, stats=True)
    assert torch.equal(mean, v)
    assert torch.equal(y, beta.to(yt).expand(T, d))


def test_means_of_infinite_sums():
    """A row with an infinity has an infinite mean, one with both or with a NaN none."""
    from omega_ai_b200 import layer_norm

    for d in (64, 328, 1001, 20000):
        x = torch.randn(4, d, device="cuda")
        x[0, d // 2], x[1, 0], x[2, 1], x[2, d - 1], x[3, 3] = float("inf"), -float("inf"), float("inf"), -float("inf"), float("nan")
        _, mean, _ = layer_norm(x, stats=True)
        assert mean[0] == float("inf") and mean[1] == -float("inf") and mean[2:].isnan().all()


@pytest.mark.parametrize("xt,yt", [(BF, BF), (F32, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("d", [8, 264, 520, 776, 1024, 2224, 4096, 5120, 8192, 9000, 16384, 20000])
def test_parameters_at_any_address(d, xt, yt):
    """Aligned rows with gamma and beta at odd elements of a buffer, or at 16 bytes, which go another way than with aligned parameters."""
    from omega_ai_b200 import layer_norm, layer_norm_backward

    T = 40
    x, _ = rows(T, d, xt, "packed", 1)
    dy, _ = rows(T, d, yt, "packed", 2)
    gen = torch.Generator(device="cuda").manual_seed(3)
    gamma, beta = torch.randn(d, generator=gen, device="cuda"), torch.randn(d, generator=gen, device="cuda")
    D = d / 32 + 40
    for a, b in ((1, 0), (0, 1), (4, 4), (3, 2), (8, 5)):
        flat = torch.full((2 * d + 64,), float("nan"), device="cuda")  # what lies beside the parameters is not used
        g, s = flat[a:a + d], flat[d + 32 + b:][:d]
        g.copy_(gamma)
        s.copy_(beta)
        y, mean, rstd = layer_norm(x, g, s, dtype=yt, stats=True)
        m, m_off, r, r_off, ref, off = forward_bounds(x, gamma, beta, 1e-5, yt)
        assert ((mean.double() - m[:, 0]).abs() <= m_off[:, 0] * 1.01 + U * m[:, 0].abs()).all()
        assert ((rstd.double() - r[:, 0]).abs() <= r_off[:, 0]).all()
        assert ((y.double() - ref).abs() <= off).all()
        dx, dgamma, dbeta = layer_norm_backward(dy, x, g, mean, rstd)
        m, r = mean.double().unsqueeze(1), rstd.double().unsqueeze(1)
        gr, h = dy.double() * gamma.double(), (x.double() - m) * r
        H = h.abs() + r * U * m.abs()
        mg, mh = gr.mean(1, keepdim=True), (gr * h).mean(1, keepdim=True)
        mg_off, mh_off = ((D + 4) * U * t.abs().mean(1, keepdim=True) for t in (gr, gr.abs() * H))
        ref = r * (gr - mg - h * mh)
        off = r * (mg_off + H * mh_off + 8 * U * (gr.abs() + mg.abs() + H * mh.abs()))
        assert ((dx.double() - ref).abs() <= off * 1.01 + HALF[xt] * (ref.abs() + off)).all()
        n = (T / 8 + 80) * U
        assert ((dgamma.double() - (dy.double() * h).sum(0)).abs() <= n * (dy.double().abs() * H).sum(0)).all()
        assert ((dbeta.double() - dy.double().sum(0)).abs() <= n * dy.double().abs().sum(0)).all()


@pytest.mark.parametrize("T,d", [(1, 1), (3, 7), (5, 1001), (8, 1024)])
def test_gradients_and_statistics_are_aligned(T, d):
    """dgamma and dbeta, mean and rstd lie side by side, apart and each on a vector of its own, whatever the sizes."""
    from omega_ai_b200 import GradList, layer_norm, layer_norm_backward

    x = torch.randn(T, d, device="cuda")
    _, mean, rstd = layer_norm(x, stats=True)
    _, dgamma, dbeta = layer_norm_backward(x, x, None, mean, rstd)
    assert all(t.data_ptr() % 32 == 0 and t.is_contiguous() for t in (mean, rstd, dgamma, dbeta))
    assert mean.shape == rstd.shape == (T,) and dgamma.shape == dbeta.shape == (d,)
    want, beta = dgamma.clone(), dbeta.clone()
    GradList([dbeta]).clip(0.0)
    assert torch.equal(dgamma, want) and (dbeta == 0).all()
    dbeta.copy_(beta)
    dgamma.zero_()
    assert torch.equal(dbeta, beta)
