"""Forms of the operators that the sizes of the other tests pass over: every table of a list of gradients, windows of wider rows in every form of
layer norm, one of its two parameters' gradients, column sums beyond 2^31 elements.  Bounds as in the tests that these add to."""
import ctypes as C

import pytest
import torch
from test_grad_norm_gpu import check_norm, check_scaled, make, norm64
from test_layer_norm_gpu import BF, F32, U, test_forward_and_backward as forward_and_backward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 15, 16, 17, 63, 64, 65, 255, 256, 257, 499, 500, 501, 999, 1000, 1001, 2001])
@pytest.mark.parametrize("empty", [0, 40])
def test_lists_of_any_length(n, empty):
    """n tensors with elements, around the sizes of the tables, and others without between them."""
    from omega_ai_b200 import GradList

    sizes = [(1 + (i * 37) % 300 + (20000 if i % 97 == 5 else 0), F32 if i % 3 else BF) for i in range(n)]
    for i in range(empty):
        sizes.insert((i * 53) % (len(sizes) + 1), (0, BF if i % 2 else F32))
    grads = make(sizes, n)
    ref = float(norm64(grads))
    limit = float(torch.tensor(0.25 * ref, dtype=F32))
    c = limit / (ref + 1e-6)
    out = [torch.full_like(g, 7.0) for g in grads]
    before = [g.clone() for g in grads]
    check_norm(GradList(grads).norm(), grads)
    check_norm(GradList(grads, out=out).clip(limit), grads)
    check_scaled(out, grads, c)
    assert all(torch.equal(g, b) for g, b in zip(grads, before))
    check_norm(GradList(grads).clip(limit), before)
    assert all(torch.equal(g, o) for g, o in zip(grads, out))
    GradList(before).scale(torch.tensor(ref, dtype=F32, device="cuda"), limit)
    check_scaled(before, make(sizes, n), c)


@pytest.mark.parametrize("xt,yt", [(BF, BF), (F32, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("T,d,layout", [
    (4001, 520, "aligned"), (13, 768, "aligned"), (8001, 648, "aligned"), (8001, 896, "aligned"), (3001, 1528, "aligned"), (2500, 2560, "aligned"),
    (901, 4352, "aligned"), (77, 7000, "aligned"), (301, 8184, "aligned"), (33, 16384, "aligned"), (65, 9000, "aligned"), (700, 256, "aligned"),
    (600, 4096, "aligned"), (8001, 648, "odd"), (77, 7000, "odd"), (901, 2224, "odd")])
def test_windows_of_wider_rows(T, d, layout, xt, yt):
    forward_and_backward(T, d, xt, yt, layout, "both", 1.0, 0.5)


@pytest.mark.parametrize("T,d", [(1, 8), (5, 1001), (300, 1024), (40, 9000), (40, 20000), (0, 64)])
def test_one_of_the_parameters_gradients(T, d):
    """dgamma or dbeta may be left out: the other one is the same."""
    from omega_ai_b200 import layer_norm, layer_norm_backward, native

    L = native.lib()
    g = torch.Generator(device="cuda").manual_seed(d)
    x, dy, gamma = (torch.randn(*s, generator=g, device="cuda") for s in ((T, d), (T, d), (d,)))
    _, mean, rstd = layer_norm(x, gamma, stats=True)
    dx, dgamma, dbeta = layer_norm_backward(dy, x, gamma, mean, rstd)
    size = L.omoe_layer_norm_backward_workspace(T, d)
    for which in (0, 1):
        got, to, ws = torch.full((d,), 7.0, device="cuda"), torch.empty_like(x), torch.empty(size, dtype=torch.uint8, device="cuda")
        outs = [None, None]
        outs[which] = got.data_ptr()
        rc = L.omoe_layer_norm_backward(dy.data_ptr(), d, 0, x.data_ptr(), d, 0, gamma.data_ptr(), mean.data_ptr(), rstd.data_ptr(), to.data_ptr(), d,
                                        *outs, T, d, ws.data_ptr(), size, C.c_void_p(torch.cuda.current_stream().cuda_stream))
        assert rc == 0
        assert torch.equal(to, dx) and torch.equal(got, (dgamma, dbeta)[which])


def test_column_sums_beyond_32_bits_of_elements():
    """dy is zero but in forty rows at the front, around element 2^31 and at the end: each of them is a fortieth of every column's sums, whose
    chains have at most forty terms and the joins."""
    from omega_ai_b200 import layer_norm_backward

    T, d = 530001, 4096
    at = list(range(8)) + list(range(2**31 // d - 4, 2**31 // d + 4)) + list(range(T - 24, T))
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = torch.empty(T, d, dtype=BF, device="cuda"), torch.zeros(T, d, dtype=BF, device="cuda")
    for part in x.split(1 << 16):
        part.normal_(generator=g)
    rows = torch.tensor(at, device="cuda")
    dy[rows] = torch.randn(len(at), d, generator=g, device="cuda").to(BF)
    mean, rstd = torch.randn(T, generator=g, device="cuda"), 0.5 + torch.rand(T, generator=g, device="cuda")
    dx, dgamma, dbeta = layer_norm_backward(dy, x, None, mean, rstd)
    few, h = dy[rows].double(), (x[rows].double() - mean[rows].double().unsqueeze(1)) * rstd[rows].double().unsqueeze(1)
    n = (40 + 80) * U
    assert ((dbeta.double() - few.sum(0)).abs() <= n * few.abs().sum(0)).all()
    assert ((dgamma.double() - (few * h).sum(0)).abs() <= n * (few * h).abs().sum(0)).all()
    part, _, _ = layer_norm_backward(dy[rows], x[rows], None, mean[rows], rstd[rows])
    assert torch.equal(dx[rows], part)
    assert all((dx[a:b] == 0).all() for a, b in ((8, 1000), (2**31 // d + 4, T - 24)))
