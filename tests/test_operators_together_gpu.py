"""The operators in a row, as a training step uses them around experts of its own: layer norm, routing, rows to the experts,
a product per expert, weighted rows back, the backward pass, gradient clipping.  The gradients are compared with
64-bit automatic differentiation of the same step on the routing the library chose.

fp32 throughout.  A gradient passes seven operators of at most (d / 32 + 80) roundings each, some on the way of the other factor
too; errors are measured against the largest magnitude of each result, of which sums of random terms stay a part: 2 * 7 * (d / 32 + 80)
u = 1.1e-4 is the bound."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,d,E,k,align", [(1, 64, 4, 2, 1), (203, 256, 8, 2, 16), (130, 128, 64, 6, 128)])
def test_training_step(T, d, E, k, align):
    from omega_ai_b200 import GradList, TokenSort, layer_norm, layer_norm_backward, native

    L = native.lib()
    g = torch.Generator(device="cuda").manual_seed(T)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, dy = rn(T, d) + 0.5, rn(T, d)
    gamma, beta, w_r, w_e = 1 + 0.1 * rn(d), 0.1 * rn(d), 0.05 * rn(E, d), rn(E, d, d) * d ** -0.5
    idx, w = torch.empty(T, k, dtype=torch.int32, device="cuda"), torch.empty(T, k, device="cuda")
    counts = torch.empty(E, dtype=torch.int32, device="cuda")

    h, mean, rstd = layer_norm(x, gamma, beta, stats=True)
    rc = L.omoe_route_noalloc(h.data_ptr(), w_r.data_ptr(), None, T, d, E, k, 1, native.OMOE_F32, idx.data_ptr(), w.data_ptr(),
                              counts.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    sort = TokenSort(T, k, E, row_align=align).plan(idx)
    assert torch.equal(sort.counts, counts)
    xs = sort.sort(h)
    start = sort.offsets.tolist()
    ys = torch.zeros_like(xs)
    for e in range(E):
        ys[start[e]:start[e + 1]] = (xs[start[e]:start[e + 1]].double() @ w_e[e].double().T).float()
    y = sort.unsort(ys, w)
    # backward
    dys, dw = sort.unsort_backward(dy, ys, w)
    dxs, dwe = torch.zeros_like(xs), torch.zeros_like(w_e)
    for e in range(E):
        part = slice(start[e], start[e + 1])  # padding rows are zeros on both sides: whole segments go into the products
        dxs[part] = (dys[part].double() @ w_e[e].double()).float()
        dwe[e] = (dys[part].double().T @ xs[part].double()).float()
    dh = sort.sort_backward(dxs)
    dx, dgamma, dbeta = layer_norm_backward(dh, x, gamma, mean, rstd)
    grads = [dwe, dgamma, dbeta]
    unclipped = [t.clone() for t in grads]
    norm = GradList(grads).clip(0.5)

    X, G, B, W, WE = (t.double().requires_grad_() for t in (x, gamma, beta, w, w_e))
    var, m = torch.var_mean(X, dim=1, correction=0, keepdim=True)
    H = (X - m) / (var + 1e-5).sqrt() * G + B
    Y = torch.zeros_like(H)
    for j in range(k):
        Y = Y + W[:, j:j + 1] * torch.einsum("tod,td->to", WE[idx[:, j].long()], H)
    grads64 = torch.autograd.grad(Y, [X, G, B, W, WE], dy.double())
    bound = 2 * 7 * (d / 32 + 80) * 2.0 ** -24
    for got, want in zip((y, dx, unclipped[1], unclipped[2], dw, unclipped[0]), (Y.detach(), *grads64)):
        assert (got.double() - want).abs().max() <= bound * want.abs().max()
    norm64 = torch.stack([grads64[i].square().sum() for i in (4, 1, 2)]).sum().sqrt()
    assert abs(float(norm) - float(norm64)) <= bound * float(norm64)
    for got, want in zip(grads, (grads64[4], grads64[1], grads64[2])):
        want = want * min(1.0, 0.5 / (float(norm64) + 1e-6))
        assert (got.double() - want).abs().max() <= 3 * bound * want.abs().max()


def test_norm_in_front_of_the_layer_and_its_gradients_clipped():
    """LayerNorm -> MoELayer forward and backward -> LayerNorm backward, the layer's own gradients clipped with the norm's."""
    from omega_ai_b200 import GradList, MoELayer, layer_norm, layer_norm_backward

    T, d, dff, E, k = 96, 128, 256, 8, 2
    layer = MoELayer(d, dff, E, k, t_max=T, compute_dtype=torch.bfloat16)
    layer.initParam(seed=3)
    layer.set_training(True)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(T, d, generator=g, device="cuda") for _ in range(2))
    gamma, beta = 1 + 0.1 * torch.randn(d, generator=g, device="cuda"), torch.zeros(d, device="cuda")
    h, mean, rstd = layer_norm(x, gamma, beta, dtype=torch.bfloat16, stats=True)
    y = layer.forward_device(h)
    dh = layer.backward(h, dy.to(torch.bfloat16))
    dx, dgamma, dbeta = layer_norm_backward(dh, x, gamma, mean, rstd)
    grads = list(layer.weight_grads().values()) + [dgamma, dbeta]
    ref = torch.stack([t.double().square().sum() for t in grads]).sum().sqrt()
    before = [t.clone() for t in grads]
    norm = GradList(grads).clip(0.01 * float(ref))
    assert y.isfinite().all() and dx.isfinite().all()
    assert abs(float(norm) - float(ref)) <= 5 * 2.0 ** -24 * float(ref)
    after = torch.stack([t.double().square().sum() for t in grads]).sum().sqrt()
    assert abs(float(after) / (0.01 * float(ref)) - 1) <= 1e-4
    assert all(((a == 0) == (b == 0)).all() for a, b in zip(grads, before))
    layer.close()


FIRST_CALLS = """
import sys
sys.path.insert(0, {root!r})
import torch
from omega_ai_b200 import GradList, TokenSort, layer_norm, layer_norm_backward
torch.manual_seed(0)
x, g, b = torch.randn(300, 264, device="cuda"), torch.randn(264, device="cuda"), torch.randn(264, device="cuda")
idx = torch.randint(0, 8, (300, 2), dtype=torch.int32, device="cuda")
w, grads = torch.rand(300, 2, device="cuda"), [torch.randn(5000, device="cuda"), torch.randn(7, device="cuda")]
sort = TokenSort(300, 2, 8, row_align=16)
out = [torch.empty_like(t) for t in grads]
clip = GradList(grads, out=out)
def step():
    h, mean, rstd = layer_norm(x, g, b, stats=True)
    sort.plan(idx)
    xs = sort.sort(h)
    y = sort.unsort(xs, w)
    dys, dw = sort.unsort_backward(y, xs, w)
    dh = sort.sort_backward(dys)
    return (y, dw, clip.clip(0.5), *layer_norm_backward(dh, x, g, mean, rstd))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in got] + [t.clone() for t in out]
want = list(step()) + out
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("same")
"""


def test_first_calls_of_a_process_may_be_captured():
    """Nothing has to be called once before a capture: attributes and occupancy are asked for while one is on."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(root=root)], capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "same" in p.stdout, p.stderr[-2000:]


def test_eager_and_captured_calls_side_by_side():
    """A captured step is replayed on one stream while the same operators run eagerly on another, on other data."""
    from omega_ai_b200 import TokenSort, layer_norm, layer_norm_backward

    def build(T, d, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x, dy = torch.randn(T, d, generator=g, device="cuda"), torch.randn(T, d, generator=g, device="cuda")
        idx = torch.randint(0, 16, (T, 3), generator=g, dtype=torch.int32, device="cuda")
        w, sort = torch.rand(T, 3, generator=g, device="cuda"), TokenSort(T, 3, 16)

        def step():
            h, mean, rstd = layer_norm(x, stats=True)
            sort.plan(idx)
            xs = sort.sort(h)
            dys, dw = sort.unsort_backward(dy, xs, w)
            return (sort.unsort(xs, w), dw, *layer_norm_backward(sort.sort_backward(dys), x, None, mean, rstd))

        return step

    one, two = build(3000, 1024, 1), build(1777, 520, 2)
    want_one, want_two = [t.clone() for t in one()], [t.clone() for t in two()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got_one = one()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        with torch.cuda.stream(a):
            graph.replay()
        with torch.cuda.stream(b):
            got_two = two()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got_one, want_one))
    assert all(torch.equal(x, y) for x, y in zip(got_two, want_two))


def test_captured_across_streams_that_part_and_join():
    """A capture that forks to a second stream and joins it again: the operators' launches depend on kernels, copies and events."""
    from omega_ai_b200 import GradList, TokenSort, layer_norm

    T, d = 500, 512
    g = torch.Generator(device="cuda").manual_seed(4)
    x, source = torch.zeros(T, d, device="cuda"), torch.randn(T, d, generator=g, device="cuda")
    idx = torch.randint(0, 8, (T, 2), generator=g, dtype=torch.int32, device="cuda")
    sort, grads = TokenSort(T, 2, 8, row_align=8), [torch.randn(30000, generator=g, device="cuda")]
    clipped = [torch.zeros_like(grads[0])]
    clip = GradList(grads, out=clipped)
    side = torch.cuda.Stream()

    def step():
        main = torch.cuda.current_stream()
        x.copy_(source)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            sort.plan(idx)
            norm = clip.clip(0.5)
        h = layer_norm(x)
        main.wait_stream(side)
        xs = sort.sort(h, out=torch.zeros(sort.rows_cap, d, device="cuda"))
        return h, sort.unsort(xs), norm

    want = [t.clone() for t in step()] + [clipped[0].clone()]
    torch.cuda.synchronize()
    clipped[0].zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        x.zero_()
        sort.pos.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip([*got, clipped[0]], want))
