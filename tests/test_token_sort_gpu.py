"""Token rows sorted by expert and back, and the gradients, against a plain implementation in 64 bits.

Integers, copies and zeros have to be equal.  Bounds for the others, with u = 2^-24 and h half a step of the output's type
(2^-8 for bf16, u for fp32): a sum over k picks of products is off by at most (k + 1) u of the sum of its terms' magnitudes;
a product of two fp32 numbers by u; a dot product over d columns by (chain + 40) u of the sum of magnitudes, where
chain = d / 32 + 32 is more than the longest run of additions a thread makes and 40 more than the joins; and every output by h of
itself for its rounding."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
BF, F32 = torch.bfloat16, torch.float32


def picks(T, k, E, seed, kind="random"):
    rng = np.random.default_rng(seed)
    if kind == "one":            # every pick the same expert, more than once by a token
        idx = np.full((T, k), E - 1)
    elif kind == "none":
        idx = np.full((T, k), -1)
    elif kind == "twice":        # experts drawn with replacement
        idx = rng.integers(0, E, (T, k))
    elif kind == "outside":      # padded tokens, dropped picks, numbers beyond the experts on either side
        idx = rng.integers(0, E, (T, k))
        idx[rng.random((T, k)) < 0.3] = -1
        idx[rng.random((T, k)) < 0.1] = E
        idx[rng.random((T, k)) < 0.05] = -2**31
        idx[rng.random((T, k)) < 0.05] = 2**31 - 1
        idx[T - T // 4:] = -1
    else:
        idx = np.argsort(rng.random((T, E)), axis=1)[:, :k]
    return idx.astype(np.int32)


def plain_plan(idx, E, align, cap):
    flat = idx.reshape(-1)
    pos, perm = np.full(flat.size, -1, np.int64), np.full(cap, -1, np.int64)
    counts, offsets = np.zeros(E, np.int64), np.zeros(E + 1, np.int64)
    for e in range(E):
        mine = np.nonzero(flat == e)[0]
        counts[e] = mine.size
        pos[mine] = offsets[e] + np.arange(mine.size)
        perm[offsets[e]:offsets[e] + mine.size] = mine
        offsets[e + 1] = offsets[e] + -(-mine.size // align) * align
    return pos.reshape(idx.shape), perm, counts, offsets


def make(idx, E, align):
    from omega_ai_b200 import TokenSort

    T, k = idx.shape
    sort = TokenSort(T, k, E, row_align=align)
    for t in (sort.pos, sort.perm, sort.counts, sort.offsets):
        t.fill_(-77)
    sort.plan(torch.from_numpy(idx).cuda())
    return sort, plain_plan(idx, E, align, sort.rows_cap)


@pytest.mark.parametrize("T,k,E,align,kind", [
    (1, 1, 1, 1, "random"), (1, 6, 64, 128, "random"), (5, 2, 8, 1, "random"), (33, 3, 12, 16, "outside"), (64, 1, 3, 7, "one"),
    (300, 2, 8, 128, "none"), (1000, 4, 60, 128, "outside"), (2049, 2, 8, 1, "one"), (1531, 16, 128, 1, "twice"),
    (4096, 6, 1024, 128, "random"), (4097, 8, 1024, 3, "outside"), (20000, 8, 64, 128, "random"), (70001, 2, 5, 1, "twice"),
    (300000, 4, 160, 16, "outside"),
])
def test_plan(T, k, E, align, kind):
    idx = picks(T, k, E, 5, kind)
    sort, (pos, perm, counts, offsets) = make(idx, E, align)
    for got, want in ((sort.counts, counts), (sort.offsets, offsets), (sort.pos, pos), (sort.perm, perm)):
        np.testing.assert_array_equal(got.cpu().numpy(), want)


def test_plan_of_no_tokens():
    from omega_ai_b200 import TokenSort

    sort = TokenSort(0, 2, 8)
    sort.counts.fill_(-7)
    sort.offsets.fill_(-7)
    sort.plan(torch.empty(0, 2, dtype=torch.int32, device="cuda"))
    assert sort.counts.tolist() == [0] * 8 and sort.offsets.tolist() == [0] * 9
    assert sort.sort(torch.empty(0, 16, device="cuda")).shape == (0, 16)
    assert sort.unsort(torch.empty(0, 16, device="cuda")).shape == (0, 16)


def test_more_rows_than_needed_and_none_at_all():
    """rows_cap may be larger than it has to be: the plan marks the rows behind the last expert's, with no tokens too."""
    import ctypes as C

    from omega_ai_b200 import native

    L = native.lib()
    for T in (0, 3):
        new = lambda n: torch.full((n,), -77, dtype=torch.int32, device="cuda")
        pos, perm, counts, offsets = new(max(1, 2 * T)), new(1000), new(8), new(9)
        idx = torch.tensor([[1, 7], [0, 9], [7, 1]], dtype=torch.int32, device="cuda")
        p = native.Sort(T, 2, 8, 4, 1000, pos.data_ptr(), perm.data_ptr(), counts.data_ptr(), offsets.data_ptr())
        assert L.omoe_sort_plan(C.byref(p), idx.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
        want = plain_plan(idx[:T].cpu().numpy().reshape(T, 2), 8, 4, 1000)
        for got, ref in zip((pos[:2 * T].reshape(T, 2), perm, counts, offsets), want):
            np.testing.assert_array_equal(got.cpu().numpy(), ref)


def matrix(rows, d, dtype, layout, seed):
    """[rows, d] of N(0, 1) in one of several layouts, and the whole buffer it lies in."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    if layout == "packed":
        whole = torch.randn(rows, d, generator=g, device="cuda").to(dtype)
        return whole, whole
    left, right = {"aligned": (8, 16), "odd": (3, 2)}[layout]
    whole = torch.randn(rows, left + d + right, generator=g, device="cuda").to(dtype)
    return whole[:, left:left + d], whole


CASES = [
    # T, k, E, d, align, kind, token rows, sorted rows, layout
    (1, 1, 1, 1, 1, "random", F32, F32, "packed"),
    (1, 6, 64, 2048, 1, "random", BF, BF, "packed"),
    (7, 2, 8, 8, 128, "random", BF, F32, "packed"),
    (33, 3, 12, 1544, 16, "outside", F32, F32, "packed"),
    (130, 2, 8, 257, 16, "outside", BF, BF, "packed"),
    (130, 4, 8, 1000, 1, "twice", F32, BF, "aligned"),
    (65, 5, 16, 1031, 128, "random", F32, BF, "odd"),
    (65, 8, 16, 264, 3, "outside", BF, BF, "odd"),
    (300, 16, 128, 520, 1, "random", BF, F32, "aligned"),
    (300, 2, 8, 512, 128, "none", BF, BF, "packed"),
    (257, 3, 4, 4096, 128, "one", BF, BF, "packed"),
    (2, 2, 4, 20008, 16, "random", F32, BF, "packed"),
    (1000, 6, 64, 1024, 128, "outside", BF, BF, "packed"),
]


@pytest.mark.parametrize("T,k,E,d,align,kind,xt,rt,layout", CASES)
def test_rows_there_and_back(T, k, E, d, align, kind, xt, rt, layout):
    idx = picks(T, k, E, 9, kind)
    sort, (pos, perm, counts, offsets) = make(idx, E, align)
    cap, used = sort.rows_cap, int(offsets[E])
    x, _ = matrix(T, d, xt, layout, 1)
    ys, _ = matrix(cap, d, rt, layout, 2)
    dy, _ = matrix(T, d, xt, layout, 3)
    w = torch.rand(T, k, device="cuda")
    pads = np.nonzero(perm < 0)[0]
    ys[torch.from_numpy(pads).cuda()] = float("nan")   # what no pick owns is not read
    w[torch.from_numpy(pos < 0).cuda()] = float("inf")  # nor the weights of picks without a row
    at = torch.from_numpy(np.where(pos < 0, 0, pos)).cuda()
    there = torch.from_numpy(pos >= 0).cuda()
    w0 = torch.where(there, w.double(), 0.0)
    rows = torch.where(there.unsqueeze(2), ys[at].double(), 0.0)  # [T, k, d]
    owned = torch.from_numpy(np.nonzero(perm >= 0)[0]).cuda()
    token = torch.from_numpy(perm[perm >= 0] // k).cuda()

    # there: whole buffer, margins of the layout included
    xs, xs_whole = matrix(cap, d, rt, layout, 4)
    want, want_whole = matrix(cap, d, rt, layout, 4)
    want[:used] = 0
    want[owned] = x[token].to(rt)
    assert sort.sort(x, out=xs) is xs
    assert torch.equal(xs_whole, want_whole)

    # back, with and without weights
    for weights, ww in ((w, w0), (None, there.double())):
        y, whole = matrix(T, d, xt, layout, 5)
        _, before = matrix(T, d, xt, layout, 5)
        sort.unsort(ys, weights, out=y)
        ref = (ww.unsqueeze(2) * rows).sum(1)
        mag = (ww.unsqueeze(2) * rows).abs().sum(1)
        assert ((y.double() - ref).abs() <= HALF[xt] * ref.abs() + (1 + HALF[xt]) * (k + 1) * U * mag).all()
        y.copy_(before if layout == "packed" else before[:, {"aligned": 8, "odd": 3}[layout]:][:, :d])
        assert torch.equal(whole, before)  # nothing outside the window
    assert torch.equal(sort.sort_backward(ys, dtype=xt), sort.unsort(ys, None, dtype=xt))

    # gradient of the way back
    dys, dys_whole = matrix(cap, d, rt, layout, 6)
    want, want_whole = matrix(cap, d, rt, layout, 6)
    out, dw = sort.unsort_backward(dy, ys, w, out=dys)
    assert out is dys
    flat = torch.from_numpy(perm[perm >= 0]).cuda()
    prod = w.reshape(-1)[flat].double().unsqueeze(1) * dy[token].double()
    err = (dys[owned].double() - prod).abs()
    assert (err <= (HALF[rt] + 2 * U) * prod.abs()).all()
    pad = torch.from_numpy(pads[pads < used]).cuda()
    assert (dys[pad] == 0).all()
    dys[:used] = want[:used]
    assert torch.equal(dys_whole, want_whole)
    ref = (dy.double().unsqueeze(1) * rows).sum(2)
    mag = (dy.double().unsqueeze(1) * rows).abs().sum(2)
    assert ((dw.double() - ref).abs() <= (d / 32 + 72) * U * mag).all()
    assert (dw[~there] == 0).all()
    unweighted, none = sort.unsort_backward(dy, ys, None)
    assert none is None and torch.equal(unweighted[owned], dy[token].to(rt))


def test_same_bits_every_time():
    idx = picks(777, 6, 64, 3)
    sort, _ = make(idx, 64, 16)
    g = torch.Generator(device="cuda").manual_seed(1)
    ys, dy = torch.randn(sort.rows_cap, 520, generator=g, device="cuda"), torch.randn(777, 520, generator=g, device="cuda")
    w = torch.rand(777, 6, generator=g, device="cuda")
    y, (dys, dw) = sort.unsort(ys, w), sort.unsort_backward(dy, ys, w, out=torch.zeros_like(ys))
    for _ in range(5):
        assert torch.equal(sort.unsort(ys, w), y)
        again, dw2 = sort.unsort_backward(dy, ys, w, out=torch.zeros_like(ys))
        assert torch.equal(again, dys) and torch.equal(dw2, dw)


def test_gradients_against_differences():
    """L = <c, unsort(sort(x) * s, w)> with fixed c and s, differentiated by x and w: central differences of the plain
    formula in 64 bits.  L is linear in each, so the differences are exact up to 64-bit rounding."""
    T, k, E, d = 19, 3, 5, 24
    idx = picks(T, k, E, 11, "outside")
    sort, (pos, perm, _, _) = make(idx, E, 16)
    g = torch.Generator().manual_seed(2)
    rn = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    x, w, c, scale = rn(T, d), rn(T, k), rn(T, d), rn(sort.rows_cap, d)
    x, w, c, scale = (t.float().double() for t in (x, w, c, scale))
    there, at = torch.from_numpy(pos >= 0), torch.from_numpy(np.where(pos < 0, 0, pos))

    def L(x, w):
        ys = torch.where(there.unsqueeze(2), x.unsqueeze(1) * scale[at], 0.0)
        return float((c * (w.unsqueeze(2) * ys).sum(1)).sum())

    xs = sort.sort(x.float().cuda(), out=torch.zeros(sort.rows_cap, d, device="cuda"))
    ys = xs * scale.float().cuda()
    dys, dw = sort.unsort_backward(c.float().cuda(), ys, w.float().cuda(), out=torch.zeros_like(ys))
    dx = sort.sort_backward(dys * scale.float().cuda())
    for seed in range(3):
        vx, vw = torch.randn(T, d, dtype=torch.float64), torch.randn(T, k, dtype=torch.float64)
        for v, grad, f in ((vx, dx, lambda h: L(x + h * vx, w)), (vw, dw, lambda h: L(x, w + h * vw))):
            num = (f(0.5) - f(-0.5))
            got = float((grad.double().cpu() * v).sum())
            # k + 3 roundings of every term on the way to dx, (d / 32 + 75) of every term of dw: d T k terms at most 30 in size
            terms = float((grad.double().cpu().abs() * v.abs()).sum()) + T * d
            assert abs(got - num) <= 100 * U * terms


def test_plan_and_moves_replay_from_a_graph_and_on_another_stream():
    T, k, E, d, align = 200, 2, 8, 264, 16
    first, second = picks(T, k, E, 1), picks(T, k, E, 2, "outside")
    sort, _ = make(first, E, align)
    idx = torch.from_numpy(first).cuda()
    x, w = torch.randn(T, d, device="cuda"), torch.rand(T, k, device="cuda")
    xs = torch.zeros(sort.rows_cap, d, device="cuda")
    y, dxs = torch.empty(T, d, device="cuda"), torch.zeros(sort.rows_cap, d, device="cuda")

    def step():
        sort.plan(idx)
        sort.sort(x, out=xs)
        sort.unsort(xs, w, out=y)
        sort.unsort_backward(y, xs, w, out=dxs)
        return sort.sort_backward(dxs)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dx = step()
    idx.copy_(torch.from_numpy(second))
    graph.replay()
    torch.cuda.synchronize()
    got = [t.clone() for t in (y, dx, sort.pos, sort.counts)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        dx2 = step()
    side.synchronize()
    for a, b in zip(got, (y, dx2, sort.pos, sort.counts)):
        assert torch.equal(a, b)


def test_more_than_32_bits_of_elements():
    """2.3e9 elements of sorted rows: the last rows move as the first do."""
    T, k, E, d = 140001, 4, 8, 4104
    idx = picks(T, k, E, 3)
    sort, (pos, perm, counts, offsets) = make(idx, E, 1)
    x = torch.randn(T, d, device="cuda").to(BF)
    xs = sort.sort(x)
    assert xs.numel() > 2**31
    for r in (0, sort.rows_cap // 2, sort.rows_cap - 2, sort.rows_cap - 1):
        assert torch.equal(xs[r], x[int(perm[r]) // k])
    w = torch.rand(T, k, device="cuda")
    y = sort.unsort(xs, w)
    dys, dw = sort.unsort_backward(x, xs, w)
    for t in (0, T // 2, T - 1):
        ref = x[t].double() * w[t].double().sum()
        assert ((y[t].double() - ref).abs() <= (HALF[BF] + 6 * U) * ref.abs()).all()
        for j in range(k):
            p = int(pos[t, j])
            ref = x[t].double() * w[t, j].double()
            assert ((dys[p].double() - ref).abs() <= (HALF[BF] + 2 * U) * ref.abs()).all()
            ref = float(x[t].double().square().sum())
            assert abs(float(dw[t, j]) - ref) <= (d / 32 + 72) * U * ref
