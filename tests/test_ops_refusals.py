"""What the operators without a handle refuse, before anything is launched: runs without a GPU (addresses are never read)."""
import ctypes as C

import pytest

INVALID, TOO_LARGE = -1, -3
P = 1 << 20  # an aligned address that nothing dereferences


@pytest.fixture(scope="module")
def native():
    from omega_ai_b200 import native as n

    n.build()
    return n


def plan(native, T=4, k=2, E=8, align=1, cap=None, pos=P, perm=2 * P, counts=3 * P, offsets=4 * P):
    cap = native.lib().omoe_sort_rows_cap(T, k, E, align) if cap is None else cap
    return native.Sort(T, k, E, align, cap, pos, perm, counts, offsets)


def refused(native, rc, code, words):
    assert rc == code
    assert words in native.lib().omoe_ops_error().decode()


def test_rows_cap(native):
    cap = native.lib().omoe_sort_rows_cap
    assert cap(0, 2, 8, 128) == 0
    assert cap(4, 2, 8, 1) == 8
    assert cap(1, 2, 8, 128) == 256          # two experts can hold a row
    assert cap(100, 2, 8, 128) == 1280       # 200 + 8 * 127 = 1216, in whole segments
    assert cap(4, 17, 64, 1) == TOO_LARGE and cap(4, 2, 1025, 1) == TOO_LARGE
    assert cap(-1, 2, 8, 1) == INVALID and cap(4, 0, 8, 1) == INVALID and cap(4, 2, 0, 1) == INVALID and cap(4, 2, 8, 0) == INVALID
    assert cap(1 << 30, 2, 8, 1) == TOO_LARGE and cap(2**31 - 1, 16, 1024, 2**31 - 1) == TOO_LARGE


@pytest.mark.parametrize("change,code,words", [
    (dict(T=-1, cap=8), INVALID, "sizes"), (dict(k=0, cap=8), INVALID, "sizes"), (dict(E=0, cap=8), INVALID, "sizes"),
    (dict(align=0, cap=8), INVALID, "sizes"), (dict(k=17, E=64, cap=1000), TOO_LARGE, "limits"),
    (dict(E=1025, cap=1000), TOO_LARGE, "limits"), (dict(cap=7), TOO_LARGE, "smaller"), (dict(cap=2**31), TOO_LARGE, "limit"),
    (dict(pos=None), INVALID, "null"), (dict(perm=None), INVALID, "null"), (dict(counts=None), INVALID, "null"),
    (dict(offsets=None), INVALID, "null"), (dict(pos=P + 2), INVALID, "aligned"),
])
def test_plan_refusals(native, change, code, words):
    L = native.lib()
    p = C.byref(plan(native, **change))
    refused(native, L.omoe_sort_plan(p, P, None), code, words)
    refused(native, L.omoe_sort_rows(p, P, 8, 0, 9 * P, 8, 0, 8, None), code, words)
    refused(native, L.omoe_unsort_rows(p, P, 8, 0, None, 9 * P, 8, 0, 8, None), code, words)


def test_sort_refusals(native):
    L, p = native.lib(), C.byref(plan(native))
    refused(native, L.omoe_sort_plan(None, P, None), INVALID, "null plan")
    refused(native, L.omoe_sort_plan(p, None, None), INVALID, "null")
    # no tokens, but rows that the plan marks as empty
    refused(native, L.omoe_sort_plan(C.byref(plan(native, T=0, cap=64, pos=None, perm=None)), None, None), INVALID, "null")
    refused(native, L.omoe_sort_plan(p, P + 1, None), INVALID, "aligned")
    for idx in (P, P + 28, 2 * P, 3 * P + 28, 4 * P + 32):  # the picks in a buffer of the plan
        refused(native, L.omoe_sort_plan(p, idx, None), INVALID, "overlaps")
    refused(native, L.omoe_sort_plan(C.byref(plan(native, counts=4 * P + 4)), 8 * P, None), INVALID, "overlaps")
    good = [6 * P, 8, 0, 9 * P, 8, 0, 8]
    for at, value, words in ((0, None, "null"), (3, None, "null"), (1, 7, "leading"), (4, 7, "leading"), (1, 2**31, "leading"),
                             (2, 2, "dtype"), (5, -1, "dtype"), (6, 0, "d must"), (6, -8, "d must"), (0, 6 * P + 2, "aligned"),
                             (3, 6 * P, "overlaps"), (3, 6 * P + 16, "overlaps"), (3, P - 32, "overlaps")):
        args = list(good)
        args[at] = value
        refused(native, L.omoe_sort_rows(p, *args, None), INVALID, words)
        refused(native, L.omoe_sort_rows_backward(p, *args, None), INVALID, words)
        refused(native, L.omoe_unsort_rows(p, *args[:3], None, *args[3:], None), INVALID, words)
    refused(native, L.omoe_unsort_rows(p, 6 * P, 8, 0, P + 1, 9 * P, 8, 0, 8, None), INVALID, "aligned")
    refused(native, L.omoe_unsort_rows(p, 6 * P, 8, 0, 9 * P + 32, 9 * P, 8, 0, 8, None), INVALID, "overlaps")
    back = lambda **v: L.omoe_unsort_rows_backward(p, v.get("dy", 6 * P), v.get("lddy", 8), 0, v.get("ys", 9 * P), 8, v.get("t", 0),
                                                   v.get("w"), v.get("dys", 17 * P), 8, v.get("dw", 30 * P), v.get("d", 8), None)
    refused(native, back(dw=17 * P), INVALID, "overlaps")
    refused(native, back(dw=30 * P, w=30 * P), INVALID, "overlaps")
    refused(native, back(dw=4 * P), INVALID, "overlaps")
    refused(native, back(dy=None), INVALID, "null")
    refused(native, back(ys=None), INVALID, "null")
    refused(native, back(dys=None), INVALID, "null")
    refused(native, back(dys=9 * P), INVALID, "overlaps")
    refused(native, back(lddy=4), INVALID, "leading")
    refused(native, back(t=3), INVALID, "dtype")
    refused(native, back(dw=30 * P + 2), INVALID, "aligned")
    refused(native, back(d=0), INVALID, "d must")


def test_layer_norm_refusals(native):
    L = native.lib()
    good = [P, 8, 0, None, None, 1e-5, 9 * P, 8, 0, None, None, 4, 8]
    for at, value, words in ((0, None, "null"), (6, None, "null"), (1, 7, "leading"), (7, 7, "leading"), (2, 5, "dtype"),
                             (8, 5, "dtype"), (11, -1, "T must"), (12, 0, "d must"), (5, -1e-5, "eps"), (5, float("nan"), "eps"),
                             (0, P + 2, "aligned"), (3, P + 1, "aligned"), (9, P + 2, "aligned"), (6, P, "overlaps"),
                             (6, P + 64, "overlaps"), (9, P, "overlaps"), (10, 9 * P + 124, "overlaps")):
        args = list(good)
        args[at] = value
        refused(native, L.omoe_layer_norm(*args, None), INVALID, words)
    ws = L.omoe_layer_norm_backward_workspace
    assert ws(-1, 8) == INVALID and ws(4, 0) == INVALID and 0 < ws(0, 8) <= ws(4, 8) <= ws(100000, 8) and ws(4, 8) < ws(4, 16)
    good = [P, 8, 0, 9 * P, 8, 0, None, 17 * P, 18 * P, 19 * P, 8, 27 * P, 28 * P, 4, 8, 30 * P, ws(4, 8)]
    for at, value, words in ((0, None, "null"), (3, None, "null"), (9, None, "null"), (7, None, "null"), (8, None, "null"),
                             (1, 7, "leading"), (4, 7, "leading"), (10, 7, "leading"), (2, 5, "dtype"), (5, 5, "dtype"),
                             (13, -1, "T must"), (14, 0, "d must"), (9, P, "overlaps"), (9, 9 * P, "overlaps"), (11, P + 2, "aligned"), (11, 28 * P, "overlaps"), (12, 17 * P, "overlaps"),
                             (15, 19 * P, "overlaps"), (11, 30 * P, "overlaps"),
                             (15, None, "workspace"), (15, P + 8, "workspace"), (16, ws(4, 8) - 1, "workspace")):
        args = list(good)
        args[at] = value
        refused(native, L.omoe_layer_norm_backward(*args, None), INVALID, words)


def refs(native, *items):
    return (native.TensorRef * max(1, len(items)))(*[native.TensorRef(p, n, t, 0) for p, n, t in items])


def test_gradient_refusals(native):
    L, size = native.lib(), native.GRAD_WORKSPACE_BYTES
    one = refs(native, (P, 100, 0))
    refused(native, L.omoe_grad_norm(one, -1, 5 * P, 6 * P, size, None), INVALID, "list")
    refused(native, L.omoe_grad_norm(None, 1, 5 * P, 6 * P, size, None), INVALID, "list")
    for bad, words in (((P, 100, 2), "dtype"), ((P, -1, 0), "count"), ((P, 2**43, 0), "count"), ((None, 4, 0), "null"),
                       ((P + 2, 4, 0), "aligned"), ((P + 1, 4, 1), "aligned")):
        r = refs(native, bad)
        refused(native, L.omoe_grad_norm(r, 1, 5 * P, 6 * P, size, None), INVALID, words)
        refused(native, L.omoe_grad_scale(r, None, 1, 5 * P, 1.0, None), INVALID, words)
        refused(native, L.omoe_grad_clip(r, None, 1, 1.0, 5 * P, 6 * P, size, None), INVALID, words)
    N, W = 5 * P, 6 * P
    for norm, ws, n in ((None, W, size), (N + 2, W, size), (N, None, size), (N, W + 8, size), (N, W, size - 1), (W, W, size), (W + size - 4, W, size)):
        words = "workspace" if norm == N or norm and norm >= W else "norm_dev"
        refused(native, L.omoe_grad_norm(one, 1, norm, ws, n, None), INVALID, words)
        refused(native, L.omoe_grad_clip(one, None, 1, 1.0, norm, ws, n, None), INVALID, words)
    for limit in (-1.0, float("nan")):
        refused(native, L.omoe_grad_scale(one, None, 1, N, limit, None), INVALID, "max_norm")
        refused(native, L.omoe_grad_clip(one, None, 1, limit, N, W, size, None), INVALID, "max_norm")
    refused(native, L.omoe_grad_scale(one, None, 1, None, 1.0, None), INVALID, "norm_dev")
    scale = lambda g, o: L.omoe_grad_scale(refs(native, *g), None if o is None else refs(native, *o), len(g), N, 1.0, None)
    # the same tensor twice, overlapping tensors in any order, outputs that meet another's gradient
    for g, o in (([(P, 100, 0), (P, 100, 0)], None), ([(P + 396, 100, 0), (P, 100, 0)], None),
                 ([(P, 100, 0), (2 * P, 100, 0)], [(9 * P, 100, 0), (9 * P + 4, 100, 0)]),
                 ([(P, 100, 0), (2 * P, 100, 0)], [(2 * P, 100, 0), (9 * P, 100, 0)]),
                 ([(P, 100, 0)], [(P + 4, 100, 0)])):
        refused(native, scale(g, o), INVALID, "overlap")
    # the norm or the workspace among the gradients
    for norm, ws in ((P + 396, W), (N, P + 384), (N, P - size + 16)):
        refused(native, L.omoe_grad_norm(one, 1, norm, ws, size, None), INVALID, "overlaps a tensor")
        refused(native, L.omoe_grad_clip(one, None, 1, 1.0, norm, ws, size, None), INVALID, "overlaps a tensor")
    refused(native, L.omoe_grad_scale(one, None, 1, P, 1.0, None), INVALID, "overlaps a tensor")
    refused(native, L.omoe_grad_scale(refs(native, (P, 100, 0)), refs(native, (9 * P, 100, 0)), 1, 9 * P + 4, 1.0, None), INVALID, "overlaps a tensor")
    refused(native, scale([(P, 100, 0)], [(9 * P, 99, 0)]), INVALID, "count and dtype")
    refused(native, scale([(P, 100, 0)], [(9 * P, 100, 1)]), INVALID, "count and dtype")
    refused(native, scale([(P, 100, 0)], [(None, 100, 0)]), INVALID, "null")
    refused(native, scale([(P, 100, 0)], [(9 * P + 2, 100, 0)]), INVALID, "aligned")


def test_host_mirror_refuses_tensors_on_the_cpu(native):
    import torch

    from omega_ai_b200 import GradList, OmoeError, TokenSort, layer_norm

    with pytest.raises(OmoeError):
        layer_norm(torch.zeros(4, 8))
    with pytest.raises(OmoeError):
        layer_norm(torch.zeros(8))
    with pytest.raises(OmoeError):
        TokenSort(4, 17, 64)
    sort = TokenSort(4, 2, 8, device="cpu")
    with pytest.raises(OmoeError):
        sort.plan(torch.zeros(4, 2, dtype=torch.int32))
    with pytest.raises(OmoeError):
        sort.plan(torch.zeros(4, 2, dtype=torch.int64))
    with pytest.raises(OmoeError):
        GradList([torch.zeros(4)]).norm()
    with pytest.raises(OmoeError):
        GradList([torch.zeros(4, 4).t()[1:]])
    with pytest.raises(OmoeError):
        GradList([torch.zeros(4, dtype=torch.float16)])
    with pytest.raises(OmoeError):
        GradList([torch.zeros(4)], out=[torch.zeros(5)])
