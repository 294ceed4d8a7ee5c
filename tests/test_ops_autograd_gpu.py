"""The operators beside torch's autograd: what they write is seen, so that a backward pass over an overwritten tensor is refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def calls():
    """(name, the tensor that is written, a call that writes it)"""
    from omega_ai_b200 import GradList, TokenSort, layer_norm, layer_norm_backward

    T, d, k, E = 12, 64, 2, 4
    new = lambda rows=T: torch.ones(rows, d, device="cuda")
    x, idx = torch.randn(T, d, device="cuda"), torch.randint(0, E, (T, k), dtype=torch.int32, device="cuda")
    _, mean, rstd = layer_norm(x, stats=True)
    sort = TokenSort(T, k, E)
    sort.plan(idx)
    xs, w = sort.sort(x), torch.rand(T, k, device="cuda")
    norm = torch.ones((), device="cuda")
    out = new()
    yield "layer_norm", out, lambda: layer_norm(x, out=out)
    dx = new()
    yield "layer_norm_backward", dx, lambda: layer_norm_backward(x, x, None, mean, rstd, out=dx)
    o = new(sort.rows_cap)
    yield "sort", o, lambda: sort.sort(x, out=o)
    s = new()
    yield "sort_backward", s, lambda: sort.sort_backward(xs, out=s)
    u = new()
    yield "unsort", u, lambda: sort.unsort(xs, w, out=u)
    b = new(sort.rows_cap)
    yield "unsort_backward", b, lambda: sort.unsort_backward(x, xs, w, out=b)
    g, g2, h, h2 = new(), new(), new(), new()
    yield "clip in place", g, lambda: GradList([g]).clip(0.5)
    yield "scale in place", g2, lambda: GradList([g2]).scale(norm, 0.5)
    yield "clip", h, lambda: GradList([x], out=[h]).clip(0.5)
    yield "scale", h2, lambda: GradList([x], out=[h2]).scale(norm, 0.5)


def test_written_tensors_are_known_to_autograd():
    for name, t, call in calls():
        leaf = torch.ones(t.shape, device="cuda", requires_grad=True)
        before = t._version
        y = (leaf * t).sum()  # saves t
        call()
        assert t._version > before, name
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


def test_tensors_of_inference_mode_are_written():
    with torch.inference_mode():
        for name, t, call in calls():
            call()
            assert (t != 1).any(), name


def test_read_tensors_stay_as_they_were():
    from omega_ai_b200 import GradList, layer_norm

    x = torch.randn(12, 64, device="cuda")
    version = x._version
    layer_norm(x)
    GradList([x]).norm()
    GradList([x], out=[torch.empty_like(x)]).clip(0.5)
    assert x._version == version


def test_a_new_plan_is_known_to_autograd():
    """Rows gathered by a plan's perm have a gradient by that perm: not by the next plan's."""
    from omega_ai_b200 import TokenSort

    sort = TokenSort(6, 2, 4)
    idx = torch.randint(0, 4, (6, 2), dtype=torch.int32, device="cuda")
    before = [t._version for t in (sort.pos, sort.perm, sort.counts, sort.offsets)]
    sort.plan(idx)
    assert all(t._version > v for t, v in zip((sort.pos, sort.perm, sort.counts, sort.offsets), before))
    picks = torch.randn(12, 8, device="cuda", requires_grad=True)
    y = picks.index_select(0, sort.perm).sum()  # saves perm
    sort.plan(idx.flip(0).contiguous())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
