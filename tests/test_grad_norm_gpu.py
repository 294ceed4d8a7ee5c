"""The global gradient norm and clipping against the same in 64 bits.

With u = 2^-24: squares are summed sixteen at a time in fp32 (each term rounded at most 7 times), then in 64 bits, so the norm is off
by at most 3.5 u relative, and u for its own rounding; the factor adds u, the product u, and the output half a step of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
BF, F32 = torch.bfloat16, torch.float32


def norm64(grads):
    return torch.stack([g.double().square().sum() for g in grads] or [torch.zeros((), dtype=torch.float64, device="cuda")]).sum().sqrt()


def check_norm(got, grads):
    ref = float(norm64(grads))
    assert got.dtype == F32 and abs(float(got) - ref) <= 5 * U * ref


def check_scaled(got, grads, c, types=None):
    for o, g in zip(got, grads):
        ref = g.double() * c
        assert ((o.double() - ref).abs() <= (HALF[g.dtype] + 8 * U) * ref.abs() + 2.0 ** -149).all()


def make(sizes, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(n, generator=g, device="cuda").mul_(10.0 ** -(i % 4)).to(t) for i, (n, t) in enumerate(sizes)]


LISTS = {
    "one element": [(1, F32)],
    "odd": [(7, F32), (4095, BF), (4096, F32), (4097, BF), (1, BF), (100003, F32)],
    "empty ones": [(0, F32), (5, F32), (0, BF), (0, F32), (9000, BF), (0, F32)],
    "full table": [(10 + i % 50, F32 if i % 3 else BF) for i in range(48)],
    "next table": [(10 + i % 50, F32 if i % 3 else BF) for i in range(49)],
    "two launches": [(1 + (i * 37) % 5000, F32 if i % 3 else BF) for i in range(1001)],
    "three launches": [(1 + (i * 37) % 100, F32 if i % 3 else BF) for i in range(2500)],
    "large": [(30_000_001, BF), (3, F32), (20_000_000, F32)],
}


@pytest.mark.parametrize("name", LISTS)
@pytest.mark.parametrize("limit", [0.25, 4.0])
def test_clip(name, limit):
    from omega_ai_b200 import GradList

    grads = make(LISTS[name])
    before = [g.clone() for g in grads]
    ref = float(norm64(before))
    max_norm = float(torch.tensor(limit * ref, dtype=F32))
    c = min(1.0, max_norm / (ref + 1e-6))
    check_norm(GradList(grads).norm(), before)
    # into other tensors
    out = [torch.full_like(g, 7.0) for g in grads]
    check_norm(GradList(grads, out=out).clip(max_norm), before)
    assert all(torch.equal(g, b) for g, b in zip(grads, before))
    if limit > 1:
        assert all(torch.equal(o, g) for o, g in zip(out, grads))
    check_scaled(out, before, c)
    # in place, and by a norm handed over
    check_norm(GradList(grads).clip(max_norm), before)
    assert all(torch.equal(g, o) for g, o in zip(grads, out))
    again = [b.clone() for b in before]
    GradList(again).scale(torch.tensor(ref, dtype=F32, device="cuda"), max_norm)
    check_scaled(again, before, c)


def test_empty_list():
    from omega_ai_b200 import GradList

    assert float(GradList([]).norm()) == 0.0 and float(GradList([]).clip(1.0)) == 0.0
    assert float(GradList([torch.empty(0, device="cuda")]).clip(1.0)) == 0.0
    GradList([]).scale(torch.ones((), device="cuda"), 1.0)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_views_at_any_element_and_their_neighbours(dtype):
    from omega_ai_b200 import GradList

    flat = torch.randn(300_000, device="cuda").to(dtype)
    before = flat.clone()
    spans = [(1, 5000), (5001, 12289), (20003, 3), (20006, 8192), (100_000, 4096), (150_002, 70_001)]
    grads = [flat[a:a + n] for a, n in spans]
    norm = GradList(grads).clip(0.5)
    views = [before[a:a + n] for a, n in spans]
    check_norm(norm, views)
    check_scaled(grads, views, 0.5 / (float(norm64(views)) + 1e-6))
    for a, n in spans:
        flat[a:a + n] = before[a:a + n]
    assert torch.equal(flat, before)


def test_outputs_at_other_alignments():
    from omega_ai_b200 import GradList

    grads = make([(9001, F32), (9001, BF), (9001, F32)])
    room = [torch.full((9010,), 3.0, dtype=g.dtype, device="cuda") for g in grads]
    out = [r[a:a + 9001] for r, a in zip(room, (1, 3, 4))]
    GradList(grads, out=out).clip(1.0)
    check_scaled(out, grads, 1.0 / (float(norm64(grads)) + 1e-6))
    for r, a in zip(room, (1, 3, 4)):
        assert (r[:a] == 3).all() and (r[a + 9001:] == 3).all()


@pytest.mark.parametrize("size", [2.0 ** 66, 2.0 ** 100, 2.0 ** -80, 2.0 ** -140, 0.0])
def test_squares_neither_overflow_nor_vanish(size):
    from omega_ai_b200 import GradList

    grads = [torch.full((5000,), size, device="cuda"), torch.full((300,), size, device="cuda").to(BF)]
    check_norm_floor = GradList(grads).norm()
    ref = float(norm64(grads))
    assert abs(float(check_norm_floor) - ref) <= 5 * U * ref + 2.0 ** -149
    mixed = [torch.full((3,), size, device="cuda"), torch.ones(7, device="cuda")]
    check_norm(GradList(mixed).norm(), mixed)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_a_norm_that_is_not_finite_leaves_the_gradients(value):
    from omega_ai_b200 import GradList

    grads = make([(5000, F32), (70, BF)])
    grads[0][4999] = value
    before = [g.clone() for g in grads]
    out = [torch.zeros_like(g) for g in grads]
    norm = GradList(grads, out=out).clip(0.1)
    assert not norm.isfinite()
    GradList(grads).clip(0.1)
    for g, o, b in zip(grads, out, before):
        assert torch.equal(g.nan_to_num(5.0), b.nan_to_num(5.0)) and torch.equal(o.nan_to_num(5.0), b.nan_to_num(5.0))


def test_limits_of_zero_and_infinity():
    from omega_ai_b200 import GradList

    grads = make([(5000, F32), (70, BF)])
    before = [g.clone() for g in grads]
    GradList(grads).clip(float("inf"))
    assert all(torch.equal(g, b) for g, b in zip(grads, before))
    GradList(grads).clip(0.0)
    assert all((g == 0).all() for g in grads)
    assert float(GradList(grads).clip(1.0)) == 0.0


def test_same_bits_every_time_and_from_graphs():
    from omega_ai_b200 import GradList

    grads = make([(3_000_001, F32), (70_000, BF)] + [(100 + i, F32) for i in range(60)])
    out = [torch.empty_like(g) for g in grads]
    gl = GradList(grads, out=out)
    norm = gl.clip(0.5)
    want = [o.clone() for o in out]
    for _ in range(5):
        assert torch.equal(gl.clip(0.5), norm) and all(torch.equal(o, w) for o, w in zip(out, want))
    # two captured norms share no workspace
    graphs, norms = [], []
    for limit in (0.5, 0.25):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(gl.norm())
        graphs.append(g)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(n, norm) for n in norms)


def test_more_than_32_bits_of_elements():
    from omega_ai_b200 import GradList

    n = 2**31 + 12345
    g = torch.zeros(n, dtype=BF, device="cuda")
    at = [0, 5, 2**31 - 1, 2**31, n - 1]
    g[at] = torch.tensor([3.0, 1.0, 4.0, 1.0, 5.0], dtype=BF, device="cuda")
    norm = GradList([g]).clip(0.5)
    ref = 52.0 ** 0.5
    assert abs(float(norm) - ref) <= 5 * U * ref
    want = torch.tensor([3.0, 1.0, 4.0, 1.0, 5.0], dtype=torch.float64) * (0.5 / (ref + 1e-6))
    assert ((g[at].double().cpu() - want).abs() <= (HALF[BF] + 8 * U) * want).all()
