"""Arguments that contradict each other or the plan are refused before anything else: runs without a GPU."""
import pytest
import torch


@pytest.fixture(scope="module", autouse=True)
def built():
    from omega_ai_b200 import native

    native.build()


def test_picks_and_weights_of_another_shape():
    """[k, T] has as many elements as [T, k], in another order."""
    from omega_ai_b200 import OmoeError, TokenSort

    T, k = 6, 2
    sort = TokenSort(T, k, 8, device="cpu")
    idx, w = torch.zeros(k, T, dtype=torch.int32), torch.zeros(k, T)
    y, ys = torch.zeros(T, 8), torch.zeros(sort.rows_cap, 8)
    for call in (lambda: sort.plan(idx), lambda: sort.plan(idx.reshape(4, 3)), lambda: sort.unsort(ys, w), lambda: sort.unsort_backward(y, ys, w)):
        with pytest.raises(OmoeError, match=r"expected \[6, 2\]"):
            call()
    for call in (lambda: sort.plan(idx.reshape(T, k)), lambda: sort.plan(idx.reshape(-1)), lambda: sort.unsort(ys, w.reshape(-1))):
        with pytest.raises(OmoeError, match="on a GPU"):  # the next check
            call()


def test_a_dtype_that_is_not_that_of_out():
    from omega_ai_b200 import OmoeError, TokenSort, layer_norm

    sort = TokenSort(6, 2, 8, device="cpu")
    x, rows, bf = torch.zeros(6, 8), torch.zeros(sort.rows_cap, 8), torch.bfloat16
    for call in (lambda dt: layer_norm(x, out=torch.zeros(6, 8), dtype=dt), lambda dt: sort.sort(x, out=rows, dtype=dt),
                 lambda dt: sort.sort_backward(rows, out=x, dtype=dt), lambda dt: sort.unsort(rows, out=x, dtype=dt)):
        with pytest.raises(OmoeError, match="dtype"):
            call(bf)
        with pytest.raises(OmoeError, match="on a GPU"):
            call(torch.float32)
