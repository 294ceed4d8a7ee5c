"""A list of gradients keeps its tensors' addresses: once a tensor has other memory, a call must not touch the old one.  Runs without a GPU
(the check comes before everything else)."""
import pytest
import torch


@pytest.fixture(scope="module", autouse=True)
def built():
    from omega_ai_b200 import native

    native.build()


@pytest.mark.parametrize("change", [
    lambda t: t.set_(torch.zeros(8)), lambda t: t.resize_(100000), lambda t: t.untyped_storage().resize_(0),
    lambda t: setattr(t, "data", torch.zeros(8)), lambda t: t.resize_(4),
])
@pytest.mark.parametrize("which", ["grads", "out"])
def test_tensors_that_moved_are_refused(change, which):
    from omega_ai_b200 import GradList, OmoeError

    grads, out = [torch.zeros(3), torch.zeros(8)], [torch.zeros(3), torch.zeros(8)]
    lists = [GradList(grads, out=out)] + ([GradList(grads)] if which == "grads" else [])
    change((grads if which == "grads" else out)[1])
    for gl in lists:
        for call in (lambda: gl.clip(1.0), lambda: gl.scale(torch.ones(()), 1.0), *([gl.norm] if which == "grads" else [])):
            with pytest.raises(OmoeError, match="another storage or size"):
                call()
