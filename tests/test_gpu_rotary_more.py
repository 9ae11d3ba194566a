"""rotate where the first tests of it do not look: tensors that a backward pass has saved."""
import pytest
import torch

from polar_pack_amd.rotary import Rotary, rotate
from serving import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("place", ["x", "other"])
def test_a_saved_tensor_that_is_written_over_is_noticed(place):
    leaf = torch.randn(3, 2, 64, device=DEV, requires_grad=True)
    saved = leaf * 2.0
    loss = (saved * saved).sum()                              # keeps `saved` for its gradient
    x, r, pos = (saved if place == "x" else torch.randn(3, 2, 64, device=DEV)), Rotary(64), torch.arange(3, device=DEV)
    want = rotate(x.detach().clone(), r, pos)
    assert torch.equal(rotate(x, r, pos, out=saved), want)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_tensors_without_versions():
    """Made in inference mode they have none, in or outside of it."""
    r, pos = Rotary(64), torch.arange(3, device=DEV)
    with torch.inference_mode():
        x = torch.randn(3, 2, 64, device=DEV)
        want = rotate(x, r, pos)
        assert torch.equal(rotate(x, r, pos, out=torch.empty_like(x)), want)
    other = torch.empty(3, 2, 64, device=DEV)
    assert torch.equal(rotate(x, r, pos, out=other), want)
    assert torch.equal(rotate(x, r, pos, out=x), want)
