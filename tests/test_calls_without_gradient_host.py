"""CPU checks of scene.without_gradient: what it marks is the tensor itself, and only a backward pass that reaches it raises."""
import pytest
import torch

from onereel_amd import _lib as L
from onereel_amd.scene import without_gradient


def test_marked_output_is_the_tensor_itself():
    x, other, out = torch.ones(4, requires_grad=True), torch.ones(4, requires_grad=True), torch.zeros(4)
    got = without_gradient('this call', out, None, x)
    assert got is out and out.requires_grad
    out.add_(2)                                   # takes in-place operations
    assert torch.equal(out, torch.full((4,), 2.0))
    with pytest.raises(L.HipValueError, match='this call has no gradient'):
        (out * other).sum().backward()
    assert x.grad is None
    rest = torch.ones(4, requires_grad=True)
    (out.detach() * rest).sum().backward()        # a caller who wants the rest of the gradient alone detaches it
    assert torch.equal(rest.grad, torch.full((4,), 2.0))


def test_unmarked_where_nothing_is_lost():
    x, leaf = torch.ones(4), torch.ones(4, requires_grad=True)
    assert not without_gradient('', torch.zeros(4), x, None).requires_grad and without_gradient('', None, leaf) is None
    with torch.no_grad():
        assert not without_gradient('', torch.zeros(4), leaf).requires_grad
    with torch.inference_mode():
        assert not without_gradient('', torch.zeros(4), leaf).requires_grad
