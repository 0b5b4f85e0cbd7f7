"""CPU checks of scene.without_gradient and overwritten: what they mark is the tensor itself, and only a backward pass that
reaches it, or that needs what it held, raises."""
import pytest
import torch

from onereel_amd import _lib as L
from onereel_amd.scene import overwritten, without_gradient


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


def test_overwritten_tensors():
    leaf = torch.ones(4, requires_grad=True)
    x = leaf.exp()                                # keeps its result
    assert overwritten('this call', x, x, None) is x and x._version == 1
    with pytest.raises(L.HipValueError, match='this call has no gradient'):
        x.sum().backward()
    x = leaf.exp()
    with torch.no_grad():                         # unrecorded, but what exp has kept is gone
        overwritten('this call', x, x)
    with pytest.raises(RuntimeError, match='inplace'):
        x.sum().backward()
    y = leaf.exp()
    overwritten('this call', y.view(2, 2)[1:], torch.ones(2))     # a view of it, updated from tensors without gradients
    with pytest.raises(RuntimeError, match='inplace'):
        y.sum().backward()
    with torch.inference_mode():
        z = torch.ones(4)
        assert overwritten('this call', z, z) is z
    assert overwritten('this call', z, z) is z
