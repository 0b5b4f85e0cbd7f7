"""Calls on leaves that require gradients are refused with the errors of the calls on other tensors, on a machine without a GPU
too."""
import pytest
import torch

from onereel_amd import _lib as L
from onereel_amd import attention as A
from onereel_amd import wan
from onereel_amd.linear import linear


def bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16, requires_grad=True)


CU, ROWS = torch.tensor([0, 4], dtype=torch.int32), [(0, 4)]
CALLS = {
    'varlen': lambda x, w: A.varlen(x, x, x, CU, CU, 4, 4),
    'varlen_lse': lambda x, w: A.varlen_lse(x, x, x, CU, CU, 4, 4),
    'packed': lambda x, w: A.packed([(x, x, x)]),
    'packed_lse': lambda x, w: A.packed_lse([(x, x, x)]),
    'overlapping_ranges': lambda x, w: A.overlapping_ranges(x, x, x, ROWS, ROWS),
    'dense': lambda x, w: A.dense(x[None], x[None], x[None]),
    'rms_norm': lambda x, w: wan.rms_norm(x.view(1, 512), w, 1e-6),
    'qk': lambda x, w: wan._qk(x.view(4, 128), x.view(4, 128), w[:128], w[:128], 1e-6, torch.ones(4, 64), torch.ones(4, 64), 2),
    'linear': lambda x, w: linear(x.view(4, 128), bf(64, 128)),
}


@pytest.mark.parametrize('call', CALLS)
def test_leaves_on_the_cpu(call):
    with torch.no_grad(), pytest.raises((L.HipPathError, ValueError)) as plain:
        CALLS[call](bf(4, 2, 64), torch.ones(512, requires_grad=True))
    with pytest.raises((L.HipPathError, ValueError)) as recorded:
        CALLS[call](bf(4, 2, 64), torch.ones(512, requires_grad=True))
    assert recorded.type is plain.type and str(recorded.value) == str(plain.value)
