"""One timestep for all tokens of a WanDiT pass as a tensor or array of one element, of any shape and on the CPU or the GPU: the pass is
that of the number, bit for bit."""
import warnings

import numpy as np
import pytest
import torch

from test_gpu_dit_operators import DEV, inputs, model

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
KINDS = {'CPU [1]': lambda: torch.tensor([300.0]), 'CPU [1, 1]': lambda: torch.tensor([[300.0]]),
         'CPU 0-d': lambda: torch.tensor(300.0), 'CPU whole [1]': lambda: torch.tensor([300]),
         'GPU [1]': lambda: torch.tensor([300.0], device=DEV), 'GPU [1, 1]': lambda: torch.tensor([[300.0]], device=DEV),
         'GPU [1, 1, 1]': lambda: torch.full((1, 1, 1), 300.0, device=DEV), 'GPU whole [1, 1]': lambda: torch.full((1, 1), 300, device=DEV),
         'array [1]': lambda: np.array([300.0]), 'array [1, 1]': lambda: np.array([[300]])}


@pytest.mark.parametrize('kind', KINDS)
def test_one_element(kind):
    print(f'one timestep: {kind}', flush=True)
    m = model()
    tokens, text, axes, _ = inputs()
    t = KINDS[kind]()
    with torch.no_grad(), warnings.catch_warnings():
        warnings.simplefilter('error', DeprecationWarning)         # of arrays taken as numbers
        assert torch.equal(m.forward(tokens, t, text, axes), m.forward(tokens, 300.0, text, axes))
        assert torch.equal(m.differentiable_forward(tokens, t, text, axes), m.differentiable_forward(tokens, 300.0, text, axes))
