"""The dims of a head past the rotated ones: handed on as they are, bit for bit, whatever their neighbours hold, and none of what they
hold reaches a rotated dim."""
import math

import pytest
import torch

from onereel_amd import rotary

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'
TYPES = [torch.bfloat16, torch.float16, torch.float32]
BITS = {2: torch.int16, 4: torch.int32}
# dims of a head, of its axes; of interleaved pairs the last unit of 8 dims may be rotated in part
CASES = [(64, (16, 8), 'interleaved'), (64, (10, 6, 2), 'interleaved'), (40, (2,), 'interleaved'), (64, (16, 8), 'half'),
         (96, (40,), 'half')]


def case(D, dims, pairs, dtype, S=11, H=3):
    g = torch.Generator(device=DEV).manual_seed(D + sum(dims))
    axes = rotary.Axes(torch.randint(0, 50, (S, len(dims)), generator=g, device=DEV).int(), dims, pairs=pairs)
    x = torch.randn(S, H, D, generator=g, device=DEV).to(dtype)
    at = sum(dims)
    # infinities of both signs, NaN, negative zeros and the type's largest value, beside finite values and one another
    special = torch.tensor([math.inf, 1.0, -math.inf, -math.inf, math.nan, -2.0, -0.0, -1.0, torch.finfo(dtype).max, math.inf], device=DEV)
    y = x.clone()
    for r in range(S):
        for i in range(D - at):
            if (r + i) % 3:
                y[r, :, at + i] = special[(2 * r + i) % 10].to(dtype)
    return axes, x, y, at


def bits(t):
    return t.contiguous().view(BITS[t.element_size()])


@pytest.mark.parametrize('D,dims,pairs', CASES)
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_rotate(D, dims, pairs, dtype):
    print(f'rotate past {dims} of {D} {pairs} {dtype}', flush=True)
    axes, x, y, at = case(D, dims, pairs, dtype)
    for call in (rotary.rotate, rotary.rotate_backward):
        clean, got = call(x, axes), call(y, axes)
        assert torch.equal(bits(clean[..., at:]), bits(x[..., at:]))
        finite = ~y[..., at:].isnan()
        assert torch.equal(bits(got[..., at:])[finite], bits(y[..., at:])[finite])
        assert bool(got[..., at:][~finite].isnan().all())
        assert torch.equal(bits(got[..., :at]), bits(clean[..., :at]))


@pytest.mark.parametrize('D,dims,pairs', CASES)
@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_norm_rotate_with_weights_that_are_not_finite(D, dims, pairs, dtype):
    """an infinite weight of an unrotated dim makes that dim infinite and no other"""
    print(f'norm_rotate past {dims} of {D} {pairs} {dtype}', flush=True)
    axes, x, _, at = case(D, dims, pairs, dtype)
    S, H = x.shape[:2]
    rows = x.reshape(S, H * D)
    w = torch.ones(H, D, dtype=dtype, device=DEV)
    clean, _ = rotary.norm_rotate(rows, rows, w.reshape(-1), w.reshape(-1), 1e-6, axes, H)
    w[:, at] = math.inf
    w[:, D - 2] = math.nan
    got, _ = rotary.norm_rotate(rows, rows, w.reshape(-1), w.reshape(-1), 1e-6, axes, H)
    hit = torch.zeros(D, dtype=torch.bool, device=DEV)
    hit[at] = hit[D - 2] = True
    assert torch.equal(got[..., ~hit], clean[..., ~hit])
    assert bool(got[..., D - 2].isnan().all())
    if at != D - 2:
        assert bool(got[..., at].isinf().all())
