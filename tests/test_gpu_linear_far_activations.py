"""SiLU's derivative far from 0, where it is small but no zero.

Tolerance. d = p + z p (1 - p), p = 1 / (1 + 2^x), x = -z log2(e): x is off by half a step, as is log2(e), so 2^x, and p where it
is small, by 2 |z| 2^-24 relative; exp2 and the reciprocal add 2^-21. Where p is near 1, 1 - p is off by 2^-24. So
|error| <= (1 + |z|) (p (2 |z| + 8) 2^-24 + 2^-23 where z > 0), and fp32 has no numbers below 2^-126 with all their bits: p below
that is lost, (1 + |z|) 2^-126 < 2^-119."""
import pytest
import torch

from onereel_amd.linear import linear, linear_backward

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'


def test_silu_gradient_far_out():
    print('silu far out', flush=True)
    z = torch.tensor([-3e38, -1e20, -200, -104, -99, -85, -60, -41, -30, -25, -22, -20.5, -20, -19.5, -17, -9, -2, 0, 2, 9, 20,
                      22, 60, 3e38], device=DEV).bfloat16()
    x, w = torch.zeros(2, 8, dtype=torch.bfloat16, device=DEV), torch.zeros(24, 8, dtype=torch.bfloat16, device=DEV)
    x[:, 0], w[:, 0] = 1, z
    kept = linear(x, w, activation='silu', keep_preactivation=True)[1]
    assert torch.equal(kept[0], z)
    dy = torch.ones(2, 24, dtype=torch.bfloat16, device=DEV)
    db = linear_backward(dy, x, w, bias=True, activation='silu', preactivation=kept)[2].double() / 2
    zd = z.double().clamp(-700, 700)
    p = torch.sigmoid(zd)
    want = p * (1 + zd * torch.sigmoid(-zd))
    room = (1 + zd.abs()) * (p * (2 * zd.abs() + 8) * 2 ** -24 + (zd > 0) * 2 ** -23) + 2 ** -119
    off = (db - want).abs() - room
    assert bool(torch.isfinite(db).all()) and off.max().item() <= 0, (z[off > 0], db[off > 0], want[off > 0])
