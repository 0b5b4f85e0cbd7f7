"""Gradients of the RMSNorm + RoPE at the width of the Wan-shaped DiT, against float64 with the tolerances of
test_gpu_norm_backward.py: q and k with rotary tables, and the RMSNorm alone on strided rows."""
import pytest
import torch

from helpers import rand_bf16
from onereel_amd import wan
from onereel_amd.wan_dit import DiTConfig
from test_gpu_norm_backward import check, reference, tables

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'


@pytest.mark.parametrize('S', [1, 3, 77, 2049, 5000])
def test_model_width(S):
    C, H = DiTConfig().dim, DiTConfig().heads
    D = C // H
    print(f'norm backward S={S} C={C}', flush=True)
    q, k, dq, dk = (rand_bf16((S, C), 3 + i).to(DEV) for i in range(4))
    dq, dk = dq.view(S, H, D), (dk / 64).view(S, H, D)
    wq, wk = ((1 + 0.2 * torch.randn(C, generator=torch.Generator().manual_seed(i))).bfloat16().to(DEV) for i in range(2))
    cos, sin = tables(S, D, 1)
    got = wan.qk_backward(dq, dk, q, k, wq, wk, 1e-6, cos, sin, H)
    for i, (d, x, w) in enumerate(((dq, q, wq), (dk, k, wk))):
        check(got[i], got[2 + i], *reference(d, x, w, 1e-6, cos, sin, H))
    again = wan.qk_backward(dq, dk, q, k, wq, wk, 1e-6, cos, sin, H)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    wide = rand_bf16((S, C + 64), 9).to(DEV)[:, 32:32 + C]
    check(*wan.rms_norm_backward(dq.view(S, C), wide, wq, 1e-5), *reference(dq, wide, wq, 1e-5))
