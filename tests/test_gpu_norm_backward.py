"""Gradients of the RMSNorm + RoPE and of the RMSNorm alone against float64.

Tolerance. g itself is a sum e0 c + e1 s of the rotation, each product and the sum off by 2^-24 relative: its error goes by
G = |e0 c| + |e1 s| (up to 2 * 2^-24 G), which cancellation leaves while g gets small. So every bound below is in G, not in
|g| (a first form of this file had |g|: one row of 512, where g = 2e-3 of G, already passes it). dx is rounded to bf16 once (half a step, 2^-8 relative) from fp32 arithmetic on at most 8192-element sums:
2^-8 |dx| + 2^-18 of the terms it is the difference of (G |w| inv, and |n| inv times the mean of G |w n|). dw is a fp32 sum over
the rows: 2^-20 of the sum of G |n| (each term is good to a few 2^-24, and no partial sum adds more than 2^7 terms in a
row without being an order of magnitude below this)."""
import pytest
import torch

from helpers import rand_bf16
from onereel_amd import wan

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'


def reference(dy, x, w, eps, cos=None, sin=None, heads=1):
    """float64 (dx, dw) and the magnitudes their rounding errors go by; all on the GPU"""
    S, C = x.shape
    g, x, w = dy.double().reshape(S, C), x.double(), w.double().reshape(C)
    G = g.abs()
    if cos is not None:
        c, s = cos.double()[:, None, 0::2], sin.double()[:, None, 1::2]
        g = g.view(S, heads, -1)
        G = torch.stack([(g[..., 0::2] * c).abs() + (g[..., 1::2] * s).abs(),
                         (g[..., 1::2] * c).abs() + (g[..., 0::2] * s).abs()], 3).reshape(S, C)
        g = torch.stack([g[..., 0::2] * c + g[..., 1::2] * s, g[..., 1::2] * c - g[..., 0::2] * s], 3).reshape(S, C)
    inv = (x.square().mean(1, keepdim=True) + eps).rsqrt()
    t, n = g * w, x * inv
    dx = inv * (t - n * (t * n).mean(1, keepdim=True))
    T = G * w.abs()
    mag = inv * (T + n.abs() * (T * n.abs()).mean(1, keepdim=True))
    return (dx, (g * n).sum(0)), (mag, (G * n.abs()).sum(0))


def check(dx, dw, ref, mags):
    assert bool(torch.isfinite(dx.float()).all()) and bool(torch.isfinite(dw).all()) and dw.dtype == torch.float32
    off = (dx.double().view_as(ref[0]) - ref[0]).abs() - (2 ** -8 * ref[0].abs() + 2 ** -18 * mags[0] + 1e-38)
    assert off.numel() == 0 or off.max().item() <= 0, f'dx {off.max().item():.3e} past its bound'
    off = (dw.double() - ref[1]).abs() - (2 ** -20 * mags[1] + 1e-38)
    assert off.max().item() <= 0, f'dw {off.max().item():.3e} past its bound'


def tables(S, D, seed):
    a = torch.rand(S, D // 2, generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * 6.3
    return tuple(t.float().repeat_interleave(2, 1).to(DEV) for t in (a.cos(), a.sin()))


@pytest.mark.parametrize('S,C', [(1, 512), (3, 1024), (4, 1536), (5, 2048), (77, 2560), (2049, 2048), (6000, 512), (9, 4096),
                                 (130, 6144), (131, 8192)])
@pytest.mark.parametrize('D', [64, 128])
def test_qk_backward(S, C, D):
    print(f'qk backward S={S} C={C} D={D}', flush=True)
    H = C // D
    q, k, dq, dk = (rand_bf16((S, C), 3 + i).to(DEV) for i in range(4))
    dq, dk = dq.view(S, H, D), (dk / 64).view(S, H, D)
    wq, wk = ((1 + 0.2 * torch.randn(C, generator=torch.Generator().manual_seed(i))).bfloat16().to(DEV) for i in range(2))
    cos, sin = tables(S, D, 1)
    got = wan.qk_backward(dq, dk, q, k, wq, wk, 1e-6, cos, sin, H)
    for i, (d, x, w) in enumerate(((dq, q, wq), (dk, k, wk))):
        check(got[i], got[2 + i], *reference(d, x, w, 1e-6, cos, sin, H))
    again = wan.qk_backward(dq, dk, q, k, wq, wk, 1e-6, cos, sin, H)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_rows_that_are_zero_large_and_small():
    print('norm extremes', flush=True)
    x = torch.zeros(5, 512, dtype=torch.bfloat16)
    x[1], x[2], x[3, 7] = 1e15, 1e-15, 3e4
    x[4] = rand_bf16((512,), 1)
    dy, w = rand_bf16((5, 512), 2), rand_bf16((512,), 3)
    g = [t.to(DEV) for t in (dy, x, w)]
    check(*wan.rms_norm_backward(*g, 1e-6), *reference(*g, 1e-6))


def test_strided_inputs_and_expanded_gradient():
    print('norm strides', flush=True)
    x = rand_bf16((40, 2048), 5).to(DEV)[:, 512:1536]
    w = torch.ones(1024, device=DEV)
    dy = torch.full((1, 1), 0.25, dtype=torch.bfloat16, device=DEV).expand(40, 1024)
    check(*wan.rms_norm_backward(dy, x, w, 1e-5), *reference(dy, x, w, 1e-5))


def test_no_rows():
    x = torch.zeros(0, 512, dtype=torch.bfloat16, device=DEV)
    dx, dw = wan.rms_norm_backward(x, x, torch.ones(512, device=DEV), 1e-6)
    assert dx.shape == (0, 512) and not dw.any()


def test_autograd_and_differences():
    print('norm autograd', flush=True)
    S, H, D = 50, 8, 64
    C = H * D
    q, k, dq, dk = (rand_bf16((1, S, C), 11 + i).to(DEV) for i in range(4))
    dq, dk = (t.view(1, S, H, D) for t in (dq, dk))
    wq, wk = torch.rand(C, device=DEV) + 0.5, (torch.rand(C, device=DEV) + 0.5).bfloat16()
    cos, sin = (t.view(1, S, 1, D) for t in tables(S, D, 4))
    x = [t.clone().requires_grad_() for t in (q, k, wq, wk)]
    out = wan._qk(*x, 1e-6, cos, sin, H)
    plain = wan._qk(q, k, wq, wk, 1e-6, cos, sin, H)
    assert all(torch.equal(a, b) for a, b in zip(out, plain)) and not plain[0].requires_grad
    grads = torch.autograd.grad(out, x, (dq, dk))
    want = wan.qk_backward(dq, dk, q, k, wq, wk, 1e-6, cos, sin, H)
    assert all(torch.equal(a, b.to(a.dtype)) and a.shape == t.shape and a.dtype == t.dtype
               for a, b, t in zip(grads, want, x))
    y = [t.clone().requires_grad_() for t in (q, wk)]
    g = torch.autograd.grad(wan.rms_norm(y[0], y[1], 1e-6), y, q)
    assert all(torch.equal(a, b.to(a.dtype)) for a, b in zip(g, wan.rms_norm_backward(q, q, wk, 1e-6)))
    # along a direction, against the central difference of the formula in float64: each of the S C rounded products is off by
    # at most 2^-8 |dx d|, dw by far less
    d = torch.randn(S, C, generator=torch.Generator().manual_seed(8), dtype=torch.float64).to(DEV)

    def f(x):
        n = x * (x.square().mean(1, keepdim=True) + 1e-6).rsqrt() * wk.double()
        return (n * q[0].double()).sum()

    e = 1e-6
    num = (f(q[0].double() + e * d) - f(q[0].double() - e * d)) / (2 * e)
    assert (num - (g[0][0].double() * d).sum()).abs() <= 2 ** -8 * (g[0][0].double() * d).abs().sum() + 1e-5


def test_graph_replays():
    print('norm graph', flush=True)
    S, C = 300, 1024
    bufs = [rand_bf16((S, C), i).to(DEV) for i in range(2)]
    w = rand_bf16((C,), 9).to(DEV)
    wan.rms_norm_backward(*bufs, w, 1e-6)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = wan.rms_norm_backward(*bufs, w, 1e-6)
    for seed in (20, 30, 40):
        for b in bufs:
            b.copy_(rand_bf16((S, C), seed))
        want = wan.rms_norm_backward(*bufs, w, 1e-6)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
