"""Rotary positions with several axes, alone and behind the RMSNorm over all heads, and their gradients, against float64.

Tolerances, u = eps / 2 of the type, e = 2^-24. The turns of a pair are taken in fp64 and reach fp32 within half a turn of 0: off by
2^-26 turns, an angle off by under 2^-23; with the cosine and sine of it rounded, each is off by at most 2^-21. A rotated value
a c - b s is then off by 2^-20 (|a| + |b|). The RMSNorm's factor is good to 64 e (sums of at most 30 additions in a row and what
is around them): 2^-18 of its value, which multiplies. The gradient's bounds are those of the norm's gradient in fp32, 2^-17 of
the terms it is the difference of; the weights' sums over rows pass at most 256 + 48 additions: 2^-15 of the sum of magnitudes."""
import math

import pytest
import torch

from onereel_amd import _lib as L
from onereel_amd import rotary, wan
from onereel_amd.wan_dit import wan_rope_table

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'
TYPES = [torch.bfloat16, torch.float16, torch.float32]
EPS = 1e-6


def rounding(v, dtype):
    f = torch.finfo(dtype)
    return f.eps / 2 * v.abs() + f.smallest_normal * f.eps / 2


def angles(axes):
    """[S, pairs] in fp64"""
    freq = [t ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d) for d, t in zip(axes.dims, axes.theta)]
    return torch.cat([axes.positions[:, a:a + 1].double() * f for a, f in enumerate(freq)], 1)


def turned(axes, y, sign=1):
    """(y [.., S, H, D] rotated, the sum |a| + |b| of every value's pair)"""
    t = angles(axes)[:, None]
    c, s, n = t.cos(), sign * t.sin(), sum(axes.dims)
    out, mag = y.clone(), y.abs()
    pick = (slice(0, n // 2), slice(n // 2, n)) if axes.pairs == 'half' else (slice(0, n, 2), slice(1, n, 2))
    a, b = y[..., pick[0]], y[..., pick[1]]
    out[..., pick[0]], out[..., pick[1]] = a * c - b * s, a * s + b * c
    for p in pick:
        mag[..., p] = a.abs() + b.abs()
    return out, mag


def check(got, want, bound, what):
    assert bool(torch.isfinite(got.float()).all()), what
    past = (got.double().reshape(want.shape) - want).abs() - 1.001 * bound - 1e-30
    assert past.numel() == 0 or past.max().item() <= 0, f'{what}: {past.max().item():.3e} past its bound'


def positions(S, n, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(0, 60, (S, n), generator=g)
    if kind == 'far':
        p = p + torch.tensor([2 ** 24 + 1, 1000003, 99991, 5][:n])
    if kind == 'negative':
        p = p - 30
    p = p.float() * 0.37 - 3.3 if kind == 'fractional' else p.int()
    return p.to(DEV)


def rows(shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dtype)


CASES = [(1, 1, 8, (8,)), (5, 3, 16, (2, 4, 8)), (77, 2, 64, (16, 24, 24)), (33, 5, 96, (48, 48)), (130, 24, 128, (44, 42, 42)),
         (9, 40, 128, (32, 32, 32, 32)), (1001, 1, 72, (40, 32)), (3, 2, 512, (512,)), (64, 7, 40, (8, 16))]


@pytest.mark.parametrize('S,H,D,dims', CASES)
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('pairs', ['interleaved', 'half'])
@pytest.mark.parametrize('kind', ['near', 'far', 'fractional'])
def test_rotate(S, H, D, dims, dtype, pairs, kind):
    if pairs == 'half' and sum(dims) % 8:
        dims = (sum(dims) // 8 * 8,)
    print(f'rotate {S} x {H} x {D} {dims} {pairs} {kind} {dtype}', flush=True)
    axes = rotary.Axes(positions(S, len(dims), kind), dims, pairs=pairs)
    x = rows((S, H, D), dtype, S + H)
    for call, sign in ((rotary.rotate, 1), (rotary.rotate_backward, -1)):
        want, mag = turned(axes, x.double(), sign)
        check(call(x, axes), want, 2 ** -20 * mag + rounding(want, dtype), call.__name__)


def test_theta_per_axis_batches_and_strides():
    print('rotate strides', flush=True)
    axes = rotary.Axes(positions(50, 3, 'negative'), (16, 24, 24), theta=(256.0, 10000.0, 1.0))
    x = rows((2, 50, 6, 64), torch.bfloat16, 1)
    want, mag = turned(axes, x.double())
    got = rotary.rotate(x, axes)
    check(got, want, 2 ** -20 * mag + rounding(want, torch.bfloat16), 'batch')
    heads_first = x.transpose(1, 2).contiguous().transpose(1, 2)                  # [2, 6, 50, 64] in memory
    assert torch.equal(rotary.rotate(heads_first, axes), got)
    assert torch.equal(rotary.rotate(heads_first[0], axes), got[0])               # no copy: strides of its own
    wide = torch.zeros(50, 6, 128, dtype=torch.bfloat16, device=DEV)
    wide[..., 64:] = x[0]
    assert torch.equal(rotary.rotate(wide[..., 64:], axes), got[0])
    odd = torch.zeros(50 * 6 * 64 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(50, 6, 64)
    odd.copy_(x[0])
    assert torch.equal(rotary.rotate(odd, axes), got[0])
    one = x[0, :, :1].expand(50, 6, 64)                                             # a shared head
    assert torch.equal(rotary.rotate(one, axes)[:, 3], rotary.rotate(x[0, :, :1], axes)[:, 0])
    assert rotary.rotate(x[:0], axes).shape == (0, 50, 6, 64)


def test_many_rows():
    print('rotate many rows', flush=True)
    axes = rotary.grid(40, 30, 53, 128)
    x = rows((63600, 2, 128), torch.bfloat16, 4)
    want, mag = turned(axes, x.double())
    check(rotary.rotate(x, axes), want, 2 ** -20 * mag + rounding(want, torch.bfloat16), 'many')


def test_the_grid_is_the_tables():
    """the Axes of a grid against _qk with the tables of wan_rope_table: two roundings to bf16 of the same values to 2^-18"""
    print('rotary grid', flush=True)
    F, Hh, Ww, H, D = 5, 6, 7, 4, 128
    S, C = F * Hh * Ww, H * D
    q, k, w = rows((1, S, C), torch.bfloat16, 1), rows((1, S, C), torch.bfloat16, 2), 1 + 0.1 * rows((C,), torch.bfloat16, 3)
    table = [t.to(DEV) for t in wan_rope_table(F, Hh, Ww, D)]
    old = wan._qk(q, k, w, w, EPS, *table, H)
    new = rotary.norm_rotate(q, k, w, w, EPS, rotary.grid(F, Hh, Ww, D), H)
    for a, b in zip(old, new):
        assert a.shape == b.shape
        assert ((a.float() - b.float()).abs() <= 2 ** -7 * a.float().abs() + 1e-5).all()
        assert (a == b).float().mean() > 0.99


def reference(x, w, axes, H, dy):
    """float64 of one tensor: (y, bound), (dx, bound), (dw, bound)"""
    dtype, shape = x.dtype, x.shape
    S, C = axes.positions.shape[0], shape[-1]
    x, w, dy = x.double().reshape(-1, S, C), w.to(dtype).double(), dy.double().reshape(-1, S, H, C // H)
    inv = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
    n = x * inv
    y, mag = turned(axes, (n * w).unflatten(-1, (H, -1)))
    g, G = (t.flatten(-2) for t in turned(axes, dy, -1))
    mean = lambda t: t.mean(-1, keepdim=True)
    dx = inv * (g * w - n * mean(g * w * n))
    terms = inv * (G * w.abs() + n.abs() * mean(G * (w * n).abs()))
    return (y, 2 ** -18 * mag + rounding(y, dtype)), (dx, 2 ** -17 * terms + rounding(dx, dtype)), \
        ((g * n).sum((0, 1)), 2 ** -15 * (G * n.abs()).sum((0, 1)))


@pytest.mark.parametrize('S,H,D,dims', CASES[:3] + [(33, 5, 96, (48, 48)), (130, 24, 128, (44, 42, 42)), (700, 64, 128, (44, 42, 42)),
                                                    (7, 16, 512, (512,)), (2049, 4, 64, (20, 22, 22))])
@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('pairs', ['interleaved', 'half'])
def test_norm_rotate(S, H, D, dims, dtype, pairs):
    if pairs == 'half' and sum(dims) % 8:
        dims = (sum(dims) // 8 * 8,)
    print(f'norm rotate {S} x {H} x {D} {dims} {pairs} {dtype}', flush=True)
    axes, C = rotary.Axes(positions(S, len(dims), 'near'), dims, pairs=pairs), H * D
    q, k = rows((S, C), dtype, 1) * 3, rows((S, C), dtype, 2)
    wq, wk = 1 + 0.2 * rows((C,), torch.float32, 3), 1 + 0.2 * rows((C,), dtype, 4)
    dq, dk = rows((S, H, D), dtype, 5), rows((S, H, D), dtype, 6)
    y = rotary.norm_rotate(q, k, wq, wk, EPS, axes, H)
    grads = rotary.norm_rotate_backward(dq, dk, q, k, wq, wk, EPS, axes, H)
    for i, (x, w, d) in enumerate(((q, wq, dq), (k, wk, dk))):
        want = reference(x, w, axes, H, d)
        for got, (value, bound), what in zip((y[i], grads[i], grads[2 + i]), want, ('y', 'dx', 'dw')):
            check(got, value, bound, what)
    again = rotary.norm_rotate_backward(dq, dk, q, k, wq, wk, EPS, axes, H)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_norm_rotate_zero_rows_batches_strides_and_no_rows():
    print('norm rotate strides', flush=True)
    S, H, D = 40, 4, 64
    axes, C = rotary.Axes(positions(S, 2, 'far'), (32, 16)), H * D
    fused = rows((3, S, 3 * C), torch.bfloat16, 1)                     # views of a projection to q, k and v
    q, k = fused[..., :C], fused[..., C:2 * C]
    q[0, 3] = 0
    w = torch.ones(C, device=DEV)
    dq, dk = rows((3, S, H, D), torch.bfloat16, 5), torch.ones(1, 1, 1, 1, dtype=torch.bfloat16, device=DEV).expand(3, S, H, D)
    y = rotary.norm_rotate(q, k, w, w, EPS, axes, H)
    grads = rotary.norm_rotate_backward(dq, dk, q, k, w, w, EPS, axes, H)
    for i, (x, d) in enumerate(((q, dq), (k, dk))):
        want = reference(x, w, axes, H, d)
        for got, (value, bound), what in zip((y[i], grads[i], grads[2 + i]), want, ('y', 'dx', 'dw')):
            check(got, value, bound, what)
    none = rotary.norm_rotate_backward(dq[:0], dk[:0], q[:0], k[:0], w, w, EPS, axes, H)
    assert none[0].shape == (0, S, C) and not none[2].any()


def test_autograd_and_differences():
    print('rotary autograd', flush=True)
    S, H, D = 50, 3, 48
    axes, C = rotary.Axes(positions(S, 3, 'fractional'), (16, 8, 16), pairs='half'), 3 * 48
    q, k, dq, dk = (rows((1, S, C), torch.float32, i) for i in range(4))
    wq, wk = torch.rand(C, device=DEV) + 0.5, (torch.rand(C, device=DEV) + 0.5).double()
    dq, dk = (t.view(1, S, H, D) for t in (dq, dk))
    x = [t.clone().requires_grad_() for t in (q, k, wq, wk)]
    out = rotary.norm_rotate(*x, EPS, axes, H)
    plain = rotary.norm_rotate(q, k, wq, wk, EPS, axes, H)
    assert all(torch.equal(a, b) for a, b in zip(out, plain)) and not plain[0].requires_grad
    grads = torch.autograd.grad(out, x, (dq, dk))
    want = rotary.norm_rotate_backward(dq, dk, q, k, wq, wk, EPS, axes, H)
    assert all(torch.equal(a, b.to(a.dtype)) and a.dtype == t.dtype and a.shape == t.shape for a, b, t in zip(grads, want, x))
    y = q.view(S, H, D).clone().requires_grad_()
    r = rotary.rotate(y, axes)
    g, = torch.autograd.grad(r, y, dq[0])
    assert torch.equal(g, rotary.rotate_backward(dq[0], axes)) and torch.equal(r, rotary.rotate(q.view(S, H, D), axes))
    # along a direction, against the central difference of the formula in float64: fp32 gradients, 2^-15 of the magnitudes
    d = torch.randn(S, C, generator=torch.Generator().manual_seed(8), dtype=torch.float64).to(DEV)

    def f(x):
        n = x * (x.square().mean(1, keepdim=True) + EPS).rsqrt() * wk.float().double()
        return (turned(axes, n.view(S, H, D))[0] * dk[0].double()).sum()

    e = 1e-5
    num = (f(k[0].double() + e * d) - f(k[0].double() - e * d)) / (2 * e)
    assert (num - (grads[1][0].double() * d).sum()).abs() <= 2 ** -15 * (grads[1][0].double() * d).abs().sum()
    axes.positions.add_(1)
    r = rotary.rotate(y, axes)
    axes.positions.add_(1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        r.sum().backward()


def test_graph_replays_and_streams():
    print('rotary graph', flush=True)
    S, H, D = 300, 8, 128
    axes = rotary.Axes(positions(S, 3, 'near'), (44, 42, 42))
    bufs = [rows((S, H * D), torch.bfloat16, i) for i in range(4)]
    w = rows((H * D,), torch.bfloat16, 9)

    def step():
        q, k, dq, dk = bufs
        a = rotary.norm_rotate(q, k, w, w, EPS, axes, H)
        b = rotary.norm_rotate_backward(dq.view(S, H, D), dk.view(S, H, D), q, k, w, w, EPS, axes, H)
        return (*a, *b, rotary.rotate(q.view(S, H, D), axes))

    step()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for seed in (10, 20, 30):
        for i, b in enumerate(bufs):
            b.copy_(rows((S, H * D), torch.bfloat16, seed + i))
        want = step()
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for out in outs for a, b in zip(out, want)), seed
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for out in got for a, b in zip(out, want))


def test_refusals():
    p = torch.zeros(6, 2, dtype=torch.int32, device=DEV)
    axes = rotary.Axes(p, (8, 8))
    x, w = torch.zeros(6, 2, 16, dtype=torch.bfloat16, device=DEV), torch.ones(32, device=DEV)
    q = x.view(6, 32)
    bad = [lambda: rotary.Axes(p.long(), (8, 8)), lambda: rotary.Axes(p, (8, 8, 8)), lambda: rotary.Axes(p, (8, 8), pairs='rows'),
           lambda: rotary.Axes(p, (8, 8), theta=(1.0,)), lambda: rotary.rotate(x, rotary.Axes(p, (7, 9))),
           lambda: rotary.rotate(x, rotary.Axes(p, (8, 10))), lambda: rotary.rotate(x, rotary.Axes(p, (8, 0))),
           lambda: rotary.rotate(x, rotary.Axes(p, (8, 8), theta=math.inf)), lambda: rotary.rotate(x, rotary.Axes(p, (8, 8), theta=-1.0)),
           lambda: rotary.rotate(x, rotary.Axes(p, (4, 8), pairs='half')), lambda: rotary.rotate(x[:5], axes),
           lambda: rotary.rotate(x[..., :12], axes), lambda: rotary.rotate(x.double(), axes), lambda: rotary.rotate(q, axes),
           lambda: rotary.rotate(x, (p, p)), lambda: rotary.Axes(p.float().requires_grad_(), (8, 8)), lambda: rotary.rotate(x, rotary.Axes(p.cpu(), (8, 8))),
           lambda: rotary.norm_rotate(q, q, w, w, EPS, axes, 3), lambda: rotary.norm_rotate(q, q[:, :16], w, w, EPS, axes, 2),
           lambda: rotary.norm_rotate(q, q, w[:16], w, EPS, axes, 2), lambda: rotary.norm_rotate(q, q.float(), w, w, EPS, axes, 2),
           lambda: rotary.norm_rotate(q, q, w, w.cpu(), EPS, axes, 2), lambda: rotary.norm_rotate(q[:4], q[:4], w, w, EPS, axes, 2),
           lambda: rotary.norm_rotate_backward(x, x[:, :1], q, q, w, w, EPS, axes, 2)]
    for k, f in enumerate(bad):
        with pytest.raises(L.HipPathError):
            f()
            print(k)
