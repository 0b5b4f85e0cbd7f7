"""Norms before and after a sub-block with gate, residual and modulation, and their gradient, against float64.

Tolerances, u = eps / 2 of the rows' type, e = 2^-24. A sum over C <= 8192 columns passes at most 8 + 6 + 16 additions one after
the other (a thread's, a wavefront's, the wavefronts'), so with the divisions and products around it each statistic is good to
under 64 e of the sum of its terms' magnitudes:
  xh = (v - m) inv is off by at most X = 2^-17 (inv (|v| + mean |v|) + |xh|);
  of v itself off by D (a norm of a computed row) by inv (D + mean D + |xh| mean(|xh| D)) more;
  a gradient inv (t - mean t - xh mean(t xh)) by N = 2^-17 inv (|t| + mean |t| + |xh| mean |t xh|) + inv (X mean |t xh| + |xh|
  mean(|t| X)), and of t off by D by inv (D + mean D + |xh| mean(|xh| D)) more.
A column's sum over rows passes at most 256 + 64 + 16 additions (a thread's rows, the work-groups' sums, their wavefronts'), then
those over groups: 2^-15 of the sum of magnitudes and the errors of its terms. Every result is rounded to its type once: u of
it, or half a step of the smallest numbers."""
import pytest
import torch

from onereel_amd import _lib as L
from onereel_amd import norms

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'
TYPES = [torch.bfloat16, torch.float16, torch.float32]
EPS = 1e-6


def rounding(v, dtype):
    f = torch.finfo(dtype)
    return f.eps / 2 * v.abs() + f.smallest_normal * f.eps / 2


def mean(v):
    return v.mean(1, keepdim=True)


def standard(v, kind, D=None):
    """xh, inv and the error of xh, of rows v that are themselves off by D"""
    m = mean(v) if kind == 'layer' else torch.zeros_like(mean(v))
    inv = (mean((v - m).square()) + EPS).rsqrt()
    xh = (v - m) * inv
    off = 2 ** -17 * (inv * (v.abs() + mean(v.abs())) + xh.abs())
    if D is not None:
        off = off + inv * (D + mean(D) + xh.abs() * mean(xh.abs() * D))
    return xh, inv, off


def standard_grad(t, xh, inv, X, kind, D=None):
    a, p = t.abs(), mean(t.abs() * xh.abs())
    g = inv * (t - xh * mean(t * xh) - (mean(t) if kind == 'layer' else 0))
    off = 2 ** -17 * inv * (a + mean(a) + xh.abs() * p) + inv * (X * p + xh.abs() * mean(a * X))
    if D is not None:
        off = off + inv * (D + mean(D) + xh.abs() * mean(xh.abs() * D))
    return g, off


def wide(t, rows):
    """a parameter as fp64 rows, one for every row"""
    if t is None:
        return None
    t = t.double().reshape(-1, t.shape[-1])
    return t.repeat_interleave(rows // t.shape[0], 0)


def forward(x, a, norm, gate, r, post, wp, w, b, scale, shift):
    """(h, its bound, n, its bound)"""
    rows, C = x.numel() // x.shape[-1], x.shape[-1]
    dtype, h, D = x.dtype, x.double().reshape(rows, C), None
    one = torch.ones(1, C, dtype=torch.float64, device=DEV)
    if a is not None:
        p = a.double().reshape(rows, C)
        X = torch.zeros_like(p)
        if post:
            p, _, X = standard(p, post)
        G = (one if gate is None else wide(gate, rows)) * (1 if wp is None else wp.double())
        D = G.abs() * X + 2 ** -21 * ((r * h).abs() + (p * G).abs())
        h = r * h + p * G
    xh, _, X = standard(h, norm, D)
    s = one if scale is None else 1 + wide(scale, rows)
    W = (one if w is None else w.double()) * s
    B = (0 if b is None else b.double()) * s + (0 if shift is None else wide(shift, rows))
    n = xh * W + B
    parts = (0 if b is None else (b.double() * s).abs()) + (0 if shift is None else wide(shift, rows).abs())
    off = X * W.abs() + 2 ** -20 * ((xh * W).abs() + parts)
    return h, rounding(h, dtype) + (0 if D is None else D), n, rounding(n, dtype) + off


def backward(dh, dn, h, a, norm, gate, r, post, wp, w, b, scale, shift):
    """[(gradient, bound)] in the order of the call's results"""
    rows, C, dtype = h.numel() // h.shape[-1], h.shape[-1], h.dtype
    flat = lambda t: t.double().reshape(rows, C)
    one = torch.ones(1, C, dtype=torch.float64, device=DEV)
    groups = max([t.numel() // C for t in (gate, scale, shift) if t is not None] or [1])
    per_group = lambda t: t.view(groups, -1, C).sum(1)
    xh, inv, X = standard(flat(h), norm)
    n = flat(dn)
    s = one if scale is None else 1 + wide(scale, rows)
    W = (one if w is None else w.double()) * s
    d, D = standard_grad(n * W, xh, inv, X, norm, 2 ** -22 * (n * W).abs())
    A, A_off = n * xh, n.abs() * X + 2 ** -15 * (n * xh).abs()
    B_off = 2 ** -15 * n.abs()
    out = []
    if a is not None:
        d, D = (d, D) if dh is None else (d + flat(dh), D + 2 ** -23 * flat(dh).abs())
        out.append((r * d, abs(r) * D + 2 ** -23 * (r * d).abs() + rounding(r * d, dtype)))
        p, X = flat(a), torch.zeros_like(d)
        if post:
            p, pinv, X = standard(p, post)
        gate_rows = one if gate is None else wide(gate, rows)
        G = gate_rows * (1 if wp is None else wp.double())
        u, U = d * G, D * G.abs() + 2 ** -22 * (d * G).abs()
        da, E = standard_grad(u, p, pinv, X, post, U) if post else (u, U)
        out.append((da, E + rounding(da, dtype)))
        y = d * p
        Y = D * p.abs() + (d.abs() + D) * X + 2 ** -15 * y.abs()
        v = 1 if wp is None else wp.double()
        out.append(None if gate is None else (per_group(y) * v, per_group(Y) * abs(v)))
        out.append(None if wp is None else ((y * gate_rows).sum(0), (Y * gate_rows.abs()).sum(0)))
    else:
        out.append((d, D + rounding(d, dtype)))
    out.append(None if w is None else ((A * s).sum(0), (A_off * s.abs()).sum(0)))
    out.append(None if b is None else ((n * s).sum(0), (B_off * s.abs()).sum(0)))
    w, b = (0 if t is None else t.double() for t in (one if w is None else w, b))
    out.append(None if scale is None else (per_group(A) * w + per_group(n) * b, per_group(A_off) * abs(w) + per_group(B_off) * abs(b)))
    out.append(None if shift is None else (per_group(n), per_group(B_off)))
    return out


def check(got, want, bound, what):
    assert bool(torch.isfinite(got.float()).all()), what
    got = got.double().reshape(want.shape)
    past = (got - want).abs() - 1.001 * bound - 1e-30
    assert past.numel() == 0 or past.max().item() <= 0, f'{what}: {past.max().item():.3e} past its bound'


def inputs(rows, C, groups, dtype, residual, gated, post, affine, modulated, bias=True, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x = (randn(rows, C) * (1 + 9 * (randn(C) > 2).float()) + 0.5 * randn(C)).to(dtype)
    some = lambda wanted, *s: 0.3 * randn(*s) if wanted else None
    return dict(x=x, a=randn(rows, C).to(dtype) if residual else None, gate=some(gated, groups, C),
                wp=1 + 0.2 * randn(C) if post and affine else None, w=1 + 0.2 * randn(C) if affine else None,
                b=some(affine and bias, C), scale=some(modulated, groups, C), shift=some(modulated, groups, C),
                dn=randn(rows, C).to(dtype), dh=randn(rows, C).to(dtype) if residual else None)


def run(i, norm, post, r):
    pre = dict(norm=norm, weight=i['w'], bias=i['b'], scale=i['scale'], shift=i['shift'])
    add = dict(gate=i['gate'], residual_scale=r, post_norm=post, post_weight=i['wp'])
    how = (norm, i['gate'], r, post, i['wp'], i['w'], i['b'], i['scale'], i['shift'])
    h, hb, n, nb = forward(i['x'], i['a'], *how)
    if i['a'] is None:
        check(norms.norm_modulate(i['x'], EPS, **pre), n, nb, 'n')
        got = norms.norm_modulate_backward(i['dn'], i['x'], EPS, **pre)
        at = i['x']
    else:
        at, m = norms.residual_norm_modulate(i['x'], i['a'], EPS, **pre, **add)
        check(at, h, hb, 'h')
        check(m, n, nb, 'n')
        got = norms.residual_norm_modulate_backward(i['dh'], i['dn'], at, i['a'], EPS, **pre, **add)
    want = backward(i['dh'], i['dn'], at, i['a'], *how)
    assert len(got) == len(want)
    for k, (x, y) in enumerate(zip(got, want)):
        assert (x is None) == (y is None), k
        if y is not None:
            check(x, *y, f'gradient {k}')
    return got


SHAPES = [(1, 8, 1), (3, 64, 1), (5, 72, 5), (7, 512, 1), (77, 520, 7), (513, 1000, 3), (96, 1024, 96), (2, 2560, 1),
          (33, 4096, 3), (9, 8192, 1), (6, 8184, 2), (3001, 256, 1)]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows,C,groups', SHAPES)
@pytest.mark.parametrize('norm,post', [('layer', None), ('rms', 'rms'), ('layer', 'layer'), ('rms', 'layer')])
def test_residual(rows, C, groups, dtype, norm, post):
    print(f'norms {rows} x {C}, {groups} groups, {dtype}, {norm} after {post}', flush=True)
    if post == 'layer' and rows == 1:
        rows, groups = 2, 1
    i = inputs(rows, C, groups, dtype, True, True, post, True, True, seed=rows + C)
    got = run(i, norm, post, 0.75)
    again = run(i, norm, post, 0.75)
    assert all(x is None or torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('norm', ['layer', 'rms'])
@pytest.mark.parametrize('affine,modulated,residual,gated', [(0, 0, 0, 0), (1, 0, 0, 0), (0, 1, 0, 0), (1, 1, 0, 0), (0, 0, 1, 0),
                                                             (1, 0, 1, 1), (0, 1, 1, 0)])
def test_options(dtype, norm, affine, modulated, residual, gated):
    print(f'norms options {norm} {affine} {modulated} {residual} {gated} {dtype}', flush=True)
    run(inputs(150, 640, 5, dtype, residual, gated, None, affine, modulated, bias=norm == 'layer'), norm, None, 1.0)


def test_many_groups_and_long_groups():
    print('norms groups', flush=True)
    run(inputs(2400, 128, 2400, torch.bfloat16, True, True, None, True, True), 'layer', None, 1.0)    # one row each
    run(inputs(20000, 64, 5000, torch.bfloat16, False, False, None, True, True), 'rms', None, 1.0)    # more than one grid of sums
    run(inputs(140001, 64, 1, torch.bfloat16, True, True, 'rms', True, False), 'rms', 'rms', 1.0)


def test_rows_that_are_zero_constant_large_and_small():
    print('norms extremes', flush=True)
    i = inputs(6, 512, 1, torch.bfloat16, True, True, None, True, True)
    i['x'][0], i['a'][0] = 0, 0
    i['x'][1], i['a'][1] = 3.5, 0
    i['x'][2] *= 1e15
    i['x'][3], i['a'][3] = i['x'][3] * 1e-15, i['a'][3] * 1e-15
    run(i, 'layer', None, 1.0)
    run(i, 'rms', None, 1.0)


def test_missing_gradients_and_a_residual_nothing_else_reads():
    print('norms no dh', flush=True)
    i = inputs(70, 256, 2, torch.bfloat16, True, True, None, False, True)
    i['dh'] = None
    run(i, 'layer', None, 1.0)


def test_strides_types_of_parameters_and_an_expanded_gradient():
    print('norms strides', flush=True)
    i = inputs(40, 512, 4, torch.bfloat16, True, True, None, True, True)
    base = torch.zeros(40, 1200, dtype=torch.bfloat16, device=DEV)
    views = {}
    for k, off in (('x', 0), ('a', 640)):
        base[:, off:off + 512] = i[k]
        views[k] = base[:, off:off + 512]
    odd = torch.zeros(40 * 512 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(40, 512)     # off its 16 bytes
    odd.copy_(i['dn'])
    i['w'], i['scale'] = i['w'].bfloat16(), i['scale'].half()
    i['dh'] = torch.full((1, 1), 0.25, dtype=torch.bfloat16, device=DEV).expand(40, 512)
    want = run(i, 'layer', None, 1.0)
    i.update(views, dn=odd)
    got = run(i, 'layer', None, 1.0)
    assert all(x is None or torch.equal(x, y) for x, y in zip(got, want))


def test_leading_dimensions_and_no_rows():
    x = torch.randn(2, 3, 5, 64, device=DEV).bfloat16()
    s = torch.randn(2, 1, 1, 64, device=DEV)
    y = norms.norm_modulate(x, EPS, scale=s, shift=s)
    assert y.shape == x.shape
    assert torch.equal(y[1], norms.norm_modulate(x[1], EPS, scale=s[1], shift=s[1]))
    h, n = norms.residual_norm_modulate(x[:0], x[:0], EPS, weight=s[0, 0, 0])
    assert h.shape == n.shape == (0, 3, 5, 64)
    grads = norms.residual_norm_modulate_backward(None, n, h, h, EPS, weight=s[0, 0, 0], gate=s[0, 0, 0])
    assert grads[0].shape == (0, 3, 5, 64) and not grads[2].any() and not grads[4].any()


def test_autograd_and_differences():
    print('norms autograd', flush=True)
    i = inputs(60, 256, 3, torch.float32, True, True, 'rms', True, True)
    names = ('x', 'a', 'gate', 'wp', 'w', 'b', 'scale', 'shift')
    leaves = {k: i[k].clone().requires_grad_() for k in names}

    def call(t):
        return norms.residual_norm_modulate(t['x'], t['a'], EPS, norm='layer', gate=t['gate'], residual_scale=0.5,
                                            post_norm='rms', post_weight=t['wp'], weight=t['w'], bias=t['b'], scale=t['scale'],
                                            shift=t['shift'])

    h, n = call(leaves)
    plain = call(i)
    assert torch.equal(h, plain[0]) and torch.equal(n, plain[1]) and not plain[0].requires_grad
    grads = torch.autograd.grad((h, n), list(leaves.values()), (i['dh'], i['dn']))
    want = norms.residual_norm_modulate_backward(i['dh'], i['dn'], plain[0], i['a'], EPS, norm='layer', gate=i['gate'],
                                                 residual_scale=0.5, post_norm='rms', post_weight=i['wp'], weight=i['w'],
                                                 bias=i['b'], scale=i['scale'], shift=i['shift'])
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    # along a direction in every argument, against the central difference of the formula in float64. The two differ by what the
    # gradients are off in fp32 (2^-15 of the magnitudes, above) and by the difference's own error, e^2 of a smooth function
    step = {k: torch.randn(i[k].shape, generator=torch.Generator().manual_seed(4), dtype=torch.float64).to(DEV) for k in names}

    def f(e):
        t = {k: i[k].double() + e * step[k] for k in names}
        h, _, n, _ = forward(t['x'], t['a'], 'layer', t['gate'], 0.5, 'rms', t['wp'], t['w'], t['b'], t['scale'], t['shift'])
        return (h * i['dh'].double()).sum() + (n * i['dn'].double()).sum()

    e = 1e-5
    num = (f(e) - f(-e)) / (2 * e)
    terms = [(g.double() * step[k]) for k, g in zip(names, grads)]
    assert (num - sum(t.sum() for t in terms)).abs() <= 2 ** -15 * sum(t.abs().sum() for t in terms)


def test_autograd_with_one_output_used_and_in_place():
    print('norms one output', flush=True)
    i = inputs(20, 128, 1, torch.bfloat16, True, True, None, True, False)
    for which in range(2):
        x, a, gate = (i[k].clone().requires_grad_() for k in ('x', 'a', 'gate'))
        out = norms.residual_norm_modulate(x, a, EPS, gate=gate, weight=i['w'])
        got = torch.autograd.grad(out[which], (x, a, gate), i['dn'])
        zero = torch.zeros_like(i['dn'])
        want = norms.residual_norm_modulate_backward(i['dn'] if which == 0 else None, zero if which == 0 else i['dn'],
                                                     out[0].detach(), i['a'], EPS, gate=i['gate'], weight=i['w'])
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    x = i['x'].clone().requires_grad_()
    y = norms.norm_modulate(x, EPS)
    y.mul_(2)                        # a result takes in-place operations
    y.sum().backward()
    h, n = norms.residual_norm_modulate(i['x'].clone().requires_grad_(), i['a'], EPS)
    h.add_(1)                        # the gradient reads h
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        n.sum().backward()


def test_graph_replays_and_streams():
    print('norms graph', flush=True)
    i = inputs(300, 1024, 4, torch.bfloat16, True, True, 'rms', True, True)

    def step():
        kw = dict(norm='layer', gate=i['gate'], post_norm='rms', post_weight=i['wp'], weight=i['w'], bias=i['b'],
                  scale=i['scale'], shift=i['shift'])
        h, n = norms.residual_norm_modulate(i['x'], i['a'], EPS, **kw)
        return (h, n, *norms.residual_norm_modulate_backward(i['dh'], i['dn'], h, i['a'], EPS, **kw))

    step()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for seed in (1, 2, 3):
        new = inputs(300, 1024, 4, torch.bfloat16, True, True, 'rms', True, True, seed=seed)
        for k, t in i.items():
            t.copy_(new[k])
        want = step()
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for out in outs for a, b in zip(out, want)), seed
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for out in got for a, b in zip(out, want))


def test_a_captured_leaf_is_not_recorded():
    x = torch.randn(8, 64, device=DEV).bfloat16().requires_grad_()
    norms.norm_modulate(x.detach(), EPS)
    g = torch.cuda.CUDAGraph()
    with pytest.warns(UserWarning, match='not recorded'):
        with torch.cuda.graph(g):
            y = norms.norm_modulate(x, EPS)
    g.replay()
    torch.cuda.synchronize()
    assert not y.requires_grad and torch.equal(y, norms.norm_modulate(x.detach(), EPS))


def test_refusals():
    x, w = torch.zeros(6, 64, dtype=torch.bfloat16, device=DEV), torch.ones(64, device=DEV)
    bad = [lambda: norms.norm_modulate(x, EPS, norm='batch'), lambda: norms.norm_modulate(x, EPS, norm=None),
           lambda: norms.norm_modulate(x[:, :60], EPS), lambda: norms.norm_modulate(x.double(), EPS),
           lambda: norms.norm_modulate(x, EPS, weight=w[:32]), lambda: norms.norm_modulate(x, EPS, weight=w.int()),
           lambda: norms.norm_modulate(x, EPS, scale=torch.zeros(4, 64, device=DEV)),
           lambda: norms.norm_modulate(x, EPS, scale=torch.zeros(2, 64, device=DEV), shift=w),
           lambda: norms.norm_modulate(x, EPS, weight=w.cpu()),
           lambda: norms.residual_norm_modulate(x, None, EPS), lambda: norms.residual_norm_modulate(x, x[:5], EPS),
           lambda: norms.residual_norm_modulate(x, x.half(), EPS), lambda: norms.residual_norm_modulate(x, x, EPS, post_weight=w),
           lambda: norms.residual_norm_modulate(x, x, EPS, post_norm='group'),
           lambda: norms.norm_modulate_backward(x[:, :32], x, EPS), lambda: norms.norm_modulate_backward(x.half(), x, EPS),
           lambda: norms.norm_modulate(torch.zeros(2, 8200, device=DEV), EPS)]
    for k, f in enumerate(bad):
        with pytest.raises(L.HipPathError):
            f()
            print(k)


@pytest.mark.parametrize('rows,C,groups', [(2100, 64, 2100), (1400, 8192, 700), (3 * 1300, 520, 1300), (30 * 40, 1000, 40), (7 * 170, 2048, 170),
                                           (20 * 5, 8, 5), (9 * 600, 4096, 600)])
@pytest.mark.parametrize('norm,post,dtype', [('layer', None, torch.bfloat16), ('rms', 'layer', torch.float32)])
def test_many_groups(rows, C, groups, norm, post, dtype):
    """as many groups as fill the GPU, each one work-group's, and numbers of them on both sides of that"""
    print(f'norms {rows} x {C}, {groups} groups, {dtype}', flush=True)
    i = inputs(rows, C, groups, dtype, True, True, post, True, True, seed=rows)
    got = run(i, norm, post, 0.7)
    # the parameters' gradients are the same whichever of them are asked for
    x, a = (i[k].clone().requires_grad_(k == 'x') for k in ('x', 'a'))
    for wanted in (('scale',), ('w',), ('gate', 'b'), ()):
        p = {k: (v if v is None else v.clone().requires_grad_(k in wanted)) for k, v in i.items() if k in ('gate', 'wp', 'w', 'b', 'scale', 'shift')}
        h, n = norms.residual_norm_modulate(x, a, EPS, norm, p['gate'], 0.7, post, p['wp'], p['w'], p['b'], p['scale'], p['shift'])
        grads = torch.autograd.grad((h, n), [x] + [p[k] for k in wanted], (i['dh'], i['dn']))
        order = {'gate': 2, 'wp': 3, 'w': 4, 'b': 5, 'scale': 6, 'shift': 7}
        for g, k in zip(grads, ('x', *wanted)):
            assert torch.equal(g, got[order[k] if k != 'x' else 0]), (wanted, k)
