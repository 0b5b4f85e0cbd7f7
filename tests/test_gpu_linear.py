"""Linear layers with a fused epilogue, and their gradients, against float64.

Tolerance. z: bf16 products are exact in fp32, their sum over K of them is off by at most 2^-24 K of the sum of |x w| (taken
as 2^-22 sqrt(K), four standard deviations of K roundings of half a step of a partial sum), then one rounding to bf16 of
2^-8. y: the same, through gate * act with |act'| <= 1.13, plus exp's error (2^-20 of z) and one rounding of y. dx, dW:
dz is rounded to bf16 (2^-8 of every term: 2^-8 of the sum of |dz w|) where there is an activation or a gate, the sums and the
result as above. db, dgate: fp32 sums, 2^-19 of the sum of the terms (2^-20 each from exp).
"""
import math

import pytest
import torch

from helpers import rand_bf16
from onereel_amd import linear as F

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'
HALF = 2 ** -8


def act(z, name):
    if name == 'silu':
        return z * torch.sigmoid(z)
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))) if name else z


def inputs(M, K, N, seed=0, bias=True, gate=True, residual=True):
    g = torch.Generator().manual_seed(seed + 100)
    x, w = rand_bf16((M, K), seed).to(DEV), (rand_bf16((N, K), seed + 1) * K ** -0.5).to(DEV)
    b = torch.randn(N, generator=g).to(DEV) if bias else None
    t = (0.5 + 0.5 * torch.randn(N, generator=g)).to(DEV) if gate else None
    r = rand_bf16((M, N), seed + 2).to(DEV) if residual else None
    return x, w, b, t, r


def near(got, want, slack, what):
    assert got.shape == want.shape and bool(torch.isfinite(got.float()).all()), what
    half = HALF if got.dtype == torch.bfloat16 else 0
    off = (got.double() - want).abs() - (half * want.abs() + (1 + half) * slack + 1e-37)
    assert off.numel() == 0 or off.max().item() <= 0, f'{what}: {off.max().item():.3e} past its bound'


def check_forward(y, z, x, w, b, t, r, name):
    zr = x.double() @ w.double().T
    slack = 2 ** -22 * math.sqrt(x.shape[1]) * (x.double().abs() @ w.double().abs().T)
    if b is not None:
        zr = zr + b.double()
    slack = slack + 2 ** -22 * zr.abs()
    if z is not None:
        near(z, zr, slack, 'z')
    a = act(zr, name)
    gate = 1.0 if t is None else t.double()
    want = gate * a + (0 if r is None else r.double())
    near(y, want, 1.13 * slack * (1 if t is None else gate.abs()) + 2 ** -20 * (gate * zr).abs() + 2 ** -22 * want.abs(), 'y')


def check_backward(got, dy, x, w, z, t, name, bias):
    dx, dw, db, dg = got
    dyd = dy.double()
    if z is None:
        dz, rounding = dyd, 0.0
    else:
        zz = z.double().requires_grad_()
        dz = torch.autograd.grad(act(zz, name), zz, dyd * (1.0 if t is None else t.double()))[0] if name else dyd * t.double()
        rounding = 1.01 * HALF
    # exp's error in act' (2^-20 of terms up to 1.13)
    exps = 2 ** -19 * (dyd * (1.0 if t is None else t.double())).abs() if name else torch.zeros_like(dyd)
    mag = rounding * dz.abs() + exps
    if dx is not None:
        near(dx, dz @ w.double(), (2 ** -22 * math.sqrt(dz.shape[1]) * dz.abs() + mag) @ w.double().abs(), 'dx')
    if dw is not None:
        rows = max(dz.shape[0], 1)
        near(dw, dz.T @ x.double(), (2 ** -22 * math.sqrt(rows) * dz.abs() + mag).T @ x.double().abs(), 'dw')
    assert (db is not None) == bias and (dg is not None) == (t is not None)
    if db is not None:
        near(db, dz.sum(0), 2 ** -19 * dz.abs().sum(0) + exps.sum(0), 'db')
    if dg is not None:
        a = act(z.double(), name)
        near(dg, (dyd * a).sum(0), 2 ** -19 * (dyd * z.double()).abs().sum(0), 'dgate')


SIZES = [(1, 64, 64), (1, 2048, 520), (1, 8, 8), (2, 4104, 24), (3, 520, 136), (4, 2560, 72), (5, 512, 40), (9, 4096, 48),
         (32, 4096, 64), (16, 72, 8), (17, 256, 1000), (32, 1000, 128), (33, 8, 72), (64, 64, 64), (65, 72, 136),
         (127, 200, 1032), (300, 520, 264), (1000, 1024, 256), (257, 4096, 96), (4100, 264, 2056), (3333, 136, 3336)]


@pytest.mark.parametrize('M,K,N', SIZES)
@pytest.mark.parametrize('name', [None, 'gelu_tanh', 'silu'])
def test_forward_and_backward(M, K, N, name):
    print(f'linear {M} x {K} -> {N} {name}', flush=True)
    x, w, b, t, r = inputs(M, K, N, bias=M % 2 == 1 or name is None, gate=name != 'silu', residual=name != 'gelu_tanh')
    y, z = F.linear(x, w, b, activation=name, gate=t, residual=r, keep_preactivation=True)
    check_forward(y, z, x, w, b, t, r, name)
    assert torch.equal(F.linear(x, w, b, activation=name, gate=t, residual=r), y)
    dy = rand_bf16((M, N), 7).to(DEV)
    got = F.linear_backward(dy, x, w, bias=b is not None, activation=name, gate=t, preactivation=z)
    check_backward(got, dy, x, w, z if name or t is not None else None, t, name, b is not None)
    again = F.linear_backward(dy, x, w, bias=b is not None, activation=name, gate=t, preactivation=z)
    assert all(torch.equal(p, q) for p, q in zip(got, again) if p is not None)


def test_plain_product_and_single_gradients():
    print('plain', flush=True)
    x, w, *_ = inputs(500, 320, 136, 3)
    check_forward(F.linear(x, w), None, x, w, None, None, None, None)
    dy = rand_bf16((500, 136), 1).to(DEV)
    both = F.linear_backward(dy, x, w, bias=True)
    check_backward(both, dy, x, w, None, None, None, True)
    assert F.linear_backward(dy, x, w, needs=(False, False)) == (None,) * 4
    a, b = F.linear_backward(dy, x, w, needs=(True, False)), F.linear_backward(dy, x, w, needs=(False, True))
    assert a[1] is None and b[0] is None and torch.equal(a[0], both[0]) and torch.equal(b[1], both[1])


def test_strides_leading_dims_and_no_rows():
    print('strides', flush=True)
    wide = rand_bf16((3, 50, 400), 1).to(DEV)
    x, w = wide[..., 64:264], rand_bf16((72, 400), 2).to(DEV)[:, 8:208]
    y = F.linear(x, w)
    assert y.shape == (3, 50, 72)
    check_forward(y.view(150, 72), None, x.reshape(150, 200), w, None, None, None, None)
    dy = torch.full((1, 1, 72), 0.5, dtype=torch.bfloat16, device=DEV).expand(3, 50, 72)
    dx, dw, _, _ = F.linear_backward(dy, x, w)
    check_backward((dx.view(150, 200), dw, None, None), dy.reshape(150, 72), x.reshape(150, 200), w, None, None, None, False)
    none = x[:0]
    assert F.linear(none, w).shape == (0, 50, 72)
    dx, dw, db, _ = F.linear_backward(dy[:0], none, w, bias=True)
    assert dx.shape == (0, 50, 200) and not dw.any() and not db.any()


def test_rows_and_columns_beside_the_operands_never_enter():
    """what lies behind a row's end, a tensor's last row and between strided rows may be anything"""
    print('neighbours', flush=True)
    M, K, N = 70, 72, 40
    big = torch.full((M + 60, K + 56), math.nan, dtype=torch.bfloat16, device=DEV)
    x, w, *_ = inputs(M, K, N, 5)
    big[:M, :K] = x
    bw = torch.full((N + 90, K + 120), math.inf, dtype=torch.bfloat16, device=DEV)
    bw[:N, :K] = w
    by = torch.full((M + 60, N + 88), math.nan, dtype=torch.bfloat16, device=DEV)
    dy = rand_bf16((M, N), 6).to(DEV)
    by[:M, :N] = dy
    assert torch.equal(F.linear(big[:M, :K], bw[:N, :K]), F.linear(x, w))
    got, want = F.linear_backward(by[:M, :N], big[:M, :K], bw[:N, :K], bias=True), F.linear_backward(dy, x, w, bias=True)
    assert all(torch.equal(p, q) for p, q in zip(got[:3], want[:3]))


def test_activations_far_out():
    print('far', flush=True)
    z = torch.tensor([-3e38, -1e20, -200, -20.5, -9, -1e-3, 0, 1e-3, 9, 20.5, 200, 1e20, 3e38, 1, -1, 2.5], device=DEV)
    x = torch.zeros(2, 8, dtype=torch.bfloat16, device=DEV)
    x[:, 0] = 1
    w = torch.zeros(16, 8, dtype=torch.bfloat16, device=DEV)
    w[:, 0] = z.bfloat16()
    zr = w[:, 0].double()
    for name, lo in (('gelu_tanh', 1e-4), ('silu', 2e-2)):
        y, kept = F.linear(x, w, activation=name, keep_preactivation=True)
        assert torch.equal(kept[0], w[:, 0])
        inner = zr.clamp(-300, 300)
        want = torch.where(zr.abs() > 300, zr.clamp(min=0), act(inner, name))
        near(y, want.expand(2, 16), 2 ** -18 * zr.clamp(-30, 30).abs().expand(2, 16), name)
        dy = torch.ones(2, 16, dtype=torch.bfloat16, device=DEV)
        db = F.linear_backward(dy, x, w, bias=True, activation=name, preactivation=kept)[2]
        i2 = inner.clone().requires_grad_()
        near(db, 2 * torch.autograd.grad(act(i2, name).sum(), i2)[0], torch.full((16,), 2 ** -17, device=DEV, dtype=torch.float64),
             name)


def test_autograd():
    print('autograd', flush=True)
    x, w, b, t, r = inputs(90, 64, 48, 9)
    x, r = x.view(2, 45, 64), r.view(2, 45, 48)
    dy = rand_bf16((2, 45, 48), 3).to(DEV)
    leaves = [v.clone().requires_grad_() for v in (x, w, b.bfloat16(), t, r)]
    y, z = F.linear(leaves[0], leaves[1], leaves[2], activation='gelu_tanh', gate=leaves[3], residual=leaves[4],
                    keep_preactivation=True)
    assert not z.requires_grad
    z2 = z.clone()
    z.zero_()                               # the caller's copy: the gradient does not read it
    grads = torch.autograd.grad(y, leaves, dy)
    want = F.linear_backward(dy, x, w, bias=True, activation='gelu_tanh', gate=t, preactivation=z2)
    for g, v, like in zip(grads, (*want, dy), leaves):
        assert g.shape == like.shape and g.dtype == like.dtype and torch.equal(g, v.to(g.dtype).view(g.shape))
    # a plain layer, the weight alone; then differences along a direction in float64
    wl = w.clone().requires_grad_()
    F.linear(x, wl).backward(dy)
    assert torch.equal(wl.grad, F.linear_backward(dy, x, w)[1])
    d = torch.randn(90, 64, generator=torch.Generator().manual_seed(2), dtype=torch.float64).to(DEV)

    def loss(v):
        out = r.double().view(90, 48) + t.double() * act(v @ w.double().T + b.bfloat16().double(), 'gelu_tanh')
        return (out * dy.double().view(90, 48)).sum()

    x0, e = x.double().view(90, 64), 1e-6
    num = (loss(x0 + e * d) - loss(x0 - e * d)) / (2 * e)
    # z, dz and dx are rounded to bf16: 2^-8 each of terms |dy gate w d|, and |act''| <= 1.13 |z| over z's rounding
    room = ((dy.double().view(90, 48) * t.double()).abs() @ w.double().abs() * d.abs()).sum() * HALF * 5
    assert (num - (grads[0].double().view(90, 64) * d).sum()).abs() <= room


def test_capture_refuses_leaves():
    print('capture of leaves', flush=True)
    x, w, *_ = inputs(40, 64, 48)
    w.requires_grad_()
    keep = torch.ones(4, device=DEV)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        keep.add_(1)
        with pytest.raises(F.L.HipValueError, match='leaf'):
            F.linear(x, w)
    g.replay()
    torch.cuda.synchronize()


def test_transposed_weight_and_one_row_of_a_wider_tensor():
    print('odd layouts', flush=True)
    x, w, *_ = inputs(70, 64, 48, 2)
    wt = w.t().contiguous().t()
    assert torch.equal(F.linear(x, wt), F.linear(x, w))
    one = x[:1, :].expand(5, 64)[2:3]
    assert torch.equal(F.linear(one, w), F.linear(x[:1], w))
    dy = rand_bf16((70, 48), 1).to(DEV)
    got = F.linear_backward(dy.t().contiguous().t(), x, wt, bias=True)
    assert all(torch.equal(a, b) for a, b in zip(got[:3], F.linear_backward(dy, x, w, bias=True)))


def test_graph_replays():
    print('graph', flush=True)
    M, K, N = 700, 1024, 136                   # few tiles: both passes split their k axis
    x, w, b, t, _ = inputs(M, K, N, 11)
    dy = rand_bf16((M, N), 4).to(DEV)

    def step():
        y, z = F.linear(x, w, b, activation='silu', gate=t, keep_preactivation=True)
        return (y, z, *F.linear_backward(dy, x, w, bias=True, activation='silu', gate=t, preactivation=z))

    step()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for seed in (1, 2, 3):
        x.copy_(rand_bf16((M, K), seed))
        dy.copy_(rand_bf16((M, N), seed + 9))
        want = step()
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for out in outs for p, q in zip(out, want))
