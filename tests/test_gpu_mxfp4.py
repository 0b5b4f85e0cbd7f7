"""Microscaled 4-bit floating point: quantisation bit for bit against the definition, reading back, and the linear layers on it
against float64 of the values that codes and scales stand for.

Tolerance of the layers, e = 2^-24: the products of 4-bit values and scales are exact, their sum is rounded to fp32 once for every
64 of them at most (2 e of it, which is at most S = sum |x| |w|): z is off by (n_in / 64 + 64) 2 e S, 64 for the joining of split
sums and what a matrix instruction does inside. The activations have slopes up to 1.13 and are good to 2^-20 of their value; the
result is rounded to bf16 once, 2^-8."""
import math

import pytest
import torch

from onereel_amd import _lib as L
from onereel_amd import mxfp4
from onereel_amd.mxfp4 import MXFP4

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'
TYPES = [torch.bfloat16, torch.float16, torch.float32]
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def quantized(x):
    """codes (one an element) and scales by the definition, on the CPU: the nearest level found by distance, ties to the even code"""
    b = x.double().cpu().reshape(-1, 32)
    top = b.abs().amax(1)
    exponent = torch.tensor([max(math.frexp(t)[1] - 3, -127) if 0 < t < math.inf else -127 for t in top.tolist()]).double()
    bad = ~torch.isfinite(b).all(1)
    v = b / torch.tensor([2.0 ** e for e in exponent.tolist()], dtype=torch.float64)[:, None]
    v = torch.where(bad[:, None], torch.zeros_like(v), v)
    d = (v.abs()[..., None] - torch.tensor(LEVELS, dtype=torch.float64)).abs()
    code = d.argmin(-1)                                        # the lower level of a tie
    tied = (d.gather(-1, (code + 1).clamp(max=7)[..., None])[..., 0] == d.gather(-1, code[..., None])[..., 0]) & (code < 7)
    code = code + (tied & (code % 2 == 1)).long()
    code = code + 8 * torch.signbit(b).long() * (~bad[:, None]).long()
    scales = torch.where(bad, torch.full_like(exponent, 255), exponent + 127)
    return code.reshape(x.shape), scales.reshape(*x.shape[:-1], x.shape[-1] // 32)


def values(codes, scales):
    level = torch.tensor(LEVELS + [-v for v in LEVELS], dtype=torch.float64)[codes.reshape(-1, 32)]
    unit = torch.tensor([2.0 ** (i - 127) for i in range(255)] + [math.nan], dtype=torch.float64)[scales.reshape(-1, 1).long()]
    return (level * unit).reshape(codes.shape)


def check_quantized(x):
    m = mxfp4.quantize(x)
    codes, scales = quantized(x)
    assert m.codes.shape == (*x.shape[:-1], x.shape[-1] // 2) and m.scales.shape == scales.shape
    got = m.codes.cpu()
    got = torch.stack([got & 15, got >> 4], -1).flatten(-2)
    assert torch.equal(m.scales.cpu().long(), scales.long())
    assert torch.equal(got.long(), codes)
    return m, values(codes, scales)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('shape', [(1, 32), (3, 64), (5, 7, 96), (1000, 160), (2, 4096), (0, 64)])
def test_quantize(shape, dtype):
    print(f'quantize {shape} {dtype}', flush=True)
    g = torch.Generator(device=DEV).manual_seed(1)
    x = (torch.randn(*shape, generator=g, device=DEV) * torch.exp(3 * torch.randn(*shape[:-1], 1, generator=g, device=DEV))).to(dtype)
    if x.numel():
        x.view(-1, 32)[0] = 0
    m, want = check_quantized(x)
    for to in TYPES:
        got = m.dequantize(to)
        # fp16 rows past its range hold infinities: NaN blocks
        assert got.dtype == to and torch.allclose(got.cpu(), want.to(to), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_ties_borders_and_ends_of_the_range(dtype):
    print(f'quantize borders {dtype}', flush=True)
    f = torch.finfo(dtype)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0], dtype=torch.float64)
    near = torch.cat([ties, ties * (1 + f.eps), ties * (1 - f.eps), torch.tensor([0, 1, 2, 3, 4, 6, 0.5, 1.5])])
    block = torch.cat([near, -near.flip(0)])[:32 * 2].reshape(2, 32)
    block[:, 0] = 7.0                                          # a scale of 1
    rows = [block * 2.0 ** e for e in (0, 5, -5, 12, -8)]
    top = torch.full((1, 32), f.max, dtype=torch.float64)
    low = torch.full((1, 32), f.smallest_normal, dtype=torch.float64)
    sub = torch.zeros(1, 32, dtype=torch.float64)
    sub[0, 3] = f.smallest_normal * f.eps
    sub[0, 4] = -f.smallest_normal * f.eps * 3
    x = torch.cat([*rows, top, -top, low, low * 1.5, sub, -sub]).to(dtype).to(DEV)
    m, want = check_quantized(x)
    assert torch.equal(m.dequantize(torch.float32).cpu(), want.float())


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize('order', ['in order', 'mixed', 'near'])
def test_every_16_bit_value(dtype, order):
    print(f'quantize every {dtype} {order}', flush=True)
    bits = torch.arange(65536, dtype=torch.int32)
    if order == 'mixed':
        bits = bits[torch.randperm(65536, generator=torch.Generator().manual_seed(2))]
    if order == 'near':              # blocks of few exponents, so that most elements are neither 0 nor at the end of the range
        bits = bits.view(512, 128).t().reshape(-1)
        bits = bits.view(-1, 16, 2).transpose(1, 2).reshape(-1)
    x = bits.to(torch.int16).view(dtype).view(64, 1024).to(DEV)
    check_quantized(x)


def test_not_finite_blocks():
    print('quantize not finite', flush=True)
    for dtype in TYPES:
        x = torch.ones(2, 96, dtype=dtype, device=DEV)
        x[0, 5], x[1, 40], x[1, 95] = math.inf, math.nan, -math.inf
        m, _ = check_quantized(x)
        back = m.dequantize()
        assert torch.equal(back.isnan().cpu().view(2, 3, 32).all(2), torch.tensor([[True, False, False], [False, True, True]]))
        assert (back[0, 32:] == 1).all()


def test_every_code_and_scale():
    print('dequantize all', flush=True)
    codes = torch.arange(256, dtype=torch.uint8, device=DEV).repeat(256, 1)
    scales = torch.arange(256, dtype=torch.uint8, device=DEV)[:, None].repeat(1, 16)
    m = MXFP4(codes, scales)
    want = values(torch.stack([codes & 15, codes >> 4], -1).flatten(1).long().cpu(), scales.cpu())
    for to in TYPES:
        # past fp32 an infinity, which bf16 and fp16 keep
        assert torch.equal(m.dequantize(to).cpu().nan_to_num(nan=3.25), want.float().to(to).nan_to_num(nan=3.25))


def test_strides_of_x():
    wide = torch.randn(30, 300, device=DEV).bfloat16()
    for x in (wide[:, 8:136], wide[:, 3:131], wide.t()[:288].t(), wide[:1, :64].expand(5, 64)):
        a, b = mxfp4.quantize(x), mxfp4.quantize(x.contiguous())
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


def act(z, name):
    return z * torch.sigmoid(z) if name == 'silu' else torch.nn.functional.gelu(z, approximate='tanh') if name else z


def check_linear(y, xv, wv, b, name, gate, residual):
    z = xv @ wv.T
    S = xv.abs() @ wv.abs().T
    off = (xv.shape[-1] / 64 + 64) * 2 ** -23 * S
    if b is not None:
        z = z + b.double()
        off = off + 2 ** -23 * z.abs()
    f = act(z, name)
    gate = 1.0 if gate is None else gate.double()
    want, bound = f * gate, (1.13 * off + 2 ** -20 * f.abs() + 2 ** -20 * z.abs() * 0.5) * abs(gate)
    if residual is not None:
        want = want + residual.double()
        bound = bound + 2 ** -22 * residual.double().abs()
    assert y.dtype == torch.bfloat16 and bool(torch.isfinite(y).all())
    past = (y.double() - want).abs() - bound - 2 ** -8 * (want.abs() + bound) - 1e-30
    assert past.numel() == 0 or past.max().item() <= 0, f'{past.max().item():.3e} past its bound'


def layer(M, K, N, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(M, K, generator=g, device=DEV) * (1 + 9 * (torch.randn(K, generator=g, device=DEV) > 2).float())).bfloat16()
    w = mxfp4.quantize(torch.randn(N, K, generator=g, device=DEV) * K ** -0.5)
    b = 0.2 * torch.randn(N, generator=g, device=DEV)
    gate = 1 + 0.5 * torch.randn(N, generator=g, device=DEV)
    return x, w, b, gate, torch.randn(M, N, generator=g, device=DEV).bfloat16()


SIZES = [(1, 32, 8), (1, 2048, 264), (2, 96, 40), (4, 4096, 512), (5, 64, 8), (16, 2080, 128), (17, 256, 72), (31, 544, 1000),
         (33, 32, 256), (64, 512, 64), (65, 288, 136), (130, 1056, 520), (256, 256, 256), (257, 2048, 264), (300, 8192, 512),
         (1000, 224, 1032), (2100, 736, 2064)]


@pytest.mark.parametrize('M,K,N', SIZES)
@pytest.mark.parametrize('how', ['plain', 'all', 'silu'])
def test_linear(M, K, N, how):
    print(f'mx linear {M} x {K} -> {N} {how}', flush=True)
    x, w, b, gate, r = layer(M, K, N)
    b, name, gate, r = (None, None, None, None) if how == 'plain' else (b, 'gelu_tanh', gate, r) if how == 'all' else \
        (b.bfloat16(), 'silu', gate.bfloat16(), None)
    y = mxfp4.linear(x, w, b, activation=name, gate=gate, residual=r)
    q = mxfp4.quantize(x)
    check_linear(y, q.dequantize(torch.float32).double(), w.dequantize(torch.float32).double(), b, name, gate, r)
    assert torch.equal(y, mxfp4.linear(q, w, b, activation=name, gate=gate, residual=r))
    assert torch.equal(y, mxfp4.linear(x, w, b, activation=name, gate=gate, residual=r))


def test_rows_and_columns_stand_where_they_belong():
    """one element of x and one of W at a time reach one element of y"""
    print('mx linear places', flush=True)
    M, K, N = 70, 320, 72
    for m, k, n in [(0, 0, 0), (69, 319, 71), (33, 31, 40), (32, 32, 31), (5, 64, 9), (64, 255, 64), (1, 256, 8)]:
        x, w = torch.zeros(M, K, device=DEV), torch.zeros(N, K, device=DEV)
        x[m, k], w[n, k] = 3.0, -0.5
        y = mxfp4.linear(x.bfloat16(), mxfp4.quantize(w))
        want = torch.zeros(M, N, device=DEV)
        want[m, n] = -1.5
        assert torch.equal(y.float(), want), (m, k, n)


def test_scales_over_their_range():
    print('mx linear scales', flush=True)
    M, K, N = 40, 256, 48
    g = torch.Generator().manual_seed(3)
    codes = [torch.randint(0, 256, (r, K // 2), generator=g, dtype=torch.uint8).to(DEV) for r in (M, N)]
    scales = [torch.randint(90, 160, (r, K // 32), generator=g, dtype=torch.uint8).to(DEV) for r in (M, N)]
    x, w = (MXFP4(c, s) for c, s in zip(codes, scales))
    check_linear(mxfp4.linear(x, w), x.dequantize(torch.float32).double(), w.dequantize(torch.float32).double(), None, None, None, None)


def test_not_finite_rows_stay_in_their_rows():
    print('mx linear not finite', flush=True)
    for M in (3, 20, 300):
        x, w, b, _, _ = layer(M, 512, 136)
        clean = mxfp4.linear(x, w, b)
        x[2, 100], x[1, 0] = math.nan, math.inf
        y = mxfp4.linear(x, w, b)
        assert y[1:3].isnan().all()
        keep = torch.ones(M, dtype=torch.bool, device=DEV)
        keep[1:3] = False
        assert torch.equal(y[keep], clean[keep])


def test_strides_leading_dimensions_and_no_rows():
    print('mx linear strides', flush=True)
    x, w, b, gate, r = layer(60, 256, 128)
    y = mxfp4.linear(x, w, b, residual=r)
    wide = torch.zeros(60, 400, dtype=torch.bfloat16, device=DEV)
    wide[:, 16:272] = x
    more = torch.zeros(60, 200, dtype=torch.bfloat16, device=DEV)
    more[:, 64:192] = r
    assert torch.equal(mxfp4.linear(wide[:, 16:272], w, b, residual=more[:, 64:192]), y)
    assert torch.equal(mxfp4.linear(x.view(3, 20, 256), w, b, residual=r.view(3, 20, 128)), y.view(3, 20, 128))
    assert torch.equal(mxfp4.linear(mxfp4.quantize(x.view(3, 20, 256)), w, b, residual=r.view(3, 20, 128)), y.view(3, 20, 128))
    assert mxfp4.linear(x[:0], w, b).shape == (0, 128)
    assert mxfp4.linear(mxfp4.quantize(x[:0]), w).shape == (0, 128)


def test_graph_replays_and_streams():
    print('mx graph', flush=True)
    for M in (1, 3, 333):
        x, w, b, gate, r = layer(M, 1024, 520)
        step = lambda: mxfp4.linear(x, w, b, activation='gelu_tanh', gate=gate, residual=r)
        step()
        graphs, outs = [], []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(step())
            graphs.append(g)
        for seed in (1, 2, 3):
            x.copy_(layer(M, 1024, 520, seed)[0])
            want = step()
            torch.cuda.synchronize()
            for g in graphs:
                g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(o, want) for o in outs), (M, seed)
        got = []
        for s in [torch.cuda.Stream() for _ in range(2)] * 2:
            with torch.cuda.stream(s):
                got.append(step())
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in got)


def test_a_backward_pass_raises():
    x, w, _, _, _ = layer(4, 64, 16)
    y = mxfp4.linear(x.requires_grad_(), w)
    with pytest.raises(L.HipValueError, match='no gradient'):
        y.sum().backward()


def test_a_backward_pass_through_quantised_tensors_raises():
    x, w, b, _, _ = layer(4, 64, 16)
    made = [mxfp4.linear(mxfp4.quantize(x.clone().requires_grad_()), w), mxfp4.quantize(x.clone().requires_grad_()).dequantize(),
            mxfp4.linear(x, mxfp4.quantize(torch.ones(16, 64, device=DEV, requires_grad=True))),
            mxfp4.linear(x, w, b.clone().requires_grad_())]
    for y in made:
        with pytest.raises(L.HipValueError, match='no gradient'):
            y.float().sum().backward()
    with torch.no_grad():
        assert not mxfp4.linear(mxfp4.quantize(x.clone().requires_grad_()), w).requires_grad
    assert not mxfp4.linear(mxfp4.quantize(x), w, b).requires_grad


def test_refusals():
    x, w, b, gate, r = layer(4, 64, 16)
    c, s = w.codes, w.scales
    bad = [lambda: mxfp4.quantize(x[:, :40]), lambda: mxfp4.quantize(x.double()), lambda: mxfp4.quantize(x.cpu()),
           lambda: MXFP4(c.int(), s), lambda: MXFP4(c, s[:, :1]), lambda: MXFP4(c[:, :9], s), lambda: MXFP4(c, s.cpu()),
           lambda: MXFP4(c[:15], s), lambda: w.dequantize(torch.float64), lambda: mxfp4.linear(x, c),
           lambda: mxfp4.linear(x[:, :32], w), lambda: mxfp4.linear(x.float(), w), lambda: mxfp4.linear(x, w, b[:8]),
           lambda: mxfp4.linear(x, w, activation='relu'), lambda: mxfp4.linear(x, w, residual=r[:2]),
           lambda: mxfp4.linear(x, w, residual=r.float()), lambda: mxfp4.linear(x, w, gate=gate.cpu()),
           lambda: mxfp4.linear(x, MXFP4(c[:12], s[:12]))]
    for k, f in enumerate(bad):
        with pytest.raises(L.HipPathError):
            f()
            print(k)
