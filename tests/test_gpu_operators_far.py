"""Tensors of more than 2^31 elements: the last rows of a large call are those of a small one, bit for bit (rows are independent of one
another), and a norm over them is the sum of its parts."""
import math

import pytest
import torch

from onereel_amd import clip, mxfp4, norms, rotary

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'
C = 8192
ROWS = (1 << 31) // C + 5000


@pytest.fixture(scope='module')
def rows():
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.empty(ROWS, C, dtype=torch.bfloat16, device=DEV)
    for a in range(0, ROWS, 1 << 15):
        x[a:a + (1 << 15)] = torch.randn(min(1 << 15, ROWS - a), C, generator=g, device=DEV)
    yield x
    del x
    torch.cuda.empty_cache()


def test_norms(rows):
    print('far norms', flush=True)
    s = torch.randn(C, device=DEV)
    n = norms.norm_modulate(rows, 1e-6, scale=s, shift=s)
    assert torch.equal(n[-7:], norms.norm_modulate(rows[-7:], 1e-6, scale=s, shift=s))
    del n
    h, n = norms.residual_norm_modulate(rows, rows, 1e-6, norm='rms', gate=s)
    hs, ns = norms.residual_norm_modulate(rows[-7:], rows[-7:], 1e-6, norm='rms', gate=s)
    assert torch.equal(h[-7:], hs) and torch.equal(n[-7:], ns)
    del n
    dx, da = norms.residual_norm_modulate_backward(None, rows, h, rows, 1e-6, norm='rms', gate=s)[:2]
    dxs, das = norms.residual_norm_modulate_backward(None, rows[-7:], hs, rows[-7:], 1e-6, norm='rms', gate=s)[:2]
    assert torch.equal(dx[-7:], dxs) and torch.equal(da[-7:], das)


def test_rotary(rows):
    print('far rotary', flush=True)
    p = torch.arange(ROWS, dtype=torch.int32, device=DEV)
    y = rotary.rotate(rows.view(ROWS, 64, 128), rotary.Axes(p, (128,)))
    assert torch.equal(y[-7:], rotary.rotate(rows[-7:].view(7, 64, 128), rotary.Axes(p[-7:], (128,))))
    del y
    w = torch.ones(C, device=DEV)
    q, k = rotary.norm_rotate(rows, rows, w, w, 1e-6, rotary.Axes(p, (128,)), 64)
    qs, _ = rotary.norm_rotate(rows[-7:], rows[-7:], w, w, 1e-6, rotary.Axes(p[-7:], (128,)), 64)
    assert torch.equal(q[-7:], qs) and torch.equal(k[-7:], qs)


def test_clipping(rows):
    print('far clip', flush=True)
    out = torch.empty_like(rows)
    halves = [clip.grad_norm([t]).double().item() for t in (rows[:ROWS // 2], rows[ROWS // 2:])]
    norm = clip.clip_grads_([rows], 1.0, out=[out])
    assert abs(norm.double().item() - math.hypot(*halves)) <= 2 ** -22 * norm.item()
    want = (rows[-7:].double() / (norm.double() + 1e-6))
    assert ((out[-7:].double() - want).abs() <= (2 ** -8 + 2 ** -20) * want.abs()).all()


def test_4_bits(rows):
    print('far 4 bits', flush=True)
    w = mxfp4.quantize(torch.randn(64, C, device=DEV))
    m = mxfp4.quantize(rows)
    s = mxfp4.quantize(rows[-300:])
    assert torch.equal(m.codes[-300:], s.codes) and torch.equal(m.scales[-300:], s.scales)
    assert torch.equal(m.dequantize()[-300:], s.dequantize())
    y = mxfp4.linear(rows, w)
    assert torch.equal(y, mxfp4.linear(m, w))
    del m
    # more than 2^31 elements of results, of tiles as the small call has them
    wide = mxfp4.quantize(torch.randn(C, 256, device=DEV))
    x = rows[:, :256]
    y = mxfp4.linear(x, wide)
    for a in (0, 200000, ROWS - 512):
        at = a // 256 * 256
        # sums over n_in in one step of the matrix cores are the same in every tile
        assert torch.equal(y[at:at + 512], mxfp4.linear(x[at:at + 512], wide)[:y[at:at + 512].shape[0]])
