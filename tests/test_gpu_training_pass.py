"""The differentiable pass of the Wan-shaped DiT: linear layers, RMSNorm + RoPE, ranged attention and cross-attention with their
gradients together, on two blocks with halo scopes, against the same formulas in float64 with torch's autograd.

Tolerance. A gradient passes at most 14 roundings to bf16 a block on its way (forward and backward: every product's
result, P or dS, dz, the norms' results), each off by at most 2^-8 relative and independent of the others: 2 blocks and the
embedding and output layers, 40 of them, give sqrt(40) 2^-8 = 2.5e-2 relative in the 2-norm where all of them are at
their worst. The forward pass has half as many.

A bias's gradient is the sum over S rows of dz. The rows' errors, 2.5e-2 of each row and independent of one another, add up
to 2.5e-2 of sqrt(sum |dz_row|^2), which is not small next to the sum where the rows cancel: a bias of the keys moves all keys
of a query alike, which softmax does not see, so that sum is 0 but for the norm and the rotation behind it (a first form
without this term failed there by 4%). So a bias may be off by 2.5e-2 (|sum| + sqrt(sum |dz_row|^2))."""
import math

import pytest
import torch
import torch.nn.functional as F

from onereel_amd import _lib as L
from onereel_amd import wan_dit as WD
from onereel_amd.layout import SceneLayout

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'
LENGTHS, T, TEXT_LEN, HALO = [2, 3, 2], 16, 8, 1


def model(**layout):
    cfg = WD.DiTConfig(dim=512, heads=4, ffn=1024, blocks=2, in_channels=4, text_dim=256, std=0.05)
    return WD.WanDiT(cfg, SceneLayout(LENGTHS, **(layout or dict(halo=HALO))), T, TEXT_LEN, DEV, seed=3)


def inputs():
    g = torch.Generator(device=DEV).manual_seed(5)
    S = sum(LENGTHS) * T
    tokens = torch.randn(S, 16, generator=g, device=DEV).bfloat16()
    text = torch.randn(3 * TEXT_LEN, 256, generator=g, device=DEV).bfloat16()
    rotary = tuple(x.to(DEV) for x in WD.wan_rope_table(sum(LENGTHS), 4, 4, 128))
    return tokens, text, rotary, torch.randn(S, 16, generator=g, device=DEV).bfloat16()


def exact_forward(m, w, tokens, t, text, rotary, rows):
    """the same pass in float64; w: the model's parameters in double, by identity of the original; rows: takes, for every
    bias, a zero added to its layer's output, whose gradient is the rows that the bias's gradient is the sum of"""
    P = lambda p: w[id(p)]

    def lin(l, x):
        y = x @ P(l.weight).T + P(l.bias)
        rows[id(l.bias)] = torch.zeros_like(y, requires_grad=True)
        return y + rows[id(l.bias)]

    eps, H = m.cfg.eps, m.cfg.heads
    silu = lambda x: x * torch.sigmoid(x)
    gelu = lambda x: 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    rms = lambda x, n: x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * P(n.weight)
    ln = lambda x, a, b: F.layer_norm(x, x.shape[-1:], eps=eps) * a + b
    cos, sin = (r[0].double() for r in rotary)

    def rope(x):
        x = x.unflatten(1, (H, -1))
        a, b, c, s = x[..., 0::2], x[..., 1::2], cos[..., 0::2], sin[..., 1::2]
        return torch.stack([a * c - b * s, a * s + b * c], 3).flatten(2)

    def attend(q, k, v, q_ranges, k_ranges):
        out = []
        for (a, b), (c, d) in zip(q_ranges, k_ranges):
            s = torch.einsum('qhd,khd->hqk', q[a:b], k[c:d]) * q.shape[2] ** -0.5
            out.append(torch.einsum('hqk,khd->qhd', torch.softmax(s, 2), v[c:d]))
        return torch.cat(out).flatten(1)

    lay = m.ctx.layout
    q_ranges = [(T * a, T * b) for a, b in lay.ranges]
    k_ranges = [tuple(T * f for f in lay.key_range(j)) for j in range(lay.n_scenes)]
    sentences = [(TEXT_LEN * j, TEXT_LEN * (j + 1)) for j in range(lay.n_scenes)]
    heads = lambda x: x.unflatten(1, (H, -1))
    x = lin(m.patch_embed, tokens)
    f = WD.timestep_features(t, m.cfg.freq_dim, DEV).bfloat16().double()
    temb = lin(m.time_out, silu(lin(m.time_in, f)))
    temb6 = lin(m.time_proj, silu(temb)).view(6, -1)
    c = lin(m.text_out, gelu(lin(m.text_in, text)))
    for b in m.blocks:
        shift, scale, gate, c_shift, c_scale, c_gate = P(b.scale_shift_table) + temb6
        n = ln(x, 1 + scale, shift)
        a1, a2 = b.attn1, b.attn2
        q, k = rope(rms(lin(a1.to_q, n), a1.norm_q)), rope(rms(lin(a1.to_k, n), a1.norm_k))
        x = x + gate * lin(a1.to_out[0], attend(q, k, heads(lin(a1.to_v, n)), q_ranges, k_ranges))
        n = ln(x, P(b.norm2_w), P(b.norm2_b))
        q, k = heads(rms(lin(a2.to_q, n), a2.norm_q)), heads(rms(lin(a2.to_k, c), a2.norm_k))
        x = x + lin(a2.to_out[0], attend(q, k, heads(lin(a2.to_v, c)), q_ranges, sentences))
        x = x + c_gate * lin(b.ffn_out, gelu(lin(b.ffn_in, ln(x, 1 + c_scale, c_shift))))
    shift, scale = P(m.scale_shift_table) + temb
    return lin(m.proj_out, ln(x, 1 + scale, shift))


def test_gradients_of_every_weight():
    print('training pass', flush=True)
    m = model()
    tokens, text, rotary, dy = inputs()
    params = m.parameters()
    assert len({id(p) for p in params}) == len(params) == 14 + 2 * 27 + 1
    for p in params:
        p.requires_grad_()
    tokens.requires_grad_()
    text.requires_grad_()
    out = m.differentiable_forward(tokens, 300.0, text, rotary)
    out.backward(dy)
    exact = {id(p): p.detach().double().requires_grad_() for p in [*params, tokens, text]}
    rows = {}
    want = exact_forward(m, exact, exact[id(tokens)], 300.0, exact[id(text)], rotary, rows)
    assert ((out.double() - want).norm() / want.norm()).item() <= 2.5e-2
    want.backward(dy.double())
    for i, p in enumerate([*params, tokens, text]):
        g = exact[id(p)].grad
        assert p.grad.dtype == p.dtype and bool(torch.isfinite(p.grad).all()), i
        size = g.norm() + (rows[id(p)].grad.norm() if id(p) in rows else 0)
        off = ((p.grad.double() - g).norm() / size).item()
        assert off <= 2.5e-2, f'parameter {i} {tuple(p.shape)}: {off:.3e}'


def test_forward_agrees_with_the_inference_pass():
    print('inference pass', flush=True)
    m = model()
    tokens, text, rotary, _ = inputs()
    a, b = m.differentiable_forward(tokens, 20.0, text, rotary), m.forward(tokens, 20.0, text, rotary)
    assert not a.requires_grad and ((a.double() - b.double()).norm() / b.double().norm()).item() <= 2.5e-2


def test_gradients_of_some_weights():
    """weights that require no gradient get none, and those that do get the ones they had with all of them"""
    print('some weights', flush=True)
    m = model()
    tokens, text, rotary, dy = inputs()
    tables = [b.scale_shift_table for b in m.blocks]
    for p in tables:
        p.requires_grad_()
    m.differentiable_forward(tokens, 10.0, text, rotary).backward(dy)
    first = [p.grad.clone() for p in tables]
    for p in m.parameters():
        p.requires_grad_()
        p.grad = None
    m.differentiable_forward(tokens, 10.0, text, rotary).backward(dy)
    assert all(torch.equal(p.grad, g) for p, g in zip(tables, first))


def test_scopes_without_a_gradient_are_refused():
    m = model(halo=0, extra={0: [3], 1: [0]})
    tokens, text, rotary, _ = inputs()
    with pytest.raises(L.HipValueError, match='halo'):
        m.differentiable_forward(tokens, 1.0, text, rotary)
