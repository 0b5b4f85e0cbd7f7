"""The norms, rotary positions, 4-bit linear layers and gradient clipping together, as a pass of the Wan-shaped DiT runs them.

Tolerance of a pass: as in test_gpu_training_pass.py, 2.5e-2 relative in the 2-norm for two blocks, in whose 40 roundings to bf16 each
result is off by at most 2^-8; with the feed forward's and attention's outputs rounded before their gates two more a block:
sqrt(44) 2^-8 = 2.6e-2. A bias's gradient may be off by as much of |sum| + sqrt(sum |dz_row|^2), and so may a gradient summed over
rows in general (the modulation's tables)."""
import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from onereel_amd import clip, mxfp4, rotary
from onereel_amd import wan_dit as WD
from onereel_amd.layout import SceneLayout

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'
LENGTHS, T, TEXT_LEN, HALO = [2, 3, 2], 16, 8, 1
STEPS = [0.0, 300.0, 300.0, 10.0, 700.0, 900.0, 0.0]
BOUND = 2.6e-2


def model(extra=None, seed=3):
    cfg = WD.DiTConfig(dim=512, heads=4, ffn=1024, blocks=2, in_channels=4, text_dim=256, std=0.05)
    lay = SceneLayout(LENGTHS, halo=0, extra=extra) if extra else SceneLayout(LENGTHS, halo=HALO)
    return WD.WanDiT(cfg, lay, T, TEXT_LEN, DEV, seed=seed)


def inputs():
    g = torch.Generator(device=DEV).manual_seed(5)
    S = sum(LENGTHS) * T
    tokens = torch.randn(S, 16, generator=g, device=DEV).bfloat16()
    text = torch.randn(3 * TEXT_LEN, 256, generator=g, device=DEV).bfloat16()
    return tokens, text, rotary.grid(sum(LENGTHS), 4, 4, 128), torch.randn(S, 16, generator=g, device=DEV).bfloat16()


def tables():
    return tuple(x.to(DEV) for x in WD.wan_rope_table(sum(LENGTHS), 4, 4, 128))


def relative(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


def exact_forward(m, w, tokens, steps, text, rows):
    """the pass in float64 with a timestep for each frame; w: the model's parameters in double by identity; rows: a zero added to
    every layer's output, whose gradient is the rows that its bias's gradient is the sum of"""
    P = lambda p: w[id(p)]

    def lin(l, x):
        y = x @ P(l.weight).T + P(l.bias)
        rows[id(l.bias)] = torch.zeros_like(y, requires_grad=True)
        return y + rows[id(l.bias)]

    eps, H, lay = m.cfg.eps, m.cfg.heads, m.ctx.layout
    silu = lambda x: x * torch.sigmoid(x)
    gelu = lambda x: 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)))
    rms = lambda x, n: x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * P(n.weight)
    ln = lambda x, a, b: F.layer_norm(x, x.shape[-1:], eps=eps) * a + b
    cos, sin = (t[0].double() for t in tables())

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

    q_ranges = [(T * a, T * b) for a, b in lay.ranges]
    k_ranges = [tuple(T * f for f in lay.key_range(j)) for j in range(lay.n_scenes)]
    sentences = [(TEXT_LEN * j, TEXT_LEN * (j + 1)) for j in range(lay.n_scenes)]
    heads = lambda x: x.unflatten(1, (H, -1))
    per_row = lambda v: v.repeat_interleave(T, 0)
    x = lin(m.patch_embed, tokens)
    f = torch.stack([WD.timestep_features(t, m.cfg.freq_dim, DEV) for t in steps]).bfloat16().double()
    temb = lin(m.time_out, silu(lin(m.time_in, f)))
    temb6 = lin(m.time_proj, silu(temb)).view(len(steps), 6, -1)
    c = lin(m.text_out, gelu(lin(m.text_in, text)))
    for b in m.blocks:
        shift, scale, gate, c_shift, c_scale, c_gate = (per_row(t) for t in (P(b.scale_shift_table) + temb6).unbind(1))
        n = ln(x, 1 + scale, shift)
        a1, a2 = b.attn1, b.attn2
        q, k = rope(rms(lin(a1.to_q, n), a1.norm_q)), rope(rms(lin(a1.to_k, n), a1.norm_k))
        x = x + gate * lin(a1.to_out[0], attend(q, k, heads(lin(a1.to_v, n)), q_ranges, k_ranges))
        n = ln(x, P(b.norm2_w), P(b.norm2_b))
        q, k = heads(rms(lin(a2.to_q, n), a2.norm_q)), heads(rms(lin(a2.to_k, c), a2.norm_k))
        x = x + lin(a2.to_out[0], attend(q, k, heads(lin(a2.to_v, c)), q_ranges, sentences))
        x = x + c_gate * lin(b.ffn_out, gelu(lin(b.ffn_in, ln(x, 1 + c_scale, c_shift))))
    shift, scale = (per_row(t) for t in (P(m.scale_shift_table) + temb[:, None]).unbind(1))
    return lin(m.proj_out, ln(x, 1 + scale, shift))


def test_gradients_with_a_timestep_for_each_frame():
    print('dit operators: gradients', flush=True)
    m = model()
    tokens, text, axes, dy = inputs()
    params = m.parameters()
    for p in params:
        p.requires_grad_()
    tokens.requires_grad_()
    text.requires_grad_()
    out = m.differentiable_forward(tokens, STEPS, text, axes)
    out.backward(dy)
    exact = {id(p): p.detach().double().requires_grad_() for p in [*params, tokens, text]}
    rows = {}
    want = exact_forward(m, exact, exact[id(tokens)], STEPS, exact[id(text)], rows)
    assert relative(out, want) <= BOUND
    want.backward(dy.double())
    for i, p in enumerate([*params, tokens, text]):
        g = exact[id(p)].grad
        assert p.grad.dtype == p.dtype and bool(torch.isfinite(p.grad).all()), i
        size = g.norm() + (rows[id(p)].grad.norm() if id(p) in rows else 0)
        off = ((p.grad.double() - g).norm() / size).item()
        assert off <= BOUND, f'parameter {i} {tuple(p.shape)}: {off:.3e}'
    # and the clipping that follows, against float64 of the gradients themselves
    keep = [p.grad.clone() for p in params]
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in keep))
    got = m.clip_gradients(norm / 3)
    assert abs(got.double().item() - norm) <= 1e-6 * norm
    for p, g in zip(params, keep):
        w = g.double() / 3
        assert ((p.grad.double() - w).abs() <= (torch.finfo(g.dtype).eps / 2 + 2 ** -20) * w.abs() + 1e-30).all()
    assert abs(clip.grad_norm([p.grad for p in params]).item() - norm / 3) <= 2 ** -9 * norm / 3


def test_equal_timesteps_and_positions_are_the_pass_with_one_and_tables():
    print('dit operators: equal timesteps', flush=True)
    m = model()
    tokens, text, axes, _ = inputs()
    want = m.forward(tokens, 300.0, text, tables())
    for t in (300.0, torch.tensor(300.0), [300.0] * 7, torch.full((7,), 300.0)):
        assert relative(m.forward(tokens, t, text, axes), want) <= BOUND
        assert relative(m.differentiable_forward(tokens, t, text, axes), want) <= BOUND


def test_frame_memory_scopes_with_a_timestep_for_each_frame():
    print('dit operators: frame memory', flush=True)
    m = model(extra={0: [3, 6], 1: [0], 2: [0, 4]})
    tokens, text, axes, _ = inputs()
    want = m.forward(tokens, 300.0, text, tables())
    assert relative(m.forward(tokens, [300.0] * 7, text, axes), want) <= BOUND
    assert relative(m.forward(tokens, STEPS, text, axes), want) > BOUND


def test_a_wrong_count_of_timesteps_is_refused():
    m = model()
    tokens, text, axes, _ = inputs()
    for call in (m.forward, m.differentiable_forward):
        with pytest.raises(ValueError, match='timesteps'):
            call(tokens, [1.0, 2.0], text, axes)


@pytest.mark.parametrize('steps', [300.0, STEPS], ids=['one', 'each'])
@pytest.mark.parametrize('extra', [None, {0: [3, 6], 1: [0], 2: [0, 4]}], ids=['halo', 'memory'])
def test_a_pass_in_4_bits(steps, extra, monkeypatch):
    """every layer of the blocks runs in 4 bits, each call against float64 of what it was given: (n_in / 64 + 64) 2^-23 of the
    product's magnitudes and 2^-8 of the result"""
    print('dit operators: 4 bits', flush=True)
    m = model(extra)
    tokens, text, axes, _ = inputs()
    plain = m.forward(tokens, steps, text, axes)
    assert m.quantize() is m
    real, calls = mxfp4.linear, []

    def checked(x, weight, bias=None, activation=None):
        y = real(x, weight, bias, activation=activation)
        q = x if isinstance(x, mxfp4.MXFP4) else mxfp4.quantize(x)
        xv, wv = (t.dequantize(torch.float32).double() for t in (q, weight))
        z = xv @ wv.T + bias.double()
        want = F.gelu(z, approximate='tanh') if activation else z
        off = 1.13 * (xv.shape[-1] / 64 + 66) * 2 ** -23 * (xv.abs() @ wv.abs().T + bias.double().abs()) + 2 ** -20 * z.abs()
        assert ((y.double() - want).abs() <= off + 2 ** -8 * (want.abs() + off) + 1e-30).all()
        calls.append(isinstance(x, mxfp4.MXFP4))
        return y

    monkeypatch.setattr(mxfp4, 'linear', checked)
    out = m.forward(tokens, steps, text, axes)
    assert len(calls) == 2 * 10 and sum(calls) == 2 * 3          # queries, keys and values share their rows in 4 bits
    assert bool(torch.isfinite(out).all()) and out.shape == plain.shape
    monkeypatch.undo()
    assert torch.equal(m.forward(tokens, steps, text, axes), out)
    if extra is None:
        # training keeps the bf16 weights
        assert relative(m.differentiable_forward(tokens, steps, text, axes), plain) <= BOUND


def test_norm_rotate_in_the_processor_shares_scenes_positions():
    """positions that restart at every scene (scene-wise RoPE) against tables gathered the same way"""
    print('dit operators: scene positions', flush=True)
    m = model()
    tokens, text, axes, _ = inputs()
    starts = [a for a, _ in m.ctx.layout.ranges]
    frame = torch.arange(sum(LENGTHS)).repeat_interleave(T)
    scene = torch.bucketize(frame, torch.tensor(starts[1:]), right=True)
    within = axes.positions.clone()
    within[:, 0] -= torch.tensor(starts, device=DEV, dtype=torch.int32)[scene.to(DEV)]
    row = within[:, 0].long() * T + torch.arange(T, device=DEV).repeat(sum(LENGTHS))
    table = tuple(t[:, row] for t in tables())
    a = m.forward(tokens, 20.0, text, table)
    b = m.forward(tokens, 20.0, text, rotary.Axes(within, axes.dims))
    assert relative(b, a) <= BOUND and not torch.equal(m.forward(tokens, 20.0, text, tables()), a)


def test_what_one_timestep_may_come_as():
    """numbers of any kind and tensors or arrays of one element are one timestep for all; a tensor on the GPU is one for each frame
    without the host reading it, so that such a pass can be captured"""
    print('dit operators: kinds of timesteps', flush=True)
    m = model()
    tokens, text, axes, _ = inputs()
    with torch.no_grad():
        want = m.forward(tokens, 300.0, text, axes)
        for t in (300, np.float32(300), np.int64(300), np.array(300.0), torch.tensor(300.0, device=DEV), torch.tensor([300.0], device=DEV)):
            assert torch.equal(m.forward(tokens, t, text, axes), want)
        want = m.forward(tokens, STEPS, text, axes)
        steps = torch.tensor(STEPS, device=DEV)
        for t in (tuple(STEPS), np.array(STEPS), torch.tensor(STEPS), steps):
            assert torch.equal(m.forward(tokens, t, text, axes), want)
        for t in (steps[:3], steps[None], steps.repeat(2), []):
            with pytest.raises(ValueError, match='timesteps'):
                m.forward(tokens, t, text, axes)


def test_a_model_is_quantised_whole_or_not_at_all():
    """a feed forward of 1032 columns does not divide into blocks of 32: no layer is left in 4 bits"""
    cfg = WD.DiTConfig(dim=512, heads=4, ffn=1032, blocks=1, in_channels=4, text_dim=256, std=0.05)
    m = WD.WanDiT(cfg, SceneLayout(LENGTHS, halo=HALO), T, TEXT_LEN, DEV, seed=3)
    with pytest.raises(ValueError, match='multiple of 32'):
        m.quantize()
    assert all(l.quantized is None for b in m.blocks for l in b.linears())
