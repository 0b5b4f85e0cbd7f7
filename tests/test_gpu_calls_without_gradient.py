"""Scopes and calls that have no gradient: they run as they do without autograd, and a backward pass that reaches their outputs
says so, where it would leave out a part of the gradient."""
import pytest
import torch

from helpers import rand_bf16
from onereel_amd import _lib as L
from onereel_amd import attention as A
from onereel_amd import hunyuan15 as HY
from onereel_amd import wan
from onereel_amd import wan_dit as WD
from onereel_amd.layout import SceneLayout

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'
LENGTHS, T, H, D = [2, 3, 2], 16, 2, 128
S = sum(LENGTHS) * T


def refused(call, inputs, what):
    """call(*inputs)'s outputs: the bits of the call without autograd, and a gradient of each that raises"""
    with torch.no_grad():
        want = call(*inputs)
    some = [[x.clone().requires_grad_(i in on) for i, x in enumerate(inputs)]
            for on in ([0], [len(inputs) - 1], range(len(inputs)))]
    for xs in some:
        for i, w in enumerate(want):
            out = call(*xs)
            assert torch.equal(out[i], w)
            with pytest.raises(L.HipValueError, match=what):
                (out[i].float() * 2).sum().backward()
            assert all(x.grad is None for x in xs)


@pytest.mark.parametrize('extra,memory', [({0: [3, 6], 1: [0], 2: [0, 4]}, 0), ({}, 4)])
def test_wan_scopes(extra, memory):
    print(f'wan scopes extra={bool(extra)} memory={memory}', flush=True)
    ctx = lambda: wan.Context(SceneLayout(LENGTHS, halo=0, extra=extra), memory=memory, T=T)
    q, k, v = (rand_bf16((S, H, D), i).to(DEV) for i in range(3))
    if memory:
        refused(lambda *x: [wan.memory_self(ctx(), *x, 0)], [q, k, v], 'bounded memory')
    else:
        refused(lambda *x: [wan.self_ranges(ctx(), *x)], [q, k, v], 'extra frames')


@pytest.mark.parametrize('extra,memory', [({0: [3, 6], 1: [0], 2: [0, 4]}, 0), ({}, 4)])
def test_wan_processor(extra, memory):
    """through the hook: the norms before the attention are recorded, the projections are trained"""
    print(f'wan processor extra={bool(extra)} memory={memory}', flush=True)
    m = WD.WanDiT(WD.DiTConfig(dim=512, heads=4, ffn=1024, blocks=1, in_channels=4, text_dim=256),
                  SceneLayout(LENGTHS, halo=0, extra=extra), T, 8, DEV, seed=3)
    m.ctx.memory = memory
    x, rot = rand_bf16((1, S, 512), 1).to(DEV), tuple(t.to(DEV) for t in WD.wan_rope_table(sum(LENGTHS), 4, 4, 128))
    attn = m.blocks[0].attn1
    with torch.no_grad():
        want = m.p_self(attn, x, rotary_emb=rot)
    m.ctx._mem = None
    for p in (attn.to_q.weight, attn.norm_k.weight):
        p.requires_grad_()
        out = m.p_self(attn, x, rotary_emb=rot)
        m.ctx._mem = None
        assert torch.equal(out, want)
        with pytest.raises(L.HipValueError, match='no gradient'):
            out.sum().backward()
        p.requires_grad_(False)
    attn.to_out[0].weight.requires_grad_()          # behind the attention: nothing of its gradient is left out
    out = m.p_self(attn, x, rotary_emb=rot)
    out.sum().backward()
    assert attn.to_out[0].weight.grad is not None and attn.to_out[0].weight.grad.any()


@pytest.mark.parametrize('memory', [0, 4])
@pytest.mark.parametrize('fused', [True, False])
def test_hunyuan_scopes(memory, fused):
    print(f'hunyuan scopes memory={memory} fused={fused}', flush=True)
    counts, Le = [5, 3, 4], 16
    extra = {} if memory else {0: [3, 6], 1: [0], 2: [0, 4]}
    q, k, v = (rand_bf16((S, H, D), i).to(DEV) for i in range(3))
    eq, ek, ev = (rand_bf16((Le, H, D), 5 + i).to(DEV) for i in range(3))
    cos, sin = (t[0, :, 0].to(DEV) for t in WD.wan_rope_table(sum(LENGTHS), 4, 4, D))

    def call(*x):
        ctx = HY.Context(SceneLayout(LENGTHS, halo=0, extra=extra), T=T, counts={True: counts, False: counts}, memory=memory,
                         fused=fused, fwd=1)
        p = HY.Processor(ctx, 0)
        if not memory:
            return p.scene_raw(*x, cos, sin)
        return p.memory(HY.rotate_tokens(ctx, x[0], cos, sin), HY.rotate_tokens(ctx, x[1], cos, sin), *x[2:])

    refused(call, [q, k, v, eq, ek, ev], 'no gradient')


def test_merge_of_partial_results():
    """merge_lse updates its first two arguments in place, the log-sum-exp that varlen_lse kept for its gradient among them"""
    print('merge', flush=True)
    n = 50
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    xs = [rand_bf16((n, H, D), i).to(DEV) for i in range(5)]

    def parts(q, k1, v1, k2, v2):
        o, lse = A.varlen_lse(q, k1, v1, cu, cu, n, n)
        return (o, o.float(), lse, *A.varlen_lse(q, k2, v2, cu, cu, n, n))

    with torch.no_grad():
        _, o, lse, *rest = parts(*xs)
        want = A.merge_lse(o, lse, *rest)
    leaves = [x.clone().requires_grad_() for x in xs]
    for i in range(2):
        _, o, lse, *rest = parts(*leaves)
        got = A.merge_lse(o, lse, *rest)
        assert got[0] is o and got[1] is lse and all(torch.equal(a, b) for a, b in zip(got, want))
        with pytest.raises(L.HipValueError, match='merge_lse'):
            got[i].sum().backward()
    # what the first call kept has changed, also where the merge itself was not recorded
    first, o, lse, *rest = parts(*leaves)
    with torch.no_grad():
        A.merge_lse(o, lse, *rest)
    with pytest.raises(RuntimeError, match='inplace'):
        first.sum().backward()
    with torch.inference_mode():
        _, o, lse, *rest = parts(*xs)
        assert all(torch.equal(a, b) for a, b in zip(A.merge_lse(o, lse, *rest), want))


def test_inference_pass_of_the_model():
    """WanDiT.forward updates its rows in place: it has the gradient of the output projection alone"""
    print('inference pass', flush=True)
    m = WD.WanDiT(WD.DiTConfig(dim=512, heads=4, ffn=1024, blocks=2, in_channels=4, text_dim=256),
                  SceneLayout(LENGTHS, halo=1), T, 8, DEV, seed=3)
    tokens, text = rand_bf16((S, 16), 1).to(DEV), rand_bf16((24, 256), 2).to(DEV)
    rot = tuple(t.to(DEV) for t in WD.wan_rope_table(sum(LENGTHS), 4, 4, 128))
    run = lambda: m.forward(tokens, 20.0, text, rot)
    with torch.no_grad():
        want = run()
    m.proj_out.weight.requires_grad_()
    run().sum().backward()
    assert m.proj_out.weight.grad.any()
    for p in (m.blocks[0].ffn_in.weight, m.blocks[1].norm2_w, m.time_in.weight, m.blocks[0].attn2.to_v.weight):
        p.requires_grad_()
        out = run()
        assert torch.equal(out, want)
        with pytest.raises(L.HipValueError, match='no gradient'):
            out.sum().backward()
        p.requires_grad_(False)
    x, a = rand_bf16((6, 512), 1).to(DEV).requires_grad_(), rand_bf16((6, 512), 2).to(DEV)
    with pytest.raises(L.HipValueError, match='layernorm_modulate'):
        WD.layernorm_modulate(x, 1e-6, scale=torch.zeros(512, device=DEV), shift=torch.zeros(512, device=DEV)).sum().backward()
    with pytest.raises(L.HipValueError, match='gated_residual_'):
        WD.gated_residual_(x * 1, a).sum().backward()
    # what an earlier call kept has changed
    y = (x * 1).mul(3)
    z = y.exp()
    WD.gated_residual_(z.detach(), a)
    with pytest.raises(RuntimeError, match='inplace'):
        z.sum().backward()
