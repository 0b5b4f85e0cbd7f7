"""Outputs of calls that autograd records take in-place operations, as they do without autograd: they are no views made inside
a custom autograd function, nor several views of one output."""
import pytest
import torch

from helpers import rand_bf16
from onereel_amd import attention as A
from onereel_amd import wan
from onereel_amd.linear import linear, linear_backward

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'


def doubled(call, leaves, grads):
    """call(*leaves)'s outputs doubled in place: twice the values, and twice the gradients (exact in bf16 and fp32). The inputs
    need no gradient for the plain call, only the weights as in a model whose parameters have theirs switched on"""
    plain = [t.clone() for t in call(*(t.detach() for t in leaves))]
    want = torch.autograd.grad(call(*leaves), leaves, grads)
    out = call(*leaves)
    for y in out:
        y.mul_(2)
    assert all(torch.equal(y, 2 * p) for y, p in zip(out, plain))
    got = torch.autograd.grad(out, leaves, grads)
    assert all(torch.equal(a, 2 * b) for a, b in zip(got, want))


@pytest.mark.parametrize('lead', [(), (1,), (2, 1)])
def test_norms(lead):
    print(f'in place: norms {lead}', flush=True)
    S, H, D = 40, 8, 64
    C, n = H * D, S * len(lead or (1,))
    q, k, dq, dk = (rand_bf16((n, C), i).to(DEV).view(*lead, -1, C) for i in range(4))
    wq, wk = (rand_bf16((C,), 7 + i).to(DEV).requires_grad_() for i in range(2))
    a = torch.rand(n, D // 2, generator=torch.Generator().manual_seed(1), dtype=torch.float64) * 6.3
    cos, sin = (t.float().repeat_interleave(2, 1).to(DEV) for t in (a.cos(), a.sin()))
    heads = lambda t: t.view(*t.shape[:-1], H, D)
    doubled(lambda x, y: wan._qk(q, k, x, y, 1e-6, cos, sin, H), [wq, wk], [heads(dq), heads(dk)])
    doubled(lambda x: [wan.rms_norm(q, x, 1e-6)], [wq], [dq])
    x = q.clone().requires_grad_()
    doubled(lambda x: [wan.rms_norm(x, wq.detach(), 1e-6)], [x], [dq])


@pytest.mark.parametrize('shape', [(48,), (5, 48), (2, 3, 48)])
@pytest.mark.parametrize('activation', [None, 'silu'])
def test_linear(shape, activation):
    print(f'in place: linear {shape} {activation}', flush=True)
    x, w = rand_bf16(shape, 1).to(DEV), rand_bf16((64, 48), 2).to(DEV)
    dy = rand_bf16((*shape[:-1], 64), 3).to(DEV)
    leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
    doubled(lambda a, b: [linear(a, b, activation=activation)], leaves, [dy])
    y, z = linear(*leaves, activation=activation, keep_preactivation=True)
    kept = z.clone()
    z.add_(1)                               # the caller's own
    assert y.shape == z.shape == dy.shape and torch.equal(z, kept + 1)
    want = linear_backward(dy, x, w, activation=activation, preactivation=kept)[:2]
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, dy), want))


@pytest.mark.parametrize('lse', [False, True])
def test_packed(lse):
    """every sequence's output takes in-place operations; the gradient, which reads the outputs, then says that they changed
    (as torch's own operations that keep their result do)"""
    print(f'in place: packed lse={lse}', flush=True)
    H, D = 2, 64
    segments = [tuple(rand_bf16((n, H, D), 10 * s + i).to(DEV).requires_grad_() for i, n in enumerate((nq, nk, nk)))
                for s, (nq, nk) in enumerate(((9, 33), (1, 4), (70, 20)))]
    call = lambda: [t for pair in A.packed_lse(segments) for t in pair] if lse else list(A.packed(segments))
    with torch.no_grad():
        want = call()
    out = call()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    out[0].mul_(2)
    assert torch.equal(out[0], 2 * want[0]) and all(torch.equal(a, b) for a, b in zip(out[1:], want[1:]))
    with pytest.raises(RuntimeError, match='inplace'):
        out[-2 if lse else -1].sum().backward()
    if lse:                                 # the log-sum-exps are the caller's own
        out = call()
        want = torch.autograd.grad(out[0::2], segments[0], [torch.ones_like(t) for t in out[0::2]], retain_graph=True)
        for t in out[1::2]:
            t.mul_(2)
        got = torch.autograd.grad(out[0::2], segments[0], [torch.ones_like(t) for t in out[0::2]])
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    out = call()
    torch.autograd.backward(out, [torch.ones_like(t) for t in out])
    assert all(bool(torch.isfinite(t.grad.float()).all()) for s in segments for t in s)
