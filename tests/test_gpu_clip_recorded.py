"""Clipping where autograd records: neither the norm nor what is scaled has a gradient, and a backward pass that reaches them raises, as
behind grad_norm; a leaf that requires a gradient is not overwritten."""
import pytest
import torch

from onereel_amd import _lib as L
from onereel_amd import clip

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'


def pair():
    g = torch.Generator(device=DEV).manual_seed(1)
    return torch.randn(40, generator=g, device=DEV, requires_grad=True), torch.randn(9, 5, generator=g, device=DEV)


def test_into_others():
    print('clip recorded: out', flush=True)
    w, t = pair()
    want = [torch.empty_like(w), torch.empty_like(t)]
    with torch.no_grad():
        wanted = clip.clip_grads_([w, t], 1.0, out=want)
    assert not wanted.requires_grad and not any(o.requires_grad for o in want)
    for pick in (lambda norm, out: norm, lambda norm, out: out[0].sum(), lambda norm, out: out[1].sum()):
        out = [torch.empty_like(t) for t in want]
        norm = clip.clip_grads_([w, t], 1.0, out=out)
        assert torch.equal(norm, wanted) and all(torch.equal(a, b) for a, b in zip(out, want))
        w.grad = None
        with pytest.raises(L.HipValueError, match='clip.clip_grads_'):
            (pick(norm, out) + w.sum()).backward()
    # one of many outputs that a recorded tensor is behind, in another type and as views of one buffer
    flat = torch.empty(85, dtype=torch.bfloat16, device=DEV)
    out = [flat[:40], flat[40:].view(9, 5)]
    clip.clip_grads_([w, t], 1.0, out=out)
    with pytest.raises(L.HipValueError, match='clip.clip_grads_'):
        flat.float().sum().backward()


def test_in_place():
    print('clip recorded: in place', flush=True)
    w, t = pair()
    made, beside = 2 * w, t.clone()
    keep = [made.detach().clone(), beside.clone()]
    with torch.no_grad():
        wanted = clip.clip_grads_(keep, 1.0)
    norm = clip.clip_grads_([made, beside], 1.0)
    assert torch.equal(norm, wanted) and torch.equal(made, keep[0]) and torch.equal(beside, keep[1])
    for y in (norm, made.sum(), beside.sum()):
        with pytest.raises(L.HipValueError, match='clip.clip_grads_'):
            (y + w.sum()).backward()
    square = 2 * w
    y = square.square().sum()                       # keeps what square held
    clip.clip_grads_([square], 1.0)
    with pytest.raises(RuntimeError):
        y.backward()


def test_what_autograd_cannot_follow_is_not_overwritten():
    print('clip recorded: leaves', flush=True)
    w, t = pair()
    before = [w.detach().clone(), t.clone()]
    other = torch.zeros(40, device=DEV, requires_grad=True)
    flat = torch.zeros(85, device=DEV)
    with torch.inference_mode():
        made = torch.zeros(40, device=DEV)
    for f in (lambda: clip.clip_grads_([t, w], 1.0), lambda: clip.clip_grads_([t, w[:20]], 1.0),
              lambda: clip.clip_grads_([w.detach(), t], 1.0, out=[other, torch.empty_like(t)]),
              lambda: clip.clip_grads_([w], 1.0, out=[flat.split([40, 45])[0]]), lambda: clip.clip_grads_([w], 1.0, out=[made])):
        with pytest.raises(L.HipValueError, match='no_grad'):
            f()
    # a refusal for another reason leaves autograd's share undone too
    with pytest.raises(L.HipPathError, match='share memory'):
        clip.clip_grads_([w, w.detach()], 1.0, out=[flat[:40], flat[20:60]])
    assert torch.equal(w, before[0]) and torch.equal(t, before[1]) and not other.any() and not flat.any() and not made.any()
    assert w.is_leaf and not t.requires_grad and not flat.requires_grad
    with torch.no_grad():
        clip.clip_grads_([w], 1.0, out=[flat.split([40, 45])[0]])
        assert flat[:40].any()
        clip.clip_grads_([t, w], 1.0)
    assert not torch.equal(w, before[0]) and w.is_leaf
    # views of several where nothing requires a gradient, as a data-parallel program has its buckets
    clip.clip_grads_(flat.split([40, 45]), 0.1)


def test_gradients_of_parameters():
    """as torch's function of that name: no graph, whether or not the gradients have one"""
    print('clip recorded: parameters', flush=True)
    p = torch.nn.Parameter(torch.arange(1.0, 5.0, device=DEV))
    (g,) = torch.autograd.grad((p ** 3).sum(), p, create_graph=True)
    assert g.requires_grad
    q = torch.nn.Parameter(p.detach().clone())
    p.grad, q.grad = g, g.detach().clone()
    want = torch.nn.utils.clip_grad_norm_([q], 1.0)
    norm = clip.clip_grad_norm_([p], 1.0)
    assert not norm.requires_grad and abs(norm.item() - want.item()) <= 2 ** -22 * want.item()
    assert ((p.grad - q.grad).abs() <= 2 ** -21 * q.grad.abs()).all()
    with torch.inference_mode():
        made = torch.randn(10, device=DEV)
        keep = made.clone()
        clip.clip_grads_([made], 0.1)
        assert not torch.equal(made, keep)
