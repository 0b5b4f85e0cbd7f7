"""The global norm of many gradients and their clipping, against float64.

Tolerances: squares are exact in fp64 and summed there (relative 2^-52 times the additions, nothing here), so the norm is off by its
rounding to fp32, 2^-24, and 1e-12. The factor is rounded to fp32 and multiplies in fp32: 2^-23 of a result before its own
rounding (half a step of its type)."""
import math

import pytest
import torch

from onereel_amd import _lib as L
from onereel_amd import clip

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def tensors(sizes, seed=0, types=TYPES, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(scale * torch.randn(n, generator=g, device=DEV)).to(types[i % len(types)]) for i, n in enumerate(sizes)]


def exact_norm(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


def check_norm(got, ts):
    want = exact_norm(ts)
    assert got.dtype == torch.float32 and got.shape == () and got.is_cuda
    assert abs(got.double().item() - want) <= (2 ** -24 + 1e-12) * want


def check_scaled(out, ts, max_norm):
    c = min(1.0, max_norm / (exact_norm(ts) + 1e-6))
    for o, t in zip(out, ts):
        f = torch.finfo(o.dtype)
        want = t.double() * c
        past = (o.double() - want).abs() - (f.eps / 2 * (1 + 2 ** -10) + 2 ** -23) * want.abs() - f.smallest_normal * f.eps / 2
        assert past.numel() == 0 or past.max().item() <= 0


SIZES = [[1], [8], [4096], [4097, 1], [0, 5, 0], [7] * 300, [1, 100000, 3, 65537, 8191], list(range(1, 400)), [3000000, 17],
         [129] * 128, [129] * 129]


@pytest.mark.parametrize('sizes', SIZES, ids=lambda s: f'{len(s)}x{max(s)}')
def test_norm_and_clipping(sizes):
    print(f'clip {len(sizes)} tensors, largest {max(sizes)}', flush=True)
    ts = tensors(sizes)
    keep = [t.clone() for t in ts]
    check_norm(clip.grad_norm(ts), keep)
    for limit in (0.3, 0.999, 1.5):
        max_norm = limit * exact_norm(keep)
        out = [torch.full_like(t, 7, dtype=TYPES[(i + 1) % 3]) for i, t in enumerate(ts)]
        check_norm(clip.clip_grads_(ts, max_norm, out=out), keep)
        check_scaled(out, keep, max_norm)
        assert all(torch.equal(a, b) for a, b in zip(ts, keep))
        mine = [t.clone() for t in keep]
        norm = clip.clip_grads_(mine, max_norm)
        check_norm(norm, keep)
        check_scaled(mine, keep, max_norm)
        if limit > 1:
            assert all(torch.equal(a, b) for a, b in zip(mine, keep))
        again = [t.clone() for t in keep]
        assert torch.equal(norm, clip.clip_grads_(again, max_norm)) and all(torch.equal(a, b) for a, b in zip(mine, again))


@pytest.mark.parametrize('dtype', TYPES, ids=str)
def test_views_of_a_bucket_at_any_alignment(dtype):
    print(f'clip bucket {dtype}', flush=True)
    sizes = [1, 2, 3, 5, 4096, 4099, 12289, 7, 20000]
    flat = tensors([sum(sizes) + 2], 3, [dtype])[0]
    keep = flat.clone()
    inner = flat[1:-1]
    check_norm(clip.clip_grads_(inner.split(sizes), 0.5), [keep[1:-1]])
    check_scaled([inner], [keep[1:-1]], 0.5)
    assert flat[0] == keep[0] and flat[-1] == keep[-1]
    out = torch.full((flat.numel() + 1,), 9.0, device=DEV)
    clip.clip_grads_(keep[1:-1].split(sizes), 0.5, out=out[2:-1].split(sizes))
    check_scaled([out[2:-1]], [keep[1:-1]], 0.5)
    assert out[0] == out[1] == out[-1] == 9


def test_layouts():
    print('clip layouts', flush=True)
    t = torch.randn(40, 30, device=DEV)
    turned = t.clone().t()                                   # not contiguous, fills its memory
    check_norm(clip.clip_grads_([turned], 1.0), [t])
    check_scaled([turned.t()], [t], 1.0)
    part = t.clone()[:, :7]
    check_norm(clip.grad_norm([part, t.sum().expand(3, 5)]), [part, t.sum().expand(3, 5)])
    out = torch.empty(40, 7, device=DEV)
    clip.clip_grads_([part], 1.0, out=[out])
    check_scaled([out], [part], 1.0)
    with pytest.raises(L.HipValueError, match='fill'):
        clip.clip_grads_([part], 1.0)


def test_large_and_small_values():
    print('clip extremes', flush=True)
    big = torch.full((100000,), 1e30, device=DEV)            # squares past fp32
    keep = big.clone()
    check_norm(clip.clip_grads_([big], 1.0), [keep])
    check_scaled([big], [keep], 1.0)
    small = torch.full((1000,), 1e-30, device=DEV)
    check_norm(clip.clip_grads_([small], 1.0), [small])
    none = torch.zeros(5000, device=DEV)
    assert clip.clip_grads_([none], 0.0).item() == 0 and not none.any()
    t = torch.randn(100, device=DEV)
    clip.clip_grads_([t], 0.0)
    assert not t.any()
    t = torch.randn(100, device=DEV)
    keep = t.clone()
    clip.clip_grads_([t], math.inf)
    assert torch.equal(t, keep)


@pytest.mark.parametrize('value', [math.inf, math.nan])
def test_not_finite_as_torch(value):
    print(f'clip {value}', flush=True)
    ts = [torch.randn(1000, device=DEV) for _ in range(3)]
    ts[1][17] = value
    ps = [torch.nn.Parameter(torch.zeros_like(t)) for t in ts]
    for p, t in zip(ps, ts):
        p.grad = t.clone()
    want = torch.nn.utils.clip_grad_norm_(ps, 1.0)
    got = clip.clip_grads_(ts, 1.0)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    for t, p in zip(ts, ps):
        assert torch.equal(t.isnan(), p.grad.isnan()) and torch.equal(t.nan_to_num(5), p.grad.nan_to_num(5))


def test_parameters():
    print('clip parameters', flush=True)
    ps = [torch.nn.Parameter(t) for t in tensors([300, 5000, 7], 1)]
    ps[2].requires_grad_()
    for i, p in enumerate(ps[:2]):
        p.grad = 3 * p.detach().clone()
    keep = [p.grad.clone() for p in ps[:2]]
    version = ps[0].grad._version
    check_norm(clip.clip_grad_norm_(iter(ps), 2.0), keep)
    check_scaled([p.grad for p in ps[:2]], keep, 2.0)
    assert ps[2].grad is None and ps[0].grad._version > version
    check_norm(clip.clip_grad_norm_(ps[0], 100.0), [ps[0].grad])
    assert clip.clip_grad_norm_([], 1.0).item() == 0 and clip.grad_norm([]).item() == 0 and clip.grad_norm([ps[0][:0]]).item() == 0


def test_shared_memory_is_refused():
    t = torch.randn(100, device=DEV)
    other = torch.empty(100, device=DEV)
    bad = [lambda: clip.clip_grads_([t, t], 1.0), lambda: clip.clip_grads_([t[:60], t[50:]], 1.0),
           lambda: clip.clip_grads_([t[:50], t[50:]], 1.0, out=[t[50:], t[:50]]),
           lambda: clip.clip_grads_([t[:50], t[50:]], 1.0, out=[other[:50], other[:50]]),
           lambda: clip.clip_grads_([t], 1.0, out=[t.view(torch.bfloat16)[:100]])]
    for f in bad:
        with pytest.raises(L.HipPathError, match='share memory|another type'):
            f()
    keep = t.clone()
    clip.clip_grads_([t, t], 1.0, out=[other, torch.empty_like(t)])      # read twice, written apart
    check_norm(clip.grad_norm([t, t]), [keep, keep])
    clip.clip_grads_([t[:50], t[50:]], 0.1, out=[t[:50], t[50:]])        # in place by name
    check_scaled([t], [keep], 0.1)


def test_refusals():
    t = torch.randn(10, device=DEV)
    bad = [lambda: clip.grad_norm([t.double()]), lambda: clip.grad_norm([t.int()]), lambda: clip.grad_norm([t, t.cpu()]),
           lambda: clip.clip_grads_([t], -1.0), lambda: clip.clip_grads_([t], math.nan),
           lambda: clip.clip_grads_([t], 1.0, out=[]), lambda: clip.clip_grads_([t], 1.0, out=[torch.empty(9, device=DEV)]),
           lambda: clip.clip_grads_([t], 1.0, out=[torch.empty(10)]),
           lambda: clip.clip_grads_([t], 1.0, out=[torch.empty(20, device=DEV)[::2]])]
    for f in bad:
        with pytest.raises(L.HipPathError):
            f()


def test_graph_replays_and_streams():
    print('clip graph', flush=True)
    ts = tensors([5000] * 150 + [300001, 3], 5)
    outs = [torch.empty_like(t) for t in ts]

    def step():
        return clip.clip_grads_(ts, 100.0, out=outs)

    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        norm = step()
    for seed in (6, 7, 8):
        for t, n in zip(ts, tensors([5000] * 150 + [300001, 3], seed)):
            t.copy_(n)
        want = step()
        keep = [o.clone() for o in outs]
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(outs, keep))
    sets = [[t.clone() for t in ts] for _ in range(2)]
    for s, mine in zip([torch.cuda.Stream() for _ in range(2)], sets):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            clip.clip_grads_(mine, 100.0)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for mine in sets for a, b in zip(mine, keep))


def test_a_norm_that_autograd_would_record_has_no_gradient():
    w = torch.randn(40, device=DEV, requires_grad=True)
    norm = clip.grad_norm([w, torch.ones(3, device=DEV)])
    want = torch.cat([w.detach().double(), torch.ones(3, device=DEV, dtype=torch.float64)]).norm()
    assert abs(norm.item() - want.item()) <= 1e-6 * want.item()
    with pytest.raises(L.HipValueError, match='clip.grad_norm'):
        (norm + w.sum()).backward()
    with torch.no_grad():
        assert not clip.grad_norm([w]).requires_grad
    assert not clip.grad_norm([w.detach()]).requires_grad
