"""Gradients of the varlen attention over many segments, with the ordinary kernels: more than 256 segments (planned by a launch of
their own) past the size up to which operands carry their rounding, and key ranges of 65 to 4096 segments that are shuffled,
nested, equal and empty. Against the float64 formula, with the tolerances of test_gpu_attention_backward.py."""
import random

import pytest
import torch

from onereel_amd import attention as A
from test_gpu_attention_backward import check, cut, inputs, reference

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'


@pytest.mark.parametrize('n,H,D', [(257, 2, 128), (300, 3, 64), (600, 16, 128), (65, 2, 64), (256, 2, 128), (4096, 1, 64)])
def test_many_segments(n, H, D):
    print(f'{n} segments H={H} D={D}', flush=True)
    rng = random.Random(n)
    lq = [rng.choice([0, 1, rng.randrange(2, 40), rng.randrange(60, 90)]) for _ in range(n)]
    lk = [rng.choice([0, 1, rng.randrange(2, 40), rng.randrange(60, 90)]) for _ in range(n)]
    lq[n // 2], lk[n // 2], lk[n // 3] = 300, 200, 700
    assert H * sum(lq) * max(lk) > 1 << 18
    (qr, cq), (kr, ck) = cut(lq), cut(lk)
    q, k, v, do = inputs(sum(lq), sum(lk), H, D)
    g = [x.to(DEV) for x in (q, k, v, do)]
    args = (cq.to(DEV), ck.to(DEV), max(lq), max(lk))
    o, lse = A.varlen_lse(*g[:3], *args)
    got = A.varlen_backward(g[3], *g[:3], o, lse, *args)
    check(got, *reference(q, k, v, do, qr, kr, o=o.cpu(), lse=lse.cpu()))
    again = A.varlen_backward(g[3], *g[:3], o, lse, *args)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.parametrize('n,H,D', [(64, 3, 64), (65, 2, 128), (100, 2, 64), (256, 1, 128), (257, 2, 64), (300, 2, 128), (4096, 1, 128)])
def test_many_shared_ranges(n, H, D):
    """every key row is read by none, one or many segments, neighbours in the order of the keys or far apart in that of the
    segments"""
    print(f'{n} ranges H={H} D={D}', flush=True)
    rng, n_k, kr = random.Random(n), 1500, []
    for i in range(n):
        lo = rng.randrange(20, n_k - 60)
        kr.append(rng.choice([(lo, lo), (lo, lo + 1), (lo, min(lo + rng.randrange(1, 200), n_k - 30)),
                              kr[rng.randrange(len(kr))] if kr else (40, 900)]))
    kr[n // 2], kr[-1], kr[0] = (30, n_k - 40), (100, 612), (31, 33)
    lq = [rng.choice([0, 1, rng.randrange(2, 50), 33]) for _ in range(n)]
    lq[n // 2] = 150
    assert H * sum(lq) * max(hi - lo for lo, hi in kr) > 1 << 18
    qr, _ = cut(lq)
    q, k, v, do = inputs(sum(lq), n_k, H, D, 7)
    dlse = torch.randn(H, sum(lq), generator=torch.Generator().manual_seed(9))
    g = [x.to(DEV) for x in (q, k, v, do)]
    o, lse = A.overlapping_ranges_lse(*g[:3], qr, kr)
    got = A.overlapping_ranges_backward(g[3], *g[:3], o, lse, qr, kr, dlse=dlse.to(DEV))
    check(got, *reference(q, k, v, do, qr, kr, dlse, o.cpu(), lse.cpu()))
    assert not got[1][:20].any() and not got[2][n_k - 30:].any()
    again = A.overlapping_ranges_backward(g[3], *g[:3], o, lse, qr, kr, dlse=dlse.to(DEV))
    assert all(torch.equal(x, y) for x, y in zip(got, again))
