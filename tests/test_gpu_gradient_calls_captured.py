"""The plain gradient calls that take their offsets or tables from the host, captured and replayed, and gradient calls on two
streams at once: each has a workspace of its own."""
import pytest
import torch

from helpers import rand_bf16
from onereel_amd import attention as A
from onereel_amd import wan

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'


def replayed(step, bufs, seeds=(50, 60, 70)):
    """two graphs of step, replayed after eager passes on other inputs"""
    step()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for seed in seeds:
        for i, b in enumerate(bufs):
            b.copy_(rand_bf16(tuple(b.shape), seed + i))
        want = step()
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for out in outs for a, b in zip(out, want)), seed


@pytest.mark.parametrize('n', [3, 300])
def test_ranges(n):
    print(f'captured: {n} ranges', flush=True)
    H, D, each = 2, 64, 900 // n
    q, k, v, do = (rand_bf16((m, H, D), i).to(DEV) for i, m in enumerate((n * each, 700, 700, n * each)))
    qr, kr = [(i * each, (i + 1) * each) for i in range(n)], [(i * 2 % 90, 100 + 600 * i // n) for i in range(n)]

    def step():
        o, lse = A.overlapping_ranges_lse(q, k, v, qr, kr)
        return A.overlapping_ranges_backward(do, q, k, v, o, lse, qr, kr)

    replayed(step, [q, k, v, do])


def test_queries_and_keys():
    print('captured: qk', flush=True)
    S, H, D = 300, 8, 128
    q, k, dq, dk = (rand_bf16((S, H * D), i).to(DEV) for i in range(4))
    w = rand_bf16((H * D,), 9).to(DEV)
    cos, sin = torch.rand(2, S, D, device=DEV)
    replayed(lambda: wan.qk_backward(dq, dk, q, k, w, w, 1e-6, cos, sin, H), [q, k, dq, dk])


def test_two_streams_at_once():
    print('two streams', flush=True)
    H, D = 4, 128
    sets = []
    for seed, (nq, nk) in enumerate(((5000, 700), (90, 6000))):       # split keys and split queries
        q, k, v, do = (rand_bf16((m, H, D), 10 * seed + i).to(DEV) for i, m in enumerate((nq, nk, nk, nq)))
        cq, ck = (torch.tensor([0, m], dtype=torch.int32, device=DEV) for m in (nq, nk))
        o, lse = A.varlen_lse(q, k, v, cq, ck, nq, nk)
        sets.append((do, q, k, v, o, lse, cq, ck, nq, nk))
    want = [A.varlen_backward(*s, check=False) for s in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for _ in range(5):
        for s, args in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(A.varlen_backward(*args, check=False))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, want[i % 2])), i
