"""Gradients of the varlen attention against the formula in float64 on the CPU: head dims, tile edges, one row, empty
segments, uncovered and shared key rows, row strides, split axes, the lse's gradient, autograd and graph replay.

Tolerance: P (for dv) and dS (for dq, dk) are rounded to bf16 once, half a step of 2^-8 relative each, and every gradient is
rounded to bf16 once more. So |error| <= 2^-8 |g| + 2^-8 sum_j |term_j|, the terms being P do, dS k and dS q, with a
quarter on top for the fp32 arithmetic around them (scores of 128 products, exp2, delta: about 2^-16 of the terms) and for
terms whose dS is itself a difference: its fp32 error is 2^-16 (|do v| + |delta|) P, added term by term.
"""
import math

import pytest
import torch

from helpers import rand_bf16
from onereel_amd import attention as A

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'
HALF = torch.finfo(torch.bfloat16).eps / 2


def reference(q, k, v, do, q_ranges, k_ranges, dlse=None, o=None, lse=None):
    """float64 gradients, and the sums of their terms' absolute values with the terms' fp32 errors folded in. o, lse:
    the forward pass's own (delta is taken from the rounded o, as in the kernel)"""
    q, k, v, do = (x.double() for x in (q, k, v, do))
    scale = q.shape[2] ** -0.5
    grads = [torch.zeros_like(x) for x in (q, k, v)]
    mags = [torch.zeros_like(x) for x in (q, k, v)]
    for (a, b), (c, d) in zip(q_ranges, k_ranges):
        if b == a or d == c:
            continue
        qh, doh = (x[a:b].transpose(0, 1) for x in (q, do))
        kh, vh = (x[c:d].transpose(0, 1) for x in (k, v))
        oh, l = o[a:b].double().transpose(0, 1), lse[:, a:b].double()
        p = torch.exp(qh @ kh.transpose(1, 2) * scale - l[:, :, None])
        dp, delta = doh @ vh.transpose(1, 2), (doh * oh).sum(2)
        if dlse is not None:
            delta = delta - dlse[:, a:b].double()
        ds = p * (dp - delta[:, :, None])
        # what bounds the rounding of a term: dS itself, and 2^-16 / 2^-8 of what it is the difference of
        ds_mag = ds.abs() + 2 ** -8 * p * (doh.abs() @ vh.abs().transpose(1, 2) + (doh * oh).abs().sum(2)[:, :, None])
        for i, (lo, hi, g, m) in enumerate(((a, b, ds @ kh * scale, ds_mag @ kh.abs() * scale),
                                            (c, d, ds.transpose(1, 2) @ qh * scale, ds_mag.transpose(1, 2) @ qh.abs() * scale),
                                            (c, d, p.transpose(1, 2) @ doh, p.transpose(1, 2) @ doh.abs()))):
            grads[i][lo:hi] += g.transpose(0, 1)
            mags[i][lo:hi] += m.transpose(0, 1)
    return grads, mags


def check(got, grads, mags):
    for name, x, g, m in zip(('dq', 'dk', 'dv'), got, grads, mags):
        x = x.cpu().double()
        assert torch.isfinite(x).all(), name
        worst = ((x - g).abs() - 1.25 * (HALF * g.abs() + HALF * m)).max().item()
        assert worst <= 1e-30, f'{name}: {worst:.3e} past the bound (max error {(x - g).abs().max():.3e})'


def cut(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return list(zip(at, at[1:])), torch.tensor(at, dtype=torch.int32)


def inputs(nq, nk, H, D, seed=0):
    q, k, v, do = (rand_bf16((n, H, D), seed + i) for i, n in enumerate((nq, nk, nk, nq)))
    return q, k, v, do


CASES = [
    ([1], [1], 1, 128),
    ([1, 77, 33], [64, 77, 0], 2, 64),                      # a segment without keys
    ([33, 0, 129], [40, 50, 1], 3, 128),                    # a segment without queries: its keys get zeros
    ([31, 32, 33, 127, 128], [33, 31, 128, 127, 32], 2, 128),
    ([129, 255, 256, 257], [257, 256, 255, 129], 2, 128),   # tiles of 256
    ([300, 5], [513, 700], 2, 64),
    ([8], [5000], 2, 128),                                  # few queries: keys split
    ([4000], [16], 1, 64),                                  # few keys: queries split
    ([3] * 90, [7] * 90, 1, 128),
    ([1] * 300 + [2] * 213, [3] * 513, 1, 64),               # planned by a launch of its own
    ([2] * 255 + [130], [3] * 255 + [140], 2, 128),          # the most segments that are not
    ([2] * 256 + [130], [3] * 256 + [140], 2, 128),
    # one long segment among short ones: some tiles split, their neighbours not
    ([8, 1, 1000, 130, 40], [3000, 7000, 40, 900, 0], 2, 128),
    ([3000, 7000, 40, 900, 0], [8, 1, 1000, 130, 40], 2, 64),
    ([4] * 30 + [700] + [5] * 33, [3] * 30 + [5000] + [6] * 33, 1, 64),    # the most segments that are sorted and split
    ([4] * 30 + [700] + [5] * 34, [3] * 30 + [5000] + [6] * 34, 1, 128),
    # heads of 64 whose tiles of 256 queries fill the GPU
    ([700, 33, 256, 1100, 90], [130, 257, 64, 33, 100], 64, 64),
    ([8] * 300, [5] * 300, 64, 64),
    # many heads and segments: more than one round of work-groups
    ([130] * 33 + [300, 1], [70] * 33 + [513, 200], 16, 64),
    ([130] * 33 + [300, 1], [70] * 33 + [513, 200], 16, 128),
    ([33] * 30, [1, 2, 31, 32, 33, 64, 65, 95, 96, 97] * 3, 64, 128),
    ([1, 2, 31, 32, 33, 64, 65, 95, 96, 97] * 3, [33] * 30, 64, 64),
]


@pytest.mark.parametrize('lq,lk,H,D', CASES)
def test_varlen_backward(lq, lk, H, D):
    print(f'varlen backward lq={lq[:6]} lk={lk[:6]} H={H} D={D}', flush=True)
    (qr, cq), (kr, ck) = cut(lq), cut(lk)
    q, k, v, do = inputs(sum(lq), sum(lk), H, D)
    g = [x.to(DEV) for x in (q, k, v, do)]
    args = (cq.to(DEV), ck.to(DEV), max(lq), max(lk))
    o, lse = A.varlen_lse(*g[:3], *args)
    got = A.varlen_backward(g[3], *g[:3], o, lse, *args)
    check(got, *reference(q, k, v, do, qr, kr, o=o.cpu(), lse=lse.cpu()))
    again = A.varlen_backward(g[3], *g[:3], o, lse, *args)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.parametrize('n,m,H,D', [(1, 3, 2, 64), (64, 64, 2, 64), (111, 77, 3, 128), (300, 5, 4, 64), (5, 700, 8, 128)])
def test_few_scores_round_only_the_result(n, m, H, D):
    """P and dS as two bf16 numbers each: what is left out of an operand is 2^-16 of it, half a step of half a step. fp32 around
    them: scores, dP and delta of D products and a sum, at most (D + 2) 2^-24 of their terms' sum (for a score: its absolute
    error, hence the relative error of P), 2^-20 for the exponent's own arithmetic (lse and scores below 16, exp2, the
    factor log2 e) and (n + 2) 2^-24 for the sums over rows. So beside the result's own half step:
    |error| <= e_p sum P |do| for dv, e_p sum |dS| |k| + (D + 2) 2^-24 sum P (|do| |v| + |do o|) |k| for dq, and so for dk."""
    print(f'few scores {n} x {m} H={H} D={D}', flush=True)
    q, k, v, do = inputs(n, m, H, D)
    g = [x.to(DEV) for x in (q, k, v, do)]
    (_, cq), (_, ck) = cut([n]), cut([m])
    args = (cq.to(DEV), ck.to(DEV), n, m)
    o, lse = A.varlen_lse(*g[:3], *args)
    got = A.varlen_backward(g[3], *g[:3], o, lse, *args)
    qh, kh, vh, doh, oh = (x.cpu().double().transpose(0, 1) for x in (q, k, v, do, o))
    scale = D ** -0.5
    p = torch.exp(qh @ kh.transpose(1, 2) * scale - lse.cpu().double()[:, :, None])
    ds = p * (doh @ vh.transpose(1, 2) - (doh * oh).sum(2)[:, :, None])
    fp32 = (D + 2) * 2 ** -24
    e_p = 2 ** -16 + fp32 * scale * (qh.abs() @ kh.abs().transpose(1, 2)).max().item() + 2 ** -20 + (max(n, m) + 2) * 2 ** -24
    ds_err = e_p * ds.abs() + fp32 * p * (doh.abs() @ vh.abs().transpose(1, 2) + (doh * oh).abs().sum(2)[:, :, None])
    for name, x, want, err in (('dq', got[0], ds @ kh * scale, ds_err @ kh.abs() * scale),
                               ('dk', got[1], ds.transpose(1, 2) @ qh * scale, ds_err.transpose(1, 2) @ qh.abs() * scale),
                               ('dv', got[2], p.transpose(1, 2) @ doh, e_p * p.transpose(1, 2) @ doh.abs())):
        off = (x.cpu().double().transpose(0, 1) - want).abs()
        worst = (off - HALF * want.abs() - (1 + HALF) * err).max().item()
        assert worst <= 1e-30, f'{name}: {worst:.3e} past the bound (max error {off.max():.3e})'


@pytest.mark.parametrize('H', [2, 96])
@pytest.mark.parametrize('D', [64, 128])
def test_ranges_backward_shares_key_rows(D, H):
    """rows read by none, one, two and three ranges; a range inside another, equal ones, an empty one"""
    lq, kr = [70, 140, 1, 300, 33], [(10, 200), (150, 600), (150, 600), (20, 20), (180, 181)]
    print(f'ranges D={D} H={H}', flush=True)
    qr, _ = cut(lq)
    q, k, v, do = inputs(sum(lq), 700, H, D, 5)
    dlse = torch.randn(H, sum(lq), generator=torch.Generator().manual_seed(9))
    g = [x.to(DEV) for x in (q, k, v, do)]
    o, lse = A.overlapping_ranges_lse(*g[:3], qr, kr)
    got = A.overlapping_ranges_backward(g[3], *g[:3], o, lse, qr, kr, dlse=dlse.to(DEV))
    check(got, *reference(q, k, v, do, qr, kr, dlse, o.cpu(), lse.cpu()))
    assert not got[1][:10].any() and not got[2][600:].any() and not got[0][211:511].any()


@pytest.mark.parametrize('D', [64, 128])
def test_ranges_backward_splits_shared_key_rows(D):
    """key rows read by several segments of long queries: parts that begin and end inside any of them"""
    lq, kr = [700, 1, 1500, 0, 333], [(0, 90), (30, 250), (60, 200), (0, 250), (80, 81)]
    print(f'shared and split D={D}', flush=True)
    qr, _ = cut(lq)
    q, k, v, do = inputs(sum(lq), 260, 2, D)
    g = [x.to(DEV) for x in (q, k, v, do)]
    o, lse = A.overlapping_ranges_lse(*g[:3], qr, kr)
    got = A.overlapping_ranges_backward(g[3], *g[:3], o, lse, qr, kr)
    check(got, *reference(q, k, v, do, qr, kr, o=o.cpu(), lse=lse.cpu()))
    assert not got[1][250:].any() and not got[2][250:].any()


def test_rows_behind_the_last_segment_and_neighbours_that_are_not_finite():
    """rows of other segments never enter a segment's sums, whatever they hold; rows behind the last one get zeros"""
    print('neighbours', flush=True)
    lq, lk, H, D = [40, 50, 20], [70, 33, 90], 2, 128
    (qr, cq), (kr, ck) = cut(lq), cut(lk)
    q, k, v, do = inputs(150, 230, H, D, 3)
    q[40:90], k[70:103], v[70:103], do[40:90] = math.nan, math.inf, math.nan, math.inf
    q[110:], do[110:] = math.nan, math.nan
    g = [x.to(DEV) for x in (q, k, v, do)]
    args = (cq.to(DEV), ck.to(DEV), max(lq), max(lk))
    o, lse = A.varlen_lse(*g[:3], *args)
    dq, dk, dv = A.varlen_backward(g[3], *g[:3], o, lse, *args)
    assert not dq[110:].any() and not dk[193:].any() and not dv[193:].any()
    keep = [0, 2]
    grads, mags = reference(q, k, v, do, [qr[i] for i in keep], [kr[i] for i in keep], o=o.cpu(), lse=lse.cpu())
    dq[40:90], dk[70:103], dv[70:103] = 0, 0, 0
    check((dq, dk, dv), grads, mags)


def test_strided_rows_and_an_expanded_gradient():
    print('strides', flush=True)
    H, D, n = 2, 64, 200
    wide = rand_bf16((n, 4 * H, D), 8).to(DEV)
    q, k, v = wide[:, :H], wide[:, H:2 * H], wide[:, 2 * H:3 * H]
    cu = torch.tensor([0, 90, n], dtype=torch.int32, device=DEV)
    o, lse = A.varlen_lse(q, k, v, cu, cu, 110, 110)
    do = torch.full((1, 1, 1), 0.5, dtype=torch.bfloat16, device=DEV).expand(n, H, D)
    got = A.varlen_backward(do, q, k, v, o, lse, cu, cu, 110, 110)
    r = [(0, 90), (90, n)]
    check(got, *reference(q.cpu(), k.cpu(), v.cpu(), do.cpu(), r, r, o=o.cpu(), lse=lse.cpu()))


def test_autograd_of_every_entry_point():
    print('autograd', flush=True)
    H, D = 2, 128
    q, k, v, do = (x.to(DEV) for x in inputs(160, 160, H, D, 2))
    leaves = lambda: [x.clone().requires_grad_() for x in (q, k, v)]
    cu = torch.tensor([0, 60, 160], dtype=torch.int32, device=DEV)
    r = [(0, 60), (60, 160)]
    o, lse = A.varlen_lse(q, k, v, cu, cu, 100, 100)
    assert not o.requires_grad
    want = A.varlen_backward(do, q, k, v, o, lse, cu, cu, 100, 100)
    calls = [lambda x: A.varlen(*x, cu, cu, 100, 100), lambda x: A.varlen_lse(*x, cu, cu, 100, 100)[0],
             lambda x: A.overlapping_ranges(*x, r, r), lambda x: A.overlapping_ranges_lse(*x, r, r)[0],
             lambda x: torch.cat(A.packed([tuple(t[a:b] for t in x) for a, b in r])),
             lambda x: torch.cat([y for y, _ in A.packed_lse([tuple(t[a:b] for t in x) for a, b in r])])]
    for i, call in enumerate(calls):
        x = leaves()
        out = call(x)
        assert torch.equal(out, o), i
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, x, do), want)), i
    x = leaves()
    out = A.dense(*(t.view(2, 80, H, D) for t in x))
    half = torch.tensor([0, 80, 160], dtype=torch.int32, device=DEV)
    o2, lse2 = A.varlen_lse(q, k, v, half, half, 80, 80)
    grads = torch.autograd.grad(out, x, do.view(2, 80, H, D))
    assert all(torch.equal(a, b) for a, b in zip(grads, A.varlen_backward(do, q, k, v, o2, lse2, half, half, 80, 80)))
    # the lse's gradient alone, and only one input that wants one
    x = leaves()
    dlse = torch.randn(H, 160, generator=torch.Generator().manual_seed(1)).to(DEV)
    got = torch.autograd.grad(A.varlen_lse(*x, cu, cu, 100, 100)[1], x, dlse)
    check(got, *reference(q.cpu(), k.cpu(), v.cpu(), 0 * do.cpu(), r, r, dlse.cpu(), o.cpu(), lse.cpu()))
    kk = k.clone().requires_grad_()
    A.varlen(q, kk, v, cu, cu, 100, 100).backward(do)
    assert torch.equal(kk.grad, want[1])


def test_gradient_against_differences():
    """the gradient along a direction against the central difference of the float64 forward formula: bf16 gradients of 60 rows,
    relative error of the inner product at most 2 roundings of half a step on sums of |g d|"""
    print('differences', flush=True)
    H, D, n = 1, 64, 30
    q, k, v, do = inputs(n, n, H, D, 21)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    g = [x.to(DEV) for x in (q, k, v, do)]
    o, lse = A.varlen_lse(*g[:3], cu, cu, n, n)
    got = [x.cpu().double() for x in A.varlen_backward(g[3], *g[:3], o, lse, cu, cu, n, n)]

    def loss(a, b, c):
        s = torch.einsum('qhd,khd->hqk', a, b) * D ** -0.5
        return (torch.einsum('hqk,khd->qhd', torch.softmax(s, 2), c) * do.double()).sum()

    base = [x.double() for x in (q, k, v)]
    for i in range(3):
        d = torch.randn(n, H, D, generator=torch.Generator().manual_seed(40 + i), dtype=torch.float64)
        e = 1e-5
        up, down = ([b + s * e * d if j == i else b for j, b in enumerate(base)] for s in (1, -1))
        num = (loss(*up) - loss(*down)) / (2 * e)
        # delta from the rounded o adds 2^-8 |do . o| P to dS: bounded by the same term sums as above
        _, mags = reference(q, k, v, do, [(0, n)], [(0, n)], o=o.cpu(), lse=lse.cpu())
        slack = (mags[i] * d.abs()).sum() * HALF * 4
        assert (num - (got[i] * d).sum()).abs() <= slack, i


def test_graph_replays_and_two_graphs():
    print('graph', flush=True)
    H, D, lq, lk = 2, 128, [100, 30], [600, 20]
    (qr, cq), (kr, ck) = cut(lq), cut(lk)
    bufs = [x.to(DEV) for x in inputs(130, 620, H, D, 1)]
    cq, ck = cq.to(DEV), ck.to(DEV)

    def step():
        q, k, v, do = bufs
        o, lse = A.varlen_lse(q, k, v, cq, ck, 100, 600, check=False)
        return A.varlen_backward(do, q, k, v, o, lse, cq, ck, 100, 600, check=False)

    step()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for seed in (50, 60, 70):
        for b, x in zip(bufs, inputs(130, 620, H, D, seed)):
            b.copy_(x)
        want = step()
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), seed


def test_capture_does_not_record_leaves():
    """a captured call on leaves that require gradients runs as without autograd, and says so"""
    print('capture of leaves', flush=True)
    x = [t.to(DEV).requires_grad_() for t in inputs(40, 40, 1, 64)[:3]]
    cu = torch.tensor([0, 40], dtype=torch.int32, device=DEV)
    with torch.no_grad():
        want = A.varlen(*x, cu, cu, 40, 40)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.warns(UserWarning, match='leaves'):
            out = A.varlen(*x, cu, cu, 40, 40, check=False)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert not out.requires_grad and torch.equal(out, want)


@pytest.mark.parametrize('call', ['dense', 'packed', 'packed_lse'])
def test_capture_does_not_record_what_is_made_of_leaves(call):
    """as above, where the call reshapes or concatenates the leaves first"""
    print(f'capture of leaves through {call}', flush=True)
    x = [t.to(DEV).requires_grad_() for t in inputs(40, 40, 1, 64)[:3]]
    y = [t.to(DEV).requires_grad_() for t in inputs(9, 33, 1, 64, 5)[:3]]
    z = [t.detach()[None].requires_grad_() for t in x]
    run = {'dense': lambda: [A.dense(*z)], 'packed': lambda: list(A.packed([x, y])),
           'packed_lse': lambda: [t for pair in A.packed_lse([x, y]) for t in pair]}[call]
    with torch.no_grad():
        want = run()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.warns(UserWarning, match='leaves'):
            out = run()
    assert not any(t.requires_grad for t in out)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize('more_k,more_v', [(7, 0), (0, 200)])
def test_rows_that_only_k_or_v_has(more_k, more_v):
    """the forward call takes such k and v, so does its gradient: zeros there"""
    print(f'k + {more_k}, v + {more_v} rows', flush=True)
    q, k, v, do = (x.to(DEV) for x in inputs(70, 300, 2, 64))
    cu_q, cu_k = (torch.tensor([0, n], dtype=torch.int32, device=DEV) for n in (70, 100))
    xs = [x.detach().requires_grad_() for x in (q, k[:100 + more_k], v[:100 + more_v])]
    A.varlen(*xs, cu_q, cu_k, 70, 100).backward(do)
    o, lse = A.varlen_lse(q, k[:100], v[:100], cu_q, cu_k, 70, 100)
    want = A.varlen_backward(do, q, k[:100], v[:100], o, lse, cu_q, cu_k, 70, 100)
    assert all(x.grad.shape == x.shape for x in xs)
    assert all(torch.equal(x.grad[:len(w)], w) and not x.grad[len(w):].any() for x, w in zip(xs, want))


@pytest.mark.parametrize('nq,nk', [(0, 70), (70, 0), (0, 0)])
def test_no_rows_at_all(nq, nk):
    print(f'no rows {nq} {nk}', flush=True)
    q, k, v, do = (x.to(DEV) for x in inputs(nq, nk, 2, 128))
    cq, ck = (torch.tensor([0, n, n], dtype=torch.int32, device=DEV) for n in (nq, nk))
    got = A.varlen_backward(do, q, k, v, q.clone(), torch.zeros(2, nq, device=DEV), cq, ck, nq, nk)
    assert [x.shape for x in got] == [q.shape, k.shape, v.shape] and not any(x.any() for x in got)


def test_another_stream():
    print('stream', flush=True)
    q, k, v, do = (x.to(DEV) for x in inputs(300, 300, 2, 128, 4))
    cu = torch.tensor([0, 300], dtype=torch.int32, device=DEV)
    o, lse = A.varlen_lse(q, k, v, cu, cu, 300, 300)
    want = A.varlen_backward(do, q, k, v, o, lse, cu, cu, 300, 300)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = A.varlen_backward(do, q, k, v, o, lse, cu, cu, 300, 300)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
