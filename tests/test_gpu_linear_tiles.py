"""Every kernel that the products of a linear layer and of its gradient are computed with, against float64: tiles of 256, 128 and
64, rings of two and four buffers, whole and split sums, in all three layouts, at ragged sizes whose rings wrap; the sums over
rows ride with the first product. Tolerances are those of test_gpu_linear.py."""
import ctypes

import pytest
import torch

from helpers import rand_bf16
from onereel_amd import _lib as L
from onereel_amd import linear as F
from test_gpu_linear import check_backward, check_forward, inputs

DEV = 'cuda'
gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
FORWARD, DX, DW = 0, 1, 2
# product, (tile, buffers, split), (rows, n_in, n_out)
CASES = [
    (FORWARD, (64, 4, 1), (37, 344, 72)), (FORWARD, (64, 4, 3), (37, 952, 72)),
    (FORWARD, (128, 4, 1), (4205, 328, 456)), (FORWARD, (128, 4, 16), (69, 4616, 1352)),
    (FORWARD, (128, 2, 1), (593, 328, 6600)), (FORWARD, (128, 2, 3), (387, 2640, 4768)),
    (FORWARD, (256, 2, 1), (7357, 336, 1040)), (FORWARD, (256, 2, 8), (139, 5080, 5840)),
    (DX, (64, 4, 1), (37, 72, 336)), (DX, (64, 4, 3), (37, 72, 904)),
    (DX, (128, 4, 1), (323, 5488, 328)), (DX, (128, 4, 8), (65, 2912, 2328)),
    (DX, (128, 2, 1), (6007, 664, 328)), (DX, (128, 2, 4), (129, 5576, 4744)),
    (DX, (256, 2, 1), (1693, 4616, 328)), (DX, (256, 2, 8), (129, 5704, 5040)),
    (DW, (64, 4, 1), (327, 72, 72)), (DW, (64, 4, 3), (901, 72, 72)),
    (DW, (128, 4, 1), (323, 5488, 328)), (DW, (128, 4, 16), (5703, 1376, 72)),
    (DW, (128, 2, 1), (321, 5960, 648)), (DW, (128, 2, 4), (5347, 152, 5512)),
    (DW, (256, 2, 1), (323, 1296, 6136)), (DW, (256, 2, 8), (5423, 136, 5536)),
]


def plan(product, rows, n_in, n_out):
    out = [ctypes.c_int32() for _ in range(3)]
    L.dit_check(L.dit_lib().or_linear_plan(rows, n_in, n_out, product, *map(ctypes.byref, out)), 'or_linear_plan')
    return tuple(x.value for x in out)


@pytest.mark.parametrize('product,want,size', CASES)
def test_sizes_choose_the_kernel_they_stand_for(product, want, size):
    assert plan(product, *size) == want


def test_every_kernel_has_a_case():
    have = {(p, tile, buffers, split > 1) for p, (tile, buffers, split), _ in CASES}
    rings = ((64, 4), (128, 4), (128, 2), (256, 2))
    assert have == {(p, *ring, split) for p in (FORWARD, DX, DW) for ring in rings for split in (False, True)}


def test_plan_query_refuses():
    for args in ((-1, 64, 64, 0), (10, 60, 64, 0), (10, 64, 64, 3), (10, 64, 64, -1)):
        with pytest.raises(L.HipPathError, match='or_linear_plan'):
            plan(args[3], *args[:3])
    assert L.dit_lib().or_linear_plan(10, 64, 64, 0, None, None, None) < 0
    assert plan(FORWARD, 1, 64, 64) == plan(FORWARD, 20, 512, 512) == (0, 0, 1)    # the kernels for few rows


def near_sizes(test):
    for mark in gpu:
        test = mark(test)
    return pytest.mark.parametrize('product,want,size', CASES)(test)


@near_sizes
def test_against_float64(product, want, size):
    M, K, N = size
    print(f'linear tiles {M} x {K} -> {N}', flush=True)
    x, w, b, t, r = inputs(M, K, N, seed=M)
    y, z = F.linear(x, w, b, activation='gelu_tanh', gate=t, residual=r, keep_preactivation=True)
    if product == FORWARD:
        check_forward(y, z, x, w, b, t, r, 'gelu_tanh')
        assert torch.equal(F.linear(x, w, b, activation='gelu_tanh', gate=t, residual=r), y)
        plain = F.linear(x, w)
        check_forward(plain, None, x, w, None, None, None, None)
        return
    dy = rand_bf16((M, N), 7).to(DEV)
    call = lambda needs: F.linear_backward(dy, x, w, bias=True, activation='gelu_tanh', gate=t, preactivation=z, needs=needs)
    got = call((True, True))
    check_backward(got, dy, x, w, z, t, 'gelu_tanh', True)
    assert all(torch.equal(p, q) for p, q in zip(call((True, True)), got))
    alone = call((product == DX, product == DW))     # the sums ride with this product
    assert all(torch.equal(p, q) for p, q in zip(alone, got) if p is not None) and sum(p is None for p in alone) == 1
    raw = F.linear_backward(dy, x, w, bias=True, needs=(product == DX, product == DW))
    check_backward(raw, dy, x, w, None, None, None, True)


@near_sizes
def test_rows_and_columns_beside_the_operands_never_enter(product, want, size):
    """strided operands inside tensors that are not finite around them: the same bits"""
    M, K, N = size
    print(f'linear tiles beside {M} x {K} -> {N}', flush=True)
    x, w, b, *_ = inputs(M, K, N, seed=N)
    dy = rand_bf16((M, N), 3).to(DEV)

    def inside(t, fill):
        big = torch.full((t.shape[0] + 40, t.shape[1] + 24), fill, dtype=t.dtype, device=DEV)
        big[8:8 + t.shape[0], 8:8 + t.shape[1]] = t
        return big[8:8 + t.shape[0], 8:8 + t.shape[1]]

    bx, bw, by = inside(x, float('nan')), inside(w, float('inf')), inside(dy, float('nan'))
    if product == FORWARD:
        assert torch.equal(F.linear(bx, bw, b), F.linear(x, w, b))
        return
    needs = (product == DX, product == DW)
    got, want = (F.linear_backward(*ops, bias=True, needs=needs) for ops in ((by, bx, bw), (dy, x, w)))
    assert all(torch.equal(p, q) for p, q in zip(got, want) if p is not None)


@pytest.mark.gpu
@pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')
@pytest.mark.parametrize('size', [(65, 2912, 2328), (5703, 1376, 72)])
def test_split_gradients_replay(size):
    """two captured graphs of a pass whose dx or dw sums in parts, each replayed after eager passes on other inputs"""
    M, K, N = size
    print(f'linear tiles graph {size}', flush=True)
    assert any(plan(p, *size)[2] > 1 for p in (DX, DW))
    x, w, b, t, _ = inputs(M, K, N, 11)
    dy = rand_bf16((M, N), 4).to(DEV)

    def step():
        y, z = F.linear(x, w, b, activation='silu', gate=t, keep_preactivation=True)
        return (y, z, *F.linear_backward(dy, x, w, bias=True, activation='silu', gate=t, preactivation=z))

    step()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for seed in (1, 2, 3):
        x.copy_(rand_bf16((M, K), seed))
        dy.copy_(rand_bf16((M, N), seed + 9))
        want = step()
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for out in outs for p, q in zip(out, want))
