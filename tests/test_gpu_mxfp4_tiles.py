"""Every kernel that a product of 4-bit values is computed with, against float64: the kernel for few rows, tiles of 256, 128 and 64, rings
of two and four buffers that wrap, whole and split sums, at sizes that leave a remainder of rows, columns and k; scales over all their
range, and blocks that stand for NaN in either operand. Tolerances are those of test_gpu_mxfp4.py."""
import ctypes

import pytest
import torch

from onereel_amd import _lib as L
from onereel_amd import mxfp4
from onereel_amd.mxfp4 import MXFP4
from test_gpu_mxfp4 import LEVELS, check_linear, layer

DEV = 'cuda'
gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
# (tile, buffers, parts of n_in), (rows, n_in, n_out)
CASES = [
    ((0, 0, 1), (13, 1312, 1000)), ((0, 0, 1), (29, 736, 264)),
    ((64, 4, 1), (333, 1312, 200)), ((64, 4, 4), (70, 5152, 136)),
    ((128, 4, 1), (1921, 1056, 2040)), ((128, 4, 8), (66, 17472, 2760)),
    ((128, 2, 1), (11050, 800, 264)), ((128, 2, 3), (262, 15648, 6584)),
    ((256, 2, 1), (3001, 1056, 4104)), ((256, 2, 3), (8297, 16448, 472)),
]


def plan(rows, n_in, n_out):
    out = [ctypes.c_int32() for _ in range(3)]
    L.dit_check(L.dit_lib().or_mx_linear_plan(rows, n_in, n_out, *map(ctypes.byref, out)), 'or_mx_linear_plan')
    return tuple(x.value for x in out)


@pytest.mark.parametrize('want,size', CASES)
def test_sizes_choose_the_kernel_they_stand_for(want, size):
    assert plan(*size) == want


def test_every_kernel_has_a_case():
    have = {(tile, buffers, split > 1) for (tile, buffers, split), _ in CASES}
    assert have == {(0, 0, False)} | {(*ring, split) for ring in ((64, 4), (128, 4), (128, 2), (256, 2)) for split in (False, True)}
    for (tile, buffers, split), (rows, n_in, n_out) in CASES:
        steps = -(-n_in // 256)
        assert rows % max(tile, 16) and n_in % 256 and (n_out % tile if tile else n_out % 16)
        assert not tile or steps // split > buffers and (split == 1 or steps % split)


def test_plan_query_refuses():
    for args in ((-1, 64, 64), (10, 48, 64), (10, 64, 12)):
        with pytest.raises(L.HipPathError, match='or_mx_linear_plan'):
            plan(*args)
    assert L.dit_lib().or_mx_linear_plan(10, 64, 64, None, None, None) < 0


def near_sizes(test):
    for mark in gpu:
        test = mark(test)
    return pytest.mark.parametrize('want,size', CASES, ids=[f'{c[0]}' for c in CASES])(test)


@near_sizes
@pytest.mark.parametrize('how', ['plain', 'all', 'silu'])
def test_against_float64(want, size, how):
    M, K, N = size
    print(f'mx tiles {want} {M} x {K} -> {N} {how}', flush=True)
    x, w, b, gate, r = layer(M, K, N, seed=M)
    b, name, gate, r = (None, None, None, None) if how == 'plain' else (b, 'gelu_tanh', gate, r) if how == 'all' else \
        (b.bfloat16(), 'silu', gate.bfloat16(), None)
    call = lambda x: mxfp4.linear(x, w, b, activation=name, gate=gate, residual=r)
    y, q = call(x), mxfp4.quantize(x)
    check_linear(y, q.dequantize(torch.float32).double(), w.dequantize(torch.float32).double(), b, name, gate, r)
    assert torch.equal(y, call(q)) and torch.equal(y, call(x))


def exact(m):
    """the values of an MXFP4 in float64: those of the largest scales are past fp32"""
    codes = torch.stack([m.codes & 15, m.codes >> 4], -1).flatten(-2).int()
    level = torch.tensor(LEVELS + [-v for v in LEVELS], dtype=torch.float64, device=DEV)[codes]
    unit = torch.tensor([2.0 ** (i - 127) for i in range(255)], dtype=torch.float64, device=DEV)[m.scales.int()]
    return (level.view(*m.scales.shape, 32) * unit[..., None]).flatten(-2)


@near_sizes
def test_scales_over_all_their_range(want, size):
    """blocks of k at every scale, those of x and W together near 1, so that each block counts in the sum"""
    M, K, N = size
    print(f'mx tiles {want} scales', flush=True)
    g = torch.Generator(device=DEV).manual_seed(M)
    base = torch.randint(0, 255, (K // 32,), generator=g, device=DEV)
    base[:4] = torch.tensor([0, 1, 253, 254], device=DEV)
    some = lambda rows, n, hi: torch.randint(0, hi, (rows, n), generator=g, device=DEV)
    of = lambda rows, b: MXFP4(some(rows, K // 2, 256).to(torch.uint8), (b + some(rows, K // 32, 9) - 4).clamp(0, 254).to(torch.uint8))
    x, w = of(M, base), of(N, 254 - base)
    assert {0, 254} <= set(x.scales.unique().tolist()) & set(w.scales.unique().tolist())
    check_linear(mxfp4.linear(x, w), exact(x), exact(w), None, None, None, None)


@near_sizes
def test_not_finite_blocks_stay_in_their_rows_and_columns(want, size):
    """a NaN block of x is its row's, one of W its column's, whatever codes lie under its scale"""
    M, K, N = size
    print(f'mx tiles {want} not finite', flush=True)
    x, w, b, _, _ = layer(M, K, N, seed=M)
    clean = mxfp4.linear(x, w, b)
    rows, columns = [0, M // 2, M - 1], [1, N // 2, N - 1]
    x[rows[0], 0], x[rows[1], K - 1], x[rows[2], K // 2] = float('nan'), float('inf'), float('-inf')
    scales, codes = w.scales.clone(), w.codes.clone()
    for n, k in zip(columns, (0, K // 32 - 1, K // 64)):
        scales[n, k] = 255
        codes[n, 16 * k:16 * k + 16] = torch.arange(16, dtype=torch.uint8, device=DEV) * (n % 3)
    bad = MXFP4(codes, scales)
    hit = torch.zeros(M, N, dtype=torch.bool, device=DEV)
    hit[rows], hit[:, columns] = True, True
    for given in (x, mxfp4.quantize(x)):
        y = mxfp4.linear(given, bad, b)
        assert bool(y[hit].isnan().all()) and torch.equal(y[~hit], clean[~hit])
