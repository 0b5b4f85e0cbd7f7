"""Codes and scales of 4-bit tensors as a program has them that made them itself: bytes, or the 64-bit integers that torch makes of
sums of bytes with Python's numbers and of lists of them."""
import pytest
import torch

from onereel_amd import _lib as L
from onereel_amd import mxfp4
from onereel_amd.mxfp4 import MXFP4

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason='needs the GPU')]
DEV = 'cuda'


def stored(rows, n, seed=0):
    """(elements' codes 0 to 15 as bytes [rows, n], scales [rows, n / 32])"""
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, 16, (rows, n), generator=g, dtype=torch.uint8).to(DEV), \
        torch.randint(115, 135, (rows, n // 32), generator=g, dtype=torch.uint8).to(DEV)


def test_codes_packed_by_torch_arithmetic():
    print('mx stored: sums', flush=True)
    code, scales = stored(24, 96)
    magnitude, negative = code & 7, code > 7
    code = magnitude + 8 * negative                      # 64-bit: a truth value times a Python number
    packed = code[:, 0::2] + 16 * code[:, 1::2]
    assert packed.dtype == torch.int64
    want = MXFP4(packed.to(torch.uint8), scales)
    for codes, s in ((packed, scales), (packed, scales.long()), (packed.to(torch.uint8), scales.long())):
        got = MXFP4(codes, s)
        assert got.codes.dtype == got.scales.dtype == torch.uint8 and got.shape == (24, 96)
        assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
        assert torch.equal(got.dequantize(torch.float32), want.dequantize(torch.float32))
    before = packed.clone()
    x = torch.randn(5, 96, device=DEV).bfloat16()
    assert torch.equal(mxfp4.linear(x, MXFP4(packed, scales)), mxfp4.linear(x, want))
    assert torch.equal(packed, before)


def test_codes_of_python_numbers_and_their_layouts():
    print('mx stored: lists', flush=True)
    codes = torch.tensor([[(7 * i + j) % 256 for j in range(32)] for i in range(8)], device=DEV)
    scales = torch.tensor([[120 + i, 130 - i] for i in range(8)], device=DEV)
    want = MXFP4(codes.to(torch.uint8), scales.to(torch.uint8))
    wide = torch.zeros(8, 70, dtype=torch.int64, device=DEV)
    wide[:, 3:35] = codes
    for c in (codes, wide[:, 3:35], codes.t().contiguous().t(), codes - 256, codes + 512):     # low 8 bits
        got = MXFP4(c, scales)
        assert torch.equal(got.codes, want.codes) and got.codes.is_contiguous()
    assert MXFP4(codes[:0], scales[:0]).shape == (0, 64)


def test_other_types_are_refused():
    code, scales = stored(8, 64)
    codes = code[:, 0::2] + 16 * code[:, 1::2]
    for t in (torch.int8, torch.int16, torch.int32, torch.float32, torch.bool):
        with pytest.raises(L.HipTypeError, match='uint8'):
            MXFP4(codes.to(t), scales)
        with pytest.raises(L.HipTypeError, match='uint8'):
            MXFP4(codes, scales.to(t))
    with pytest.raises(L.HipTypeError):
        MXFP4(codes.long().cpu(), scales)
