"""Linear layers in microscaled 4-bit floating point (OCP MXFP4: e2m1 elements, one e8m0 power of two for 32 of them) for
inference: the projections and the feed forward of the DiT blocks around the scene attention (diffusers' WanTransformerBlock, in
whose blocks the processors of src/onereel/models/wan.py:77-108 are installed), on `or_mx_quantize`, `or_mx_dequantize` and
`or_mx_linear` (libonereel_dit.so).

`linear` is `onereel_amd.linear.linear` with 4-bit weights, and activations that are quantised in the call or were before it (one
`quantize` for several layers that read the same rows). It has no gradient: a backward pass that reaches its result raises. Errors
raise `onereel_amd._lib.HipPathError` (a RuntimeError).
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib as L
from .linear import _activation, _on_one_gpu, _rows, _vector
from .scene import without_gradient

BLOCK = 32


class MXFP4:
    """A tensor [.., n] in 4 bits: codes uint8 [.., n / 2], two e2m1 values a byte with the even element in the low half, and
    scales uint8 [.., n / 32], the biased exponent of each 32 elements' power of two (255: NaN). Both contiguous on one GPU; n a
    multiple of 32. `quantize` makes one; one can be made of stored codes and scales too, of bytes or of the 64-bit integers that
    torch makes of sums of bytes with Python's numbers and of lists of those (their low 8 bits, copied)."""

    def __init__(self, codes, scales):
        for t, what in ((codes, 'codes'), (scales, 'scales')):
            if t.dtype not in (torch.uint8, torch.int64) or not t.is_cuda:
                raise L.HipTypeError(f'{what} must be a uint8 (or int64) GPU tensor, got {t.dtype} on {t.device}')
        if codes.device != scales.device:
            raise L.HipTypeError('all tensors of a call must be on one GPU')
        n = 2 * codes.shape[-1] if codes.dim() else 0
        if not n or n % BLOCK or scales.shape != (*codes.shape[:-1], n // BLOCK):
            raise L.HipValueError(f'codes [.., n / 2] and scales [.., n / 32] of a multiple of 32 elements n are needed, got '
                                  f'{tuple(codes.shape)} and {tuple(scales.shape)}')
        if codes.dtype != torch.uint8:
            codes = codes.to(torch.uint8)
        if scales.dtype != torch.uint8:
            scales = scales.to(torch.uint8)
        codes = codes.contiguous()
        self.codes, self.scales = codes if codes.data_ptr() % 16 == 0 else codes.clone(), scales.contiguous()
        self.shape = torch.Size((*codes.shape[:-1], n))
        self._of = None      # what was quantised, where autograd recorded that

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype=torch.bfloat16):
        """the values that codes and scales stand for, rounded to bf16, fp16 or fp32 (exact in fp32, and in bf16 where they are
        none of its subnormals)"""
        if dtype not in L.TYPES:
            raise L.HipTypeError(f'dtype must be bf16, fp16 or fp32, got {dtype}')
        shape, dev = self.shape, self.device
        out = torch.empty(shape, dtype=dtype, device=dev)
        n = shape[-1]
        L.dit_check(L.call(dev, L.dit_lib().or_mx_dequantize, self.codes.data_ptr(), self.scales.data_ptr(), out.numel() // n, n,
                           L.TYPES[dtype], out.data_ptr()), 'or_mx_dequantize')
        return without_gradient('MXFP4.dequantize', out, self._of)


def quantize(x) -> MXFP4:
    """x [.., n] (bf16, fp16 or fp32, n a multiple of 32) in 4 bits: a block's scale is the power of two that brings its largest
    magnitude into [4, 8), elements go to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4 and 6 times it, ties to the even code, past 6 to
    6. A block with an infinity or a NaN becomes NaN. Without a gradient: a backward pass that reaches what is made of the result
    raises, where autograd records and x requires one."""
    if x.dtype not in L.TYPES or not x.is_cuda:
        raise L.HipTypeError(f'expected a bf16, fp16 or fp32 GPU tensor, got {x.dtype} on {x.device}')
    shape = x.shape
    if not shape or shape[-1] < BLOCK or shape[-1] % BLOCK:
        raise L.HipValueError(f'rows must hold a multiple of 32 elements, got {tuple(shape)}')
    n, dev = shape[-1], x.device
    x2 = x.detach().reshape(-1, n)
    row, one = x2.stride()
    if one != 1 or row < n or row % 8 or x2.data_ptr() % 16:
        x2, row = x2.clone(memory_format=torch.contiguous_format), n
    codes = torch.empty(*shape[:-1], n // 2, dtype=torch.uint8, device=dev)
    scales = torch.empty(*shape[:-1], n // BLOCK, dtype=torch.uint8, device=dev)
    L.dit_check(L.call(dev, L.dit_lib().or_mx_quantize, x2.data_ptr(), x2.shape[0], n, row, L.TYPES[x.dtype], codes.data_ptr(),
                       scales.data_ptr()), 'or_mx_quantize')
    m = MXFP4(codes, scales)
    if torch.is_grad_enabled() and x.requires_grad:
        m._of = x
    return m


_SIZES = functools.lru_cache(256)(lambda *sizes: int(L.dit_lib().or_mx_linear_workspace_size(*sizes)))


def linear(x, weight: MXFP4, bias=None, activation=None, gate=None, residual=None):
    """residual + gate * activation(x weight^T + bias) as `onereel_amd.linear.linear`, of values in 4 bits: x [.., n_in] bf16, which
    the call quantises, or MXFP4; weight MXFP4 [n_out, n_in] (n_in a multiple of 32, n_out of 8); bias and gate [n_out] bf16 or
    fp32, residual [.., n_out] bf16, activation None, 'gelu_tanh' or 'silu'. bf16 [.., n_out], fp32 from the products to the one
    rounding."""
    act = _activation(activation)
    if not isinstance(weight, MXFP4):
        raise L.HipTypeError(f'weight must be an MXFP4, got {type(weight).__name__}')
    ready = isinstance(x, MXFP4)
    rows, of = x.shape, weight.shape
    if len(of) != 2 or not rows or rows[-1] != of[1]:
        raise L.HipValueError(f'x {tuple(rows)} does not fit a weight of {tuple(of)}')
    n_out, n_in = of
    if n_out < 8 or n_out % 8:
        raise L.HipValueError(f'n_out must be a multiple of 8, got {n_out}')
    first = x.codes if ready else x
    _on_one_gpu(first, weight.codes, bias, gate, residual)
    shape = (*rows[:-1], n_out)
    if residual is not None and tuple(residual.shape) != shape:
        raise L.HipValueError(f'the residual must be {shape}, got {tuple(residual.shape)}')
    x2, xs = (None, 0) if ready else _rows(x, n_in, 'x')
    r, rs = (None, 0) if residual is None else _rows(residual, n_out, 'residual')
    (b, b16), (g, g16) = _vector(bias, n_out, 'bias'), _vector(gate, n_out, 'gate')
    dev, p = weight.device, L.ptr
    y = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    M = y.numel() // n_out
    size = _SIZES(M, n_in, n_out, int(ready))
    if size < 0:
        L.dit_check(L.dit_lib().or_mx_linear_workspace_size(M, n_in, n_out, int(ready)), 'or_mx_linear_workspace_size')
    space = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
    a = L.MxLinearArgs(p(x2), x.codes.data_ptr() if ready else None, x.scales.data_ptr() if ready else None,
                       weight.codes.data_ptr(), weight.scales.data_ptr(), p(b), p(g), p(r), y.data_ptr(), M, xs, rs, n_out, n_in,
                       n_out, act, b16, g16, p(space), size)
    L.dit_check(L.call(dev, L.dit_lib().or_mx_linear, ctypes.byref(a)), 'or_mx_linear')
    return without_gradient('mxfp4.linear', y, x._of if ready else x, weight._of, bias, gate, residual)
