"""Linear layers with bias, activation, gate and residual in the product's epilogue, and their gradient: the projections and
the feed forward of the DiT blocks around the scene attention (diffusers' WanTransformerBlock, in whose blocks the
processors of src/onereel/models/wan.py:77-108 are installed), on `or_linear` and `or_linear_bwd` (libonereel_dit.so).

`linear` is differentiable (once) in every tensor it takes when autograd records; `linear_backward` is the same gradient as a
plain call. bf16 in and out, fp32 inside. Errors raise `onereel_amd._lib.HipPathError` (a RuntimeError).
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib as L
from .attention import captured_leaves, wants_grad


def _activation(name) -> int:
    if name not in L.ACTIVATIONS:
        raise L.HipValueError(f'activation must be one of {list(L.ACTIVATIONS)}, got {name!r}')
    return L.ACTIVATIONS[name]


def _rows(t, width: int, what: str):
    """t as ([rows, width], row stride) that the kernels read: contiguous elements, whole 16-byte pieces (a copy where its
    rows are not such, e.g. an expanded gradient)"""
    if t.dtype != torch.bfloat16 or not t.is_cuda:
        raise L.HipTypeError(f'{what} must be a bf16 GPU tensor, got {t.dtype} on {t.device}')
    shape = t.shape
    if not shape or shape[-1] != width:
        raise L.HipValueError(f'{what} must have rows of {width} elements, got {tuple(shape)}')
    if len(shape) != 2:
        t = t.reshape(-1, width)
    row, one = t.stride()
    if one == 1 and row >= width and row % 8 == 0 and row <= L.MAX_LINEAR_STRIDE and t.data_ptr() % 16 == 0:
        return t, row
    return (t, width) if not t.shape[0] else (t.clone(memory_format=torch.contiguous_format), width)


def _vector(t, n: int, what: str):
    """(a parameter of n columns, contiguous at a 16-byte aligned address, whether it is bf16)"""
    if t is None:
        return None, 0
    if t.dtype not in (torch.bfloat16, torch.float32) or not t.is_cuda:
        raise L.HipTypeError(f'{what} must be a bf16 or fp32 GPU tensor, got {t.dtype} on {t.device}')
    if t.numel() != n:
        raise L.HipValueError(f'{what} must hold {n} elements, got {tuple(t.shape)}')
    v = t if t.is_contiguous() else t.reshape(n).contiguous()
    return v if v.data_ptr() % 16 == 0 else v.clone(), int(t.dtype == torch.bfloat16)


def _on_one_gpu(x, *others):
    at = x.get_device()
    for t in others:
        if t is not None and t.get_device() != at:
            raise L.HipTypeError('all tensors of a call must be on one GPU')


_SIZES = functools.lru_cache(256)(lambda name, *sizes: int(getattr(L.dit_lib(), name)(*sizes)))


def _workspace(device, name, *sizes):
    """(a workspace or None, its bytes)"""
    n = _SIZES(name, *sizes)
    if n < 0:
        L.dit_check(getattr(L.dit_lib(), name)(*sizes), name)
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None, n


def _sizes(x, weight):
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise L.HipValueError(f'x {tuple(x.shape)} does not fit a weight of {tuple(weight.shape)}')
    n_out, n_in = weight.shape
    if n_in < 8 or n_in % 8 or n_out < 8 or n_out % 8:
        raise L.HipValueError(f'a weight\'s sizes must be multiples of 8, got {tuple(weight.shape)}')
    return n_in, n_out


def _forward(x, weight, bias, act: int, gate, residual, keep: bool):
    n_in, n_out = _sizes(x, weight)
    _on_one_gpu(x, weight, bias, gate, residual)
    shape = (*x.shape[:-1], n_out)
    if residual is not None and tuple(residual.shape) != shape:
        raise L.HipValueError(f'the residual must be {shape}, got {tuple(residual.shape)}')
    x2, xs = _rows(x, n_in, 'x')
    w, ws = _rows(weight, n_in, 'weight')
    r, rs = (None, 0) if residual is None else _rows(residual, n_out, 'residual')
    (b, b16), (g, g16) = _vector(bias, n_out, 'bias'), _vector(gate, n_out, 'gate')
    M, dev, p = x2.shape[0], x.device, L.ptr
    # in its final shape: a view made inside an autograd function takes no in-place operation
    y = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    z = torch.empty_like(y) if keep else None
    space, bytes_ = _workspace(dev, 'or_linear_workspace_size', M, n_in, n_out)
    a = L.LinearArgs(x2.data_ptr(), w.data_ptr(), p(b), p(g), p(r), y.data_ptr(), p(z), M, xs, ws, rs, n_out, n_in, n_out,
                     act, b16, g16, p(space), bytes_)
    L.dit_check(L.call(dev, L.dit_lib().or_linear, ctypes.byref(a)), 'or_linear')
    return y, z


def linear(x, weight, bias=None, activation=None, gate=None, residual=None, keep_preactivation: bool = False):
    """residual + gate * activation(x weight^T + bias): x [.., n_in] and weight [n_out, n_in] bf16 (n_in and n_out multiples
    of 8), bias and gate [n_out] bf16 or fp32 (gate: one factor per column, the same for every row), residual
    [.., n_out] bf16, activation None, 'gelu_tanh' or 'silu'. fp32 from the products to the one rounding of the result.
    With keep_preactivation also returns z = x weight^T + bias in bf16, which linear_backward needs for an activation and
    for the gate's gradient."""
    act = _activation(activation)
    if wants_grad(x, weight, bias, gate, residual):
        if captured_leaves(x, weight, bias, gate, residual):
            raise L.HipValueError('linear: a leaf that requires a gradient cannot be differentiated under graph capture: '
                                  'capture the call without autograd, and linear_backward')
        y, z = _Linear.apply(x, weight, bias, activation, gate, residual, bool(keep_preactivation))
        return (y, z) if keep_preactivation else y
    y, z = _forward(x, weight, bias, act, gate, residual, bool(keep_preactivation))
    return (y, z) if keep_preactivation else y


def linear_backward(dy, x, weight, bias: bool = False, activation=None, gate=None, preactivation=None,
                    needs=(True, True)):
    """The gradient of linear: (dx bf16, dweight bf16, dbias fp32 [n_out] or None, dgate fp32 [n_out] or None). dy
    [.., n_out] bf16 is also the residual's gradient. bias: whether the call had one; preactivation: the z it kept (needed
    with an activation or a gate); needs: whether dx and dweight are wanted (None in their place otherwise). Sums are fp32
    in a fixed order; dz = dy gate act'(z) is rounded to bf16 as the operand of the two products."""
    act = _activation(activation)
    n_in, n_out = _sizes(x, weight)
    _on_one_gpu(x, dy, weight, gate, preactivation)
    if dy.shape != (*x.shape[:-1], n_out):
        raise L.HipValueError(f'dy must be {(*x.shape[:-1], n_out)}, got {tuple(dy.shape)}')
    if (act or gate is not None) and preactivation is None:
        raise L.HipValueError('an activation or a gate needs the pre-activation that the forward call kept')
    dy2, ds = _rows(dy, n_out, 'dy')
    x2, xs = _rows(x, n_in, 'x')
    w, ws = _rows(weight, n_in, 'weight')
    z = None
    if preactivation is not None and (act or gate is not None):
        if preactivation.shape != dy.shape:
            raise L.HipValueError(f'the pre-activation must be {tuple(dy.shape)}, got {tuple(preactivation.shape)}')
        z, zs = _rows(preactivation, n_out, 'preactivation')
        z = z if zs == n_out else z.contiguous()
    g, g16 = _vector(gate, n_out, 'gate')
    M, dev, p = x2.shape[0], x.device, L.ptr
    new = lambda dtype, *shape: torch.empty(shape, dtype=dtype, device=dev)
    dx, dw = new(torch.bfloat16, M, n_in) if needs[0] else None, new(torch.bfloat16, n_out, n_in) if needs[1] else None
    db, dg = new(torch.float32, n_out) if bias else None, new(torch.float32, n_out) if gate is not None else None
    space, bytes_ = _workspace(dev, 'or_linear_bwd_workspace_size', M, n_in, n_out, int(act != 0 or g is not None))
    a = L.LinearBwdArgs(dy2.data_ptr(), x2.data_ptr(), w.data_ptr(), p(z), p(g), p(dx), p(dw), p(db), p(dg), M, ds, xs, ws,
                        n_in, n_out, act, g16, p(space), bytes_)
    L.dit_check(L.call(dev, L.dit_lib().or_linear_bwd, ctypes.byref(a)), 'or_linear_bwd')
    return dx if dx is None or x.dim() == 2 else dx.view(x.shape), dw, db, dg


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation, gate, residual, keep):
        scaled = activation is not None or gate is not None
        y, z = _forward(x, weight, bias, _activation(activation), gate, residual, scaled or keep)
        ctx.save_for_backward(x, weight, z if scaled else None, gate)
        ctx.activation = activation
        ctx.bias, ctx.gate = (None if t is None else (t.shape, t.dtype) for t in (bias, gate))
        if not keep:
            return y, None
        z = z.clone() if scaled else z    # the caller's own: the saved one is not handed out
        ctx.mark_non_differentiable(z)
        return y, z

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _):
        x, weight, z, gate = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, dw, db, dg = linear_backward(dy, x, weight, bias=ctx.bias is not None and need[2], activation=ctx.activation,
                                         gate=gate, preactivation=z, needs=need[:2])
        db, dg = (g if g is None else g.view(like[0]).to(like[1]) for g, like in ((db, ctx.bias), (dg, ctx.gate)))
        return dx, dw, db, None, dg, dy if need[5] else None, None
