"""The norms before and after a sub-block of a DiT block, fused with its gate and residual, and their gradient: diffusers'
WanTransformerBlock around the attention and the feed forward (the blocks the processors of src/onereel/models/wan.py:77-108 are
installed in), on `or_block_norm` and `or_block_norm_bwd` (libonereel_dit.so).

`norm_modulate` and `residual_norm_modulate` are differentiable (once) in every tensor they take when autograd records;
`norm_modulate_backward` and `residual_norm_modulate_backward` are the same gradients as plain calls. They are what
`wan_dit.layernorm_modulate` and `wan_dit.residual_layernorm_modulate_` are for inference, without updating anything in place;
gate, scale and shift may differ from one group of rows to the next (frames at timesteps of their own), the norm may be an RMS
norm, and a norm of the sub-block's output may come before its gate. Rows are bf16, fp16 or fp32, fp32 inside. Errors raise
`onereel_amd._lib.HipPathError` (a RuntimeError).
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib as L
from .attention import records


def _rows(t, shape, dtype, what: str):
    """t as ([rows, C], row stride) that the kernels read: contiguous elements, rows of whole 16-byte pieces (a copy where its
    rows are not such, e.g. an expanded gradient)"""
    if t.shape != shape:
        raise L.HipValueError(f'{what} must be {tuple(shape)}, got {tuple(t.shape)}')
    if t.dtype != dtype:
        raise L.HipTypeError(f'{what} must be {dtype} as the rows it belongs to, got {t.dtype}')
    C = shape[-1]
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t, C
    t = t.reshape(-1, C)
    row, one = t.stride()
    if one == 1 and row >= C and row % 8 == 0 and t.data_ptr() % 16 == 0:
        return t, row
    return t.clone(memory_format=torch.contiguous_format), C


def _vector(t, C: int, what: str, groups=None):
    """a parameter as contiguous fp32 at a 16-byte aligned address; with groups, how many vectors of C it holds is written there"""
    if t is None:
        return None
    if not t.is_floating_point():
        raise L.HipTypeError(f'{what} must be floating point, got {t.dtype}')
    n = t.numel()
    if t.dim() < 1 or t.shape[-1] != C or (n != C if groups is None else not n):
        raise L.HipValueError(f'{what} must hold {"one vector" if groups is None else "vectors"} of {C} elements, got '
                              f'{tuple(t.shape)}')
    if groups is not None:
        groups.add(n // C)
    if t.dtype != torch.float32 or not t.is_contiguous():
        t = t.to(torch.float32).contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _like(t):
    """a new contiguous tensor of t's shape and type, in its final shape: a view made inside an autograd function takes no in-place
    operation"""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format)


def _norm(name, none: bool = False) -> int:
    if name not in L.NORMS or name is None and not none:
        raise L.HipValueError(f'a norm must be one of {[n for n in L.NORMS if none or n]}, got {name!r}')
    return L.NORMS[name]


def _check(x, *others):
    if x.dtype not in L.TYPES or not x.is_cuda:
        raise L.HipTypeError(f'rows must be bf16, fp16 or fp32 on the GPU, got {x.dtype} on {x.device}')
    if x.dim() < 1 or x.shape[-1] < 8 or x.shape[-1] % 8 or x.shape[-1] > 8192:
        raise L.HipValueError(f'rows must hold a multiple of 8 elements up to 8192, got {tuple(x.shape)}')
    at = x.get_device()
    for t in others:
        if t is not None and t.get_device() != at:
            raise L.HipTypeError('all tensors of a call must be on one GPU')


def _parameters(C, rows, gate, post_norm, post_weight, weight, bias, scale, shift):
    """the parameters as the kernels read them, and the rows of a group"""
    if post_weight is not None and post_norm is None:
        raise L.HipValueError('post_weight belongs to a post_norm')
    groups = set()
    given = [_vector(gate, C, 'gate', groups), _vector(post_weight, C, 'post_weight'), _vector(weight, C, 'weight'),
             _vector(bias, C, 'bias'), _vector(scale, C, 'scale', groups), _vector(shift, C, 'shift', groups)]
    if len(groups) > 1:
        raise L.HipValueError(f'gate, scale and shift must hold as many vectors, got {sorted(groups)}')
    n = groups.pop() if groups else 1
    if rows % n:
        raise L.HipValueError(f'{rows} rows do not divide into the {n} groups that gate, scale or shift hold vectors for')
    return given, max(rows // n, 1)


def _forward(x, a, eps, norm, gate, residual_scale, post_norm, post_weight, weight, bias, scale, shift):
    _check(x, a, gate, post_weight, weight, bias, scale, shift)
    shape, C = x.shape, x.shape[-1]
    kinds = _norm(norm), _norm(post_norm, True)
    rows = x.numel() // C
    (g, pw, w, b, sc, sh), per = _parameters(C, rows, gate, post_norm, post_weight, weight, bias, scale, shift)
    x2, xs = _rows(x, shape, x.dtype, 'x')
    a2, as_ = (None, 0) if a is None else _rows(a, shape, x.dtype, 'a')
    p, dev = L.ptr, x.device
    n, h = _like(x), None if a is None else _like(x)
    args = L.BlockNormArgs(x2.data_ptr(), p(a2), p(h), n.data_ptr(), p(g), p(pw), p(w), p(b), p(sc), p(sh), rows, per, xs, as_,
                           C, L.TYPES[x.dtype], *kinds, eps, residual_scale)
    L.dit_check(L.call(dev, L.dit_lib().or_block_norm, ctypes.byref(args)), 'or_block_norm')
    return h, n


_SIZES = functools.lru_cache(256)(lambda *sizes: int(L.dit_lib().or_block_norm_bwd_workspace_size(*sizes)))


def _backward(dh, dn, h, a, eps, norm, gate, residual_scale, post_norm, post_weight, weight, bias, scale, shift,
              needs=(True,) * 6):
    """(dx, da, dgate, dpost_weight, dweight, dbias, dscale, dshift), None where there is no such argument or, of the
    parameters, needs says that it is not wanted"""
    _check(h, dh, dn, a, gate, post_weight, weight, bias, scale, shift)
    shape, C, dev = h.shape, h.shape[-1], h.device
    kinds = _norm(norm), _norm(post_norm, True)
    rows = h.numel() // C
    given, per = _parameters(C, rows, gate, post_norm, post_weight, weight, bias, scale, shift)
    h2, hs = _rows(h, shape, h.dtype, 'h' if a is not None else 'x')
    n2, ns = _rows(dn, shape, h.dtype, 'dn')
    a2, as_ = (None, 0) if a is None else _rows(a, shape, h.dtype, 'a')
    d2, ds = (None, 0) if dh is None else _rows(dh, shape, h.dtype, 'dh')
    dx, da = _like(h), None if a is None else _like(h)
    make = torch.empty_like if rows else torch.zeros_like
    grads = [make(t) if t is not None and need else None for t, need in zip(given, needs)]
    p = L.ptr
    size, space = 0, None
    if any(t is not None for t in grads):
        size = _SIZES(rows, per, C)
        if size < 0:
            L.dit_check(L.dit_lib().or_block_norm_bwd_workspace_size(rows, per, C), 'or_block_norm_bwd_workspace_size')
        space = torch.empty(size, dtype=torch.uint8, device=dev)
    args = L.BlockNormBwdArgs(p(d2), n2.data_ptr(), h2.data_ptr(), p(a2), dx.data_ptr(), p(da), *map(p, given[:5]),
                              *map(p, grads), rows, per, ds, ns, hs, as_, C, L.TYPES[h.dtype], *kinds, eps, residual_scale,
                              p(space), size)
    L.dit_check(L.call(dev, L.dit_lib().or_block_norm_bwd, ctypes.byref(args)), 'or_block_norm_bwd')
    return (dx, da, *grads)


def norm_modulate(x, eps: float, norm: str = 'layer', weight=None, bias=None, scale=None, shift=None):
    """(Norm(x) weight + bias) (1 + scale) + shift over the last dimension of x [.., C] (bf16, fp16 or fp32, C a multiple of 8 up
    to 8192), rounded once. norm: 'layer' or 'rms'. weight and bias [C]; scale and shift [.., C] with G vectors, one for every
    rows / G consecutive rows of x. Parameters of any floating type, fp32 inside."""
    if records('norm_modulate', x, weight, bias, scale, shift):
        return _Norm.apply(eps, norm, None, 1.0, x, None, None, None, weight, bias, scale, shift)[1]
    return _forward(x, None, eps, norm, None, 1.0, None, None, weight, bias, scale, shift)[1]


def residual_norm_modulate(x, a, eps: float, norm: str = 'layer', gate=None, residual_scale: float = 1.0, post_norm=None,
                           post_weight=None, weight=None, bias=None, scale=None, shift=None):
    """(h, n): h = residual_scale x + gate Post(a) post_weight, rounded once, and n = norm_modulate of h before that rounding, in
    one pass. a: rows as x (a sub-block's output); post_norm None, 'layer' or 'rms' (of a, with the same eps), post_weight [C];
    gate as scale and shift of norm_modulate, the three with as many vectors. Both results are new tensors."""
    if a is None:
        raise L.HipValueError('a is required: norm_modulate is the norm alone')
    if records('residual_norm_modulate', x, a, gate, post_weight, weight, bias, scale, shift):
        return _Norm.apply(eps, norm, post_norm, residual_scale, x, a, gate, post_weight, weight, bias, scale, shift)
    return _forward(x, a, eps, norm, gate, residual_scale, post_norm, post_weight, weight, bias, scale, shift)


def norm_modulate_backward(dn, x, eps: float, norm: str = 'layer', weight=None, bias=None, scale=None, shift=None):
    """The gradient of norm_modulate: (dx in the type of x, dweight, dbias, dscale, dshift fp32 in their parameters' shapes, None
    for those not given). Sums over rows are taken in a fixed order."""
    out = _backward(None, dn, x, None, eps, norm, None, 1.0, None, None, weight, bias, scale, shift)
    return (out[0], *out[4:])


def residual_norm_modulate_backward(dh, dn, h, a, eps: float, norm: str = 'layer', gate=None, residual_scale: float = 1.0,
                                    post_norm=None, post_weight=None, weight=None, bias=None, scale=None, shift=None):
    """The gradient of residual_norm_modulate from the gradients of its h (None: nothing else read it) and n, at the h that it
    returned: (dx, da in the type of h, dgate, dpost_weight, dweight, dbias, dscale, dshift fp32)"""
    if a is None:
        raise L.HipValueError('a is required: norm_modulate_backward is the norm alone')
    return _backward(dh, dn, h, a, eps, norm, gate, residual_scale, post_norm, post_weight, weight, bias, scale, shift)


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, eps, norm, post_norm, residual_scale, x, a, *params):
        h, n = _forward(x, a, eps, norm, params[0], residual_scale, post_norm, *params[1:])
        ctx.save_for_backward(x if a is None else h, a, *params)
        ctx.set_materialize_grads(False)
        ctx.how = eps, norm, post_norm, residual_scale
        return h, n

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dn):
        h, a, gate, *params = ctx.saved_tensors
        eps, norm, post_norm, residual_scale = ctx.how
        if dh is None and dn is None:
            return (None,) * 12
        dn = torch.zeros_like(h, memory_format=torch.contiguous_format) if dn is None else dn
        need = ctx.needs_input_grad[6:]
        dx, da, *grads = _backward(dh, dn, h, a, eps, norm, gate, residual_scale, post_norm, *params, needs=need)
        grads = [g if g is None else g.view(t.shape).to(t.dtype) for g, t in zip(grads, (gate, *params))]
        return None, None, None, None, dx, da, *grads
