"""Rotary positions with several axes (time, row and column of a video's tokens) computed from the positions, without tables:
the rotation alone, and behind the RMSNorm over all heads of the Wan self-attention's queries and keys (`wan._qk`,
src/onereel/models/wan.py:64-74), on `or_rope_axes_rotate`, `or_rmsnorm_rope_axes` and `or_rmsnorm_rope_axes_bwd`.

`Axes` says where the tokens lie and how a head's dims are dealt out to the axes. `wan.Processor` and `wan_dit.WanDiT` take one
in place of the (cos, sin) tables. `rotate` and `norm_rotate` are differentiable (once) when autograd records; `rotate_backward`
and `norm_rotate_backward` are the same gradients as plain calls. bf16, fp16 or fp32, angles in fp64, fp32 inside, one rounding.
Errors raise `onereel_amd._lib.HipPathError` (a RuntimeError).
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib as L
from .attention import records

PAIRS = {'interleaved': 0, 'half': 1}


@functools.lru_cache(256)
def _four(dims: tuple, theta: tuple):
    """dims and theta of up to 4 axes as the library takes them"""
    fill = (0,) * (4 - len(dims))
    return (L.i32 * 4)(*dims, *fill), (ctypes.c_double * 4)(*theta, *fill)


class Axes:
    """Positions [S, n] of S tokens on n (1 to 4) axes, int32 or fp32 on the GPU (whole or fractional, of any size; one axis may
    come as [S]), and the dims of a head that each axis rotates: an even count, together up to the head's; the dims past them
    stay as they are. Pair i of an axis of d dims turns by position * theta^(-2 i / d). theta: one for all axes, or one each.
    pairs: 'interleaved' (dims 2 j and 2 j + 1 of the head) or 'half' (dims j and j + R / 2 of the R rotated ones, R a multiple
    of 8)."""

    def __init__(self, positions, dims, theta=10000.0, pairs: str = 'interleaved'):
        if positions.dtype not in (torch.int32, torch.float32):
            raise L.HipTypeError(f'positions must be int32 or fp32, got {positions.dtype}')
        if positions.requires_grad:
            raise L.HipValueError('positions have no gradient: detach them')
        dims = tuple(int(d) for d in dims)
        n = len(dims)
        theta = tuple(float(t) for t in theta) if isinstance(theta, (tuple, list)) else (float(theta),) * n
        if positions.dim() == 1:
            positions = positions[:, None]
        if positions.dim() != 2 or positions.shape[1] != n or not 1 <= n <= 4 or len(theta) != n:
            raise L.HipValueError(f'positions must be [S, n] for the n (1 to 4) axes of dims {dims}, got '
                                  f'{tuple(positions.shape)} and {len(theta)} theta')
        if pairs not in PAIRS:
            raise L.HipValueError(f'pairs must be one of {list(PAIRS)}, got {pairs!r}')
        self.positions, self.dims, self.theta, self.pairs = positions.contiguous(), dims, theta, pairs

    def _struct(self):
        p = self.positions
        return L.RopeAxes(p.data_ptr(), p.shape[0], len(self.dims), int(p.dtype == torch.float32), PAIRS[self.pairs],
                          *_four(self.dims, self.theta))


def split_dims(head_dim: int) -> tuple:
    """a head's dims for frame, row and column as diffusers' WanRotaryPosEmbed splits them: 2 (D // 6) for row and column each,
    the rest for the frame"""
    hw = 2 * (head_dim // 6)
    return head_dim - 2 * hw, hw, hw


def grid(frames: int, height: int, width: int, head_dim: int, theta=10000.0, pairs: str = 'interleaved', device='cuda') -> Axes:
    """the Axes of a latent's tokens in frame-major order: the angles of `wan_dit.wan_rope_table`"""
    f, y, x = (torch.arange(n, dtype=torch.int32, device=device) for n in (frames, height, width))
    shape = (frames, height, width)
    at = torch.stack([f[:, None, None].expand(shape), y[None, :, None].expand(shape), x[None, None, :].expand(shape)], 3)
    return Axes(at.reshape(-1, 3), split_dims(head_dim), theta, pairs)


def _check(axes, *xs):
    if not isinstance(axes, Axes):
        raise L.HipTypeError(f'axes must be a rotary.Axes, got {type(axes).__name__}')
    x = xs[0]
    if x.dtype not in L.TYPES or not x.is_cuda:
        raise L.HipTypeError(f'expected a bf16, fp16 or fp32 GPU tensor, got {x.dtype} on {x.device}')
    at = x.get_device()
    for t in xs[1:]:
        if t.dtype != x.dtype:
            raise L.HipTypeError(f'all tensors of a call must be {x.dtype}, got {t.dtype}')
    for t in (*xs[1:], axes.positions):
        if t.get_device() != at:
            raise L.HipTypeError('all tensors of a call must be on one GPU')


def _rows(x, C: int):
    """x as ([rows, C] rows that the kernels read, their stride), a copy where x is not such rows"""
    if x.dim() != 2 or x.shape[1] != C:
        x = x.reshape(-1, C)
    row, one = x.stride()
    if one == 1 and row >= C and row % 8 == 0 and x.data_ptr() % 16 == 0:
        return x, row
    return (x, C) if not x.shape[0] else (x.clone(memory_format=torch.contiguous_format), C)


def _rotate(x, axes, inverse: bool):
    _check(axes, x)
    if x.dim() < 3 or x.shape[-3] != axes.positions.shape[0]:
        raise L.HipValueError(f'expected [.., {axes.positions.shape[0]}, heads, dims], got {tuple(x.shape)}')
    H, D = x.shape[-2:]
    x3 = x if x.dim() == 3 else x.reshape(-1, H, D)
    s = x3.stride()
    if s[2] != 1 or s[0] % 8 or s[1] % 8 or x3.data_ptr() % 16:
        x3 = x3.clone(memory_format=torch.contiguous_format)
        s = x3.stride()
    # in its final shape: a view made inside an autograd function takes no in-place operation
    out = torch.empty_like(x) if x.is_contiguous() else torch.empty_like(x, memory_format=torch.contiguous_format)
    a = axes._struct()
    L.check(L.call(x.device, L.lib().or_rope_axes_rotate, ctypes.byref(a), x3.data_ptr(), out.data_ptr(), x3.shape[0], H, D,
                   s[0], s[1], L.TYPES[x.dtype], int(inverse)), 'or_rope_axes_rotate')
    return out


def rotate(x, axes: Axes):
    """x [.., S, heads, D] (D a multiple of 8 up to 512, any strides of tokens and heads), every token's heads rotated by its
    position: a new tensor of the shape of x. Leading dimensions share the S positions."""
    if records('rotate', x):
        return _Rotate.apply(x, axes)
    return _rotate(x, axes, False)


def rotate_backward(dy, axes: Axes):
    """The gradient of rotate: dy [.., S, heads, D] rotated back"""
    return _rotate(dy, axes, True)


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, axes):
        ctx.axes = axes
        ctx.save_for_backward(axes.positions)
        return _rotate(x, axes, False)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        ctx.saved_tensors      # raises where the positions have been changed since
        return rotate_backward(dy, ctx.axes), None


def _weight(w, like, C: int):
    """a norm's weight in the type of the rows, contiguous at a 16-byte aligned address"""
    if w.numel() != C or not w.is_floating_point():
        raise L.HipValueError(f'weights must hold {C} floating-point elements, got {tuple(w.shape)} {w.dtype}')
    if w.get_device() != like.get_device():
        raise L.HipTypeError('all tensors of a call must be on one GPU')
    if w.dtype != like.dtype or not w.is_contiguous():
        w = w.reshape(C).to(like.dtype).contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


def _sizes(q, k, axes, heads: int):
    C = q.shape[-1]
    if heads < 1 or C % heads or k.shape != q.shape:
        raise L.HipValueError(f'q of width {C} does not split into {heads} heads (k {tuple(k.shape)})')
    if q.dim() < 2 or q.shape[-2] != axes.positions.shape[0]:
        raise L.HipValueError(f'expected [.., {axes.positions.shape[0]}, {C}], got {tuple(q.shape)}')
    return C, C // heads


def _norm_rotate(q, k, wq, wk, eps, axes, heads):
    _check(axes, q, k)
    C, D = _sizes(q, k, axes, heads)
    (q2, qs), (k2, ks) = _rows(q, C), _rows(k, C)
    w = [_weight(t, q, C) for t in (wq, wk)]
    qo = torch.empty(*q.shape[:-1], heads, D, dtype=q.dtype, device=q.device)
    ko = torch.empty_like(qo)
    a = axes._struct()
    L.check(L.call(q.device, L.lib().or_rmsnorm_rope_axes, ctypes.byref(a), q2.data_ptr(), k2.data_ptr(), w[0].data_ptr(),
                   w[1].data_ptr(), qs, ks, q2.shape[0], C, D, L.TYPES[q.dtype], float(eps), qo.data_ptr(), ko.data_ptr()),
            'or_rmsnorm_rope_axes')
    return qo, ko


def norm_rotate(q, k, wq, wk, eps: float, axes: Axes, heads: int):
    """wan._qk with positions in place of tables: the RMSNorm of q and k [.., S, C] (C up to 8192, heads of a multiple of 8 dims)
    over each token row, times wq and wk [C], then the rotation; one launch. Returns q, k as [.., S, heads, D]. The weights are
    taken in the type of the rows."""
    if records('norm_rotate', q, k, wq, wk):
        return _NormRotate.apply(q, k, wq, wk, eps, axes, heads)
    return _norm_rotate(q, k, wq, wk, eps, axes, heads)


_SIZES = functools.lru_cache(256)(lambda S, C: int(L.lib().or_rmsnorm_rope_axes_bwd_workspace_size(S, C)))


def norm_rotate_backward(dq, dk, q, k, wq, wk, eps: float, axes: Axes, heads: int):
    """The gradient of norm_rotate: (q_grad, k_grad) in the type and shape of q and k, (wq_grad, wk_grad) fp32 [C]. dq, dk
    [.., S, heads, D]: the gradients of its outputs. Sums over rows are taken in a fixed order."""
    _check(axes, q, k, dq, dk)
    C, D = _sizes(q, k, axes, heads)
    shape = (*q.shape[:-1], heads, D)
    if dq.shape != shape or dk.shape != shape:
        raise L.HipValueError(f'the gradients must be {shape}, got {tuple(dq.shape)} and {tuple(dk.shape)}')
    (q2, qs), (k2, ks), (dq2, dqs), (dk2, dks) = (_rows(t, C) for t in (q, k, dq, dk))
    w = [_weight(t, q, C) for t in (wq, wk)]
    S, dev = q2.shape[0], q.device
    gq = torch.empty(q.shape, dtype=q.dtype, device=dev)
    gk, gw = torch.empty_like(gq), [torch.empty(C, dtype=torch.float32, device=dev) for _ in range(2)]
    n = _SIZES(S, C)
    if n < 0:
        L.check(L.lib().or_rmsnorm_rope_axes_bwd_workspace_size(S, C), 'or_rmsnorm_rope_axes_bwd_workspace_size')
    space = torch.empty(n, dtype=torch.uint8, device=dev)
    a = axes._struct()
    L.check(L.call(dev, L.lib().or_rmsnorm_rope_axes_bwd, ctypes.byref(a), dq2.data_ptr(), dk2.data_ptr(), q2.data_ptr(),
                   k2.data_ptr(), w[0].data_ptr(), w[1].data_ptr(), dqs, dks, qs, ks, S, C, D, L.TYPES[q.dtype], float(eps),
                   gq.data_ptr(), gk.data_ptr(), gw[0].data_ptr(), gw[1].data_ptr(), space.data_ptr(), n),
            'or_rmsnorm_rope_axes_bwd')
    return gq, gk, *gw


class _NormRotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, eps, axes, heads):
        out = _norm_rotate(q, k, wq, wk, eps, axes, heads)
        ctx.save_for_backward(q, k, wq, wk, axes.positions)
        ctx.how = eps, axes, heads
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        q, k, wq, wk, _ = ctx.saved_tensors
        gq, gk, gwq, gwk = norm_rotate_backward(dq, dk, q, k, wq, wk, *ctx.how)
        return gq, gk, gwq.view(wq.shape).to(wq.dtype), gwk.view(wk.shape).to(wk.dtype), None, None, None
