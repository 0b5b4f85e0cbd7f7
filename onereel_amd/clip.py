"""The global norm of a model's gradients and their clipping, between the backward pass (`wan_dit.WanDiT.differentiable_forward`,
the gradients of `onereel_amd.attention`, `linear`, `norms` and `rotary`) and an optimizer's step: torch's
`torch.nn.utils.clip_grad_norm_` on `or_clip` (libonereel_dit.so), without reading anything back to the host. Tensors are bf16, fp16
or fp32, of any number and mixture; squares are summed in fp64, in a fixed order. Errors raise `onereel_amd._lib.HipPathError` (a
RuntimeError).
"""
from __future__ import annotations

import array
import ctypes
import operator

import torch

from . import _lib as L
from .scene import without_gradient


_T = torch.Tensor
_DTYPE, _DEVICE, _ADDRESS, _NUMEL, _SHAPE = operator.attrgetter('dtype'), _T.get_device, _T.data_ptr, _T.numel, operator.attrgetter('shape')


def _dense(t) -> bool:
    """whether t's elements fill one run of memory, each once, in whatever order of its dimensions"""
    if t.is_contiguous():
        return True
    n = 1
    for stride, size in sorted((s, z) for s, z in zip(t.stride(), t.shape) if z > 1):
        if stride != n:
            return False
        n *= size
    return True


def _addresses(tensors, what: str, at: int):
    """(addresses, lengths, types) of the tensors as the library takes them, and their GPU's index (at: the one it has to be,
    None for any)"""
    # one C call for each tensor and question: a model has hundreds of them, and their launches take less than a loop over them
    dtypes, devices = list(map(_DTYPE, tensors)), set(map(_DEVICE, tensors))
    distinct = set(dtypes)
    if not L.TYPES.keys() >= distinct or devices and min(devices) < 0:
        t = next(t for t in tensors if t.dtype not in L.TYPES or t.get_device() < 0)
        raise L.HipTypeError(f'{what} must be bf16, fp16 or fp32 GPU tensors, got {t.dtype} on {t.device}')
    if at is not None:
        devices.add(at)
    if len(devices) > 1:
        raise L.HipTypeError('all tensors of a call must be on one GPU')
    kinds = array.array('i', map(L.TYPES.__getitem__, distinct if len(distinct) == 1 else dtypes))
    if len(distinct) == 1:
        kinds *= len(tensors)
    return (array.array('Q', map(_ADDRESS, tensors)), array.array('q', map(_NUMEL, tensors)), kinds), \
        devices.pop() if devices else None


def _refuse(changed):
    """what autograd cannot follow a change of, where it records one"""
    for t in changed:
        view = t._is_view()
        if t.is_inference() or t.requires_grad and (t._base if view else t).is_leaf or \
                view and torch._C._autograd._get_creation_meta(t) != torch._C._autograd.CreationMeta.DEFAULT:
            raise L.HipValueError('where autograd records a call, it scales no leaf that requires a gradient, no inference tensor and no '
                                  'view that was made without autograd or as one of several: call it under torch.no_grad()')


def _norm_on(at: int):
    return torch.empty((), dtype=torch.float32, device=torch.device('cuda', at))


def _call(sources, out, norm, max_norm: float = 0.0):
    """or_clip of two results of _addresses (out None: the norm alone) into the scalar norm"""
    p = lambda values: values.buffer_info()[0]
    n, device = len(sources[0]), norm.device
    args = L.ClipArgs(*map(p, sources), out and p(out[0]), out and p(out[2]), n, max_norm, norm.data_ptr(), None, 0)
    size = L.dit_lib().or_clip_workspace_size(ctypes.byref(args))
    if size < 0:
        L.dit_check(size, 'or_clip_workspace_size')
    if size:
        space = torch.empty(size, dtype=torch.uint8, device=device)
        args.workspace, args.workspace_bytes = space.data_ptr(), size
    L.dit_check(L.call(device, L.dit_lib().or_clip, ctypes.byref(args)), 'or_clip')
    return norm


def _zero():
    return torch.zeros((), dtype=torch.float32, device='cuda')


def grad_norm(tensors):
    """The 2-norm of all elements of the tensors (an iterable; 0 without any), an fp32 scalar on their GPU. It has no gradient: where
    autograd records and one of them requires a gradient, a backward pass that reaches it raises."""
    given = tensors = list(tensors)
    if not all(map(_T.is_contiguous, tensors)):
        tensors = [t if _dense(t) else t.detach().contiguous() for t in tensors]
    sources, at = _addresses(tensors, 'tensors', None)
    return _zero() if at is None else without_gradient('clip.grad_norm', _call(sources, None, _norm_on(at)), *given)


def clip_grads_(tensors, max_norm: float, out=None):
    """Scales the tensors by c = min(1, max_norm / (norm + 1e-6)), norm being the 2-norm of all their elements together, in place
    or, with out (one tensor of the same shape for each, of any of the types), into those. Returns the norm before clipping, an
    fp32 scalar on the GPU. A norm that is infinite or NaN does to the tensors what the formula says, as in torch: zeros and NaN, or
    NaN throughout. Tensors that are written must not share memory with one another or with what is read (but for the tensor that
    they take the place of), and each fill its own. Nothing here has a gradient: where autograd records and one of the tensors requires
    one, a backward pass that reaches the norm or what was written raises, and what autograd could not follow a change of (a leaf
    that requires one) is refused."""
    given = tensors = list(tensors)
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise L.HipValueError(f'max_norm must be 0 or more, got {max_norm}')
    if out is None:
        if not all(map(_T.is_contiguous, tensors)) and not all(map(_dense, tensors)):
            raise L.HipValueError('tensors that are scaled in place must fill their memory: expanded or strided ones do not')
        sources, at = _addresses(tensors, 'tensors', None)
        written = sources
    else:
        if not all(map(_T.is_contiguous, tensors)):
            tensors = [t.detach().contiguous() for t in tensors]
        out = list(out)
        if len(out) != len(tensors) or list(map(_SHAPE, out)) != list(map(_SHAPE, tensors)):
            raise L.HipValueError('out must hold a tensor of the same shape for each of the tensors')
        if not all(map(_T.is_contiguous, out)):
            raise L.HipValueError('out must be contiguous')
        sources, at = _addresses(tensors, 'tensors', None)
        written, _ = _addresses(out, 'out', at)
    if at is None:
        return _zero()
    changed, norm = tensors if out is None else out, _norm_on(at)
    # one C call for all, as above
    recorded = torch.is_grad_enabled() and torch._C._any_requires_grad(*given, *(out or ()))
    if recorded:
        _refuse(changed)
    _call(sources, written, norm, max_norm)
    if recorded:
        norm = without_gradient('clip.clip_grads_', norm, *given, *changed)
        for t in changed:              # which counts their versions up too
            without_gradient('clip.clip_grads_', t, norm)
        return norm
    try:
        torch.autograd.graph.increment_version(changed)
    except RuntimeError:               # inference tensors among them, which have no version
        torch.autograd.graph.increment_version([t for t in changed if not t.is_inference()])
    return norm


def clip_grad_norm_(parameters, max_norm: float):
    """torch.nn.utils.clip_grad_norm_ of the parameters' gradients (those that have one): scaled in place, returns their norm
    before that, an fp32 scalar on the GPU. As there, autograd does not record it. A parameter is given once."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    with torch.no_grad():
        return clip_grads_([p.grad for p in parameters if p.grad is not None], max_norm)
