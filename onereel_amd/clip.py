"""The global norm of a model's gradients and their clipping, between the backward pass (`wan_dit.WanDiT.differentiable_forward`,
the gradients of `onereel_amd.attention`, `linear`, `norms` and `rotary`) and an optimizer's step: torch's
`torch.nn.utils.clip_grad_norm_` on `or_clip` (libonereel_dit.so), without reading anything back to the host. Tensors are bf16, fp16
or fp32, of any number and mixture; squares are summed in fp64, in a fixed order. Errors raise `onereel_amd._lib.HipPathError` (a
RuntimeError).
"""
from __future__ import annotations

import array
import ctypes

import torch

from . import _lib as L


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


def _check(tensors, what: str, device=None):
    for t in tensors:
        if t.dtype not in L.TYPES or not t.is_cuda:
            raise L.HipTypeError(f'{what} must be bf16, fp16 or fp32 GPU tensors, got {t.dtype} on {t.device}')
        device = t.device if device is None else device
        if t.device != device:
            raise L.HipTypeError('all tensors of a call must be on one GPU')
    return device


def _apart(written, read):
    """raises where a tensor to write shares memory with another one, or with one to read that it does not take the place of"""
    spans = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), True) for t in written if t.numel()]
    spans += [(r.data_ptr(), r.data_ptr() + r.numel() * r.element_size(), False) for r, w in zip(read, written)
              if r.numel() and (r.data_ptr() != w.data_ptr() or r.dtype != w.dtype)]
    end = end_written = 0
    for first, last, writes in sorted(spans):
        if first < (end if writes else end_written):
            raise L.HipValueError('tensors that are written must not share memory with one another or with what is read')
        end, end_written = max(end, last), max(end_written, last) if writes else end_written


def _call(tensors, device, max_norm=0.0, out=None):
    n = len(tensors)
    x = array.array('Q', [t.data_ptr() for t in tensors])
    numel = array.array('q', [t.numel() for t in tensors])
    types = array.array('i', [L.TYPES[t.dtype] for t in tensors])
    o = None if out is None else array.array('Q', [t.data_ptr() for t in out])
    out_types = None if out is None else array.array('i', [L.TYPES[t.dtype] for t in out])
    at = lambda values: None if values is None or not n else values.buffer_info()[0]
    norm = torch.empty((), dtype=torch.float32, device=device)
    args = L.ClipArgs(at(x), at(numel), at(types), at(o), at(out_types), n, max_norm, norm.data_ptr(), None, 0)
    size = int(L.dit_lib().or_clip_workspace_size(ctypes.byref(args)))
    if size < 0:
        L.dit_check(size, 'or_clip_workspace_size')
    space = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    args.workspace, args.workspace_bytes = L.ptr(space), size
    L.dit_check(L.call(device, L.dit_lib().or_clip, ctypes.byref(args)), 'or_clip')
    return norm


def grad_norm(tensors):
    """The 2-norm of all elements of the tensors (an iterable; 0 without any), an fp32 scalar on their GPU"""
    tensors = [t.detach() for t in tensors]
    device = _check(tensors, 'tensors')
    if device is None:
        return torch.zeros((), dtype=torch.float32, device='cuda')
    return _call([t if _dense(t) else t.contiguous() for t in tensors], device)


def clip_grads_(tensors, max_norm: float, out=None):
    """Scales the tensors by c = min(1, max_norm / (norm + 1e-6)), norm being the 2-norm of all their elements together, in place
    or, with out (one tensor of the same shape for each, of any of the types), into those. Returns the norm before clipping, an
    fp32 scalar on the GPU. A norm that is infinite or NaN does to the tensors what the formula says, as in torch: zeros and NaN, or
    NaN throughout. The tensors (those of out) must not share memory, and each fill its own."""
    tensors = [t.detach() for t in tensors]
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise L.HipValueError(f'max_norm must be 0 or more, got {max_norm}')
    device = _check(tensors, 'tensors')
    if out is None:
        written = tensors
        if not all(_dense(t) for t in tensors):
            raise L.HipValueError('tensors that are scaled in place must fill their memory: expanded or strided ones do not')
        sources = tensors
    else:
        written = [t.detach() for t in out]
        if len(written) != len(tensors) or any(a.shape != b.shape for a, b in zip(written, tensors)):
            raise L.HipValueError('out must hold a tensor of the same shape for each of the tensors')
        _check(written, 'out', device)
        if not all(t.is_contiguous() for t in written):
            raise L.HipValueError('out must be contiguous')
        sources = [t.contiguous() for t in tensors]
    _apart(written, sources)
    if device is None:
        return torch.zeros((), dtype=torch.float32, device='cuda')
    for t in out if out is not None else tensors:
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)
    return _call(sources, device, max_norm, written)


def clip_grad_norm_(parameters, max_norm: float):
    """torch.nn.utils.clip_grad_norm_ of the parameters' gradients (those that have one): scaled in place, returns their norm
    before that, an fp32 scalar on the GPU"""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    return clip_grads_([p.grad for p in parameters if p.grad is not None], max_norm)
