"""Wan2.2-TI2V-5B scene attention on one MI355X: the drop-in processor (src/onereel/models/wan.py:33-124).

Self-attention: scene j's queries read scene j's frames plus its halo frames, which are adjacent to it, so its keys
are one contiguous token range: the varlen kernel reads every scene's overlapping key range in place (per-segment
key offset and length). With extra frames (frame memory) each scene's keys are packed by the device layout and
pack-gather kernels instead. With `Context.memory` = M > 0, scene j's queries read scene j plus M representatives
per head of the other scenes' boundary keys (`onereel_amd.memory`, wan.py:100-101,154-173). Cross-attention: scene
j's queries read only sentence j, all scenes in one varlen launch. The RMSNorm + interleaved RoPE of `_qk`
(wan.py:64-74) is one HIP launch for q and k (`or_rmsnorm_rope`; with positions in place of tables, `onereel_amd.rotary`).
"""
from __future__ import annotations

import functools
from dataclasses import dataclass

import torch

from . import _lib as L
from . import attention as A
from .comm import frame_tokens  # noqa: F401  (re-exported for callers of the reference module)
from .frame_memory import FrameMemory
from .layout import SceneLayout
from .memory import BoundaryMemory, MemoryAttention, frame_plan
from .mxfp4 import MXFP4
from .rotary import Axes, norm_rotate
from .scene import ScopePlan, pack_layer, varlen, without_gradient

TEXT_LEN = 512


@dataclass
class Context:
    """the fields of the reference Context (wan.py:33-58) that the single-GPU path reads"""
    layout: SceneLayout
    memory: int = 0                      # M > 0: bounded cross-scene memory of M representatives per head (halo 0)
    frame_memory: FrameMemory = None
    _mem: MemoryAttention = None         # the bounded memory's state (centroids per layer and branch, plans)
    T: int = 0
    fwd: int = 0
    cfg: bool = False
    text_len: int = TEXT_LEN

    def cond(self) -> bool:
        return (self.fwd - 1) % 2 == 0 if self.cfg else True

    def step(self) -> int:
        return (self.fwd - 1) // 2 if self.cfg else self.fwd - 1


def _qk(q, k, wq, wk, eps: float, cos, sin, heads: int):
    """RMSNorm over each token row (all heads) and the interleaved RoPE of diffusers' Wan attention, fused: one HIP
    launch for q and k, fp32 inside, one rounding to bf16 (wan.py:64-74, compiled there with torch.compile).
    q, k [..., S, C] bf16 with contiguous rows; wq, wk [C]; cos / sin of S rows of D = C / heads entries
    (e.g. [1, S, 1, D]). Returns q, k as [..., S, heads, D] bf16."""
    C = q.shape[-1]
    D = C // heads
    if heads * D != C or k.shape != q.shape:
        raise L.HipValueError(f'q / k of width {C} do not split into {heads} heads (k {tuple(k.shape)})')
    if q.dtype != torch.bfloat16 or k.dtype != torch.bfloat16:
        raise L.HipTypeError('q and k must be bfloat16')
    if A.records('_qk', q, k, wq, wk):
        return _QK.apply(q, k, wq, wk, eps, cos, sin, heads)
    return _qk_forward(q, k, wq, wk, eps, cos, sin, heads)


def _qk_forward(q, k, wq, wk, eps, cos, sin, heads):
    C = q.shape[-1]
    D = C // heads
    lead = q.shape[:-1]
    q2, k2 = q.reshape(-1, C), k.reshape(-1, C)
    if q2.stride(1) != 1 or k2.stride(1) != 1:
        raise L.HipValueError('q / k rows must be contiguous')
    S = q2.shape[0]
    c = cos.reshape(-1, D).to(torch.float32).contiguous()
    s = sin.reshape(-1, D).to(torch.float32).contiguous()
    if c.shape[0] != S or s.shape[0] != S:
        raise L.HipValueError(f'rotary tables hold {c.shape[0]} rows for {S} tokens')
    w1, w2 = (w.to(torch.bfloat16).contiguous() for w in (wq, wk))
    # in their final shape: a view made inside an autograd function takes no in-place operation
    qo = torch.empty(*lead, heads, D, dtype=torch.bfloat16, device=q.device)
    ko = torch.empty_like(qo)
    L.check(L.lib().or_rmsnorm_rope(q2.data_ptr(), k2.data_ptr(), w1.data_ptr(), w2.data_ptr(), q2.stride(0),
                                    k2.stride(0), S, C, D, float(eps), c.data_ptr(), s.data_ptr(), None, S,
                                    qo.data_ptr(), ko.data_ptr(), C, C, L.stream_handle(q.device)),
            'or_rmsnorm_rope')
    return qo, ko


def rms_norm(x, weight, eps: float):
    """RMSNorm over the last dimension (C a multiple of 512) with a bf16 weight [C]: x / sqrt(mean(x^2) + eps) * w,
    fp32 inside, one rounding to bf16; one HIP launch (or_rmsnorm_rope without rotary tables). The norm_q / norm_k
    of diffusers' Wan attention, as the cross-attention processor applies them."""
    C = x.shape[-1]
    if x.dtype != torch.bfloat16:
        raise L.HipTypeError('x must be bfloat16')
    if A.records('rms_norm', x, weight):
        return _RMSNorm.apply(x, weight, eps)
    x2 = x.reshape(-1, C)
    if x2.stride(1) != 1:
        raise L.HipValueError('x rows must be contiguous')
    w = weight.to(torch.bfloat16).contiguous()
    out = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    L.check(L.lib().or_rmsnorm_rope(x2.data_ptr(), None, w.data_ptr(), None, x2.stride(0), 0, x2.shape[0], C, 128,
                                    float(eps), None, None, None, 0, out.data_ptr(), None, C, 0,
                                    L.stream_handle(x.device)), 'or_rmsnorm_rope')
    return out


def _grad_rows(x, C: int):
    """x as ([rows, C] bf16 rows that the gradient kernel reads, their stride): contiguous elements, whole 16-byte pieces (a
    copy where x is not such rows, e.g. an expanded gradient)"""
    if x.dtype != torch.bfloat16 or not x.is_cuda:
        raise L.HipTypeError(f'expected a bf16 GPU tensor, got {x.dtype} on {x.device}')
    if x.dim() != 2 or x.shape[1] != C:
        x = x.reshape(-1, C)
    row, one = x.stride()
    if one == 1 and row >= C and row % 8 == 0 and x.data_ptr() % 16 == 0:
        return x, row
    return (x, C) if not x.shape[0] else (x.clone(memory_format=torch.contiguous_format), C)


def _weight(w, C: int):
    if w.numel() != C:
        raise L.HipValueError(f'weights must hold {C} elements, got {tuple(w.shape)}')
    if w.dtype != torch.bfloat16 or not w.is_contiguous():
        w = w.reshape(C).to(torch.bfloat16).contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


_SIZES = functools.lru_cache(256)(lambda S, C: int(L.lib().or_rmsnorm_rope_bwd_workspace_size(S, C)))


def _norm_backward(dys, xs, ws, eps, C: int, D: int, cos=None, sin=None):
    """or_rmsnorm_rope_bwd of one or two tensors: ([dx, ..] [rows, C] bf16, [dw, ..] [C] fp32)"""
    at, dev = xs[0].get_device(), xs[0].device
    for t in (*dys, *xs, *ws, *(() if cos is None else (cos, sin))):
        if t.get_device() != at:
            raise L.HipTypeError('all tensors of a call must be on one GPU')
    both = len(xs) == 2
    (x0, xs0), (d0, ds0), w0 = _grad_rows(xs[0], C), _grad_rows(dys[0], C), _weight(ws[0], C)
    (x1, xs1), (d1, ds1), w1 = (_grad_rows(xs[1], C), _grad_rows(dys[1], C), _weight(ws[1], C)) if both else \
        ((None, 0), (None, 0), None)
    S = x0.shape[0]
    if d0.shape[0] != S or both and (x1.shape[0] != S or d1.shape[0] != S):
        raise L.HipValueError('gradients and inputs must have the same rows')
    new = lambda: (torch.empty(S, C, dtype=torch.bfloat16, device=dev), torch.empty(C, dtype=torch.float32, device=dev))
    (dx0, dw0), (dx1, dw1) = new(), new() if both else (None, None)
    n = _SIZES(S, C)
    if n < 0:
        L.check(L.lib().or_rmsnorm_rope_bwd_workspace_size(S, C), 'or_rmsnorm_rope_bwd_workspace_size')
    space = torch.empty(n, dtype=torch.uint8, device=dev)
    p = L.ptr
    L.check(L.call(dev, L.lib().or_rmsnorm_rope_bwd, d0.data_ptr(), p(d1), x0.data_ptr(), p(x1), w0.data_ptr(), p(w1), ds0,
                   ds1, xs0, xs1, S, C, D, float(eps), p(cos), p(sin), None, S if cos is not None else 0,
                   dx0.data_ptr(), p(dx1), dw0.data_ptr(), p(dw1), space.data_ptr(), n), 'or_rmsnorm_rope_bwd')
    return ([dx0, dx1], [dw0, dw1]) if both else ([dx0], [dw0])


def qk_backward(dq, dk, q, k, wq, wk, eps: float, cos, sin, heads: int):
    """The gradient of _qk: (q_grad, k_grad) bf16 in the shapes of q and k, (wq_grad, wk_grad) fp32 [C]. dq, dk
    [..., S, heads, D] bf16: the gradients of its outputs; the other arguments are the call's own. fp32 inside, one
    rounding; the weights' sums over rows are taken in a fixed order."""
    C = q.shape[-1]
    D = C // heads
    if heads * D != C or k.shape != q.shape or dq.numel() != q.numel() or dk.numel() != q.numel():
        raise L.HipValueError(f'q, k and their gradients must have one size of {heads} heads (q {tuple(q.shape)}, '
                              f'k {tuple(k.shape)}, dq {tuple(dq.shape)}, dk {tuple(dk.shape)})')
    S = q.numel() // C if C else 0
    c, s = (t.reshape(-1, D).to(torch.float32).contiguous() for t in (cos, sin))
    if c.shape[0] != S or s.shape[0] != S:
        raise L.HipValueError(f'rotary tables hold {c.shape[0]} rows for {S} tokens')
    (gq, gk), (gwq, gwk) = _norm_backward([dq, dk], [q, k], [wq, wk], eps, C, D, c, s)
    return gq.view(q.shape), gk.view(k.shape), gwq, gwk


def rms_norm_backward(dy, x, weight, eps: float):
    """The gradient of rms_norm: (dx bf16 in the shape of x, dw fp32 [C])"""
    C = x.shape[-1]
    if dy.shape != x.shape:
        raise L.HipValueError(f'x {tuple(x.shape)} and its output\'s gradient {tuple(dy.shape)} must have one shape')
    (dx,), (dw,) = _norm_backward([dy], [x], [weight], eps, C, 128)
    return dx if x.dim() == 2 else dx.view(x.shape), dw


class _QK(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, eps, cos, sin, heads):
        ctx.save_for_backward(q, k, wq, wk, cos, sin)
        ctx.eps, ctx.heads = eps, heads
        return _qk_forward(q, k, wq, wk, eps, cos, sin, heads)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        q, k, wq, wk, cos, sin = ctx.saved_tensors
        gq, gk, gwq, gwk = qk_backward(dq, dk, q, k, wq, wk, ctx.eps, cos, sin, ctx.heads)
        return gq, gk, gwq.view(wq.shape).to(wq.dtype), gwk.view(wk.shape).to(wk.dtype), None, None, None, None


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        ctx.save_for_backward(x, weight)
        ctx.eps = eps
        return rms_norm(x, weight, eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        dx, dw = rms_norm_backward(dy, x, weight, ctx.eps)
        return dx, dw.view(weight.shape).to(weight.dtype), None


def _token_ranges(lay, T: int) -> list:
    """[first, end) token rows of every scene (T tokens per latent frame)"""
    return [(T * first, T * end) for first, end in lay.ranges]


def self_ranges(ctx: Context, q, k, v):
    """all tokens: every scene's keys are one contiguous range read in place, or packed per scene when it reads extra
    frames (wan.py:110-124); those packed scopes have no gradient, a backward pass that reaches their output raises"""
    T, lay = ctx.T, ctx.layout
    if any(lay.extra.get(j) for j in range(lay.n_scenes)):
        key = ('wan_plan', tuple(lay.lengths), lay.halo, lay.sides,
               tuple((j, tuple(x)) for j, x in sorted(lay.extra.items())), T, str(q.device))
        cache = ctx.__dict__.setdefault('_cache', {})
        if key not in cache:
            cache[key] = ScopePlan(lay, T, None, 0, False, None, False, False, q.device)
        plan = cache[key]
        # keys packed; the values of each scene's own frames and of its first shared frames read in place from v
        # (the others packed; with head_dim 128, as the runs past the leading one need)
        in_place = v.is_contiguous() and q.shape[2] == 128
        kp, vp, _ = pack_layer(plan, k, None, v, None, mode='none', values_in_place=in_place)
        o = torch.empty_like(q)
        vi = dict(v_tok=v, v_lead=plan.v_lead, v_row=plan.v_row, v_runs=plan.v_runs) if in_place else {}
        varlen(q, kp, vp, plan.cu_q, plan.cu_k, plan.max_q, plan.max_k, out=o, seg_q_src=plan.seg_q_src,
               n_q_video=plan.n_video, sum_q=plan.sum_q, **vi)
        return without_gradient('self_ranges with extra frames', o, q, k, v)
    k_ranges = []
    for j in range(lay.n_scenes):
        first, end = lay.key_range(j)
        if end - first != len(lay.key_frames(j)):
            raise L.HipValueError(f'scene {j}: its key frames are not one contiguous run of frames')
        k_ranges.append((T * first, T * end))
    return A.overlapping_ranges(q, k, v, _token_ranges(lay, T), k_ranges)


def memory_self(ctx: Context, q, k, v, layer: int):
    """self-attention with the bounded memory on one GPU (wan.py:154-173): every scene's queries read its frames
    plus M representatives per head of the other scenes' boundary keys; q / k already normalised and rotated"""
    T, lay = ctx.T, ctx.layout
    if ctx._mem is None:
        if lay.halo != 0:
            raise L.HipValueError('the bounded memory replaces the halo frames: use halo = 0')
        ctx._mem = MemoryAttention(BoundaryMemory(ctx.memory))
    pk = (q.shape[0], k.shape[0])
    if pk not in ctx._mem.plans:
        pieces = [(j, lo * T, hi * T) for j, (lo, hi) in enumerate(lay.ranges)]
        ctx._mem.plans[pk] = frame_plan(lay, T, torch.arange(lay.n_frames * T), k.shape[0], pieces, device=q.device)
    return ctx._mem((layer, ctx.cond()), q, k, v, ctx._mem.plans[pk])


def cross_ranges(ctx: Context, q, k, v):
    """scene j's query rows read sentence j's rows [j * text_len, (j + 1) * text_len) of k / v (wan.py:84-89)"""
    T, lay, n = ctx.T, ctx.layout, ctx.text_len
    sentences = [(n * j, n * j + n) for j in range(lay.n_scenes)]
    return A.overlapping_ranges(q, k, v, _token_ranges(lay, T), sentences)


class Processor:
    """kind 'self' or 'cross' (wan.py:77-108). One GPU: the whole token range. rotary_emb: the (cos, sin) tables, or the positions
    (`rotary.Axes`); hidden_states may come in 4 bits (`mxfp4.MXFP4`) where the projections take it so."""

    def __init__(self, ctx: Context, kind: str, orig=None, layer: int = 0):
        assert kind in ('self', 'cross'), kind
        self.ctx, self.kind, self.orig, self.layer = ctx, kind, orig, layer

    def __call__(self, attn, hidden_states, encoder_hidden_states=None, attention_mask=None, rotary_emb=None):
        H = attn.heads
        if self.kind == 'cross':
            q = attn.norm_q(attn.to_q(hidden_states)).unflatten(2, (H, -1))
            k = attn.norm_k(attn.to_k(encoder_hidden_states)).unflatten(2, (H, -1))
            v = attn.to_v(encoder_hidden_states).unflatten(2, (H, -1))
            q, k, v = (x[0].to(torch.bfloat16).contiguous() for x in (q, k, v))
            o = cross_ranges(self.ctx, q, k, v)
        else:
            q, k, v = attn.to_q(hidden_states), attn.to_k(hidden_states), attn.to_v(hidden_states)
            w = attn.norm_q.weight, attn.norm_k.weight, attn.norm_q.eps
            q, k = norm_rotate(q, k, *w, rotary_emb, H) if isinstance(rotary_emb, Axes) else _qk(q, k, *w, *rotary_emb, H)
            v = v.unflatten(2, (H, -1))
            q, k, v = (x[0].to(torch.bfloat16).contiguous() for x in (q, k, v))
            o = memory_self(self.ctx, q, k, v, self.layer) if self.ctx.memory else self_ranges(self.ctx, q, k, v)
        o = o.flatten(1, 2)[None]
        return attn.to_out[1](attn.to_out[0](o if isinstance(hidden_states, MXFP4) else o.type_as(hidden_states)))
