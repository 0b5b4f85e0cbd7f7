"""Varlen attention on the gfx950 kernel: the drop-in for `onereel.attention` (src/onereel/attention.py:1-84).

Same names, shapes and semantics: packed q [Nq, H, D], k / v [Nk, H, D], bf16, non-causal, softmax scale D^-0.5;
`cu_seqlens` int32 on the device. The reference's FlashAttention backends (`BACKEND` 'fa2' / 'fa3' / 'auto') map to
the one HIP kernel; `backend()` reports 'hip'. Errors raise `onereel_amd._lib.HipPathError` (a RuntimeError).

`dense`, `varlen`, `varlen_lse`, `packed`, `packed_lse`, `overlapping_ranges` and `overlapping_ranges_lse` are
differentiable in q, k and v, as FlashAttention's are (once; the gradient itself has no graph): when autograd records and
one of them requires a gradient, the call keeps its output and log-sum-exp for `or_varlen_bwd`. `varlen_backward` and
`overlapping_ranges_backward` are the same gradients as plain calls, without autograd.
"""
from __future__ import annotations

import array
import ctypes
import functools
import operator
import warnings

import torch

from . import _lib as _L
from . import scene as _scene

BACKEND = 'hip'


_SHAPE, _DTYPE = operator.attrgetter('shape'), operator.attrgetter('dtype')


def backend() -> str:
    return 'hip'


def _offsets(lengths) -> list:
    """[0, cumsum(lengths)]"""
    c, out = 0, [0]
    for n in lengths:
        c += int(n)
        out.append(c)
    return out


def cu_seqlens(lengths, device='cuda') -> torch.Tensor:
    """[0, cumsum(lengths)] int32 (attention.py:28-29), there when the call returns: whatever stream reads it"""
    return torch.tensor(_offsets(lengths), dtype=torch.int32, device=device)


def wants_grad(*xs) -> bool:
    """whether autograd records a call on these tensors (None: no tensor)"""
    return torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in xs)


def captured_leaves(*xs) -> bool:
    """Whether this call is being captured and one of xs is a leaf that requires a gradient. A backward pass recorded into a
    graph adds into its leaves' gradients on the stream of the first pass that used them; when that is another stream (an
    eager pass whose graph still lives), the capture ends the process. So autograd records no such call; the backward entry
    points without autograd can be captured."""
    return any(x is not None and x.is_cuda and x.requires_grad and x.is_leaf for x in xs) and \
        torch.cuda.is_current_stream_capturing()


def records(what: str, *xs) -> bool:
    """whether a call on these tensors is recorded by autograd: when wants_grad says so, but for captured_leaves, whose call
    runs as it does without autograd (with a warning)"""
    if not wants_grad(*xs):
        return False
    if captured_leaves(*xs):
        warnings.warn(f'{what}: under graph capture a call on leaves that require gradients is not recorded: capture the '
                      f'backward entry point instead', stacklevel=3)
        return False
    return True


def unrecorded_capture(what: str, *xs):
    """xs, detached where records would not have autograd record a call on them, for entry points that reshape or
    concatenate them first: what that makes of a leaf is none"""
    return [x.detach() for x in xs] if wants_grad(*xs) and not records(what, *xs) else xs


_MAX_STRIDE = 1 << 24      # of or_varlen_bwd's rows


def _rows_for(x, H: int, D: int):
    """(x, row stride), x itself where its rows are as the kernels read them, else a copy (a gradient may come expanded or
    transposed)"""
    shape = x.shape    # asked for once, as in scene._rows2d: a small call's time is the host's
    if len(shape) != 3 or shape[1] != H or shape[2] != D:
        raise _L.HipValueError(f'expected [rows, {H}, {D}], got {tuple(shape)}')
    if x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x, H * D
    stride = x.stride()
    row = stride[0]
    if stride[2] == 1 and stride[1] == D and H * D <= row <= _MAX_STRIDE and row % 8 == 0 and x.data_ptr() % 16 == 0:
        return x, row
    return (x, H * D) if not shape[0] else (x.clone(memory_format=torch.contiguous_format), H * D)


_GRAD_SIZES = functools.lru_cache(256)(lambda *sizes: int(_L.lib().or_varlen_bwd_workspace_size(*sizes)))


def _index_pointers(q, *index):
    """the addresses of a call's index arrays (None: no array)"""
    at = q.get_device()
    for x in index:
        if x is not None and (x.dtype != torch.int32 or x.get_device() != at or not x.is_contiguous()):
            raise _L.HipTypeError('index arrays must be contiguous int32 tensors on the GPU of q')
    return [_L.ptr(x) for x in index]


def _backward(do, q, k, v, o, lse, index, n_seg, max_q, max_k, dlse=None):
    """or_varlen_bwd on torch tensors: (dq, dk, dv), bf16 and contiguous. index: the addresses of cu_q, cu_k, k_off, k_len,
    or an array of the ints of cu_q, k_off and k_len, which then lie behind the workspace"""
    _scene._check_bf16(do, q, k, v, o)
    if k.dim() != 3 or q.dim() != 3:
        raise _L.HipValueError('q, k and v must be [rows, heads, head_dim]')
    (n_q, H, D), more_k, more_v, dev, at = q.shape, k.shape[0], v.shape[0], q.device, q.get_device()
    if o.shape[0] != n_q or do.shape[0] != n_q:
        raise _L.HipValueError('q, o and do must have the same rows')
    n_k = min(more_k, more_v)
    if more_k != more_v:     # rows that only one of them has are read by no segment
        k, v = k[:n_k], v[:n_k]
    for x in (lse, dlse):
        if x is not None and (x.dtype != torch.float32 or x.shape != (H, n_q) or x.get_device() != at):
            raise _L.HipTypeError(f'lse and its gradient must be float32 [{H}, {n_q}] on the GPU of q')
    if do.get_device() != at or k.get_device() != at or v.get_device() != at or o.get_device() != at:
        raise _L.HipTypeError('all tensors of a call must be on one GPU')
    (q, qs), (o, os_), (do, dos) = _rows_for(q, H, D), _rows_for(o, H, D), _rows_for(do, H, D)
    (k, ks), (v, vs) = _rows_for(k, H, D), _rows_for(v, H, D)
    if ks != vs:
        (k, ks), v = (k.clone(memory_format=torch.contiguous_format), H * D), v.clone(memory_format=torch.contiguous_format)
    lse = lse.contiguous()
    dlse = None if dlse is None else dlse.contiguous()
    new = lambda n: torch.empty(n, H, D, dtype=torch.bfloat16, device=dev)
    dq, dk, dv = new(n_q), new(more_k), new(more_v)
    if more_k != more_v:
        (dk if more_k > n_k else dv)[n_k:].zero_()
    max_q, max_k = int(max_q), int(max_k)
    n = _GRAD_SIZES(n_seg, n_q, n_k, max_q, max_k, H, D)
    if n < 0:
        _L.check(_L.lib().or_varlen_bwd_workspace_size(n_seg, n_q, n_k, max_q, max_k, H, D), 'or_varlen_bwd_workspace_size')
    p = _L.ptr
    if isinstance(index, array.array):
        ws = torch.empty(n + 4 * len(index), dtype=torch.uint8, device=dev)
        to = ws.data_ptr() + n
        _L.check(_L.call(dev, _L.lib().or_index_fill, index.buffer_info()[0], len(index), to), 'or_index_fill')
        index = to, None, to + 4 * n_seg + 4, to + 8 * n_seg + 4
    else:
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
    a = _L.VarlenBwdArgs(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), do.data_ptr(), lse.data_ptr(), p(dlse),
                         dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *index, qs, ks, os_, dos, n_q, n_seg, n_q, n_k, max_q,
                         max_k, H, D, D ** -0.5, ws.data_ptr(), n)
    _L.check(_L.call(dev, _L.lib().or_varlen_bwd, ctypes.byref(a)), 'or_varlen_bwd')
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    """or_varlen_fwd with its log-sum-exp, and or_varlen_bwd"""

    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, k_off, k_len, max_q, max_k):
        lse = torch.empty(q.shape[1], q.shape[0], dtype=torch.float32, device=q.device)
        o = _scene.varlen(q, k, v, cu_q, cu_k, max_q, max_k, k_off=k_off, k_len=k_len, lse=lse)
        ctx.save_for_backward(q, k, v, o, lse, cu_q, cu_k, k_off, k_len)
        ctx.longest = max_q, max_k
        ctx.set_materialize_grads(False)
        return o, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dlse):
        q, k, v, o, lse, cu_q, cu_k, k_off, k_len = ctx.saved_tensors
        grads = (None,) * 3
        if do is not None or dlse is not None:
            do = torch.zeros_like(o) if do is None else do
            grads = _backward(do, q, k, v, o, lse, _index_pointers(q, cu_q, cu_k, k_off, k_len), cu_q.numel() - 1,
                              *ctx.longest, dlse)
        return *grads, None, None, None, None, None, None


def _attend(q, k, v, cu_q, cu_k, max_q, max_k, k_off=None, k_len=None, lse=False):
    """the varlen call of every entry point: o, or (o, lse)"""
    if records('attention', q, k, v):
        o, l = _Attention.apply(q, k, v, cu_q, cu_k, k_off, k_len, max_q, max_k)
        return (o, l) if lse else o
    l = torch.empty(q.shape[1], q.shape[0], dtype=torch.float32, device=q.device) if lse else None
    o = _scene.varlen(q, k, v, cu_q, cu_k, max_q, max_k, k_off=k_off, k_len=k_len, lse=l)
    return (o, l) if lse else o


def dense(q, k, v):
    """q, k, v [B, S, H, D] -> [B, S, H, D] (attention.py:32-36)"""
    B, S, H, D = q.shape
    Sk = k.shape[1]
    q, k, v = unrecorded_capture('dense', q, k, v)
    cu_q, cu_k = _L.device_ints([_offsets([S] * B), _offsets([Sk] * B)], q.device)
    o = _attend(q.reshape(B * S, H, D), k.reshape(B * Sk, H, D), v.reshape(B * Sk, H, D), cu_q, cu_k, S, Sk)
    return o.view(B, S, H, D)


def check_cu_seqlens(cu: torch.Tensor, n_rows: int, max_len: int, what: str):
    """cu_seqlens as the kernels read them: [0, ..., total] nondecreasing with total <= n_rows and no segment longer
    than max_len. The kernels index q / k / v rows by these offsets without bounds checks, so a bad entry is an error
    here, before any launch (one copy of n_seg + 1 int32 to the host)"""
    if cu.dim() != 1 or cu.numel() < 2:
        raise _L.HipValueError(f'{what} must be a 1-D tensor of at least 2 offsets')
    c = cu.cpu().tolist()
    lens = [b - a for a, b in zip(c, c[1:])]
    if c[0] != 0 or min(lens) < 0 or c[-1] > n_rows:
        raise _L.HipValueError(f'{what} must start at 0, not decrease and end at most at {n_rows} rows (ends at '
                               f'{c[-1]}, starts at {c[0]})')
    if max(lens) > max_len:
        raise _L.HipValueError(f'{what}: a segment of {max(lens)} rows exceeds the given maximum {max_len}')


def varlen(q, k, v, cu_q, cu_k, max_q, max_k, check: bool = True):
    """packed q [Nq, H, D], k / v [Nk, H, D] (attention.py:39-43). cu_q / cu_k are checked against the row counts
    and max_q / max_k on the host unless check=False (callers whose offsets are known to be good)"""
    if check:
        check_cu_seqlens(cu_q, q.shape[0], max_q, 'cu_q')
        check_cu_seqlens(cu_k, min(k.shape[0], v.shape[0]), max_k, 'cu_k')
        if cu_q.numel() != cu_k.numel():
            raise _L.HipValueError('cu_q and cu_k must hold one offset per segment boundary each')
    return _attend(q, k, v, cu_q, cu_k, max_q, max_k)


def varlen_lse(q, k, v, cu_q, cu_k, max_q, max_k, check: bool = True):
    """varlen with the softmax log-sum-exp: (out [Nq, H, D], lse [H, Nq] fp32) (attention.py:46-53)"""
    if check:
        check_cu_seqlens(cu_q, q.shape[0], max_q, 'cu_q')
        check_cu_seqlens(cu_k, min(k.shape[0], v.shape[0]), max_k, 'cu_k')
        if cu_q.numel() != cu_k.numel():
            raise _L.HipValueError('cu_q and cu_k must hold one offset per segment boundary each')
    return _attend(q, k, v, cu_q, cu_k, max_q, max_k, lse=True)


def varlen_backward(do, q, k, v, o, lse, cu_q, cu_k, max_q, max_k, dlse=None, check: bool = True):
    """The gradient of varlen / varlen_lse: (dq, dk, dv) bf16 from do [Nq, H, D], the call's inputs, its output o and lse
    [H, Nq] fp32, and dlse [H, Nq] fp32 when the lse was used too. Rows of q behind the last segment and rows of k / v
    that no segment reads get zeros. Sums are fp32 in a fixed order: the same bits every time. check as in varlen."""
    if check:
        check_cu_seqlens(cu_q, q.shape[0], max_q, 'cu_q')
        check_cu_seqlens(cu_k, min(k.shape[0], v.shape[0]), max_k, 'cu_k')
    if cu_q.numel() != cu_k.numel():
        raise _L.HipValueError('cu_q and cu_k must hold one offset per segment boundary each')
    return _backward(do, q, k, v, o, lse, _index_pointers(q, cu_q, cu_k, None, None), cu_q.numel() - 1, max_q, max_k,
                     dlse)


def _concat_table(xs):
    """addresses and shapes of the tensors xs when or_concat takes them (bf16 rows of one [H, D] on one GPU, contiguous and
    16-byte aligned), else None. Every test is one pass of a C function over all of them: with a Python expression per
    sequence, 300 sequences of 20 rows took 579 us a call where three torch.cat took 363."""
    shapes = list(map(_SHAPE, xs))
    if set(map(len, shapes)) != {3} or len(set(map(torch.Tensor.get_device, xs))) != 1 or not xs[0].is_cuda or \
            set(map(_DTYPE, xs)) != {torch.bfloat16} or not all(map(torch.Tensor.is_contiguous, xs)):
        return None
    rows, heads, dims = zip(*shapes)
    if len(set(heads)) != 1 or len(set(dims)) != 1 or not heads[0] * dims[0] or heads[0] * dims[0] % 8:
        return None
    at = list(map(torch.Tensor.data_ptr, xs))
    return None if functools.reduce(operator.or_, at) % 16 else (at, rows, heads[0], dims[0])


def _concat(segments):
    """the segments' q, k and v end to end, as the varlen call takes them, and the query count of each segment"""
    qs, ks, vs = zip(*segments)
    n, dev = len(qs), qs[0].device
    grad = wants_grad(*qs, *ks, *vs)
    if grad:
        xs = unrecorded_capture('packed', *qs, *ks, *vs)
        qs, ks, vs, grad = xs[:n], xs[n:2 * n], xs[2 * n:], wants_grad(*xs)
    # past one launch of or_concat (112 sequences) the host is what counts, and torch.cat needs less of it per tensor (225
    # sequences of 20 rows x 16 x 128: 297 us a call with or_concat, 258 so), unless the sequences are long enough for the
    # GPU to be the slower side (300 of 100 rows: 428 and 594, of 300: 984 and 1453)
    nq = nk = None
    if n > 112:
        nq, nk = [x.shape[0] for x in qs], [x.shape[0] for x in ks]
    long = n <= 112 or (sum(nq) + 2 * sum(nk)) * qs[0].shape[1:].numel() >= n << 19
    # autograd records torch.cat
    table = _concat_table(qs + ks + vs) if long and not grad else None
    if table is not None and table[1][n:2 * n] == table[1][2 * n:] and sum(table[1]) < 2 ** 31:
        at, rows, *row = table
        nq, nk = rows[:n], rows[n:2 * n]
        q, k, v = (torch.empty(m, *row, dtype=torch.bfloat16, device=dev) for m in (sum(nq), sum(nk), sum(nk)))
        cu_q, cu_k = torch.empty(2, n + 1, dtype=torch.int32, device=dev)
        at, rows = array.array('Q', at), array.array('i', rows)
        pa, pr = at.buffer_info()[0], rows.buffer_info()[0]
        with torch.cuda.device(dev):
            _L.check(_L.lib().or_concat(pa, pa + 8 * n, pa + 16 * n, pr, pr + 4 * n, n, 2 * row[0] * row[1], q.data_ptr(),
                                        k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(),
                                        _L.stream_handle(dev)), 'or_concat')
    else:
        if nq is None:
            nq, nk = [x.shape[0] for x in qs], [x.shape[0] for x in ks]
        q, k, v = torch.cat(qs), torch.cat(ks), torch.cat(vs)
        cu_q, cu_k = _L.device_ints([_offsets(nq), _offsets(nk)], dev)
    return (q, k, v, cu_q, cu_k, max(nq), max(nk)), nq


class _Pieces(torch.autograd.Function):
    """x.split(sizes) as tensors that take in-place operations, which the views of torch's split do not. They are x's memory,
    which the gradient of the call that made x reads: a piece that has changed is an error in the backward pass."""

    @staticmethod
    def forward(ctx, x, sizes):
        out = torch.unsafe_split_with_sizes(x, sizes)
        ctx.save_for_backward(*out)
        return tuple(out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        ctx.saved_tensors       # raises when one has changed
        return torch.cat(grads), None


def _pieces(x, sizes):
    return _Pieces.apply(x, sizes) if x.requires_grad else x.split(sizes)


def packed_lse(segments):
    """as packed, with each segment's log-sum-exp: list of (out, lse [H, n]) (attention.py:56-62)"""
    args, nq = _concat(segments)
    o, lse = varlen_lse(*args, check=False)    # offsets built here from the segments' lengths
    # a recorded lse is kept for the gradient: the segments get copies
    return list(zip(_pieces(o, nq), torch.split_with_sizes_copy(lse, nq, 1) if lse.requires_grad else lse.split(nq, dim=1)))


def packed(segments):
    """segments: list of (q, k, v) sequences -> list of outputs, one varlen call (attention.py:65-71)"""
    args, nq = _concat(segments)
    return _pieces(varlen(*args, check=False), nq)    # offsets built here from the segments' lengths


def _range_args(q, k, v, q_ranges, k_ranges):
    """(cu_q, key starts, key counts) of overlapping_ranges as lists, checked"""
    nq = [hi - lo for lo, hi in q_ranges]
    cu_q = _offsets(nq)
    if cu_q[-1] != q.shape[0] or [lo for lo, _ in q_ranges] != cu_q[:-1]:
        raise _L.HipValueError('q_ranges must tile q in order')
    if len(k_ranges) != len(q_ranges):
        raise _L.HipValueError('q_ranges and k_ranges must pair up')
    n_k = min(k.shape[0], v.shape[0])
    if any(not 0 <= lo <= hi <= n_k for lo, hi in k_ranges):
        raise _L.HipValueError(f'k_ranges must lie inside the {n_k} rows of k and v')
    return cu_q, [lo for lo, _ in k_ranges], [hi - lo for lo, hi in k_ranges]


def _ranges(q, k, v, q_ranges, k_ranges, lse):
    cu_q, starts, counts = _range_args(q, k, v, q_ranges, k_ranges)
    index = _L.device_ints([cu_q, starts, counts], q.device)
    longest = max(hi - lo for lo, hi in q_ranges)
    return _attend(q, k, v, index[0], None, longest, max(counts), *index[1:], lse=lse)


def overlapping_ranges(q, k, v, q_ranges, k_ranges):
    """attention of q rows q_ranges[j] to k / v rows k_ranges[j] without copying k / v: the kernel reads the
    overlapping contiguous key ranges in place (per-segment key offset and length, as FA3's cu_seqlens_k offsets
    with seqused_k). q_ranges must tile q in order (attention.py:74-84)."""
    return _ranges(q, k, v, q_ranges, k_ranges, False)


def overlapping_ranges_lse(q, k, v, q_ranges, k_ranges):
    """overlapping_ranges with the softmax log-sum-exp: (out, lse [H, Nq] fp32), what its backward call needs"""
    return _ranges(q, k, v, q_ranges, k_ranges, True)


def overlapping_ranges_backward(do, q, k, v, o, lse, q_ranges, k_ranges, dlse=None):
    """the gradient of overlapping_ranges / overlapping_ranges_lse, as varlen_backward: a row of k and v sums the
    gradients of every range that reads it"""
    cu_q, starts, counts = _range_args(q, k, v, q_ranges, k_ranges)
    if not q.is_cuda:
        raise _L.HipTypeError(f'expected a bf16 GPU tensor, got {q.dtype} on {q.device}')
    return _backward(do, q, k, v, o, lse, array.array('i', cu_q + starts + counts), len(starts),
                     max(hi - lo for lo, hi in q_ranges), max(counts), dlse)


def merge_lse(o, lse, o_s, lse_s):
    """fold a partial attention result into a running one, in place: o [N, H, D] fp32 and lse [H, N] fp32 are updated
    with o_s [N, H, D] bf16 and lse_s [H, N] fp32 (as varlen_lse returns them). The log-sum-exp merge of ring._merge
    (src/onereel/parallel/ring.py:63-70) and of Processor._far_lse (src/onereel/models/hunyuan15.py:270-275).
    Returns (o, lse). It has no gradient: where autograd records and an argument requires one, a backward pass that reaches
    the results raises, as does one that needs what they held before."""
    N, H, D = o.shape
    if o.dtype != torch.float32 or lse.dtype != torch.float32 or lse_s.dtype != torch.float32:
        raise _L.HipTypeError('o, lse and lse_s must be float32')
    if o_s.dtype != torch.bfloat16 or tuple(o_s.shape) != (N, H, D):
        raise _L.HipTypeError(f'o_s must be bfloat16 [{N}, {H}, {D}]')
    if tuple(lse.shape) != (H, N) or tuple(lse_s.shape) != (H, N) or not (lse.is_contiguous() and lse_s.is_contiguous()):
        raise _L.HipValueError(f'lse and lse_s must be contiguous [{H}, {N}]')
    for x in (o, o_s):
        if x.stride(2) != 1 or x.stride(1) != D:
            raise _L.HipValueError('o and o_s rows must hold contiguous [H, D]')
    for x in (o, lse):
        _scene.overwritten('merge_lse', x, o, lse, o_s, lse_s)
    _L.check(_L.lib().or_lse_merge(o.data_ptr(), lse.data_ptr(), o_s.data_ptr(), lse_s.data_ptr(), N, H, D,
                                   o.stride(0), o_s.stride(0), _L.stream_handle(o.device)), 'or_lse_merge')
    return o, lse
