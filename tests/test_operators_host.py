"""CPU checks of the norms, rotary positions, gradient clipping and 4-bit linear layers: what their entry points refuse without a GPU
(in Python and at the C ABI), and their argument structs against the headers."""
import ctypes
import subprocess

import pytest
import torch

from onereel_amd import _lib as L
from onereel_amd import build as B
from onereel_amd import clip, mxfp4, norms, rotary

X = torch.zeros(4, 64, dtype=torch.bfloat16)


def test_tensors_on_the_cpu_are_refused():
    axes = rotary.Axes(torch.zeros(4, 2, dtype=torch.int32), (16, 16))
    calls = [lambda: norms.norm_modulate(X, 1e-6), lambda: norms.residual_norm_modulate(X, X, 1e-6),
             lambda: norms.norm_modulate_backward(X, X, 1e-6), lambda: rotary.rotate(X.view(4, 2, 32), axes),
             lambda: rotary.rotate_backward(X.view(4, 2, 32), axes),
             lambda: rotary.norm_rotate(X, X, X[0], X[0], 1e-6, axes, 2), lambda: clip.grad_norm([X]),
             lambda: clip.clip_grads_([X], 1.0), lambda: mxfp4.quantize(X),
             lambda: mxfp4.MXFP4(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8))]
    for call in calls:
        with pytest.raises(L.HipTypeError):
            call()
    for leaf in (norms.norm_modulate, lambda x, e: rotary.rotate(x.view(4, 2, 32), axes)):
        with pytest.raises(L.HipTypeError):
            leaf(X.clone().requires_grad_(), 1e-6)


def test_axes():
    p = torch.zeros(5, 3, dtype=torch.int32)
    assert rotary.split_dims(128) == (44, 42, 42) and rotary.split_dims(64) == (24, 20, 20)
    a = rotary.Axes(p, [44, 42, 42], theta=256)
    assert a.dims == (44, 42, 42) and a.theta == (256.0,) * 3 and a.positions.shape == (5, 3)
    assert rotary.Axes(p[:, 0], (8,)).positions.shape == (5, 1)
    g = rotary.grid(2, 3, 4, 128, device='cpu')
    assert g.positions.tolist() == [[f, y, x] for f in range(2) for y in range(3) for x in range(4)]
    for bad in (lambda: rotary.Axes(p.long(), (8, 8, 8)), lambda: rotary.Axes(p, (8, 8)), lambda: rotary.Axes(p, ()),
                lambda: rotary.Axes(p, (8, 8, 8), theta=(1.0, 2.0)), lambda: rotary.Axes(p, (8, 8, 8), pairs='x'),
                lambda: rotary.Axes(p[None], (8, 8, 8)), lambda: rotary.Axes(torch.zeros(5, 5).int(), (2,) * 5)):
        with pytest.raises(L.HipPathError):
            bad()


STRUCTS = {'or_block_norm_args': L.BlockNormArgs, 'or_block_norm_bwd_args': L.BlockNormBwdArgs, 'or_rope_axes': L.RopeAxes,
           'or_clip_args': L.ClipArgs, 'or_mx_linear_args': L.MxLinearArgs}


def test_structs_match_the_headers(tmp_path):
    lines = [f'printf("{n} %zu\\n", sizeof({n}));' for n in STRUCTS]
    lines += [f'printf("{n}.{f[0]} %zu\\n", offsetof({n}, {f[0]}));' for n, s in STRUCTS.items() for f in s._fields_]
    src = tmp_path / 's.c'
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "onereel_hip.h"\n#include "onereel_dit.h"\n'
                   'int main(void) {\n' + '\n'.join(lines) + '\nreturn 0; }\n')
    subprocess.run(['gcc', '-I', str(B.INCLUDE), str(src), '-o', str(tmp_path / 's')], check=True)
    got = dict(l.split() for l in subprocess.run([str(tmp_path / 's')], capture_output=True, text=True, check=True).stdout.splitlines())
    for n, s in STRUCTS.items():
        assert int(got[n]) == ctypes.sizeof(s), n
        for f in s._fields_:
            assert int(got[f'{n}.{f[0]}']) == getattr(s, f[0]).offset, f'{n}.{f[0]}'


def refused(lib, name, *args, text=''):
    rc = getattr(lib, name)(*args)
    message = lib.or_last_error().decode()
    assert rc == -1 and text in message, (name, rc, message)


BUF = ctypes.create_string_buffer(1 << 12)
AT = (ctypes.addressof(BUF) + 255) & ~255


def norm_args(cls, **over):
    a = cls()
    for f in ('x', 'n', 'h', 'a', 'dn', 'dx', 'da'):
        if hasattr(cls, f):
            setattr(a, f, AT)
    a.n_rows, a.rows_per_group, a.C, a.type, a.norm, a.post_norm, a.eps, a.residual_scale = 4, 2, 64, 0, 1, 0, 1e-6, 1.0
    for f in ('x_row_stride', 'a_row_stride', 'dh_row_stride', 'dn_row_stride', 'h_row_stride'):
        if hasattr(cls, f):
            setattr(a, f, 64)
    for k, v in over.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize('over,text', [(dict(C=60), 'multiple of 8'), (dict(C=8200), 'up to 8192'), (dict(type=3), 'type'),
                                       (dict(norm=0), 'norm'), (dict(post_norm=5), 'post_norm'), (dict(n_rows=-1), 'rows'),
                                       (dict(rows_per_group=3), 'divide'), (dict(rows_per_group=0), 'divide'),
                                       (dict(a_row_stride=60), 'apart'), (dict(a=AT + 8), 'aligned'), (dict(gate=AT + 4), 'aligned'),
                                       (dict(post_weight=AT), 'post_norm'), (dict(a=None, gate=AT), 'belong')])
def test_norms_at_the_c_abi(over, text):
    d = L.dit_lib()
    refused(d, 'or_block_norm', norm_args(L.BlockNormArgs, **over), None, text=text)
    refused(d, 'or_block_norm_bwd', norm_args(L.BlockNormBwdArgs, **over), None, text=text)


def test_norms_at_the_c_abi_more():
    d = L.dit_lib()
    refused(d, 'or_block_norm', None, None)
    refused(d, 'or_block_norm_bwd', None, None)
    refused(d, 'or_block_norm', norm_args(L.BlockNormArgs, x=None), None, text='required')
    refused(d, 'or_block_norm_bwd', norm_args(L.BlockNormBwdArgs, dshift=AT), None, text='workspace')
    refused(d, 'or_block_norm_bwd', norm_args(L.BlockNormBwdArgs, a=None, dgate=AT), None, text='belong')
    assert d.or_block_norm(norm_args(L.BlockNormArgs, n_rows=0, x=None), None) == 0
    assert d.or_block_norm_bwd_workspace_size(4, 3, 64) == -1 and d.or_block_norm_bwd_workspace_size(0, 1, 64) == 0
    assert d.or_block_norm_bwd_workspace_size(12720, 1590, 2048) >= 3 * 2048 * 4 * 9


def axes_args(**over):
    a = L.RopeAxes(AT, 4, 2, 0, 0, (L.i32 * 4)(16, 16, 0, 0), (ctypes.c_double * 4)(1e4, 1e4, 0, 0))
    for k, v in over.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize('over,text', [(dict(n_axes=0), 'axes'), (dict(n_axes=5), 'axes'), (dict(pairs=2), 'pairs'),
                                       (dict(dims=(L.i32 * 4)(15, 16)), 'even'), (dict(dims=(L.i32 * 4)(20, 16)), 'of 32 dims'),
                                       (dict(dims=(L.i32 * 4)(0, 16)), 'even'), (dict(dims=(L.i32 * 4)(-2, 16)), 'even'),
                                       (dict(dims=(L.i32 * 4)(12, 16), pairs=1), 'half'),
                                       (dict(theta=(ctypes.c_double * 4)(float('nan'), 1)), 'theta'),
                                       (dict(theta=(ctypes.c_double * 4)(0.0, 1)), 'theta'), (dict(n_positions=3), 'divide'),
                                       (dict(n_positions=0), 'divide'), (dict(positions=None), 'positions'),
                                       (dict(positions=AT + 2), 'positions')])
def test_rotary_at_the_c_abi(over, text):
    h = L.lib()
    refused(h, 'or_rope_axes_rotate', axes_args(**over), AT, AT, 4, 2, 32, 64, 32, 0, 0, None, text=text)
    refused(h, 'or_rmsnorm_rope_axes', axes_args(**over), AT, AT, AT, AT, 64, 64, 4, 64, 32, 0, 1e-6, AT, AT, None, text=text)
    refused(h, 'or_rmsnorm_rope_axes_bwd', axes_args(**over), AT, AT, AT, AT, AT, AT, 64, 64, 64, 64, 4, 64, 32, 0, 1e-6, AT, AT, AT,
            AT, AT, 1 << 20, None, text=text)


def test_rotary_at_the_c_abi_more():
    h = L.lib()
    refused(h, 'or_rope_axes_rotate', None, AT, AT, 4, 2, 32, 64, 32, 0, 0, None)
    refused(h, 'or_rope_axes_rotate', axes_args(), AT, AT, 4, 0, 32, 64, 32, 0, 0, None, text='heads')
    refused(h, 'or_rope_axes_rotate', axes_args(), AT, AT, 4, 2, 36, 64, 32, 0, 0, None, text='dims')
    refused(h, 'or_rope_axes_rotate', axes_args(), AT, AT, 4, 2, 520, 64, 32, 0, 0, None, text='dims')
    refused(h, 'or_rope_axes_rotate', axes_args(), AT, AT, 4, 2, 32, 62, 32, 0, 0, None, text='strides')
    refused(h, 'or_rope_axes_rotate', axes_args(), AT, AT, 4, 2, 32, 64, 32, 3, 0, None, text='type')
    refused(h, 'or_rope_axes_rotate', axes_args(), AT + 4, AT, 4, 2, 32, 64, 32, 0, 0, None, text='aligned')
    refused(h, 'or_rmsnorm_rope_axes', axes_args(), AT, AT, AT, AT, 64, 64, 4, 80, 32, 0, 1e-6, AT, AT, None, text='whole heads')
    refused(h, 'or_rmsnorm_rope_axes', axes_args(), AT, AT, AT, None, 64, 64, 4, 64, 32, 0, 1e-6, AT, AT, None, text='weights')
    refused(h, 'or_rmsnorm_rope_axes', axes_args(), AT, AT, AT, AT, 60, 64, 4, 64, 32, 0, 1e-6, AT, AT, None, text='apart')
    refused(h, 'or_rmsnorm_rope_axes_bwd', axes_args(), AT, AT, AT, AT, AT, AT, 64, 64, 64, 64, 4, 64, 32, 0, 1e-6, AT, AT, AT, AT, AT, 8,
            None, text='workspace')
    assert h.or_rmsnorm_rope_axes_bwd_workspace_size(-1, 64) == -1 and h.or_rmsnorm_rope_axes_bwd_workspace_size(0, 64) == 0


def clip_args(x=(AT,), numel=(8,), types=(2,), out=None, out_types=None, max_norm=1.0, norm=AT, workspace=AT, size=1 << 12):
    n = len(x)
    arrays = [(ctypes.c_uint64 * n)(*x), (ctypes.c_int64 * n)(*numel), (ctypes.c_int32 * n)(*types)]
    arrays += [out and (ctypes.c_uint64 * n)(*out), out_types and (ctypes.c_int32 * n)(*out_types)]
    a = L.ClipArgs(*(None if v is None else ctypes.addressof(v) for v in arrays), n, max_norm, norm, workspace, size)
    a.keep = arrays
    return ctypes.byref(a)


def test_clipping_at_the_c_abi():
    d = L.dit_lib()
    refused(d, 'or_clip', None, None)
    refused(d, 'or_clip_workspace_size', None)
    for over, text in [(dict(types=(7,)), 'type'), (dict(numel=(-1,)), 'elements'), (dict(x=(AT + 2,)), 'address'), (dict(x=(0,)), 'address'),
                       (dict(out=(AT + 1,)), 'address'), (dict(out=(AT + 16,)), 'share memory'),
                       (dict(out=(AT,), out_types=(0,)), 'another type'), (dict(out=(AT,), max_norm=-1.0), 'max_norm'),
                       (dict(out=(AT,), max_norm=float('nan')), 'max_norm'), (dict(norm=None), 'norm'), (dict(size=4), 'workspace'),
                       (dict(workspace=AT + 8), 'workspace'),
                       (dict(x=(AT, AT + 16), numel=(8, 8), types=(2, 2), out=(AT, AT + 16)), 'share memory'),
                       (dict(x=(AT, AT + 64), numel=(8, 8), types=(2, 2), out=(AT + 64, AT)), 'share memory')]:
        refused(d, 'or_clip', clip_args(**over), None, text=text)
    assert d.or_clip_workspace_size(clip_args(x=(), numel=(), types=())) == 0
    assert d.or_clip_workspace_size(clip_args(numel=(1 << 30,))) == 512 * 8
    assert d.or_clip_workspace_size(clip_args(x=(AT,) * 300, numel=(8,) * 300, types=(2,) * 300)) == 300 * 8


def mx_args(**over):
    a = L.MxLinearArgs(AT, None, None, AT, AT, None, None, None, AT, 40, 64, 16, 16, 64, 16, 0, 0, 0, AT, 1 << 30)
    for k, v in over.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_4_bit_layers_at_the_c_abi():
    d = L.dit_lib()
    refused(d, 'or_mx_linear', None, None)
    for over, text in [(dict(n_in=48), '32'), (dict(n_in=0), '32'), (dict(n_out=12), 'n_out'), (dict(n_rows=-1), 'rows'),
                       (dict(activation=9), 'activation'), (dict(x=None), 'x_codes'), (dict(weight_codes=None), 'weight_codes'),
                       (dict(y=None), 'y'), (dict(x_row_stride=56), 'apart'), (dict(x_row_stride=68), 'apart'),
                       (dict(y_row_stride=8), 'apart'), (dict(residual=AT, residual_row_stride=12), 'apart'),
                       (dict(bias=AT + 8), 'aligned'), (dict(workspace_bytes=16), 'workspace'), (dict(workspace=None), 'workspace'),
                       (dict(n_rows=1 << 30, n_out=1 << 21, y_row_stride=1 << 21), 'tiles')]:
        refused(d, 'or_mx_linear', mx_args(**over), None, text=text)
    refused(d, 'or_mx_quantize', AT, 4, 40, 64, 0, AT, AT, None, text='32')
    refused(d, 'or_mx_quantize', AT, 4, 64, 60, 0, AT, AT, None, text='apart')
    refused(d, 'or_mx_quantize', AT, 4, 64, 64, 4, AT, AT, None, text='type')
    refused(d, 'or_mx_quantize', AT, 4, 64, 64, 0, None, AT, None, text='required')
    refused(d, 'or_mx_dequantize', AT, AT, 4, 40, 0, AT, None, text='32')
    refused(d, 'or_mx_dequantize', AT + 4, AT, 4, 64, 0, AT, None, text='aligned')
    assert d.or_mx_linear_workspace_size(4, 40, 16, 0) == -1
    assert d.or_mx_linear_workspace_size(1, 2048, 512, 0) == 0
    assert d.or_mx_linear_workspace_size(12720, 2048, 8192, 0) >= 12720 * 1024


def test_workspaces_grow_no_further_than_stated():
    d = L.dit_lib()
    for rows in (1, 16, 17, 33, 300, 5000, 100000):
        for n_in in (32, 2048, 8192):
            for n_out in (8, 2048, 8192):
                for quantized in (0, 1):
                    n = d.or_mx_linear_workspace_size(rows, n_in, n_out, quantized)
                    # codes and scales of whole tiles of 256 rows and 256 elements, and split sums of products too small for the GPU
                    whole = lambda v: (v + 255) // 256 * 256
                    assert 0 <= n <= (0 if quantized else rows * n_in // 2) + (whole(rows) + whole(n_out)) * whole(n_in) // 32 + \
                        16 * 4 * min(rows * n_out, 1 << 21) + 2048, (rows, n_in, n_out)
