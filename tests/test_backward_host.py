"""CPU checks of the gradient entry points: their argument structures match the header, and they refuse bad arguments before
any launch."""
import ctypes
import subprocess

import pytest
import torch

from conftest import ROOT
from onereel_amd import _lib as L
from onereel_amd import attention as A
from onereel_amd import linear as F
from onereel_amd import wan


@pytest.mark.parametrize('cls,name,header', [(L.VarlenBwdArgs, 'or_varlen_bwd_args', 'onereel_hip.h'),
                                             (L.LinearArgs, 'or_linear_args', 'onereel_dit.h'),
                                             (L.LinearBwdArgs, 'or_linear_bwd_args', 'onereel_dit.h')])
def test_struct_matches_the_header(cls, name, header, tmp_path):
    lines = ['#include <stddef.h>', '#include <stdio.h>', f'#include "{ROOT / "include" / header}"',
             'int main(void) {', f'printf("%zu\\n", sizeof({name}));']
    lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / 'a.c', tmp_path / 'a'
    src.write_text('\n'.join(lines + ['return 0; }']))
    subprocess.run(['gcc', str(src), '-o', str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f, _ in cls._fields_]


def bwd_args(**kw):
    a = L.VarlenBwdArgs()
    for f in ('q', 'k', 'v', 'o', 'd_o', 'lse', 'dq', 'dk', 'dv', 'cu_q', 'cu_k', 'workspace'):
        setattr(a, f, 4096)
    a.q_row_stride = a.k_row_stride = a.o_row_stride = a.do_row_stride = 256
    a.lse_stride = a.n_q = a.n_k = a.max_q = a.max_k = 100
    a.n_seg, a.H, a.D, a.scale, a.workspace_bytes = 2, 2, 128, 0.1, 1 << 40
    for f, x in kw.items():
        setattr(a, f, x)
    return a


@pytest.mark.parametrize('kw,message', [
    (dict(D=96), 'head_dim'), (dict(H=0), 'heads'), (dict(H=257), 'heads'), (dict(n_seg=0), 'segments'),
    (dict(n_seg=4097), 'segments'), (dict(n_q=-1), 'negative'), (dict(max_k=-1), 'negative'),
    (dict(scale=0.0), 'scale'), (dict(scale=float('nan')), 'scale'), (dict(scale=float('inf')), 'scale'),
    (dict(q=None), 'required'), (dict(dv=None), 'required'), (dict(cu_q=None), 'cu_q'), (dict(cu_k=None), 'cu_k'),
    (dict(cu_k=None, k_off=4096), 'cu_k'), (dict(q_row_stride=128), 'strides'), (dict(do_row_stride=260), 'strides'),
    (dict(k_row_stride=1 << 25), 'strides'), (dict(v=4100), 'aligned'), (dict(lse_stride=99), 'lse_stride'),
    (dict(workspace=None), 'workspace'), (dict(workspace_bytes=100), 'workspace'),
    (dict(n_q=1 << 29, lse_stride=1 << 29), '2\\^29'),
])
def test_varlen_bwd_refuses(kw, message):
    with pytest.raises(L.HipPathError, match=message):
        L.check(L.lib().or_varlen_bwd(ctypes.byref(bwd_args(**kw)), None), 'or_varlen_bwd')


def test_varlen_bwd_of_nothing_launches_nothing():
    assert L.lib().or_varlen_bwd(ctypes.byref(bwd_args(n_q=0, n_k=0, q=None, k=None)), None) == 0
    assert L.lib().or_varlen_bwd(None, None) == -1


def test_varlen_bwd_workspace_sizes():
    size = L.lib().or_varlen_bwd_workspace_size
    assert size(0, 10, 10, 10, 10, 2, 128) < 0 and size(1, 10, 10, 10, 10, 2, 80) < 0 and size(1, -1, 10, 10, 10, 2, 64) < 0
    few, many = size(1, 64, 12720, 64, 12720, 16, 128), size(8, 101760, 101760, 12720, 12720, 16, 128)
    # partial gradients of the split axis; with many tiles only the tables and two floats per query row and head
    assert few >= 64 * 16 * 128 * 4 and many < 3 * 101760 * 16 * 4


def test_python_refusals():
    x = torch.zeros(10, 2, 64, dtype=torch.bfloat16)
    cu, lse = torch.tensor([0, 10], dtype=torch.int32), torch.zeros(2, 10)
    with pytest.raises(L.HipTypeError):
        A.varlen_backward(x, x, x, x, x, lse, cu, cu, 10, 10)             # on the CPU
    with pytest.raises(L.HipValueError):
        A.varlen_backward(x, x, x, x, x, lse, cu + 1, cu, 10, 10)         # offsets that do not start at 0
    with pytest.raises(L.HipValueError):
        A.varlen_backward(x, x, x, x, x, lse, cu, cu, 9, 10)              # a segment longer than the maximum
    with pytest.raises(L.HipValueError):
        A.varlen_backward(x, x, x, x, x, lse, cu, torch.tensor([0, 5, 10], dtype=torch.int32), 10, 10)
    with pytest.raises(L.HipValueError):
        A.overlapping_ranges_backward(x, x, x, x, x, lse, [(0, 10)], [(5, 11)])
    with pytest.raises(L.HipValueError):
        A.overlapping_ranges_lse(x, x, x, [(0, 9)], [(0, 10)])


def test_gradient_rows_are_copied_only_where_they_must_be():
    x = torch.zeros(6, 2, 64, dtype=torch.bfloat16)
    assert A._rows_for(x, 2, 64) == (x, 128) and A._rows_for(x[::2], 2, 64)[1] == 256
    for odd in (x[:1].expand(6, 2, 64), x.transpose(1, 2).reshape(6, 64, 2).transpose(1, 2),
                torch.zeros(6, 64, 2, dtype=torch.bfloat16).transpose(1, 2)):
        y, stride = A._rows_for(odd, 2, 64)
        assert stride == 128 and y.is_contiguous() and (y.data_ptr() == odd.data_ptr()) == odd.is_contiguous()
    assert A._rows_for(x[:0], 2, 64)[1] == 128
    far = torch.zeros((1 << 24) + 136, dtype=torch.bfloat16).as_strided((2, 2, 64), ((1 << 24) + 8, 64, 1))
    y, stride = A._rows_for(far, 2, 64)     # rows further apart than or_varlen_bwd takes
    assert stride == 128 and y.is_contiguous() and torch.equal(y, far)
    with pytest.raises(L.HipValueError):
        A._rows_for(x, 2, 32)


# ------------------------------------------------------------------------------------------------------------------------
# RMSNorm + RoPE

def norm_bwd(**kw):
    v = dict(dq=4096, dk=4096, q=4096, k=4096, wq=4096, wk=4096, dqs=1024, dks=1024, qs=1024, ks=1024, n=10, C=1024, D=128,
             eps=1e-6, cos=4096, sin=4096, rope_row=None, n_rope=10, gq=4096, gk=4096, gwq=4096, gwk=4096, ws=4096,
             bytes=1 << 30)
    v.update(kw)
    L.check(L.lib().or_rmsnorm_rope_bwd(*v.values(), None), 'or_rmsnorm_rope_bwd')


@pytest.mark.parametrize('kw,message', [
    (dict(n=-1), 'n_rows'), (dict(C=1000), 'multiple of 512'), (dict(C=8704), 'multiple of 512'), (dict(D=96), 'dividing 512'),
    (dict(C=3584, dqs=4096, dks=4096, qs=4096, ks=4096), 'not instantiated'), (dict(n_rope=-1), 'n_rope_rows'), (dict(cos=None), 'tables'), (dict(q=None), 'required'),
    (dict(gwq=None), 'required'), (dict(wk=4096, dk=None), 'wk needs'), (dict(gwk=None), 'wk needs'), (dict(qs=1000), 'cover'),
    (dict(dks=1028), 'multiples of 8'), (dict(q=4100), 'aligned'), (dict(gwk=4100), 'aligned'), (dict(ws=None), 'workspace'),
    (dict(bytes=1000), 'workspace'),
])
def test_norm_bwd_refuses(kw, message):
    with pytest.raises(L.HipPathError, match=message):
        norm_bwd(**kw)


def test_norm_bwd_python_refusals():
    x, w = torch.zeros(4, 512, dtype=torch.bfloat16), torch.ones(512)
    with pytest.raises(L.HipTypeError):
        wan.rms_norm_backward(x, x, w, 1e-6)                                   # on the CPU
    with pytest.raises(L.HipValueError):
        wan.rms_norm_backward(x[:3], x, w, 1e-6)
    t = torch.zeros(4, 64)
    with pytest.raises(L.HipValueError):
        wan.qk_backward(x, x, x, x, w, w, 1e-6, t[:3], t[:3], 8)               # tables of 3 rows for 4 tokens
    with pytest.raises(L.HipValueError):
        wan.qk_backward(x, x[:2], x, x, w, w, 1e-6, t, t, 8)
    with pytest.raises(L.HipValueError):
        wan.qk_backward(x, x, x, x, w, w, 1e-6, t, t, 7)
    assert L.lib().or_rmsnorm_rope_bwd_workspace_size(-1, 512) < 0 and L.lib().or_rmsnorm_rope_bwd_workspace_size(4, 500) < 0


# ------------------------------------------------------------------------------------------------------------------------
# linear layers

def linear_args(**kw):
    a = L.LinearArgs()
    for f in ('x', 'weight', 'bias', 'gate', 'residual', 'y', 'preactivation', 'workspace'):
        setattr(a, f, 4096)
    a.n_rows, a.n_in, a.n_out, a.workspace_bytes = 100, 64, 128, 1 << 40
    a.x_row_stride = a.weight_row_stride = 64
    a.residual_row_stride = a.y_row_stride = 128
    for f, x in kw.items():
        setattr(a, f, x)
    return a


@pytest.mark.parametrize('kw,message', [
    (dict(n_rows=-1), 'rows'), (dict(n_in=60), 'multiples of 8'), (dict(n_out=0), 'multiples of 8'),
    (dict(n_in=(1 << 21) + 8), '2\\^21'), (dict(activation=3), 'activation'), (dict(x=None), 'required'), (dict(y=None), 'required'),
    (dict(x_row_stride=56), 'strides'), (dict(weight_row_stride=68), 'strides'), (dict(y_row_stride=1 << 22), 'strides'),
    (dict(residual_row_stride=64), 'strides'), (dict(bias=4100), 'aligned'), (dict(preactivation=4104), 'aligned'),
    (dict(workspace=None, n_in=8192, x_row_stride=8192, weight_row_stride=8192), 'workspace'),
    (dict(workspace_bytes=10, n_in=8192, x_row_stride=8192, weight_row_stride=8192), 'workspace'),
    (dict(n_rows=1 << 31), 'rows'), (dict(n_rows=1 << 30, n_in=1 << 12, x_row_stride=1 << 12, weight_row_stride=1 << 12), 'tiles'),
])
def test_linear_refuses(kw, message):
    with pytest.raises(L.HipPathError, match=message):
        L.dit_check(L.dit_lib().or_linear(ctypes.byref(linear_args(**kw)), None), 'or_linear')


def linear_bwd_args(**kw):
    a = L.LinearBwdArgs()
    for f in ('dy', 'x', 'weight', 'preactivation', 'gate', 'dx', 'dweight', 'dbias', 'dgate', 'workspace'):
        setattr(a, f, 4096)
    a.n_rows, a.n_in, a.n_out, a.workspace_bytes, a.activation = 100, 64, 128, 1 << 40, 1
    a.x_row_stride = a.weight_row_stride = 64
    a.dy_row_stride = 128
    for f, x in kw.items():
        setattr(a, f, x)
    return a


@pytest.mark.parametrize('kw,message', [
    (dict(n_rows=-1), 'rows'), (dict(n_out=100), 'multiples of 8'), (dict(activation=-1), 'activation'), (dict(dy=None), 'dy'),
    (dict(weight=None), 'dx needs'), (dict(x=None), 'dweight needs'), (dict(gate=None), 'dgate needs'),
    (dict(preactivation=None), 'pre-activation'), (dict(preactivation=None, activation=0), 'pre-activation'),
    (dict(dy_row_stride=120), 'strides'), (dict(x_row_stride=8), 'strides'), (dict(dx=4098), 'aligned'),
    (dict(workspace_bytes=10), 'workspace'), (dict(n_rows=(1 << 30) + 1), '2\\^30 rows'),
    (dict(n_rows=1 << 30, n_out=1 << 12, dy_row_stride=1 << 12), 'tiles'),
])
def test_linear_bwd_refuses(kw, message):
    with pytest.raises(L.HipPathError, match=message):
        L.dit_check(L.dit_lib().or_linear_bwd(ctypes.byref(linear_bwd_args(**kw)), None), 'or_linear_bwd')


def test_linear_of_nothing_launches_nothing():
    d = L.dit_lib()
    assert d.or_linear(ctypes.byref(linear_args(n_rows=0, x=None)), None) == 0
    assert d.or_linear(None, None) == -1 and d.or_linear_bwd(None, None) == -1
    nothing = dict(dx=None, dweight=None, dbias=None, dgate=None)
    assert d.or_linear_bwd(ctypes.byref(linear_bwd_args(**nothing)), None) == 0


def test_linear_workspace_sizes():
    d = L.dit_lib()
    assert d.or_linear_workspace_size(-1, 64, 64) < 0 and d.or_linear_workspace_size(4, 63, 64) < 0
    assert d.or_linear_bwd_workspace_size(4, 64, 4, 0) < 0
    # whole videos need no partial products forward; a long k with few tiles does, and never more than 32 of them
    assert d.or_linear_workspace_size(12720, 2048, 8192) == 0 and d.or_linear_workspace_size(1, 2048, 12288) == 0
    assert 64 * 128 * 4 < d.or_linear_workspace_size(64, 8192, 128) <= 32 * 64 * 128 * 4
    # dz in bf16 where there is an activation or a gate
    assert d.or_linear_bwd_workspace_size(12720, 2048, 8192, 1) - d.or_linear_bwd_workspace_size(12720, 2048, 8192, 0) == \
        12720 * 8192 * 2


def test_linear_python_refusals():
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    x, w = bf(10, 64), bf(128, 64)
    with pytest.raises(L.HipTypeError):
        F.linear(x, w)                                                # on the CPU
    with pytest.raises(L.HipValueError):
        F.linear(x, w, activation='relu')
    with pytest.raises(L.HipValueError):
        F.linear(x, bf(128, 72))
    with pytest.raises(L.HipValueError):
        F.linear(bf(10, 60), bf(128, 60))
    with pytest.raises(L.HipValueError):
        F.linear(x, w, residual=bf(10, 120))
    with pytest.raises(L.HipValueError):
        F.linear_backward(bf(9, 128), x, w)
    with pytest.raises(L.HipValueError):
        F.linear_backward(bf(10, 128), x, w, activation='silu')       # no pre-activation
