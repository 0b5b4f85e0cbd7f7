"""CPU checks of the gradient entry points: their argument structures match the header, and they refuse bad arguments before
any launch."""
import ctypes
import subprocess

import pytest
import torch

from conftest import ROOT
from onereel_amd import _lib as L
from onereel_amd import attention as A


def test_struct_matches_the_header(tmp_path):
    cls, name = L.VarlenBwdArgs, 'or_varlen_bwd_args'
    lines = ['#include <stddef.h>', '#include <stdio.h>', f'#include "{ROOT / "include" / "onereel_hip.h"}"',
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
    with pytest.raises(L.HipValueError):
        A._rows_for(x, 2, 32)
