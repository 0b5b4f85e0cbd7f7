"""Addresses that the norms' kernels read in 16-byte pieces, refused where they are not aligned so: CPU checks at the C ABI."""
import pytest

from onereel_amd import _lib as L
from test_operators_host import AT, norm_args, refused

PARAMETERS = ['gate', 'weight', 'bias', 'scale']


@pytest.mark.parametrize('name', PARAMETERS + ['shift'])
def test_parameters_of_the_norm(name):
    refused(L.dit_lib(), 'or_block_norm', norm_args(L.BlockNormArgs, **{name: AT + 4}), None, text='aligned')


@pytest.mark.parametrize('name', PARAMETERS)
def test_parameters_of_its_gradient(name):
    # a workspace that is too small comes after what is tested: nothing is launched either way
    over = {name: AT + 4, 'dscale': AT, 'workspace': AT, 'workspace_bytes': 0}
    refused(L.dit_lib(), 'or_block_norm_bwd', norm_args(L.BlockNormBwdArgs, **over), None, text='parameters must be 16-byte aligned')


@pytest.mark.parametrize('name', ['dgate', 'dweight', 'dbias', 'dscale', 'dshift'])
def test_gradients_of_parameters(name):
    over = {name: AT + 4, 'workspace': AT, 'workspace_bytes': 0}
    refused(L.dit_lib(), 'or_block_norm_bwd', norm_args(L.BlockNormBwdArgs, **over), None, text='gradients must be 16-byte aligned')
