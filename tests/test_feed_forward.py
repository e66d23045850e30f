"""The root-mean-square norm and the gated feed-forward block against float64 forms with derived bounds: on the GPU, and (small cases) on the CPU
stand-in build of the same kernel sources."""
import os

import pytest
import torch

import feed_forward_cases as cases
from feed_forward_cases import BF16, F16, F32

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope='module')
def emu():
    import sys
    sys.path.insert(0, HERE)
    from host_harness import standin
    from nerfool_amd import _lib
    if not os.path.exists(standin.CLANG):
        pytest.skip('no clang++ for the CPU stand-in build')
    keep = _lib._lib, _lib._emulated
    standin.install_emulated(build=True)
    yield 'cpu'
    _lib._lib, _lib._emulated = keep


NORM_SMALL = [(1, 1, F32), (1, 64, BF16), (5, 37, F32), (3, 129, F16), (9, 8, BF16), (2, 515, F32), (1, 2049, F16), (70, 20, F32)]
NORM_GPU = NORM_SMALL + [(1, 4096, BF16), (513, 64, F32), (2050, 520, BF16), (2100, 1023, F32), (2049, 4097, F16), (3, 8200, F32), (4, 16385, BF16),
                         (2, 40000, F32), (40, 70001, BF16), (32768, 64, F32), (4099, 1001, BF16)]
GATED_SMALL = [(1, 8, 8, F32), (3, 16, 24, BF16), (5, 33, 17, F16), (130, 40, 72, BF16), (2, 65, 130, F32), (17, 7, 5, BF16)]
GATED_GPU = GATED_SMALL + [(1, 1, 1, F32), (1, 256, 512, BF16), (7, 512, 300, F16), (40, 257, 129, BF16), (64, 64, 256, F32), (65, 1000, 520, F32),
                           (300, 264, 1032, BF16), (1025, 520, 260, F16), (513, 129, 65, F32), (129, 2048, 1000, BF16)]


@pytest.mark.parametrize('rows,dim,dtype', NORM_SMALL)
def test_norm_standin(emu, rows, dim, dtype):
    cases.check_norm(rows, dim, dtype, emu)


@pytest.mark.parametrize('rows,dim,hidden,dtype', GATED_SMALL)
def test_gated_standin(emu, rows, dim, hidden, dtype):
    cases.check_gated(rows, dim, hidden, dtype, emu, act=('silu', 'gelu', 'relu')[rows % 3])


@pytest.mark.gpu
@pytest.mark.parametrize('rows,dim,dtype', NORM_GPU)
def test_norm(rows, dim, dtype):
    cases.check_norm(rows, dim, dtype, 'cuda')


@pytest.mark.gpu
@pytest.mark.parametrize('residual,weight,use', [(False, True, ('y',)), (True, False, ('y', 'h')), (False, False, ('y',)), (True, True, ('y',))])
def test_norm_optional_inputs(residual, weight, use):
    cases.check_norm(37, 200, BF16, 'cuda', residual=residual, weight=weight, use=use)
    cases.check_norm(37, 8200, F32, 'cuda', residual=residual, weight=weight, use=use)


@pytest.mark.gpu
@pytest.mark.parametrize('act', ['silu', 'gelu', 'relu'])
@pytest.mark.parametrize('rows,dim,hidden,dtype', GATED_GPU)
def test_gated(rows, dim, hidden, dtype, act):
    cases.check_gated(rows, dim, hidden, dtype, 'cuda', act=act)


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_gated_large_tiles(dtype):
    """enough tiles for the largest tile form, with a ragged last tile each way"""
    cases.check_gated(2560 + 9, 1160, 2568, dtype, 'cuda', act='silu')


NORM_8BIT_SMALL = [(1, 32, BF16), (5, 37, F32), (3, 129, F16), (70, 20, F32), (1, 2049, BF16)]
GATED_8BIT_SMALL = [(1, 32, 32), (3, 64, 96), (33, 160, 32), (5, 96, 288)]


@pytest.mark.parametrize('rows,dim,dtype', NORM_8BIT_SMALL)
def test_norm_8bit_standin(emu, rows, dim, dtype):
    cases.check_norm_8bit(rows, dim, dtype, emu)
    cases.check_quantize(rows, dim, dtype, emu)


@pytest.mark.parametrize('rows,dim,hidden', GATED_8BIT_SMALL)
def test_gated_8bit_standin(emu, rows, dim, hidden):
    cases.check_gated_8bit(rows, dim, hidden, emu, act=('silu', 'gelu', 'relu')[rows % 3])


@pytest.mark.gpu
@pytest.mark.parametrize('rows,dim,dtype', NORM_8BIT_SMALL + [(16, 5120, BF16), (2100, 1023, F32), (2049, 4097, F16), (2, 40000, F32), (513, 64, F32)])
def test_norm_8bit(rows, dim, dtype):
    cases.check_norm_8bit(rows, dim, dtype, 'cuda')
    cases.check_norm_8bit(rows, dim, dtype, 'cuda', residual=False)
    cases.check_quantize(rows, dim, dtype, 'cuda')


@pytest.mark.gpu
@pytest.mark.parametrize('act,dtype', [('silu', BF16), ('gelu', F32), ('relu', F16)])
@pytest.mark.parametrize('rows,dim,hidden', GATED_8BIT_SMALL + [(1, 4096, 1024), (16, 256, 512), (129, 1056, 544), (700, 320, 2080), (2569, 1184, 2592)])
def test_gated_8bit(rows, dim, hidden, act, dtype):
    cases.check_gated_8bit(rows, dim, hidden, 'cuda', act=act, dtype=dtype)
