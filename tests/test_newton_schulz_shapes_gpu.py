"""newton_schulz where its forms meet: one-launch matrices with slices of more
than 128 columns, the longest that it takes, the first ones of the general
kernels. Tolerance as in test_training_ops_gpu (one rounding to bf16 and up to
1.5e-3 of the fp16 products: 4e-3)."""

import ctypes

import pytest
import torch

from llattn_b200 import _lib, newton_schulz
from test_training_ops_gpu import BF, FP, plain_ns, rel, spectrum

pytestmark = pytest.mark.gpu


def workspace(m, n, dtype):
    ptrs = (ctypes.c_void_p * 1)(1 << 20)
    a = _lib.OrthArgs(m, n, 1, 5, _lib.BF16 if dtype == BF else _lib.F32, 3.4, -4.7, 2.0, 1e-7, ptrs, 1 << 21, None, 0)
    return _lib.lib().llattn_orth_workspace_bytes(ctypes.byref(a))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("m,n", [(64, 2049), (64, 5000), (5000, 33), (3, 7001), (64, 11520), (11520, 61)])
def test_wide_slices(m, n, dtype):
    assert workspace(m, n, dtype) == 256  # one launch
    gs = [spectrum(m, n, d, dtype, i) for i, d in enumerate((0.0, 0.7))]
    for g, o in zip(gs, newton_schulz(gs)):
        assert rel(o, plain_ns(g)) <= 4e-3


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("m,n", [(64, 11700), (17000, 64), (65, 64), (65, 66)])
def test_past_one_launch(m, n, dtype):
    gs = [spectrum(m, n, d, dtype, i) for i, d in enumerate((0.0, 0.7))]
    for g, o in zip(gs, newton_schulz(gs)):
        assert rel(o, plain_ns(g)) <= 4e-3


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("m,n", [(1, 200000), (16, 100000), (300000, 5), (70, 150000)])
def test_long_sums(m, n, dtype):
    """Gram sums over hundreds of thousands of products: what the tensor cores'
    additions drop does not grow with the length."""
    gs = [spectrum(m, n, d, dtype, i) for i, d in enumerate((0.0, 0.7))]
    for g, o in zip(gs, newton_schulz(gs)):
        assert rel(o, plain_ns(g)) <= 4e-3
