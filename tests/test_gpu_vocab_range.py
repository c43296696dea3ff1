"""Vocabulary cross entropy on the GPU: precision and range, row by row and entry by entry, against the formulas in 64 bits
(tests/vocab_formula.py says what the bounds count)."""
import pytest
import torch

from tests.test_gpu_vocab import _case, _gen, _within
from tests.vocab_formula import formula
from trajnetplusplusbaselines_amd import vocab

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _check(x, w, b, t, up=None, extra=0.0):
    """losses and gradients of reduction 'none' within the bounds; returns them"""
    up = torch.ones(t.shape[0], device='cuda') if up is None else up
    loss, bound, want, bounds = formula(x, w, b, t, up, extra)
    out = vocab.vocab_cross_entropy(x, w, t, bias=b, reduction='none')
    _within(out.detach(), loss, bound)
    leaves = (x, w) if b is None else (x, w, b)
    got = torch.autograd.grad(out, leaves, up)
    for a, e, lim in zip(got, want, bounds):
        assert a.dtype == x.dtype
        _within(a, e, lim)
    return got


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('m,v,d', [(1, 9, 8), (300, 70, 24), (260, 513, 65), (700, 40, 200), (513, 1000, 130)])
def test_gradients_are_rounded_once(dtype, m, v, d):
    """G does not add a rounding of the gradients' own size (fp16: it is held in two numbers)"""
    _check(*_case(m, v, d, dtype, m + 3 * v + d, absent=0.2 if m > 4 else 0.0))
