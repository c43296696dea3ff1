"""Refusals and host-side checks of the vocabulary operators (no GPU): every call that the documentation does not allow raises before
anything is launched."""
import ctypes

import pytest
import torch

from trajnetplusplusbaselines_amd import _lib, vocab
from trajnetplusplusbaselines_amd.lstm import TokenEmbedding, VocabularyLoss


class VocabCe(ctypes.Structure):
    """struct tnp_vocab_ce of include/trajnet_hip.h"""
    _fields_ = [('dtype', ctypes.c_int32), ('reduction', ctypes.c_int32), ('M', ctypes.c_int64), ('V', ctypes.c_int32),
                ('D', ctypes.c_int32), ('hidden', ctypes.c_void_p), ('ld_hidden', ctypes.c_int64), ('weight', ctypes.c_void_p),
                ('ld_weight', ctypes.c_int64), ('bias', ctypes.c_void_p), ('target', ctypes.c_void_p), ('saved', ctypes.c_void_p)]


def test_host_tensors_are_refused():
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        vocab.token_embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8))
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        vocab.vocab_cross_entropy(torch.zeros(3, 8), torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        TokenEmbedding(4, 8)(torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        VocabularyLoss(8, 4)(torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64))


@pytest.mark.parametrize('tokens,weight,error', [
    (torch.zeros(3), torch.zeros(4, 8), TypeError), (torch.zeros(3, dtype=torch.int16), torch.zeros(4, 8), TypeError),
    ([0, 1], torch.zeros(4, 8), TypeError), (torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8, dtype=torch.float64), TypeError),
    (torch.zeros(3, dtype=torch.int64), torch.zeros(4), ValueError), (torch.zeros(3, dtype=torch.int64), torch.zeros(0, 8), ValueError)])
def test_embedding_arguments(tokens, weight, error):
    with pytest.raises(error):
        vocab.token_embedding(tokens, weight)


def _ce(**kw):
    a = dict(hidden=torch.zeros(3, 8), weight=torch.zeros(4, 8), target=torch.zeros(3, dtype=torch.int64), bias=torch.zeros(4))
    a.update(kw)
    return vocab.vocab_cross_entropy(**a)


@pytest.mark.parametrize('kw,error', [
    (dict(reduction='max'), ValueError), (dict(hidden=torch.zeros(3, 7)), ValueError), (dict(hidden=torch.zeros(2, 8)), ValueError),
    (dict(target=torch.zeros(3)), TypeError), (dict(bias=torch.zeros(5)), ValueError), (dict(bias=torch.zeros(4).half()), TypeError),
    (dict(hidden=torch.zeros(3, 8).half()), TypeError), (dict(weight=torch.zeros(4, 8).double()), TypeError),
    (dict(weight=torch.zeros(0, 8)), ValueError), (dict(target=[0, 1, 2]), TypeError), (dict(target=torch.zeros(3, 1, dtype=torch.int64)), ValueError)])
def test_cross_entropy_arguments(kw, error):
    with pytest.raises(error):
        _ce(**kw)


def test_registered_backward_operators_refuse():
    """called by hand with tensors that do not belong together"""
    from trajnetplusplusbaselines_amd import ops  # noqa: F401
    i = lambda *s: torch.zeros(*s, dtype=torch.int64)
    emb = torch.ops.trajnet.token_embedding_backward
    for grad, tok, v, error in ((torch.zeros(3, 8), i(4), 5, ValueError), (torch.zeros(3, 8), i(3), 0, ValueError),
                                (torch.zeros(3, 8), torch.zeros(3), 5, TypeError), (torch.zeros(3, 8).double(), i(3), 5, TypeError),
                                (torch.zeros(3, 8), i(3), 5, RuntimeError)):
        with pytest.raises(error):
            emb(grad, tok, v, 1.0)
    ce = torch.ops.trajnet.vocab_cross_entropy_backward
    x, w, t, b = torch.zeros(3, 8), torch.zeros(4, 8), i(3), torch.zeros(4)
    saved = torch.zeros(vocab.saved_bytes(3, 4, 8, torch.float32), dtype=torch.uint8)
    for args, error in (((torch.zeros(3), x, w, t, b, saved, 'mean'), ValueError), ((torch.zeros(()), x, w, t, b, saved, 'none'), ValueError),
                        ((torch.zeros(()), x, w, t, b, saved[1:], 'mean'), ValueError), ((torch.zeros(()), x, w, t, b, saved.char(), 'mean'), ValueError),
                        ((torch.zeros(()), x, w, i(2), b, saved, 'sum'), ValueError), ((torch.zeros(()), x, w, t, b[:3], saved, 'sum'), ValueError),
                        ((torch.zeros(()), x, w, t, b, saved, 'mean'), RuntimeError)):
        with pytest.raises(error):
            ce(*args)


def test_c_entries_refuse_on_the_host():
    L = _lib.lib()
    p = ctypes.c_void_p(1 << 20)        # never followed: every call below is refused first
    fwd = lambda **k: L.tnp_token_embedding_forward(*[k.get(n, d) for n, d in (
        ('tokens', p), ('token_bytes', 8), ('N', 4), ('weight', p), ('ldw', 8), ('V', 4), ('D', 8), ('dtype', 0), ('scale', 1.0), ('out', p),
        ('ldo', 8), ('stream', None))])
    for bad in (dict(token_bytes=2), dict(N=-1), dict(N=1 << 40), dict(V=0), dict(D=0), dict(dtype=7), dict(ldw=7), dict(ldo=1), dict(tokens=None)):
        assert fwd(**bad) == -1
        assert b'tnp_token_embedding_forward' in L.tnp_last_error()
    assert fwd(N=0, tokens=None) == 0
    assert L.tnp_token_embedding_backward_workspace_bytes(100, 50, 8) == 0          # few tokens are not sorted
    need = L.tnp_token_embedding_backward_workspace_bytes(10000, 50, 8)
    assert need > 0
    args = [p, 8, 10000, p, 8, 50, 8, 0, 1.0, p, 8, p, need - 1, None]
    assert L.tnp_token_embedding_backward(*args) == -1 and b'workspace' in L.tnp_last_error()
    a = VocabCe(dtype=0, reduction=1, M=10, V=20, D=8, hidden=1 << 20, ld_hidden=8, weight=1 << 20, ld_weight=8, target=1 << 20)
    ref = ctypes.byref(a)
    assert L.tnp_vocab_ce_saved_bytes(ref) > 0
    need = L.tnp_vocab_ce_workspace_bytes(ref, 0)
    assert L.tnp_vocab_ce_forward(ref, p, p, need - 1, None) == -1 and b'workspace' in L.tnp_last_error()
    assert L.tnp_vocab_ce_backward(ref, p, p, p, None, p, 1 << 40, None) == -1          # nothing saved
    a.saved = 1 << 20
    assert L.tnp_vocab_ce_backward(ref, p, p, p, p, p, 1 << 40, None) == -1 and b'bias' in L.tnp_last_error()
    for field, value in (('dtype', 3), ('reduction', 3), ('V', 0), ('D', 0), ('D', 20000), ('M', -1), ('ld_hidden', 7), ('ld_weight', 7)):
        b = VocabCe.from_buffer_copy(a)
        setattr(b, field, value)
        assert L.tnp_vocab_ce_saved_bytes(ctypes.byref(b)) == 0
        assert L.tnp_vocab_ce_workspace_bytes(ctypes.byref(b), 1) == 0
        assert L.tnp_vocab_ce_forward(ctypes.byref(b), p, p, 1 << 40, None) == -1
    a.M = 0
    assert L.tnp_vocab_ce_forward(ref, p, p, 1 << 40, None) == -1


def test_struct_mirror():
    assert _lib.lib().tnp_abi_sizeof(8) == ctypes.sizeof(VocabCe)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_saved_bytes_from_the_sizes(dtype):
    for m, v, d in ((1, 1, 1), (256, 256, 16), (257, 300, 33), (5000, 70000, 200)):
        a = VocabCe(dtype=(torch.float32, torch.bfloat16, torch.float16).index(dtype), M=m, V=v, D=d, ld_hidden=d, ld_weight=d)
        assert _lib.lib().tnp_vocab_ce_saved_bytes(ctypes.byref(a)) == vocab.saved_bytes(m, v, d, dtype)


def test_fake_implementations():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from trajnetplusplusbaselines_amd import ops  # noqa: F401
    with FakeTensorMode():
        w = torch.empty(30, 8, dtype=torch.bfloat16)
        tok = torch.empty(5, 7, dtype=torch.int64)
        out = torch.ops.trajnet.token_embedding(tok, w, 2.0)
        assert out.shape == (5, 7, 8) and out.dtype == torch.bfloat16
        loss, saved = torch.ops.trajnet.vocab_cross_entropy(out, w, tok, None, 'mean')
        assert loss.shape == () and loss.dtype == torch.float32 and saved.dtype == torch.uint8
        assert torch.ops.trajnet.vocab_cross_entropy(out, w, tok, torch.empty(30, dtype=torch.bfloat16), 'none')[0].shape == (5, 7)


def test_the_plans_that_the_gpu_tests_are_written_for():
    """a threshold that moves a case to other kernels shows here"""
    from tests.vocab_formula import LARGE, plan
    for m, v, d, dtype, pieces in LARGE:
        assert plan(m, v, d, dtype) == (256, 256, pieces)
    assert plan(300, 700, 65, torch.float32) == (128, 128, 1)
    assert plan(64, 700, 65, torch.float32, train=False)[0] == 0 and plan(65, 700, 65, torch.float32, train=False)[0] == 128
    assert plan(4000, 8200, 72, torch.bfloat16) == (128, 128, 1)
    assert plan(20000, 34000, 40, torch.bfloat16)[2] == 2
    assert plan(0, 0, 0, torch.float32) == (-1, -1, -1)


@pytest.mark.parametrize('entries', [32, 36, 42, 58])
def test_one_rounded_log_sum_exp_is_out_of_the_bounds_of_large_logits(entries):
    """the check of the normaliser's precision on the GPU tells the two forms apart: exp(l - top) / sum, formed here in fp32, is inside
    its bounds, exp(l - lse) with lse rounded to fp32 is not"""
    from tests.test_gpu_vocab_range import offset_case
    from tests.vocab_formula import formula
    x, w, b, t, shift = offset_case(1e4, entries, 'cpu')
    _, _, want, bounds = formula(x, w, b.detach().double() - shift, t, torch.ones(20), extra=2.0 ** -19)
    l = (b.detach() * torch.tensor(1.4426950408889634, dtype=torch.float32)).expand(20, entries)
    top = l.max(1, keepdim=True).values
    e = torch.exp2(l - top)
    total = e.sum(1, keepdim=True)
    for p, inside in ((e / total, True), (torch.exp2(l - (top + torch.log2(total))), False)):
        G = p.double().scatter_add(1, t[:, None], torch.full((20, 1), -1.0, dtype=torch.float64))
        got = (G @ w.detach().double(), G.t() @ x.detach().double(), G.sum(0))
        off = [float(((a - c).abs() / lim).max()) for a, c, lim in zip(got, want, bounds)]
        assert (max(off) < 1.0) == inside and (inside or min(off) > 1.0), off


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_what_is_held_of_the_logits_at_a_time(dtype):
    """a piece of the vocabulary: 1 GB, or 256 entries of all rows where that is more"""
    from tests.vocab_formula import plan
    each = 2 if dtype == torch.bfloat16 else 4
    for m, v in ((1, 1 << 23), (300, 70000), (16384, 65536), (100001, 50021), (1 << 20, 3000), (1 << 23, 5), (1 << 23, 1000)):
        up = lambda n: (n + 255) // 256 * 256
        pieces = plan(m, v, 64, dtype)[2]
        piece = up(-(-up(v) // pieces))
        assert up(m) * piece * each <= max(1 << 30, up(m) * 256 * each)
        assert (pieces - 1) * piece < up(v) <= pieces * piece
