"""Motions as tokens: the two operators that a model over a vocabulary of displacements or grid cells needs beside the ones for
continuous positions, on the kernels of csrc/token_embed.hip and csrc/vocab_ce.hip.

    token_embedding(tokens, weight, scale)               scale * weight[tokens]           (module: lstm.TokenEmbedding)
    vocab_cross_entropy(hidden, weight, target, bias)    cross entropy of the output layer hidden @ weight.T + bias against
                                                         ``target``, the logits never stored  (module: lstm.VocabularyLoss)

Both are differentiable, run on the current stream of the tensors' device without a host synchronisation, take fp32, bf16 and fp16
and refuse host tensors.  A negative token or target is an absent track (zero row, no loss, no gradient); one past the end of the
vocabulary gives NaN, since the host does not look at device data.
"""
import ctypes

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_REDUCTIONS = {'none': 0, 'mean': 1, 'sum': 2}


_current = torch._C._cuda_getDevice


class _On(object):
    """The device's own context where it is not the current one (the native calls take the CURRENT device's stream)."""
    __slots__ = ('ctx',)

    def __init__(self, device):
        self.ctx = None if device.index is None or device.index == _current() else torch.cuda.device(device)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *exc):
        if self.ctx is not None:
            self.ctx.__exit__(*exc)


def _rows(t):
    """(t, elements per row) with unit column stride and rows that do not overlap; a copy only where the layout asks for one.  t of
    more than two dimensions has to be, or is made, contiguous."""
    d = t.shape[-1]
    if t.is_contiguous():
        return t, d
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= d:
        return t, t.stride(0)
    return t.contiguous(), d


def _check_table(weight, what):
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError('%s must be [entries, columns] (got %s)' % (what, tuple(weight.shape)))
    if weight.dtype not in _DTYPES:
        raise TypeError('%s must be float32, bfloat16 or float16 (got %s)' % (what, weight.dtype))


# ---- token embedding ---------------------------------------------------------------------------------------------------------
def _embedding_forward(tokens, weight, scale):
    w, ld = _rows(weight)
    tok = tokens if tokens.is_contiguous() else tokens.contiguous()
    v, d = w.shape
    dev = w.device
    with _On(dev):
        out = torch.empty(tokens.shape + (d,), dtype=w.dtype, device=dev)
        _lib.check(_lib.lib().tnp_token_embedding_forward(
            tok.data_ptr(), 8 if tok.dtype == torch.int64 else 4, tok.numel(), w.data_ptr(), ld, v, d, _DTYPES[w.dtype], scale,
            out.data_ptr(), d, _lib.raw_stream()), 'tnp_token_embedding_forward')
    return out


def _embedding_backward(grad, tokens, vocab, scale):
    g, ld = _rows(grad)
    tok = tokens if tokens.is_contiguous() else tokens.contiguous()
    n, d, dev = tok.numel(), g.shape[-1], g.device
    L = _lib.lib()
    with _On(dev):
        dw = torch.empty((vocab, d), dtype=g.dtype, device=dev)
        need = L.tnp_token_embedding_backward_workspace_bytes(n, vocab, d)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        _lib.check(L.tnp_token_embedding_backward(
            tok.data_ptr(), 8 if tok.dtype == torch.int64 else 4, n, g.data_ptr(), ld, vocab, d, _DTYPES[g.dtype], scale, dw.data_ptr(),
            d, None if ws is None else ws.data_ptr(), need, _lib.raw_stream()), 'tnp_token_embedding_backward')
    return dw


class _TokenEmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale):
        ctx.save_for_backward(tokens)
        ctx.args = (weight.shape[0], scale)
        return _embedding_forward(tokens, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        return None, _embedding_backward(grad, ctx.saved_tensors[0], *ctx.args), None


def check_embedding(tokens, weight, scale):
    if not isinstance(tokens, torch.Tensor) or not isinstance(weight, torch.Tensor):
        raise TypeError('token_embedding: tokens and weight are tensors')
    if tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError('token_embedding: tokens must be int64 or int32 (got %s)' % tokens.dtype)
    _check_table(weight, 'token_embedding: weight')
    _lib.require_device(weight, 'token_embedding: weight')
    if tokens.device != weight.device:
        raise RuntimeError('token_embedding: tokens on %s, weight on %s' % (tokens.device, weight.device))
    return float(scale)


def check_embedding_backward(grad, tokens, entries):
    if grad.dtype not in _DTYPES or tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError('token_embedding_backward: gradient of %s for tokens of %s' % (grad.dtype, tokens.dtype))
    if grad.dim() < 1 or grad.shape[:-1] != tokens.shape or grad.shape[-1] < 1 or entries < 1:
        raise ValueError('token_embedding_backward: gradient %s, tokens %s, %d entries' % (tuple(grad.shape), tuple(tokens.shape), entries))
    _lib.require_device(grad, 'token_embedding_backward: grad')
    if tokens.device != grad.device:
        raise RuntimeError('token_embedding_backward: tokens on %s, gradient on %s' % (tokens.device, grad.device))


def token_embedding(tokens, weight, scale=1.0):
    """``scale * weight[tokens]``: tokens int64 / int32 of any shape, weight [V, D] -> tokens.shape + (D,) in weight's dtype, rounded
    once.  tokens < 0 (absent track): a row of zeros; tokens >= V: a row of NaN.  The gradient of ``weight`` is dense, summed in fp32
    in a fixed order (two calls give the same bits)."""
    if torch.compiler.is_compiling():
        from . import ops  # noqa: F401  (registers the operators)
        return torch.ops.trajnet.token_embedding(tokens, weight, float(scale))
    scale = check_embedding(tokens, weight, scale)
    if weight.requires_grad and torch.is_grad_enabled():
        return _TokenEmbeddingFn.apply(tokens, weight, scale)
    return _embedding_forward(tokens, weight, scale)


# ---- cross entropy over a vocabulary -----------------------------------------------------------------------------------------
class VocabCe(ctypes.Structure):
    """mirror of ``struct tnp_vocab_ce`` (include/trajnet_hip.h)"""
    _fields_ = [('dtype', ctypes.c_int32), ('reduction', ctypes.c_int32), ('M', ctypes.c_int64), ('V', ctypes.c_int32),
                ('D', ctypes.c_int32), ('hidden', ctypes.c_void_p), ('ld_hidden', ctypes.c_int64), ('weight', ctypes.c_void_p),
                ('ld_weight', ctypes.c_int64), ('bias', ctypes.c_void_p), ('target', ctypes.c_void_p), ('saved', ctypes.c_void_p)]


def saved_bytes(rows, entries, columns, dtype):
    """tnp_vocab_ce_saved_bytes() from the sizes alone (they may be symbolic while a graph is traced)"""
    panels = (columns + 15) // 16 if dtype == torch.float32 else (columns + 31) // 32
    up = lambda n: (n + 255) // 256 * 256
    return 256 + 16 * up(rows) + 64 * panels * (up(rows) + up(entries))


def _ce_args(hidden, weight, bias, target, reduction, saved):
    """(struct, the tensors in kernel layout that it points to)"""
    x, ldx = _rows(hidden)
    w, ldw = _rows(weight)
    t = target if target.dtype == torch.int64 and target.is_contiguous() else target.to(torch.int64).contiguous()
    b = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    v, d = w.shape
    return VocabCe(_DTYPES[w.dtype], reduction, t.numel(), v, d, x.data_ptr(), ldx, w.data_ptr(), ldw, None if b is None else b.data_ptr(),
                   t.data_ptr(), None if saved is None else saved.data_ptr()), (x, w, t, b)


def _ce_forward(hidden, weight, bias, target, reduction, train):
    """(loss, what the backward pass reads or None); at least one row"""
    dev = weight.device
    L = _lib.lib()
    with _On(dev):
        a, held = _ce_args(hidden, weight, bias, target, reduction, None)
        ref = ctypes.byref(a)
        saved = None
        if train:
            saved = torch.empty(L.tnp_vocab_ce_saved_bytes(ref), dtype=torch.uint8, device=dev)
            a.saved = saved.data_ptr()
        need = L.tnp_vocab_ce_workspace_bytes(ref, 0)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        loss = torch.empty(target.shape if reduction == 0 else (), dtype=torch.float32, device=dev)
        _lib.check(L.tnp_vocab_ce_forward(ref, loss.data_ptr(), ws.data_ptr(), need, _lib.raw_stream()), 'tnp_vocab_ce_forward')
    return loss, saved


def _ce_backward(grad, hidden, weight, bias, target, saved, reduction, needs):
    dev = weight.device
    L = _lib.lib()
    with _On(dev):
        a, held = _ce_args(hidden, weight, bias, target, reduction, saved)
        ref = ctypes.byref(a)
        g = grad if grad.dtype == torch.float32 and grad.is_contiguous() else grad.float().contiguous()
        dx = torch.empty(hidden.shape, dtype=hidden.dtype, device=dev) if needs[0] else None
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=dev) if needs[1] else None
        db = torch.empty(bias.shape, dtype=bias.dtype, device=dev) if needs[2] else None
        need = L.tnp_vocab_ce_workspace_bytes(ref, 1)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        _lib.check(L.tnp_vocab_ce_backward(ref, g.data_ptr(), _lib.ptr(dx), _lib.ptr(dw), _lib.ptr(db), ws.data_ptr(), need,
                                           _lib.raw_stream()), 'tnp_vocab_ce_backward')
    return dx, dw, db


class _VocabCeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, target, reduction):
        loss, saved = _ce_forward(hidden, weight, bias, target, reduction, True)
        ctx.save_for_backward(hidden, weight, bias, target, saved)
        ctx.reduction = reduction
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        hidden, weight, bias, target, saved = ctx.saved_tensors
        return _ce_backward(grad, hidden, weight, bias, target, saved, ctx.reduction, ctx.needs_input_grad) + (None, None)


def check_cross_entropy(hidden, weight, target, bias, reduction):
    if reduction not in _REDUCTIONS:
        raise ValueError("vocab_cross_entropy: reduction must be 'none', 'mean' or 'sum' (got %r)" % (reduction,))
    for name, t in (('hidden', hidden), ('weight', weight), ('target', target)):
        if not isinstance(t, torch.Tensor):
            raise TypeError('vocab_cross_entropy: %s must be a tensor' % name)
    _check_table(weight, 'vocab_cross_entropy: weight')
    if hidden.dtype != weight.dtype or (bias is not None and bias.dtype != weight.dtype):
        raise TypeError('vocab_cross_entropy: hidden, weight and bias must have one dtype')
    if target.dtype not in (torch.int64, torch.int32):
        raise TypeError('vocab_cross_entropy: target must be int64 or int32 (got %s)' % target.dtype)
    if hidden.dim() < 1 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError('vocab_cross_entropy: hidden %s does not fit weight %s' % (tuple(hidden.shape), tuple(weight.shape)))
    if hidden.shape[:-1] != target.shape:
        raise ValueError('vocab_cross_entropy: hidden %s does not fit target %s' % (tuple(hidden.shape), tuple(target.shape)))
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError('vocab_cross_entropy: bias %s does not fit weight %s' % (tuple(bias.shape), tuple(weight.shape)))
    _lib.require_device(weight, 'vocab_cross_entropy: weight')
    for name, t in (('hidden', hidden), ('target', target), ('bias', bias)):
        if t is not None and t.device != weight.device:
            raise RuntimeError('vocab_cross_entropy: %s on %s, weight on %s' % (name, t.device, weight.device))


def check_cross_entropy_backward(grad, hidden, weight, target, bias, saved, reduction):
    if grad.shape != (target.shape if reduction == 'none' else ()):
        raise ValueError('vocab_cross_entropy_backward: gradient %s of a loss with reduction %r, target %s'
                         % (tuple(grad.shape), reduction, tuple(target.shape)))
    if saved.dtype != torch.uint8 or saved.numel() != saved_bytes(target.numel(), weight.shape[0], weight.shape[-1], weight.dtype) \
            or not saved.is_contiguous():
        raise ValueError('vocab_cross_entropy_backward: saved is not the second output of this vocab_cross_entropy')
    check_cross_entropy(hidden, weight, target, bias, reduction)
    for name, t in (('grad', grad), ('saved', saved)):
        if t.device != weight.device:
            raise RuntimeError('vocab_cross_entropy_backward: %s on %s, weight on %s' % (name, t.device, weight.device))


def vocab_cross_entropy(hidden, weight, target, bias=None, reduction='mean'):
    """Cross entropy of ``softmax(hidden @ weight.T + bias)`` against ``target``, without storing the logits.

    hidden [..., D], weight [V, D], bias [V] (may hold -inf: masked entries) of one dtype, target [...] int64 / int32.  Returns fp32:
    a scalar ('mean' over the rows that are there, 0 if there are none; 'sum') or target's shape ('none').  target < 0: an absent
    row -- its hidden state is not read, its loss and gradient are 0; target >= V: NaN.  Differentiable in hidden, weight and bias.

    fp32 operands are multiplied as two fp16 numbers each, scaled by the largest finite element of their tensor: an element below
    2^-16 of that one loses relative precision (2^-40 of the largest remains), a row of valid targets that holds an infinity gives
    NaN."""
    if torch.compiler.is_compiling():
        from . import ops  # noqa: F401  (registers the operators)
        return torch.ops.trajnet.vocab_cross_entropy(hidden, weight, target, bias, reduction)[0]
    check_cross_entropy(hidden, weight, target, bias, reduction)
    red = _REDUCTIONS[reduction]
    if target.numel() == 0:                                              # no rows: an empty / zero loss with zero gradients
        zero = hidden.float().sum() + weight[:0].float().sum() + (bias[:0].float().sum() if bias is not None else 0.0)
        return zero.expand(target.shape) if red == 0 else zero
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)):
        return _VocabCeFn.apply(hidden, weight, bias, target, red)
    return _ce_forward(hidden, weight, bias, target, red, False)[0]
