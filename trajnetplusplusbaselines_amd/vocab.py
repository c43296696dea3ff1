"""Motions as tokens: the two operators that a model over a vocabulary of displacements or grid cells needs beside the ones for
continuous positions, on the kernels of csrc/token_embed.hip and csrc/vocab_ce.hip.

    token_embedding(tokens, weight, scale)               scale * weight[tokens]           (module: lstm.TokenEmbedding)
    vocab_cross_entropy(hidden, weight, target, bias)    cross entropy of the output layer hidden @ weight.T + bias against
                                                         ``target``, the logits never stored  (module: lstm.VocabularyLoss)

Both are differentiable, run on the current stream of the tensors' device without a host synchronisation, take fp32, bf16 and fp16
and refuse host tensors.  A negative token or target is an absent track (zero row, no loss, no gradient); one past the end of the
vocabulary gives NaN, since the host does not look at device data.
"""
import contextlib
import ctypes

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_REDUCTIONS = {'none': 0, 'mean': 1, 'sum': 2}


def _on(device):
    """The device's own context when it is not the current one (the native calls take the CURRENT device's stream)."""
    if device.index is None or device.index == torch._C._cuda_getDevice():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _rows(t):
    """[n, D] with unit column stride; a copy only where the layout asks for one"""
    if t.stride(-1) == 1 or t.shape[-1] == 1:
        if t.dim() == 2:
            if t.shape[0] <= 1 or t.stride(0) >= t.shape[1]:
                return t if t.stride(-1) == 1 else t.contiguous()
        elif t.is_contiguous():
            return t.reshape(-1, t.shape[-1])
    return t.contiguous().reshape(-1, t.shape[-1])


def _ld(t):
    """elements per row (a single row's stride is whatever torch left there)"""
    return max(t.stride(0), t.shape[1]) if t.shape[0] > 1 else t.shape[1]


def _workspace(nbytes, device):
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)


def _check_table(weight, what):
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError('%s must be [entries, columns] (got %s)' % (what, tuple(weight.shape)))
    if weight.dtype not in _DTYPES:
        raise TypeError('%s must be float32, bfloat16 or float16 (got %s)' % (what, weight.dtype))


# ---- token embedding ---------------------------------------------------------------------------------------------------------
def _embedding_forward(tokens, weight, scale):
    w = _rows(weight)
    tok = tokens.reshape(-1)                                   # a view where it can be
    if not tok.is_contiguous():
        tok = tok.contiguous()
    n, d = tok.shape[0], w.shape[1]
    out = torch.empty(tokens.shape + (d,), dtype=w.dtype, device=w.device)
    with _on(w.device):
        _lib.check(_lib.lib().tnp_token_embedding_forward(
            tok.data_ptr(), tok.element_size(), n, w.data_ptr(), _ld(w), w.shape[0], d, _DTYPES[w.dtype], scale, out.data_ptr(), d,
            _lib.raw_stream()), 'tnp_token_embedding_forward')
    return out


def _embedding_backward(grad, tokens, vocab, scale):
    d = grad.shape[-1]
    tok = tokens.reshape(-1).contiguous()
    g = _rows(grad) if grad.numel() else grad.reshape(0, d)
    n = tok.shape[0]
    dw = torch.empty(vocab, d, dtype=grad.dtype, device=grad.device)
    L = _lib.lib()
    with _on(grad.device):
        need = L.tnp_token_embedding_backward_workspace_bytes(n, vocab, d)
        ws = _workspace(need, grad.device)
        _lib.check(L.tnp_token_embedding_backward(
            tok.data_ptr(), tok.element_size(), n, g.data_ptr(), _ld(g) if n else d, vocab, d, _DTYPES[grad.dtype], scale, dw.data_ptr(),
            d, ws.data_ptr(), need, _lib.raw_stream()), 'tnp_token_embedding_backward')
    return dw


class _TokenEmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale):
        ctx.save_for_backward(tokens)
        ctx.args = (weight.shape[0], scale)
        return _embedding_forward(tokens, weight.detach(), scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        tokens, = ctx.saved_tensors
        return None, _embedding_backward(grad, tokens, *ctx.args), None


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


def token_embedding(tokens, weight, scale=1.0):
    """``scale * weight[tokens]``: tokens int64 / int32 of any shape, weight [V, D] -> tokens.shape + (D,) in weight's dtype, rounded
    once.  tokens < 0 (absent track): a row of zeros; tokens >= V: a row of NaN.  The gradient of ``weight`` is dense, summed in fp32
    in a fixed order (two calls give the same bits)."""
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


def _ce_args(hidden, weight, bias, target, reduction):
    a = VocabCe()
    a.dtype, a.reduction = _DTYPES[weight.dtype], reduction
    a.M, a.V, a.D = hidden.shape[0], weight.shape[0], weight.shape[1]
    a.hidden, a.ld_hidden = hidden.data_ptr(), _ld(hidden)
    a.weight, a.ld_weight = weight.data_ptr(), _ld(weight)
    a.bias = bias.data_ptr() if bias is not None else None
    a.target = target.data_ptr()
    return a


def _ce_forward(hidden, weight, bias, target, reduction, train):
    """(loss [M] or [1], what the backward pass reads or None); every operand already in kernel layout, M >= 1"""
    dev = weight.device
    L = _lib.lib()
    a = _ce_args(hidden, weight, bias, target, reduction)
    saved = None
    with _on(dev):
        if train:
            saved = _workspace(L.tnp_vocab_ce_saved_bytes(ctypes.byref(a)), dev)
            a.saved = saved.data_ptr()
        need = L.tnp_vocab_ce_workspace_bytes(ctypes.byref(a), 0)
        ws = _workspace(need, dev)
        loss = torch.empty(hidden.shape[0] if reduction == 0 else 1, dtype=torch.float32, device=dev)
        _lib.check(L.tnp_vocab_ce_forward(ctypes.byref(a), loss.data_ptr(), ws.data_ptr(), need, _lib.raw_stream()),
                   'tnp_vocab_ce_forward')
    return loss, saved


def _ce_backward(grad, hidden, weight, bias, target, saved, reduction, needs):
    dev = weight.device
    L = _lib.lib()
    a = _ce_args(hidden, weight, bias, target, reduction)
    a.saved = saved.data_ptr()
    with _on(dev):
        g = grad.detach().reshape(-1).float().contiguous()
        dx = torch.empty(hidden.shape, dtype=hidden.dtype, device=dev) if needs[0] else None
        dw = torch.empty(weight.shape, dtype=weight.dtype, device=dev) if needs[1] else None
        db = torch.empty(weight.shape[0], dtype=weight.dtype, device=dev) if needs[2] else None
        need = L.tnp_vocab_ce_workspace_bytes(ctypes.byref(a), 1)
        ws = _workspace(need, dev)
        p = lambda t: None if t is None else t.data_ptr()
        _lib.check(L.tnp_vocab_ce_backward(ctypes.byref(a), g.data_ptr(), p(dx), p(dw), p(db), ws.data_ptr(), need, _lib.raw_stream()),
                   'tnp_vocab_ce_backward')
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
        n = ctx.needs_input_grad
        return _ce_backward(grad, hidden, weight, bias, target, saved, ctx.reduction,
                            (n[0], n[1], n[2] and bias is not None)) + (None, None)


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


def vocab_cross_entropy(hidden, weight, target, bias=None, reduction='mean'):
    """Cross entropy of ``softmax(hidden @ weight.T + bias)`` against ``target``, without storing the logits.

    hidden [..., D], weight [V, D], bias [V] (may hold -inf: masked entries) of one dtype, target [...] int64 / int32.  Returns fp32:
    a scalar ('mean' over the rows that are there, 0 if there are none; 'sum') or target's shape ('none').  target < 0: an absent
    row -- its hidden state is not read, its loss and gradient are 0; target >= V: NaN.  Differentiable in hidden, weight and bias.

    fp32 operands are multiplied as two fp16 numbers each, scaled by the largest finite element of their tensor: an element below
    2^-16 of that one loses relative precision (2^-40 of the largest remains), a row of valid targets that holds an infinity gives
    NaN."""
    check_cross_entropy(hidden, weight, target, bias, reduction)
    red = _REDUCTIONS[reduction]
    shape = target.shape
    t = target.reshape(-1)
    if t.dtype != torch.int64 or not t.is_contiguous():
        t = t.to(torch.int64).contiguous()
    x, w = hidden.reshape(-1, hidden.shape[-1]) if hidden.dim() != 2 else hidden, weight
    if x.shape[0] == 0:                                                       # no rows: an empty / zero loss with zero gradients
        zero = hidden.float().sum() + weight[:0].float().sum() + (bias[:0].float().sum() if bias is not None else 0.0)
        return zero.expand(shape) if red == 0 else zero
    if x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    if w.stride(1) != 1 or (w.shape[0] > 1 and w.stride(0) < w.shape[1]):
        w = w.contiguous()
    b = bias.contiguous() if bias is not None else None
    if torch.is_grad_enabled() and (x.requires_grad or w.requires_grad or (b is not None and b.requires_grad)):
        loss = _VocabCeFn.apply(x, w, b, t, red)
    else:
        loss, _ = _ce_forward(x, w, b, t, red, False)
    return loss.reshape(shape) if red == 0 else loss[0]
