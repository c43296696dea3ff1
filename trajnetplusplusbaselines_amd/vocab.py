"""Motions as tokens: the two operators that a model over a vocabulary of displacements or grid cells needs beside the ones for
continuous positions, on the kernels of csrc/token_embed.hip and csrc/vocab_ce.hip (autograd nodes: csrc/vocab_torch.cpp).

    token_embedding(tokens, weight, scale)               scale * weight[tokens]           (module: lstm.TokenEmbedding)
    vocab_cross_entropy(hidden, weight, target, bias)    cross entropy of the output layer hidden @ weight.T + bias against
                                                         ``target``, the logits never stored  (module: lstm.VocabularyLoss)

Both are differentiable, run on the current stream of the tensors' device without a host synchronisation, take fp32, bf16 and fp16
and refuse host tensors.  A negative token or target is an absent track (zero row, no loss, no gradient); one past the end of the
vocabulary gives NaN, since the host does not look at device data.
"""
import ctypes
import importlib.util
import os

import torch

from . import _lib

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_REDUCTIONS = {'none': 0, 'mean': 1, 'sum': 2}
_ENTRIES = ('tnp_last_error', 'tnp_token_embedding_forward', 'tnp_token_embedding_backward_workspace_bytes', 'tnp_token_embedding_backward',
            'tnp_vocab_ce_saved_bytes', 'tnp_vocab_ce_workspace_bytes', 'tnp_vocab_ce_forward', 'tnp_vocab_ce_backward')
_NATIVE = None


def native():
    """csrc/vocab_torch.cpp, bound to the loaded library's entries (once)"""
    global _NATIVE
    if _NATIVE is None:
        L = _lib.lib()
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), 'lib', '_trajnet_torch.so')
        if not os.path.exists(path):
            raise RuntimeError('%s not found: build it with `python -c "import __graft_entry__ as g; g.build()"`' % path)
        spec = importlib.util.spec_from_file_location('_trajnet_torch', path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.bind([ctypes.cast(getattr(L, e), ctypes.c_void_p).value for e in _ENTRIES])
        _NATIVE = module
    return _NATIVE


def _check_table(weight, what):
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError('%s must be [entries, columns] (got %s)' % (what, tuple(weight.shape)))
    if weight.dtype not in _DTYPES:
        raise TypeError('%s must be float32, bfloat16 or float16 (got %s)' % (what, weight.dtype))


# ---- token embedding ---------------------------------------------------------------------------------------------------------
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
    return native().token_embedding(tokens, weight, check_embedding(tokens, weight, scale))


# ---- cross entropy over a vocabulary -----------------------------------------------------------------------------------------
def saved_bytes(rows, entries, columns, dtype):
    """tnp_vocab_ce_saved_bytes() from the sizes alone (they may be symbolic while a graph is traced)"""
    panels = (columns + 15) // 16 if dtype == torch.float32 else (columns + 31) // 32
    up = lambda n: (n + 255) // 256 * 256
    return 256 + 24 * up(rows) + 8 * up(entries) + 64 * panels * (up(rows) + up(entries))


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
    row -- its hidden state is not read, its loss and gradient are 0; target >= V: NaN.  Differentiable in hidden, weight and bias; until its
    backward pass a call keeps packed copies of hidden and of weight, so that one call on stacked rows keeps less than several.

    fp32 operands are multiplied as two fp16 numbers each, scaled by the largest finite element of their tensor or, where all of a row
    (of hidden or of weight) is below 2^-16 of that one, of their row: no row's result goes by another's size.  Within a row, an element below
    2^-16 of the row's largest may lose relative precision (2^-23 of the row's largest remains, usually 2^-40).  Infinities are
    multiplied as the formula says (a logit of -inf masks its entry; two infinities that meet may give NaN).  Gradients: (p - y) times the upstream gradient is rounded to fp16 (fp32 and fp16 operands: two fp16 numbers); parts of a
    row below 2^-29 of the largest lose relative precision (2^-40 of the largest upstream gradient remains, and 2^-22 of the row's own). An
    upstream gradient that is no number spoils its own row of hidden's gradient, and the sums over rows."""
    if torch.compiler.is_compiling():
        from . import ops  # noqa: F401  (registers the operators)
        return torch.ops.trajnet.vocab_cross_entropy(hidden, weight, target, bias, reduction)[0]
    check_cross_entropy(hidden, weight, target, bias, reduction)
    red = _REDUCTIONS[reduction]
    if target.numel() == 0:                                              # no rows: an empty / zero loss with zero gradients
        zero = hidden.float().sum() + weight[:0].float().sum() + (bias[:0].float().sum() if bias is not None else 0.0)
        return zero.expand(target.shape) if red == 0 else zero
    return native().vocab_cross_entropy(hidden, weight, target, bias, red)
