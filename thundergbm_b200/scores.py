"""Operators on the scores of many classes, on CUDA tensors.

Scores are a tensor of rows x classes (float32, float16 or bfloat16, any strides).  A booster keeps all rows of a class side by side:
`torch.from_numpy(booster.ypred()).cuda().t()` is such a tensor, no copy is made of it.

    adjust   penalties for classes a row was given before, a bias per class, classes a row may not have
    top      the largest scores of every row, their classes, the row's log-sum-exp
    distill  loss on a teacher's largest scores and on hard labels, with its gradient

(top and distill take several times as long by class above some 5000 classes, or where neither rows nor classes lie side by side.)

Results come on the stream that is torch's current one on the scores' device, in the layout of the scores; nothing waits.
Autograd does not record them: results require no gradient, also where the scores do (distill returns its gradient).
Every function is one call of the C interface (tgbm_scores_* in include/thundergbm.h, which defines the operators); what the
arguments may not be is refused there or here before anything is queued.
"""
from __future__ import annotations

import torch

from . import _lib

_TYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_INT = (torch.int32,)
_GIVES = {'loss': 0, 'gradient': 1, 'pairs': 2}
MAX_TOP = 128


def _refuse(what):
    raise ValueError(what)


def _scores(t, name='scores'):
    """(rows, classes, type, device)"""
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dim() == 2:
        kind = _TYPE.get(t.dtype)
        if kind is not None:
            n, k = t.shape
            if k < 1 or n >= 2 ** 31 or k >= 2 ** 31:
                _refuse(f'{name}: at least one class and fewer than 2^31 rows')
            return n, k, kind, t.get_device()
    _refuse(f'{name}: a CUDA tensor of rows x classes in float32, float16 or bfloat16')


def _beside(t, device, dtype, shape, name):
    """Address of a contiguous tensor on the scores' device."""
    if isinstance(t, torch.Tensor) and t.dtype == dtype and t.shape == shape and t.get_device() == device and t.is_contiguous():
        return t.data_ptr()
    _refuse(f'{name}: a contiguous {dtype} tensor of shape {tuple(shape)} on cuda:{device}')


def _call(f, device, *args):
    # (the calls beneath torch.cuda.current_device and current_stream(device).cuda_stream: 0.2 us instead of 1.5 of a call's 14)
    if torch._C._cuda_getDevice() == device:
        rc = f(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = f(*args, torch._C._cuda_getCurrentRawStream(device))
    if rc:
        _lib.check(rc)


def _like(scores, n, k):
    """(new memory in the layout of the scores, its strides)"""
    if scores.stride(0) < scores.stride(1):
        return scores.new_empty_strided((n, k), (1, n)), 1, n
    return scores.new_empty((n, k)), k, 1


def adjust(scores, *, out=None, bias=None, allowed=None, allowed_row=None, history=None, repetition=1.0, frequency=0.0, presence=0.0):
    """Scores after penalties, bias and mask, in their own type; `out=scores` changes them in place.

    bias: float32, one per class.  allowed: int32 words (masks x ceil(classes / 32)), class k in bit k % 32 of word k // 32, bits of
    classes that may be chosen set; allowed_row: int32, the mask of every row (-1: none), without it row n has mask n.
    history: (ptr, classes), int64 (rows + 1) and int32: what row n was given before is classes[ptr[n]:ptr[n + 1]]; a class that stands
    there c > 0 times has its score divided (above 0) or multiplied by `repetition`, less c * frequency + presence."""
    n, k, kind, device = _scores(scores)
    made = out is None
    if made:
        out, o0, o1 = _like(scores, n, k)
    else:
        _scores(out, 'out')
        o0, o1 = out.stride()
        if not (out.shape == scores.shape and out.dtype == scores.dtype and out.device == scores.device):
            _refuse('out: shape, type and device of the scores')
        if out.requires_grad and torch.is_grad_enabled():
            _refuse('out: takes part in autograd, which does not see what is written here')
    masks = words = given = 0
    mask_ptr = row_ptr = bias_ptr = ptr = ids = None
    if bias is not None:
        bias_ptr = _beside(bias, device, torch.float32, (k,), 'bias')
    if allowed is not None:
        if not (isinstance(allowed, torch.Tensor) and allowed.dim() == 2):
            _refuse('allowed: masks x words')
        masks, words = allowed.shape
        if words < (k + 31) // 32:
            _refuse('allowed: a bit for every class')
        if n and masks < (n if allowed_row is None else 1):   # (no masks have no address, which means that all classes are allowed)
            _refuse('allowed: fewer masks than rows, and none named for each row')
        mask_ptr = _beside(allowed, device, torch.int32, (masks, words), 'allowed')
        if allowed_row is not None:
            row_ptr = _beside(allowed_row, device, torch.int32, (n,), 'allowed_row')
    elif allowed_row is not None:
        _refuse('allowed_row: there are no masks')
    if history is not None:
        ptr, ids = history
        if not (isinstance(ids, torch.Tensor) and ids.dim() == 1):
            _refuse('history: (ptr, classes)')
        given = ids.numel()
        ptr = _beside(ptr, device, torch.int64, (n + 1,), 'history')
        ids = _beside(ids, device, torch.int32, (given,), 'history')
    s = scores.stride()
    _call(_lib.lib().tgbm_scores_adjust, device, n, k, kind, scores.data_ptr(), s[0], s[1], out.data_ptr(), o0, o1, bias_ptr, mask_ptr, masks, words,
          row_ptr, ptr, ids, given, repetition, frequency, presence)
    if not made:
        torch.autograd.graph.increment_version(out)   # (for operations that keep it for their backward pass)
    return out


def top(scores, k, *, temperature=1.0):
    """(values, classes, lse): the k largest scores of every row (float32, rows x k; largest first, of equal ones the lower class first),
    their classes (int32) and the log of the sum over all classes of exp(score / temperature).  Masked scores (-inf) and NaN are not
    chosen: a row that runs out of others ends in -inf and class -1."""
    n, classes, kind, device = _scores(scores)
    if not 1 <= k <= MAX_TOP:
        _refuse(f'k: 1 to {MAX_TOP}')
    values = scores.new_empty((n, k), dtype=torch.float32)
    ids = scores.new_empty((n, k), dtype=torch.int32)
    lse = scores.new_empty((n,), dtype=torch.float32)
    s = scores.stride()
    _call(_lib.lib().tgbm_scores_top, device, n, classes, kind, scores.data_ptr(), s[0], s[1], k, temperature, values.data_ptr(), ids.data_ptr(),
          lse.data_ptr())
    return values, ids, lse


def _list(t, types, n, device, name):
    if not (isinstance(t, torch.Tensor) and t.dtype in types and t.dim() == 2 and t.size(0) == n and t.get_device() == device):
        _refuse(f'{name}: rows x kept classes, {", ".join(map(str, types))}, on cuda:{device}')
    if t.stride(1) != 1 and t.size(1) > 1:
        _refuse(f'{name}: the entries of a row have to be side by side')


def distill(scores, ids, logits, *, lse=None, labels=None, weights=None, temperature=1.0, alpha=1.0, gives='gradient'):
    """(loss, gradient) of a student's scores against a teacher's largest ones.

    ids (int32) and logits (float32, float16 or bfloat16), rows x up to 128: classes and scores that are kept of the teacher, entries of
    class -1 are none; their rows may be apart (a slice of a longer list).  lse: the teacher's log-sum-exp at this temperature (from
    `top`); with it the mass that is not listed is compared as one class, without it the listed ones are taken for all.  labels:
    int32, -1 for none; the loss on them weighs 1 - alpha.  weights: float32, per row.
    gives: 'loss' (no gradient: None), 'gradient' (rows x classes, type of the scores), 'pairs' (rows x classes x 2, float32:
    gradient and hessian, what a booster grows trees from)."""
    n, k, kind, device = _scores(scores)
    if gives not in _GIVES:
        _refuse("gives: 'loss', 'gradient' or 'pairs'")
    _list(ids, _INT, n, device, 'ids')
    _list(logits, _TYPE, n, device, 'logits')
    if ids.shape != logits.shape:
        _refuse('ids and logits: one score for every class')
    lse_ptr = None if lse is None else _beside(lse, device, torch.float32, (n,), 'lse')
    label_ptr = None if labels is None else _beside(labels, device, torch.int32, (n,), 'labels')
    weight_ptr = None if weights is None else _beside(weights, device, torch.float32, (n,), 'weights')
    loss = scores.new_empty((n,), dtype=torch.float32)
    grad = grad_ptr = None
    g0 = g1 = 0
    if gives == 'pairs':
        if scores.stride(0) < scores.stride(1):
            g0, g1 = 1, n
            grad = scores.new_empty_strided((n, k, 2), (2, 2 * n, 1), dtype=torch.float32)
        else:
            g0, g1 = k, 1
            grad = scores.new_empty((n, k, 2), dtype=torch.float32)
        grad_ptr = grad.data_ptr()
    elif gives == 'gradient':
        grad, g0, g1 = _like(scores, n, k)
        grad_ptr = grad.data_ptr()
    s = scores.stride()
    _call(_lib.lib().tgbm_scores_distill, device, n, k, kind, scores.data_ptr(), s[0], s[1], ids.size(1), ids.data_ptr(), ids.stride(0),
          _TYPE[logits.dtype], logits.data_ptr(), logits.stride(0), lse_ptr, label_ptr, weight_ptr, temperature, alpha, loss.data_ptr(),
          _GIVES[gives], grad_ptr, g0, g1)
    return loss, grad
