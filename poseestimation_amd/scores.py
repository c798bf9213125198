"""Rows of scores: the readout of a network that names one of many things per row.

``get_peaks`` reads the answer of a network that draws a map per keypoint.  A network that answers
with a row of scores per question instead (over coordinate bins, classes or tokens) is read by

* ``token_logprobs``            log probabilities of given answers, the entropy of the row, the best
                                answers with theirs
* ``token_logprobs_backward``   the gradient of those with respect to the scores
* ``route_experts``             which experts (answering heads) a row goes to, and with which weights
* ``route_experts_backward``    the gradient of the weights

Scores are torch tensors on a GPU, ``(rows, columns)`` in float32, bfloat16 or float16; rows may be any
distance apart (a slice of a padded buffer, an expanded row), columns are next to each other.  Calls are
queued on the current stream of the tensors' device and do not wait; they can be captured into a graph.
A row's result depends on that row alone, not on its place or the other rows of the call; calls of other
shapes may add in another order.  The functions take no part in autograd: a training step calls the backward
form itself, and where gradients are recorded the forward ones refuse logits that require one (pass
``logits.detach()``).  Gradients have no gradient.  Bad arguments raise ``ValueError``.  Nothing here has a counterpart
in the reference.
"""
from collections import namedtuple

import torch

from . import _ffi

_DTYPES = {torch.float32: _ffi.F32, torch.bfloat16: _ffi.BF16, torch.float16: _ffi.F16}
_SCORES = {'softmax': _ffi.SCORE_SOFTMAX, 'sigmoid': _ffi.SCORE_SIGMOID}
_GROUP_SCORES = {'max': _ffi.GROUP_MAX, 'top2': _ffi.GROUP_TOP2}

TokenLogprobs = namedtuple('TokenLogprobs', 'logp entropy top_logp top_index stats')
Routes = namedtuple('Routes', 'weights index')


def _no_grad(logits):
    """Refuses logits whose gradient autograd would lose: what is made of them here carries none."""
    if isinstance(logits, torch.Tensor) and logits.requires_grad and torch.is_grad_enabled():
        raise ValueError('the logits require a gradient, which autograd does not get from here: pass logits.detach() '
                         '(or call under torch.no_grad()) and call the backward form')


def _rows(x, name):
    """``(dtype code, rows, columns, row stride)`` of a matrix of scores."""
    if not isinstance(x, torch.Tensor) or x.dim() != 2 or x.dtype not in _DTYPES:
        raise ValueError('%s must be a (rows, columns) float32, bfloat16 or float16 tensor' % name)
    if not x.is_cuda:
        raise ValueError('%s must be on a GPU' % name)
    rows, columns = x.shape
    stride, step = x.stride()
    if step != 1 and columns > 1:
        raise ValueError('the columns of %s must be next to each other (stride 1, got %d)' % (name, step))
    return _DTYPES[x.dtype], rows, columns, stride


def _like(x, name, dtype, shapes, device):
    """``x`` as a contiguous tensor of ``dtype`` with one of the shapes, on the device."""
    if isinstance(x, torch.Tensor) and x.dtype is dtype and x.shape == shapes[0] and x.device == device and x.is_contiguous():
        return x
    if not isinstance(x, torch.Tensor) or tuple(x.shape) not in shapes or x.device != device:
        raise ValueError('%s must be a tensor of shape %s on %s' % (name, ' or '.join(map(str, shapes)), device))
    if x.dtype != dtype:
        if x.is_floating_point() != dtype.is_floating_point or x.dtype in (torch.bool, torch.uint64) or x.is_complex():
            raise ValueError('%s must hold %s, got %s' % (name, 'numbers' if dtype.is_floating_point else 'whole numbers', x.dtype))
        if dtype == torch.int32 and x.dtype.itemsize >= 4:  # a larger number stays out of every range
            x = x.to(torch.int64).clamp(-1, 0x7fffffff)
        x = x.to(dtype)
    return x if x.is_contiguous() else x.contiguous()


def _tokens(tokens, rows, device):
    if not isinstance(tokens, torch.Tensor) or tokens.dim() not in (1, 2):
        raise ValueError('tokens must be a (rows,) or (rows, n) tensor of whole numbers')
    shape = (rows,) + tuple(tokens.shape[1:])
    return _like(tokens, 'tokens', torch.int64, (shape,), device), shape


def _current(device):
    """Whether ``device`` is the current one, which the library's calls work on."""
    return torch.cuda.current_device() == device.index


# The current stream's address itself: making a Stream object of it takes longer than the checks of a small call.  Not a public
# name of torch, so that it need not be there.
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None)


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream if _raw_stream is None else _raw_stream(device.index)


def _raise(rc):
    msg = _ffi.lib().pd_last_error(None).decode()
    if rc == _ffi.PD_E_INVALID:
        raise ValueError(msg)
    raise RuntimeError('libposedecode error %d: %s' % (rc, msg))


def _address(x):
    return None if x is None else x.data_ptr()


def _grad_out(out, logits):
    if out is None:
        return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device), logits.shape[1]
    if not isinstance(out, torch.Tensor) or out.dtype != logits.dtype or out.shape != logits.shape or out.device != logits.device:
        raise ValueError('out must be a tensor like the logits: %s %s on %s' % (tuple(logits.shape), logits.dtype, logits.device))
    _, rows, columns, stride = _rows(out, 'out')
    return out, columns if rows <= 1 else stride


def _written(out):
    """The kernels write to an address: tells autograd, which may have kept the tensor for a backward pass."""
    torch.autograd.graph.increment_version(out)
    return out


def token_logprobs(logits, tokens=None, top=0, widths=None):
    """Log probabilities of the given ``tokens`` (``(rows,)`` or ``(rows, n)``, n <= 64) under the softmax of
    every row, the row's entropy, and its ``top`` (<= 64) largest entries.

    ``widths`` (rows,): row r holds that many columns only; what lies behind is not read and counts as -inf.
    Returns ``TokenLogprobs(logp, entropy, top_logp, top_index, stats)``: ``logp`` shaped like ``tokens``,
    ``entropy`` (rows,), ``top_logp`` / ``top_index`` (rows, top) in descending order, equal scores by the lower
    index; what was not asked for is None.  ``stats`` (rows, 3) holds the largest score, the logarithm of the sum
    relative to it and the entropy, for the backward form.

    A negative token is not given: 0.  A token that the row does not hold: -inf.  A row with nothing above -inf:
    -inf, entropy 0, alternatives 0, 1, .. .  A row that holds a NaN or +inf: NaN, alternatives -1."""
    _no_grad(logits)
    code, rows, columns, stride = _rows(logits, 'logits')
    dev = logits.device
    if not _current(dev):
        with torch.cuda.device(dev):
            return token_logprobs(logits, tokens, top, widths)
    n_tok, shape, top = 0, None, int(top)
    if not 0 <= top <= min(_ffi.MAX_ALTERNATIVES, columns):
        raise ValueError('top must be within 0..%d and the columns, got %d' % (_ffi.MAX_ALTERNATIVES, top))
    if tokens is not None:
        tokens, shape = _tokens(tokens, rows, dev)
        n_tok = shape[1] if len(shape) == 2 else 1
    if widths is not None:
        widths = _like(widths, 'widths', torch.int32, ((rows,),), dev)
    L = _ffi.lib()
    ws_bytes = L.pd_token_logprobs_workspace(code, rows, columns, top)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    # Each result a tensor of its own: one that is kept keeps nothing else, and one that is written marks no other as changed.
    # (Sizes one by one: 1.25 us an allocation, 1.6 with a tuple.)
    logp = top_logp = top_index = None
    entropy = torch.empty(rows, dtype=torch.float32, device=dev)
    stats = torch.empty(rows, 3, dtype=torch.float32, device=dev)
    if top:
        top_logp = torch.empty(rows, top, dtype=torch.float32, device=dev)
        top_index = torch.empty(rows, top, dtype=torch.int32, device=dev)
    if shape is not None:
        logp = torch.empty(*shape, dtype=torch.float32, device=dev)
    rc = L.pd_token_logprobs(logits.data_ptr(), code, rows, columns, stride, _address(widths), _address(tokens), n_tok, top,
                             _address(logp), entropy.data_ptr(), stats.data_ptr(), _address(top_logp), _address(top_index),
                             _address(ws), ws_bytes, _stream(dev))
    if rc:
        _raise(rc)
    return TokenLogprobs(logp, entropy, top_logp, top_index, stats)


def token_logprobs_backward(logits, stats, tokens=None, grad_logp=None, grad_entropy=None, widths=None, out=None):
    """The gradient with respect to the logits, of their type, from that of ``logp`` (shaped like ``tokens``) and of
    ``entropy``; ``stats`` is the forward call's.  The alternatives' log probabilities are differentiated by passing
    ``top_index`` as tokens.  Tokens that are not given contribute nothing, one that the row does not hold what a
    masked logit would (-p_j g at every column), a token named twice counts twice;
    columns behind a row's width and rows with nothing above -inf get 0.  ``out``: where to put it; the logits
    themselves are allowed."""
    code, rows, columns, stride = _rows(logits, 'logits')
    dev = logits.device
    if not _current(dev):
        with torch.cuda.device(dev):
            return token_logprobs_backward(logits, stats, tokens, grad_logp, grad_entropy, widths, out)
    stats = _like(stats, 'stats', torch.float32, ((rows, 3),), dev)
    n_tok = 0
    if (tokens is None) != (grad_logp is None):
        raise ValueError('tokens and grad_logp go together')
    if tokens is not None:
        tokens, shape = _tokens(tokens, rows, dev)
        n_tok = shape[1] if len(shape) == 2 else 1
        grad_logp = _like(grad_logp, 'grad_logp', torch.float32, (shape,), dev)
    elif grad_entropy is None:
        raise ValueError('grad_logp or grad_entropy is required')
    if grad_entropy is not None:
        grad_entropy = _like(grad_entropy, 'grad_entropy', torch.float32, ((rows,),), dev)
    if widths is not None:
        widths = _like(widths, 'widths', torch.int32, ((rows,),), dev)
    given = out is not None
    out, out_stride = _grad_out(out, logits)
    rc = _ffi.lib().pd_token_logprobs_grad(logits.data_ptr(), code, rows, columns, stride, _address(widths), stats.data_ptr(),
                                           _address(tokens), n_tok, _address(grad_logp), _address(grad_entropy), out.data_ptr(),
                                           out_stride, _stream(dev))
    if rc:
        _raise(rc)
    return _written(out) if given else out


def _score_code(table, value, name):
    if value not in table:
        raise ValueError('%s must be one of %s, got %r' % (name, ', '.join(map(repr, table)), value))
    return table[value]


def route_experts(logits, top, score='softmax', bias=None, groups=1, top_groups=None, group_score='max', renormalise=True,
                  scale=1.0):
    """The ``top`` (<= 32) of the experts (columns, <= 1024) that each row goes to, and their weights.

    p is the softmax of the row, or 1 / (1 + exp(-x)) with ``score='sigmoid'``.  Experts are ordered by p + ``bias``
    (experts,), without bias by the logits, equal ones by the lower index; the order is that of float64 arithmetic on the
    logits and on the bias in float32, which one of another type is rounded to.
    With ``groups`` > 1 (<= 64, equal parts of consecutive experts) only the experts of the ``top_groups`` best groups are
    eligible, a group counting by its largest value (``group_score='max'``) or by the sum of its two largest
    (``'top2'``, of p or p + bias).  ``Routes(weights, index)``, both (rows, top) in descending order: weights are
    ``scale`` * p, with ``renormalise`` divided by the sum of the chosen p.

    A bias of -inf or NaN puts an expert behind all others; a group with fewer than two others has a sum of -inf, all
    such groups alike (the lower index first), and one with a bias of +inf counts as +inf.  A row whose chosen p sum to 0
    gets weights of 0 when renormalised.  A row that holds a NaN (softmax: or +inf): weights NaN, index -1."""
    _no_grad(logits)
    code, rows, experts, stride = _rows(logits, 'logits')
    dev = logits.device
    if not _current(dev):
        with torch.cuda.device(dev):
            return route_experts(logits, top, score, bias, groups, top_groups, group_score, renormalise, scale)
    score = _score_code(_SCORES, score, 'score')
    group_score = _score_code(_GROUP_SCORES, group_score, 'group_score')
    if bias is not None:
        bias = _like(bias, 'bias', torch.float32, ((experts,),), dev)
    top, groups = int(top), int(groups)
    top_groups = groups if top_groups is None else int(top_groups)
    if not 1 <= top <= min(_ffi.MAX_ROUTES, experts):
        raise ValueError('top must be within 1..%d and the experts, got %d' % (_ffi.MAX_ROUTES, top))
    weights = torch.empty((rows, top), dtype=torch.float32, device=dev)
    index = torch.empty((rows, top), dtype=torch.int32, device=dev)
    rc = _ffi.lib().pd_route_experts(logits.data_ptr(), code, rows, experts, stride, _address(bias), score, groups, top_groups,
                                     group_score, top, 1 if renormalise else 0, float(scale), weights.data_ptr(), index.data_ptr(),
                                     _stream(dev))
    if rc:
        _raise(rc)
    return Routes(weights, index)


def route_experts_backward(logits, index, grad_weights, score='softmax', renormalise=True, scale=1.0, out=None):
    """The gradient of ``weights`` with respect to the logits, of their type; ``index`` is the forward call's, the choice
    itself (bias, groups) has no gradient.  Entries of ``index`` that name no expert are skipped, an expert named twice
    counts twice.  So a row without an order (its index is -1) gets 0, but NaN where the weights are a softmax that is not
    renormalised, the one form that reads all of the row.  ``out``: where to put it; the logits themselves are allowed."""
    code, rows, experts, stride = _rows(logits, 'logits')
    dev = logits.device
    if not _current(dev):
        with torch.cuda.device(dev):
            return route_experts_backward(logits, index, grad_weights, score, renormalise, scale, out)
    score = _score_code(_SCORES, score, 'score')
    if not isinstance(index, torch.Tensor) or index.dim() != 2:
        raise ValueError('index must be a (rows, top) tensor of whole numbers')
    top = index.shape[1]
    index = _like(index, 'index', torch.int32, ((rows, top),), dev)
    grad_weights = _like(grad_weights, 'grad_weights', torch.float32, ((rows, top),), dev)
    given = out is not None
    out, out_stride = _grad_out(out, logits)
    rc = _ffi.lib().pd_route_experts_grad(logits.data_ptr(), code, rows, experts, stride, index.data_ptr(), grad_weights.data_ptr(),
                                          score, top, 1 if renormalise else 0, float(scale), out.data_ptr(), out_stride, _stream(dev))
    if rc:
        _raise(rc)
    return _written(out) if given else out
