"""The operators on rows of scores, as cases that can be timed: log probabilities of given tokens with
entropy and top alternatives, the routing of rows to experts, and the gradients of both.

``own`` chooses between the plain form (elementary torch operations, 32 bits, the order of near scores
in 64) and the calls of ``poseestimation_amd.scores``.  ``exact`` restates the definitions in 64 bits.
"""
import math
import types

import torch

own = False

DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
SIZE = {'float32': 4, 'bfloat16': 2, 'float16': 2}


# ---- the cases -----------------------------------------------------------------------------

def _logprobs(op, rows, vocab, dtype, tokens=1, top=0, ragged=False, masked=False, pad=0):
    """``pad``: unused columns behind each row; ``ragged``: rows of different widths; ``masked``: some
    scores at -inf, some rows with nothing else, some tokens not given."""
    return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, tokens=tokens, top=top, ragged=ragged, masked=masked, pad=pad)


def _route(op, rows, experts, dtype, top, score='softmax', bias=False, groups=1, top_groups=1, group_score='max',
           renormalise=True, scale=1.0):
    return dict(op=op, rows=rows, experts=experts, dtype=dtype, top=top, score=score, bias=bias, groups=groups,
                top_groups=top_groups, group_score=group_score, renormalise=renormalise, scale=scale)


def listed():
    def named(name, case):
        return dict(case, name=name)
    return [
        # a batch of 64 images of 368 x 368 read out as coordinate bins: 18 parts, two axes, one row each
        named('logp_bins_64x368', _logprobs('logprobs', 64 * 18 * 2, 368, 'float32', top=5)),
        # one row over a large vocabulary: a single token being answered, where latency counts
        named('logp_one_row_131072', _logprobs('logprobs', 1, 131072, 'bfloat16', top=20)),
        # a serving batch over an odd vocabulary, several candidates scored per row, constrained answers
        named('logp_48x32003', _logprobs('logprobs', 48, 32003, 'float16', tokens=4, top=8, masked=True)),
        # 256 images of up to 656 pixels a side, each with its own number of bins
        named('logp_ragged_256x656', _logprobs('logprobs', 256 * 18 * 2, 656, 'bfloat16', top=3, ragged=True)),
        # a long prompt (or a batch of them) scored over a large vocabulary
        named('logp_4096x131072', _logprobs('logprobs', 4096, 131072, 'bfloat16', top=5)),
        # the gradient of a small batch over an odd vocabulary, rows that start on no 16-byte border
        named('logp_grad_500x50021', _logprobs('logprobs_grad', 500, 50021, 'float32', tokens=2, masked=True)),
        # the gradient of a training batch
        named('logp_grad_8192x32768', _logprobs('logprobs_grad', 8192, 32768, 'bfloat16')),
        # one row to its experts: a single token being answered
        named('route_1x64', _route('route', 1, 64, 'bfloat16', 4)),
        # a training batch, balanced by a bias, experts in groups
        named('route_4096x256_groups', _route('route', 4096, 256, 'float32', 8, score='sigmoid', bias=True, groups=8,
                                              top_groups=4, group_score='top2', scale=2.5)),
        # a large batch, plain softmax routing
        named('route_65536x128', _route('route', 65536, 128, 'bfloat16', 8)),
        # the gradient of the balanced routing of a training batch
        named('route_grad_4096x256', _route('route_grad', 4096, 256, 'float32', 8, score='sigmoid', scale=2.5)),
        # the gradient of softmax weights that are not renormalised, which reaches every expert
        named('route_grad_32768x160', _route('route_grad', 32768, 160, 'bfloat16', 6, renormalise=False)),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['logprobs', 'logprobs', 'logprobs_grad', 'route', 'route', 'route_grad'])
    dtype = rng.choice(['bfloat16', 'bfloat16', 'float32', 'float16'])
    if op.startswith('logprobs'):
        vocab = _log_int(rng, 40, 200000)
        rows = _log_int(rng, 1, max(1, min(16384, (1 << 27) // vocab)))
        top = 0 if op == 'logprobs_grad' else rng.choice([0, 1, _log_int(rng, 2, 32)])
        return _logprobs(op, rows, vocab, dtype, tokens=rng.choice([1, 1, _log_int(rng, 2, 16)]), top=top,
                         ragged=rng.random() < 0.25, masked=rng.random() < 0.4,
                         pad=rng.choice([0, 0, _log_int(rng, 1, 64)]))
    score = rng.choice(['softmax', 'sigmoid'])
    groups = rng.choice([1, 1, 2, 4, 8])
    experts = groups * _log_int(rng, max(2, 8 // groups), 512 // groups)
    top_groups = rng.randint((groups + 1) // 2, groups)
    top = _log_int(rng, 1, min(16, top_groups * (experts // groups)))
    return _route(op, _log_int(rng, 1, 32768), experts, dtype, top, score=score, bias=rng.random() < 0.5, groups=groups,
                  top_groups=top_groups, group_score=rng.choice(['max', 'top2']), renormalise=rng.random() < 0.6,
                  scale=rng.choice([1.0, 2.5]))


def work(case):
    rows, size = case['rows'], SIZE[case['dtype']]
    if case['op'].startswith('logprobs'):
        # ragged rows hold between a half and all of the columns
        scores = rows * case['vocab'] * (0.75 if case['ragged'] else 1.0)
        if case['op'] == 'logprobs':
            return {'bytes': scores * size + rows * (12 * case['tokens'] + 4 + 8 * case['top']), 'flops': 5 * scores}
        return {'bytes': (scores + rows * case['vocab']) * size + rows * (12 * case['tokens'] + 16), 'flops': 6 * scores}
    scores = rows * case['experts']
    if case['op'] == 'route':
        return {'bytes': scores * size + rows * 8 * case['top'], 'flops': 5 * scores}
    dense = case['score'] == 'softmax' and not case['renormalise']
    return {'bytes': scores * size * (2 if dense else 1) + rows * 8 * case['top'], 'flops': 5 * scores if dense else 8 * rows * case['top']}


# ---- inputs --------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(int(seed))
    dev, rows, dtype = 'cuda', case['rows'], DTYPES[case['dtype']]

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    def uniform(*shape):
        return torch.rand(*shape, device=dev, generator=g)

    s = types.SimpleNamespace(case=case)
    if case['op'].startswith('logprobs'):
        vocab, n_tok = case['vocab'], case['tokens']
        store = torch.empty(rows, vocab + case['pad'], device=dev, dtype=dtype)
        part = max(1, (1 << 26) // vocab)
        for lo in range(0, rows, part):     # in parts: the float32 of a large batch is not needed whole
            x = normal(min(part, rows - lo), vocab).mul_(2.5)
            x[torch.arange(len(x), device=dev), torch.randint(vocab, (len(x),), device=dev, generator=g)] += 12.0
            if case['masked']:
                x[uniform(*x.shape) < 0.3] = -math.inf
            store[lo:lo + part, :vocab] = x
            store[lo:lo + part, vocab:] = math.nan      # behind the row: never read
        s.logits = store[:, :vocab]
        s.tokens = torch.randint(vocab, (rows, n_tok), device=dev, generator=g)
        s.widths = None
        if case['ragged']:
            s.widths = torch.randint(vocab // 2, vocab + 1, (rows,), device=dev, generator=g, dtype=torch.int32)
            s.tokens %= s.widths[:, None]
        # a share of the given tokens is what the row names itself, as in real answers
        s.tokens[:, 0] = torch.where(uniform(rows) < 0.5, s.logits.argmax(1) if not case['ragged'] else s.tokens[:, 0],
                                     s.tokens[:, 0])
        if case['masked'] and rows > 4:
            s.logits[rows // 3] = -math.inf
            s.tokens[uniform(rows, n_tok) < 0.1] = -1
        if case['op'] == 'logprobs_grad':
            s.grad_logp = normal(rows, n_tok)
            s.grad_entropy = normal(rows) * 0.1
            # what the forward pass left for the gradient
            s.stats = torch.empty(rows, 3, device=dev)
            for lo in range(0, rows, part):
                m, log_sum, entropy = _statistics(s, lo, min(rows, lo + part), torch.float64)
                s.stats[lo:lo + part] = torch.stack((m, log_sum, entropy), 1)
        return s
    experts, top = case['experts'], case['top']
    s.logits = normal(rows, experts).mul_(1.5).to(dtype)
    s.bias = (normal(experts) * 0.05) if case['bias'] else None
    if case['op'] == 'route_grad':
        s.index = uniform(rows, experts).argsort(1)[:, :top].to(torch.int32).contiguous()
        s.grad_weights = normal(rows, top)
    return s


# ---- one pass ------------------------------------------------------------------------------

def run(s):
    c = s.case
    if own:
        from poseestimation_amd import scores
        if c['op'] == 'logprobs':
            r = scores.token_logprobs(s.logits, s.tokens, top=c['top'], widths=s.widths)
            return {'logp': r.logp, 'entropy': r.entropy, 'top_logp': r.top_logp, 'top_index': r.top_index}
        if c['op'] == 'logprobs_grad':
            return {'grad': scores.token_logprobs_backward(s.logits, s.stats, s.tokens, s.grad_logp, s.grad_entropy,
                                                           widths=s.widths)}
        if c['op'] == 'route':
            r = scores.route_experts(s.logits, c['top'], score=c['score'], bias=s.bias, groups=c['groups'],
                                     top_groups=c['top_groups'], group_score=c['group_score'],
                                     renormalise=c['renormalise'], scale=c['scale'])
            return {'weights': r.weights, 'index': r.index}
        return {'grad': scores.route_experts_backward(s.logits, s.index, s.grad_weights, score=c['score'],
                                                      renormalise=c['renormalise'], scale=c['scale'])}
    return {'logprobs': _plain_logprobs, 'logprobs_grad': _plain_logprobs_grad, 'route': _plain_route,
            'route_grad': _plain_route_grad}[c['op']](s)


def _in_width(s, lo=0, hi=None):
    """Scores of rows [lo, hi) with -inf in the columns that a ragged row does not have."""
    x = s.logits[lo:hi]
    if s.widths is not None:
        columns = torch.arange(x.shape[1], device=x.device, dtype=torch.int32)
        x = x.masked_fill(columns >= s.widths[lo:hi, None], -math.inf)
    return x


def _statistics(s, lo, hi, dtype):
    x = _in_width(s, lo, hi).to(dtype)
    m = x.max(1).values
    empty = m == -math.inf
    v = x - m.masked_fill(empty, 0)[:, None]
    e = v.exp()
    total = e.sum(1)
    log_sum = total.log().masked_fill(empty, 0)
    entropy = (log_sum - (e * v).masked_fill(e == 0, 0).sum(1) / total).masked_fill(empty, 0)
    return m, log_sum, entropy


def _plain_logprobs(s):
    rows, vocab = s.logits.shape
    x = _in_width(s).float()
    m = x.max(1).values
    empty = m == -math.inf
    v = x - m.masked_fill(empty, 0)[:, None]
    e = v.exp()
    total = e.sum(1)
    log_sum = total.log().masked_fill(empty, 0)
    entropy = (log_sum - (e * v).masked_fill(e == 0, 0).sum(1) / total).masked_fill(empty, 0)
    del e
    given = s.tokens >= 0
    logp = v.gather(1, s.tokens.clamp(0, vocab - 1)) - log_sum[:, None]
    logp = logp.masked_fill(s.tokens >= vocab, -math.inf).masked_fill(~given, 0)
    out = {'logp': logp, 'entropy': entropy, 'top_logp': None, 'top_index': None}
    if s.case['top']:
        # one whole number an element, by score and then the lowest index: no two are alike
        bits = (x + 0.0).view(torch.int32)
        key = (torch.where(bits < 0, bits ^ 0x7fffffff, bits).long() << 32) - torch.arange(vocab, device=x.device)
        del bits
        index = key.topk(s.case['top'], 1).indices
        out['top_logp'] = v.gather(1, index) - log_sum[:, None]
        out['top_index'] = index.int()
    return out


def _plain_logprobs_grad(s):
    x = _in_width(s).float()
    m, log_sum, entropy = s.stats[:, 0:1], s.stats[:, 1:2], s.stats[:, 2:3]
    empty = m == -math.inf
    lp = x - m.masked_fill(empty, 0) - log_sum
    p = lp.exp()
    given = s.tokens >= 0
    g = s.grad_logp * given
    grad = -p * (g.sum(1, keepdim=True) + (s.grad_entropy[:, None] * (lp + entropy)).masked_fill(p == 0, 0))
    grad.scatter_add_(1, s.tokens.clamp(min=0), g)
    return {'grad': grad.masked_fill(empty, 0).to(s.logits.dtype)}


def _plain_route(s):
    c = s.case
    rows, experts = s.logits.shape
    x = s.logits.float()
    wide = s.logits.double()            # which of two near scores is larger is decided in 64 bits
    p = wide.softmax(1) if c['score'] == 'softmax' else 1 / (1 + (-wide).exp())
    order = (p + s.bias if s.bias is not None else wide).clamp(min=-1e300)
    if c['groups'] > 1:
        per_group = (p if s.bias is None else order).view(rows, c['groups'], -1)
        if c['group_score'] == 'max':
            of_group = (order.view(rows, c['groups'], -1)).max(2).values
        else:
            of_group = per_group.sort(dim=2, descending=True).values[:, :, :2].sum(2)
        chosen = of_group.sort(dim=1, descending=True, stable=True).indices[:, :c['top_groups']]
        kept = torch.zeros_like(of_group, dtype=torch.bool).scatter_(1, chosen, True)
        order = order.view(rows, c['groups'], -1).masked_fill(~kept[:, :, None], -math.inf).view(rows, experts)
    index = order.sort(dim=1, descending=True, stable=True).indices[:, :c['top']]
    if c['score'] == 'softmax':
        e = (x - x.max(1, keepdim=True).values).exp()
        weights = (e / e.sum(1, keepdim=True)).gather(1, index)
    else:
        weights = 1 / (1 + (-x.gather(1, index)).exp())
    if c['renormalise']:
        weights = weights / weights.sum(1, keepdim=True)
    return {'weights': weights * c['scale'], 'index': index.int()}


def _plain_route_grad(s):
    c = s.case
    x = s.logits.float()
    index = s.index.long()
    g = s.grad_weights * c['scale']
    if c['score'] == 'softmax':
        e = (x - x.max(1, keepdim=True).values).exp()
        p = e / e.sum(1, keepdim=True)
        at = p.gather(1, index)
    else:
        at = 1 / (1 + (-x.gather(1, index)).exp())
    if c['renormalise']:
        total = at.sum(1, keepdim=True)
        g = (g - (g * at).sum(1, keepdim=True) / total) / total
    grad = torch.zeros_like(x)
    if c['score'] == 'softmax':
        grad.scatter_add_(1, index, g)
        grad = p * (grad - (g * at).sum(1, keepdim=True))
    else:
        grad.scatter_add_(1, index, g * at / (1 + x.gather(1, index).exp()))
    return {'grad': grad.to(s.logits.dtype)}


# ---- the definitions in 64 bits ------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    parts = []
    step = max(1, (1 << 26) // s.logits.shape[1])
    with torch.no_grad():
        for lo in range(0, case['rows'], step):
            parts.append(_EXACT[case['op']](s, slice(lo, min(case['rows'], lo + step))))
    return {k: None if parts[0][k] is None else torch.cat([q[k] for q in parts]) for k in parts[0]}


def _exact_rows(s, rows):
    x = s.logits[rows].to(torch.float64, copy=True)
    if s.widths is not None:
        x[torch.arange(x.shape[1], device=x.device)[None] >= s.widths[rows][:, None]] = -math.inf
    lse = torch.logsumexp(x, 1, keepdim=True)
    return x, lse, x - torch.where(lse == -math.inf, 0.0, lse)


def _exact_logprobs(s, rows):
    x, lse, lp = _exact_rows(s, rows)
    entropy = -torch.special.xlogy(lp.exp(), lp.exp()).sum(1)
    tokens = s.tokens[rows]
    logp = torch.where(tokens < 0, 0.0, lp.gather(1, tokens.clamp(min=0)))
    out = {'logp': logp, 'entropy': entropy, 'top_logp': None, 'top_index': None}
    found, places = [], torch.arange(x.shape[1], device=x.device)
    taken = torch.zeros_like(x, dtype=torch.bool)
    for _ in range(s.case['top']):      # the largest that is left, at its first place
        best = torch.where(taken, -math.inf, x).max(1, keepdim=True).values
        at = torch.where((x == best) & ~taken, places, x.shape[1]).min(1, keepdim=True).values
        taken.scatter_(1, at, True)
        found.append(at)
    if found:
        out['top_index'] = torch.cat(found, 1).int()
        out['top_logp'] = lp.gather(1, out['top_index'].long())
    return out


def _exact_logprobs_grad(s, rows):
    x, lse, lp = _exact_rows(s, rows)
    tokens, g = s.tokens[rows], s.grad_logp[rows].double()
    p = lp.exp()
    plogp = torch.special.xlogy(p, p)
    # d logp_t / dx_j = [j = t] - p_j;   d H / dx_j = -p_j log p_j - p_j H
    g = torch.where(tokens < 0, 0.0, g)
    grad = torch.zeros_like(x).scatter_add_(1, tokens.clamp(min=0), g) - p * g.sum(1, keepdim=True)
    grad -= s.grad_entropy[rows].double()[:, None] * (plogp - p * plogp.sum(1, keepdim=True))
    return {'grad': torch.where(lse == -math.inf, 0.0, grad)}


def _exact_probability(c, x):
    if c['score'] == 'sigmoid':
        return torch.sigmoid(x)
    return (x - torch.logsumexp(x, 1, keepdim=True)).exp()


def _exact_route(s, rows):
    c, x = s.case, s.logits[rows].double()
    p = _exact_probability(c, x)
    by = x if s.bias is None else p + s.bias.double()
    size = x.shape[1] // c['groups']
    group_of = torch.arange(x.shape[1], device=x.device) // size
    if c['group_score'] == 'max':
        of_group = torch.stack([by[:, group_of == k].max(1).values for k in range(c['groups'])], 1)
    else:
        sums = p if s.bias is None else by
        of_group = torch.stack([sums[:, group_of == k].topk(min(2, size), 1).values.sum(1) for k in range(c['groups'])], 1)
    # rank of a group: how many come before it, the lower index first among equals
    before = (of_group[:, None, :] > of_group[:, :, None]) | ((of_group[:, None, :] == of_group[:, :, None]) & torch.ones(
        c['groups'], c['groups'], dtype=torch.bool, device=x.device).tril(-1))
    left = (before.sum(2) < c['top_groups'])[:, group_of]
    found, places = [], torch.arange(x.shape[1], device=x.device)
    for _ in range(c['top']):
        best = torch.where(left, by, -math.inf).max(1, keepdim=True).values
        at = torch.where((by == best) & left, places, x.shape[1]).min(1, keepdim=True).values
        left = left.scatter(1, at, False)
        found.append(at)
    index = torch.cat(found, 1)
    weights = p.gather(1, index)
    if c['renormalise']:
        weights = weights / weights.sum(1, keepdim=True)
    return {'weights': weights * c['scale'], 'index': index.int()}


def _exact_route_grad(s, rows):
    c, x, index = s.case, s.logits[rows].double(), s.index[rows].long()
    p, g = _exact_probability(c, x), s.grad_weights[rows].double() * c['scale']
    at = p.gather(1, index)
    if c['renormalise']:        # d(w_i / sum w) / dw_j = [i = j] / sum w - w_i / (sum w)^2
        total = at.sum(1, keepdim=True)
        g = g / total - (g * at).sum(1, keepdim=True) / total ** 2
    dp = torch.zeros_like(x).scatter_add_(1, index, g)
    if c['score'] == 'sigmoid':
        return {'grad': dp * p * torch.sigmoid(-x)}
    return {'grad': p * (dp - (dp * p).sum(1, keepdim=True))}


_EXACT = {'logprobs': _exact_logprobs, 'logprobs_grad': _exact_logprobs_grad, 'route': _exact_route,
          'route_grad': _exact_route_grad}
