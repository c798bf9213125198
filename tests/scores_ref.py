"""Plain float64 restatement of the operators on rows of scores, row by row, for the tests."""
import numpy as np


def _row(x, width):
    x = np.array(x, np.float64)
    x[max(0, min(len(x), width)):] = -np.inf
    return x


def _statistics(x):
    m = x.max()
    if m == -np.inf:
        return m, 0.0, 0.0
    with np.errstate(invalid='ignore', divide='ignore'):
        e = np.exp(x - m)
        s = e.sum()
        # 0 * -inf is nothing
        return m, np.log(s), np.log(s) - np.where(e == 0, 0, e * np.where(e == 0, 0, x - m)).sum() / s


def best(x, k):
    """Places of the k largest, equal ones by the lower place."""
    return np.argsort(-(x + 0.0), kind='stable')[:k]


def logprobs(x, tokens, top=0, widths=None):
    """``(logp, entropy, top_logp, top_index, stats)`` of (rows, columns) scores, tokens (rows, n)."""
    rows, columns = x.shape
    logp = np.zeros(tokens.shape)
    entropy, stats = np.zeros(rows), np.zeros((rows, 3))
    top_logp, top_index = np.zeros((rows, top)), np.zeros((rows, top), np.int32)
    for r in range(rows):
        v = _row(x[r], columns if widths is None else widths[r])
        m, log_sum, entropy[r] = _statistics(v)
        stats[r] = m, log_sum, entropy[r]
        bad = np.isnan(v).any() or m == np.inf
        if bad:
            entropy[r] = stats[r, 1] = stats[r, 2] = np.nan
        for t, tok in enumerate(tokens[r]):
            if tok < 0:
                continue
            if bad:
                logp[r, t] = np.nan
            elif tok >= columns or v[tok] == -np.inf:
                logp[r, t] = -np.inf
            else:
                logp[r, t] = v[tok] - m - log_sum
        at = best(v, top)
        if bad:
            top_index[r], top_logp[r] = -1, np.nan
        elif m == -np.inf:
            top_index[r], top_logp[r] = at, -np.inf
        else:
            top_index[r], top_logp[r] = at, v[at] - m - log_sum
    return logp, entropy, top_logp, top_index, stats


def logprobs_grad(x, tokens, g_logp, g_entropy, widths=None):
    rows, columns = x.shape
    grad = np.zeros(x.shape)
    for r in range(rows):
        v = _row(x[r], columns if widths is None else widths[r])
        m, log_sum, h = _statistics(v)
        if m == -np.inf:
            continue
        lp = v - m - log_sum
        p = np.exp(lp)
        given = tokens[r] >= 0
        grad[r] = -p * (g_logp[r][given].sum() + g_entropy[r] * (np.where(p == 0, 0, lp) + h))
        for t, tok in enumerate(tokens[r]):
            if 0 <= tok < (columns if widths is None else widths[r]):
                grad[r, tok] += g_logp[r, t]
    return grad


def probability(x, score):
    with np.errstate(over='ignore'):
        if score == 'sigmoid':
            return 1 / (1 + np.exp(-x))
    m = x.max()
    if m == -np.inf:
        return np.zeros_like(x)
    e = np.exp(x - m)
    return e / e.sum()


def route_row(x, top, score='softmax', bias=None, groups=1, top_groups=None, group_score='max'):
    """The chosen experts of one row."""
    p = probability(x, score)
    by = x + 0.0 if bias is None else p + bias
    by = np.where(np.isnan(by), -np.inf, by)
    per = len(x) // groups
    eligible = list(range(len(x)))
    if groups > 1:
        of = []
        for g in range(groups):
            part = slice(g * per, (g + 1) * per)
            if group_score == 'max':
                of.append(by[part].max())
            else:
                of.append(np.sort((p if bias is None else by)[part])[::-1][:2].sum())
        chosen = best(np.array(of), groups if top_groups is None else top_groups)
        eligible = [j for j in eligible if j // per in chosen]
    return np.array(sorted(eligible, key=lambda j: (-by[j], j))[:top])


def route(x, top, renormalise=True, scale=1.0, **how):
    rows = x.shape[0]
    weights, index = np.zeros((rows, top)), np.zeros((rows, top), np.int32)
    for r in range(rows):
        if np.isnan(x[r]).any() or (how.get('score', 'softmax') == 'softmax' and (x[r] == np.inf).any()):
            weights[r], index[r] = np.nan, -1
            continue
        index[r] = route_row(x[r], top, **how)
        weights[r] = scale * weights_of(x[r], index[r], how.get('score', 'softmax'), renormalise)
    return weights, index


def weights_of(x, index, score, renormalise):
    w = probability(x, score)[index]
    if renormalise:
        w = w / w.sum() if w.sum() > 0 else np.zeros(len(w))
    return w


def route_grad(x, index, g, score='softmax', renormalise=True, scale=1.0):
    grad = np.zeros(x.shape)
    for r in range(x.shape[0]):
        have = (index[r] >= 0) & (index[r] < x.shape[1])
        at, gr = index[r][have], g[r][have] * scale
        p = probability(x[r], score)
        w = p[at]
        if renormalise:
            if not len(at) or w.sum() == 0:
                continue
            gr = gr / w.sum() - (gr * w).sum() / w.sum() ** 2
        dp = np.zeros(x.shape[1])
        np.add.at(dp, at, gr)
        if score == 'sigmoid':
            grad[r] = dp * p * probability(-x[r], 'sigmoid')
        else:
            grad[r] = p * (dp - (dp * p).sum())
    return grad
