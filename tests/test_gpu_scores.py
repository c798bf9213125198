"""Rows of scores on the GPU, against the float64 restatement in ``scores_ref``.

Tolerances.  u = 2^-24 is half a step of float32, relative.  A statistic is a sum of n positive terms, each
off by a few u and by |t| u for the rounding of its exponent (where it counts: t e^t <= 0.6), added in at most
n / 64 + 64 steps a lane and its reductions; with the exponential, the logarithm and the rescalings that is
below (n / 64 + 96) u, absolutely, for log S, and times (1 + log n) for the entropy.  ``x - m - log S`` adds
2 u of its largest operand.  A gradient is formed from these in a dozen roundings of its parts and then
rounded to its type: half a step, or half the smallest number.
"""
import math

import numpy as np
import pytest

from tests import scores_ref as ref

torch = pytest.importorskip('torch')
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
#: half of the smallest positive number of a type
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def _scores():
    from poseestimation_amd import scores
    return scores


def _rows(rows, cols, dtype, seed=0, scale=2.5):
    g = torch.Generator().manual_seed(seed + rows * 7919 + cols)
    x = torch.randn(rows, cols, generator=g) * scale
    x[torch.arange(rows), torch.randint(cols, (rows,), generator=g)] += 6
    return x.to(TYPES[dtype]).cuda()


def _tokens(rows, cols, n, seed=0):
    g = torch.Generator().manual_seed(seed + 17)
    return torch.randint(cols, (rows, n), generator=g).cuda()


def _np(x):
    return x.double().cpu().numpy() if x.is_floating_point() else x.cpu().numpy()


def _close(got, want, tol, what):
    # a value past the largest number of the type by half a step or more (the difference of two scores near that
    # number, say) rounds to infinity
    last = torch.finfo(got.dtype).max * (1 + torch.finfo(got.dtype).eps / 4)
    want = np.where(np.abs(want) >= last, np.copysign(np.inf, want), want)
    got = _np(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]) and np.array_equal(np.isinf(got), inf), what
    fine = np.isfinite(want)
    off = np.abs(got[fine] - want[fine]) - np.broadcast_to(tol, want.shape)[fine]
    assert not off.size or off.max() <= 0, '%s: %g over its tolerance' % (what, off.max())


def _check_logprobs(x, tokens=None, top=0, widths=None):
    r = _scores().token_logprobs(x, tokens, top=top, widths=widths)
    torch.cuda.synchronize()
    rows, cols = x.shape
    tok = np.zeros((rows, 0), np.int64) if tokens is None else _np(tokens).reshape(rows, -1)
    w = None if widths is None else np.clip(_np(widths), 0, cols)
    logp, entropy, top_logp, top_index, stats = ref.logprobs(_np(x), tok, top, w)
    err = (cols / 64 + 96) * U
    if tokens is not None:
        size = np.where(np.isfinite(logp), np.abs(logp), 0)
        _close(r.logp.reshape(rows, -1), logp, err + 2 * U * (size + math.log(cols + 1)), 'logp')
        assert r.logp.shape == tokens.shape
    _close(r.entropy, entropy, err * (1 + math.log(cols + 1)), 'entropy')
    if top:
        assert np.array_equal(_np(r.top_index), top_index), 'top_index'
        size = np.where(np.isfinite(top_logp), np.abs(top_logp), 0)
        _close(r.top_logp, top_logp, err + 2 * U * (size + math.log(cols + 1)), 'top_logp')
    else:
        assert r.top_logp is None and r.top_index is None
    # a row with a NaN or +inf: the first column is the largest of what is no NaN, or a NaN
    fine = np.isfinite(entropy)
    _close(r.stats[torch.from_numpy(fine).cuda()], stats[fine],
           np.array([0, err, err * (1 + math.log(cols + 1))]), 'stats')
    return r


def _check_many(x, tokens=None, top=0, widths=None, times=19):
    """The rows of x over and over: a call of many rows, cut differently, against the restatement for the first ones
    and itself for the others."""
    one = _check_logprobs(x, tokens, top, widths)
    rows = x.shape[0]

    def again(v):
        return None if v is None else v.repeat(times, *[1] * (v.dim() - 1))
    many = _scores().token_logprobs(again(x), again(tokens), top=top, widths=again(widths))
    err = (x.shape[1] / 64 + 96) * U * (1 + math.log(x.shape[1] + 1))
    for a, b in zip(many, one):
        if a is not None:
            first = a[:rows]
            assert torch.equal(a.nan_to_num(nan=7.0), first.repeat(times, *[1] * (a.dim() - 1)).nan_to_num(nan=7.0))
            if a.dtype == torch.int32:
                assert torch.equal(first, b)
            else:
                _close(first, _np(b), 2 * err + 4 * U * np.abs(np.nan_to_num(_np(b), posinf=0, neginf=0)), 'many rows')
    return one


SHAPES = [(1, 1, 1), (3, 2, 2), (5, 63, 3), (2, 64, 64), (4, 65, 5), (300, 7, 7), (7, 368, 5), (33, 656, 3), (3, 1000, 20),
          (9, 1024, 1), (5, 1025, 9), (2, 2047, 64), (3, 2049, 8), (4, 4099, 0), (2, 8193, 17), (3, 32003, 8), (2, 50021, 33),
          (1, 131072, 20), (1, 131073, 64), (2, 262149, 5),
          (1, 1200001, 7)]


@pytest.mark.parametrize('dtype', list(TYPES))
@pytest.mark.parametrize('rows, cols, top', SHAPES)
def test_logprobs(rows, cols, top, dtype):
    _check_logprobs(_rows(rows, cols, dtype), _tokens(rows, cols, 3), top)


@pytest.mark.parametrize('rows, cols, top', [(600, 5000, 4), (1500, 513, 6), (5000, 90, 2), (2100, 1030, 0)])
def test_logprobs_of_many_rows(rows, cols, top):
    _check_logprobs(_rows(rows, cols, 'bf16'), _tokens(rows, cols, 1)[:, 0], top)


@pytest.mark.parametrize('dtype', list(TYPES))
@pytest.mark.parametrize('cols', [5, 300, 2100, 9001, 140000])
def test_logprobs_of_masked_infinite_equal_and_nan_rows(cols, dtype):
    low = torch.finfo(TYPES[dtype]).min
    high = torch.finfo(TYPES[dtype]).max
    x = _rows(15, cols, dtype, seed=3)
    x[0] = -math.inf                              # nothing left
    x[1, 1:] = -math.inf                          # one left
    x[2] = low                                    # masked by the lowest value, whole
    x[3, :-2] = low                               # and all but the last two
    x[4] = 1.5                                    # all equal
    x[5, ::2] = -0.0                              # zeros of both signs
    x[5, 1::2] = 0.0
    x[6, cols // 2] = math.nan
    x[7, cols - 1] = math.inf
    x[8] = -math.inf
    x[8, cols - 1] = math.nan
    x[9] = torch.where(torch.arange(cols, device='cuda') % 3 == 0, 2.0, -math.inf).to(x.dtype)
    x[10] = torch.arange(cols, device='cuda').float().mul_(20.0 / cols).to(x.dtype)      # rising
    x[11] = torch.arange(cols, device='cuda').float().mul_(-20.0 / cols).to(x.dtype)     # falling
    x[12, 0] = high
    x[13] = low
    x[13, cols // 3] = high
    x[14] = (torch.arange(cols, device='cuda') % 4).to(x.dtype)                          # four values, many ties
    top = min(cols, 40)
    # (thousands of rows: several to a wavefront where they are short)
    _check_many(x, _tokens(15, cols, 4, seed=cols), top, times=1200 if cols < 1000 else 19)
    _check_many(x, _tokens(15, cols, 20, seed=cols), min(5, cols), times=1200 if cols < 1000 else 300 if cols < 5000 else 19)
    _check_logprobs(x[:1], None, 0)


@pytest.mark.parametrize('cols, period', [(131072, 256), (131072, 64), (131072, 2048), (32768, 1024), (262144, 8192),
                                          (262144, 4096), (40000, 2048)])
def test_alternatives_that_all_lie_in_few_lanes(cols, period):
    """The largest entries a fixed distance apart: where columns are dealt out to threads, a few threads hold them all."""
    x = _rows(2, cols, 'f32', seed=11)
    at = torch.arange(5, cols, period, device='cuda')
    x[0, at] = 50 + torch.arange(len(at), device='cuda').float() * 0.01
    x[1, at] = 50 - torch.arange(len(at), device='cuda').float() * 0.01
    for top in (3, 64):
        _check_many(x, None, top, times=128)
    _check_many(x.bfloat16(), None, 50, times=128)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_alternatives_of_short_rows_that_lie_in_few_lanes_and_of_many(dtype):
    """Columns as they are dealt out to 16, 32 or 64 lanes in pieces of 4 or 8: all the large ones to one lane."""
    piece = 4 if dtype == 'f32' else 8
    for cols, lanes in ((500, 16), (1000, 32), (2000, 64), (500, 64)):
        x = _rows(4, cols, dtype, seed=cols)
        column = torch.arange(cols, device='cuda')
        for r, lane in enumerate((3, 0, lanes - 1, 7)):
            mine = (column // piece) % lanes == lane
            x[r] = torch.where(mine, 20 + (column if r % 2 else -column).float() / 32, x[r].float()).to(x.dtype)
        for top in (1, 5, 8, 13, 30):
            _check_many(x, None, top, times=64 * 4096 // lanes // 4)
    for rows, cols in ((5, 300), (3, 1000), (2, 2000), (4, 100), (3, 3000)):
        for top in (17, 20, 33, 50, 64):
            _check_logprobs(_rows(rows, cols, dtype, seed=top), None, top)


@pytest.mark.parametrize('cols, top', [(131072, 64), (600000, 20), (1500000, 64)])
def test_alternatives_of_long_rows_with_equal_scores(cols, top):
    """Slices whose keys are all alike: constant rows, few scores that are not masked, two values, whole steps."""
    for fill, some in ((1.0, None), (-math.inf, 5), (-math.inf, 300), (0.0, 17), (-3e38, 3)):
        x = torch.full((2, cols), fill, dtype=torch.bfloat16, device='cuda')
        if some:
            at = torch.randperm(cols, generator=torch.Generator().manual_seed(some))[:some].cuda()
            x[0, at] = 2.0
            x[1, at] = torch.arange(some, device='cuda').bfloat16()
        _check_logprobs(x, _tokens(2, cols, 2), top)
    x = torch.randint(0, 4, (2, cols), generator=torch.Generator().manual_seed(cols)).to(torch.bfloat16).cuda()
    _check_logprobs(x, None, top, torch.tensor([cols, cols // 3], dtype=torch.int32, device='cuda'))


@pytest.mark.parametrize('cols', [40, 656, 5000, 20000])
def test_logprobs_of_ragged_rows(cols):
    x = _rows(11, cols, 'bf16', seed=5)
    widths = torch.tensor([0, 1, 2, 3, cols // 2, cols - 1, cols, cols + 9, -4, 17, cols], dtype=torch.int32, device='cuda')
    for r, w in enumerate(widths.tolist()):
        x[r, max(0, min(w, cols)):] = math.nan
    x[9, :17] = -math.inf
    _check_many(x, _tokens(11, cols, 5), 20, widths, times=25)
    _check_logprobs(x, _tokens(11, cols, 5), 0, widths.long())


@pytest.mark.parametrize('dtype', list(TYPES))
def test_logprobs_of_strided_misaligned_and_expanded_rows(dtype):
    store = torch.full((6, 1300), math.nan, dtype=TYPES[dtype], device='cuda')
    for first, cols in ((1, 655), (3, 1001), (8, 64), (7, 1293)):
        x = store[:, first:first + cols]
        x.copy_(_rows(6, cols, dtype))
        _check_logprobs(x, _tokens(6, cols, 2), 4)
        _check_logprobs(x[::2], _tokens(3, cols, 2), 4)
        store.fill_(math.nan)
    one = _rows(1, 3001, dtype)
    _check_logprobs(one.expand(5, 3001), _tokens(5, 3001, 2), 7)
    _check_logprobs(one.t()[:, :1].contiguous(), None, 1)
    long = _rows(1, 600001, dtype)
    want, many = _check_logprobs(long, None, 9), _scores().token_logprobs(long.expand(300, 600001), top=9)
    assert torch.equal(many.top_index, want.top_index.expand(300, 9)) and (many.entropy - want.entropy).abs().max() < 1e-3
    _check_logprobs(_rows(50, 9, dtype)[:, 3:4], _tokens(50, 1, 1), 1)


def test_tokens_given_twice_not_given_and_out_of_the_row():
    x = _rows(6, 500, 'f32')
    tokens = _tokens(6, 500, 64)
    tokens[:, 1] = tokens[:, 0]
    tokens[:, 2] = -1
    tokens[:, 3] = 500
    tokens[:, 4] = 1 << 40
    tokens[:, 5] = -(1 << 40)
    r = _check_logprobs(x, tokens, 2)
    assert (r.logp[:, 2] == 0).all() and (r.logp[:, 3:5] == -math.inf).all() and torch.equal(r.logp[:, 0], r.logp[:, 1])
    _check_logprobs(x, tokens.int()[:, :3], 2)
    _check_logprobs(x, tokens.t().contiguous().t(), 2)


@pytest.mark.parametrize('dtype', [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64])
def test_tokens_widths_and_indices_of_every_size(dtype):
    s = _scores()
    x, tokens = _rows(9, 100, 'bf16'), _tokens(9, 100, 4)
    widths = torch.arange(9, device='cuda') * 12
    g = torch.rand(4, 9, device='cuda', dtype=torch.float64).t()
    want = s.token_logprobs(x, tokens, 3, widths.int())
    # (columns of the tokens first: copied into the order that is needed)
    got = s.token_logprobs(x, tokens.t().contiguous().t().to(dtype), 3, widths.to(dtype))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(s.token_logprobs_backward(x, got.stats, tokens.to(dtype), g, widths=widths.to(dtype)),
                       s.token_logprobs_backward(x, want.stats, tokens, g.float().contiguous(), widths=widths.int()))
    index = s.route_experts(x, 4).index
    assert torch.equal(s.route_experts_backward(x, index.to(dtype), g), s.route_experts_backward(x, index, g.float().contiguous()))


def test_rows_whose_offsets_pass_32_bits():
    store = torch.empty((1 << 32) + (1 << 20), dtype=torch.bfloat16, device='cuda')
    x = store.as_strided((3, 1000), ((1 << 31) + 8, 1))
    x.copy_(_rows(3, 1000, 'bf16'))
    tokens = _tokens(3, 1000, 2)
    r = _check_logprobs(x, tokens, 4)
    g, ge = torch.randn(3, 2, device='cuda'), torch.randn(3, device='cuda')
    want = _scores().token_logprobs_backward(x.contiguous(), r.stats, tokens, g, ge)
    got = _scores().token_logprobs_backward(x, r.stats, tokens, g, ge, out=x)
    assert got is x and torch.equal(x, want)
    x.copy_(_rows(3, 1000, 'bf16'))
    a, b = _scores().route_experts(x, 6), _scores().route_experts(x.contiguous(), 6)
    assert torch.equal(a.weights, b.weights) and torch.equal(a.index, b.index)


# ---- the gradient ----------------------------------------------------------------------------

def _grad_tolerance(x, want, tokens, g, ge, widths=None):
    """Half a step of the type, and 32 roundings of the parts on top of the statistics' own error."""
    rows, cols = x.shape
    tol = np.zeros((rows, cols))
    for r in range(rows):
        v = ref._row(_np(x)[r], cols if widths is None else widths[r])
        m, log_sum, h = ref._statistics(v)
        if m == -np.inf:
            continue
        lp = np.maximum(v - m - log_sum, -300)
        given = tokens[r] >= 0
        size = np.exp(lp) * (np.abs(g[r][given]).sum() + abs(ge[r]) * (np.abs(lp) + h)) * (1 + np.abs(lp))
        tol[r] = ((cols / 64 + 96) * U * (1 + math.log(cols + 1)) + 32 * U) * size
        for t, tok in enumerate(tokens[r]):
            if 0 <= tok < cols:
                tol[r, tok] += 64 * U * np.abs(g[r]).sum()
    kind = x.dtype
    return tol * 1.01 + np.abs(want) * torch.finfo(kind).eps / 2 + TINY[kind] + 1e-37


def _check_grad(x, tokens, widths=None, out=None, entropy=True):
    rows, cols = x.shape
    gen = torch.Generator().manual_seed(rows + cols)
    r = _scores().token_logprobs(x, tokens, widths=widths)
    g = torch.randn(tokens.shape, generator=gen).cuda()
    ge = torch.randn(rows, generator=gen).cuda() if entropy else None
    before = x.clone()
    got = _scores().token_logprobs_backward(x, r.stats, tokens, g, ge, widths=widths, out=out)
    torch.cuda.synchronize()
    assert got.dtype == x.dtype and (out is None or got is out)
    if out is None or out.data_ptr() != x.data_ptr():
        assert torch.equal(x.view(torch.uint8) if x.is_contiguous() else x.nan_to_num(), before.view(torch.uint8)
                           if x.is_contiguous() else before.nan_to_num())
    tok = _np(tokens).reshape(rows, -1)
    w = None if widths is None else np.clip(_np(widths), 0, cols)
    gg, gge = _np(g).reshape(rows, -1), np.zeros(rows) if ge is None else _np(ge)
    want = ref.logprobs_grad(_np(before), tok, gg, gge, w)
    _close(got, want, _grad_tolerance(before, want, tok, gg, gge, w), 'grad')
    return got


@pytest.mark.parametrize('dtype', list(TYPES))
@pytest.mark.parametrize('rows, cols', [(1, 1), (3, 2), (70, 63), (4, 65), (7, 368), (33, 656), (3, 1025), (2, 2049), (5, 8193),
                                        (3, 32003), (1, 131073)])
def test_logprobs_gradient(rows, cols, dtype):
    tokens = _tokens(rows, cols, 3)
    tokens[:, 1] = tokens[:, 0]
    tokens[0, 2] = -1
    _check_grad(_rows(rows, cols, dtype), tokens)
    _check_grad(_rows(rows, cols, dtype, seed=1), tokens[:, 0], entropy=False)


def test_logprobs_gradient_of_masked_ragged_strided_and_shared_buffers():
    for cols in (30, 700, 9000):
        x = _rows(8, cols, 'f32', seed=2)
        x[0] = -math.inf
        x[1, 1:] = -math.inf
        x[2, ::2] = -math.inf
        x[3] = torch.finfo(torch.float32).min
        tokens = _tokens(8, cols, 64)
        tokens[:, ::5] = tokens[:, :1]
        tokens[:, 3] = cols
        widths = torch.tensor([cols, cols, cols, cols, cols // 2, 1, 0, 3], dtype=torch.int32, device='cuda')
        tokens = torch.where((tokens < widths[:, None]) | (tokens == cols), tokens, -1)
        got = _check_grad(x, tokens, widths)
        assert not got[0].any() and not got[6].any() and not got[7, 3:].any()
        store = torch.full((8, cols + 5), 7.0, device='cuda').bfloat16()
        y = store[:, 1:cols + 1]
        y.copy_(x.bfloat16())
        _check_grad(y, tokens, widths, out=y)
        assert (store[:, 0] == 7).all() and (store[:, cols + 1:] == 7).all()
        wide = torch.full((8, cols + 9), 3.0, device='cuda').bfloat16()
        _check_grad(x.bfloat16(), tokens, widths, out=wide[:, 4:cols + 4])
        assert (wide[:, :4] == 3).all() and (wide[:, cols + 4:] == 3).all()
        _check_grad(x[2:3].expand(4, cols), tokens[:4] % cols)


def test_logprobs_gradient_against_differences():
    """Along a random direction, against central differences of the float64 restatement's values."""
    x = _rows(6, 777, 'f32', seed=9)
    tokens = _tokens(6, 777, 3)
    g, ge = torch.randn(6, 3, device='cuda'), torch.randn(6, device='cuda')
    r = _scores().token_logprobs(x, tokens)
    grad = _np(_scores().token_logprobs_backward(x, r.stats, tokens, g, ge))
    d = np.random.default_rng(1).normal(size=x.shape)

    def value(h):                       # of every row
        logp, entropy = ref.logprobs(_np(x) + h * d, _np(tokens))[:2]
        return (logp * _np(g)).sum(1) + entropy * _np(ge)
    slope = (value(1e-4) - value(-1e-4)) / 2e-4
    per_row = (grad * d).sum(1)
    # the difference is good to (1e-4)^2 times a third derivative of order |d|^3 |g|; the kernel to some hundred u
    assert np.abs(per_row - slope).max() < 1e-5 * (1 + np.abs(slope).max())


# ---- routing ---------------------------------------------------------------------------------

def _check_route(x, top, **how):
    bias = how.pop('bias', None)
    r = _scores().route_experts(x, top, bias=bias, **how)
    torch.cuda.synchronize()
    more = dict(how)
    if bias is not None:
        more['bias'] = _np(bias.float())
    weights, index = ref.route(_np(x), top, **more)
    assert np.array_equal(_np(r.index), index), 'index'
    # the exponent's rounding (|x - m| u), the exponential and the sums: 64 u and the spread of the row
    spread = np.nan_to_num(np.where(np.isfinite(_np(x)), np.abs(_np(x)), 0)).max() * 2
    _close(r.weights, weights, np.abs(np.nan_to_num(weights)) * (64 + 2 * spread) * U + 1e-37, 'weights')
    return r


WAYS = [dict(), dict(renormalise=False), dict(score='sigmoid', scale=2.5), dict(score='sigmoid', renormalise=False)]


@pytest.mark.parametrize('dtype', list(TYPES))
@pytest.mark.parametrize('rows, experts, top', [(1, 1, 1), (1, 64, 4), (5, 2, 2), (70, 8, 2), (9, 31, 31), (3, 33, 32), (130, 60, 6),
                                                (257, 128, 8), (33, 160, 6), (65, 256, 8), (5, 257, 9), (17, 384, 16), (3, 512, 10),
                                                (2, 1000, 32), (4, 1024, 1)])
def test_route(rows, experts, top, dtype):
    x = _rows(rows, experts, dtype, scale=1.5)
    bias = torch.randn(experts, generator=torch.Generator().manual_seed(experts)).mul_(0.05).cuda()
    for how in WAYS:
        _check_route(x, top, **how)
        _check_route(x, top, bias=bias, **how)
        _check_route(x, top, bias=torch.zeros_like(bias), **how)


@pytest.mark.parametrize('experts, groups, top_groups, top', [(256, 8, 4, 8), (160, 8, 3, 6), (64, 64, 5, 5), (60, 4, 1, 4),
                                                              (24, 12, 3, 6), (512, 2, 1, 32), (1024, 32, 7, 20), (96, 3, 2, 8),
                                                              (33, 11, 11, 3), (1000, 40, 2, 4)])
@pytest.mark.parametrize('group_score', ['max', 'top2'])
def test_route_in_groups(experts, groups, top_groups, top, group_score):
    bias = torch.randn(experts, generator=torch.Generator().manual_seed(experts)).mul_(0.05).cuda()
    for k, dtype in enumerate(TYPES):
        x = _rows(41, experts, dtype, seed=k, scale=1.5)
        for how in WAYS:
            how = dict(how, groups=groups, top_groups=top_groups, group_score=group_score)
            _check_route(x, top, **how)
            _check_route(x, top, bias=bias, **how)


@pytest.mark.parametrize('groups', [1, 4])
def test_route_of_masked_equal_and_nan_rows(groups):
    for experts, top in ((8, 2), (64, 8), (256, 8), (1000, 20)):
        x = _rows(12, experts, 'f32', seed=4)
        x[0] = -math.inf
        x[1, 1:] = -math.inf
        x[2] = 0.25
        x[3] = torch.finfo(torch.float32).min
        x[4, experts // 2] = math.nan
        x[5, ::2] = x[5, 1::2]                          # pairs of equals
        x[6] = -200 - torch.arange(experts, device='cuda').float() * 0.01    # a sigmoid below every normal number
        x[7] = 300
        x[8, :] = -0.0
        x[8, ::3] = 0.0
        x[9, experts - 1] = -math.inf
        x[10] = torch.arange(experts, device='cuda').float() * 1e-7
        x[11] = 1e-3 * (torch.arange(experts, device='cuda') % 5)
        zero, some = torch.zeros(experts, device='cuda'), torch.zeros(experts, device='cuda')
        some[experts // 3:] = -math.inf
        some[experts // 2] = math.nan
        for how in WAYS[:2] + WAYS[3:]:
            for group_score in ('max', 'top2'):
                how = dict(how, groups=groups, top_groups=max(1, groups // 2), group_score=group_score)
                t = min(top, experts // groups * how['top_groups'])
                keep = torch.arange(12, device='cuda') != (6 if how.get('score') == 'sigmoid' else 99)
                _check_route(x[keep], t, **how)
                _check_route(x[keep], t, bias=zero, **how)
                if group_score == 'max':
                    _check_route(x[keep], t, bias=some, **how)
    x = torch.full((2, 64), -200.0, device='cuda')
    x[1] = -200 + torch.arange(64, device='cuda') * 0.125
    r = _scores().route_experts(x, 8, score='sigmoid', scale=2.0)
    # values too small for float32 still share out the weight: e^-200 / (8 e^-200)
    assert torch.allclose(r.weights[0], torch.full((8,), 0.25, device='cuda'), rtol=1e-6)
    e = torch.exp(torch.arange(8, device='cuda') * -0.125)
    assert torch.allclose(r.weights[1], 2 * e / e.sum(), rtol=1e-5) and r.index[1, 0] == 63
    x[0, 3] = math.inf
    r = _scores().route_experts(x, 8)
    assert torch.isnan(r.weights[0]).all() and (r.index[0] == -1).all() and (r.index[1] >= 0).all()


def test_route_orders_near_scores_as_float64_does():
    """Scores that float32 cannot tell apart: p + bias with biases that undo the differences of p to 1e-9."""
    gen = torch.Generator().manual_seed(8)
    for experts, groups, top_groups in ((64, 1, 1), (256, 8, 4), (128, 1, 1)):
        x = (torch.randn(64, experts, generator=gen) * 0.8).cuda()
        for score in ('softmax', 'sigmoid'):
            for r in range(0, 64, 16):
                p = torch.from_numpy(ref.probability(_np(x)[r], score))
                bias = (0.5 - p).float().cuda()          # every p + bias of this row is 0.5, to 2^-25
                _check_route(x[r:r + 16], 8, bias=bias, score=score, groups=groups, top_groups=top_groups, group_score='top2')
                _check_route(x[r:r + 16], 8, bias=bias, score=score, groups=groups, top_groups=top_groups, group_score='max')


def test_route_orders_a_few_near_scores_in_and_around_the_list():
    """Six experts whose scores differ by less than float32 tells, at places that put them inside the list, at its end and
    beyond it, the other experts well apart."""
    gen = torch.Generator().manual_seed(21)
    for experts, groups, top_groups, top in ((64, 1, 1, 8), (256, 8, 4, 8), (256, 1, 1, 6), (160, 1, 1, 6), (1024, 1, 1, 8), (48, 1, 1, 2)):
        for above in (0, 1, 3, 5, 7, 9):
            for score in ('sigmoid', 'softmax'):
                x = (torch.randn(20, experts, generator=gen) * 0.8).cuda()
                p = torch.from_numpy(ref.probability(_np(x)[7], score))
                # apart by 2e-3, then `above` of them first and six to one value
                target = 0.25 + 2e-3 * torch.randperm(experts, generator=gen).double()
                order = target.argsort(descending=True)
                target[order[above:above + 6]] = target[order[above]].item()
                bias = (target - p).float().cuda()
                _check_route(x, top, bias=bias, score=score, groups=groups, top_groups=top_groups)


@pytest.mark.parametrize('dtype', list(TYPES))
def test_route_of_strided_misaligned_and_expanded_rows(dtype):
    store = torch.full((40, 300), math.nan, dtype=TYPES[dtype], device='cuda')
    for first, experts in ((1, 256), (3, 64), (8, 128), (16, 160), (4, 40)):
        x = store[:, first:first + experts]
        x.copy_(_rows(40, experts, dtype))
        _check_route(x, 4)
        _check_route(x[::3], 4, groups=4, top_groups=2)
        store.fill_(math.nan)
    _check_route(_rows(1, 64, dtype).expand(9, 64), 5, score='sigmoid')


def _check_route_grad(x, index, g, out=None, **how):
    before = _np(x)
    got = _scores().route_experts_backward(x, index, g, out=out, **how)
    torch.cuda.synchronize()
    assert got.dtype == x.dtype and (out is None or got is out)
    want = ref.route_grad(before, _np(index), _np(g), **how)
    # the parts: p (|g| + sum |g p|) times the scale, each with the weights' error and a dozen roundings
    spread = np.where(np.isfinite(before), np.abs(before), 0).max() * 2
    part = np.zeros_like(want)
    for r in range(len(want)):
        p = ref.probability(before[r], how.get('score', 'softmax'))
        at = _np(index)[r]
        have = (at >= 0) & (at < len(p))
        total = np.abs(_np(g)[r][have]).sum() * how.get('scale', 1.0)
        if how.get('renormalise', True):
            s = p[at[have]].sum()
            part[r] = total * (p / s if s > 0 else 0)
        else:
            part[r] = total * p
    part = np.minimum(part, np.abs(_np(g)).sum(1, keepdims=True) * how.get('scale', 1.0))
    tol = part * (128 + 4 * spread) * U * 1.01 + np.abs(want) * torch.finfo(x.dtype).eps / 2 + TINY[x.dtype] + 1e-37
    _close(got, want, tol, 'grad')
    return got


@pytest.mark.parametrize('dtype', list(TYPES))
@pytest.mark.parametrize('rows, experts, top', [(1, 1, 1), (1, 64, 4), (70, 8, 2), (9, 31, 31), (33, 160, 6), (65, 256, 8), (5, 257, 9),
                                                (2, 1000, 32), (300, 40, 3)])
def test_route_gradient(rows, experts, top, dtype):
    x = _rows(rows, experts, dtype, scale=1.5)
    gen = torch.Generator().manual_seed(rows)
    g = torch.randn(rows, top, generator=gen).cuda()
    for how in WAYS:
        index = _scores().route_experts(x, top, **how).index
        _check_route_grad(x, index, g, **how)
        twice = index.clone()
        twice[:, -1] = twice[:, 0]
        twice[0, 0] = -1
        twice[-1, 0] = experts
        _check_route_grad(x, twice, g, **how)
        store = torch.full((rows, experts + 3), 5.0, device='cuda').to(x.dtype)
        store[:, 1:experts + 1] = x
        _check_route_grad(store[:, 1:experts + 1], index, g, out=store[:, 1:experts + 1], **how)
        assert (store[:, 0] == 5).all() and (store[:, experts + 1:] == 5).all()


def test_route_gradient_of_masked_rows():
    x = _rows(6, 96, 'f32', seed=6)
    x[0] = -math.inf
    x[1, 5:] = -math.inf
    x[2] = 0.5
    x[3] = -60
    x[4] = 60
    g = torch.randn(6, 8, device='cuda')
    for how in WAYS:
        index = _scores().route_experts(x, 8, **how).index
        got = _check_route_grad(x, index, g, **how)
        assert not got[0].any()


def test_route_gradient_against_differences():
    x = _rows(5, 48, 'f32', seed=12, scale=1.0)
    g = torch.randn(5, 6, device='cuda')
    d = np.random.default_rng(2).normal(size=x.shape)
    for how in WAYS:
        score, renorm, scale = how.get('score', 'softmax'), how.get('renormalise', True), how.get('scale', 1.0)
        index = _scores().route_experts(x, 6, **how).index
        grad = _np(_scores().route_experts_backward(x, index, g, **how))

        def value(h):
            v = _np(x) + h * d
            return np.array([(scale * ref.weights_of(v[r], _np(index)[r], score, renorm) * _np(g)[r]).sum() for r in range(5)])
        slope = (value(1e-4) - value(-1e-4)) / 2e-4
        assert np.abs((grad * d).sum(1) - slope).max() < 1e-5 * (1 + np.abs(slope).max())


# ---- refusals, streams, graphs, and a run of them together --------------------------------------

def test_refusals_on_the_gpu():
    s = _scores()
    x = _rows(4, 64, 'f32')
    stats = torch.zeros(4, 3, device='cuda')
    idx, g = torch.zeros(4, 2, dtype=torch.int32, device='cuda'), torch.zeros(4, 2, device='cuda')
    bad = [lambda: s.token_logprobs(x.t()), lambda: s.token_logprobs(x[:, ::2]), lambda: s.token_logprobs(x, top=65),
           lambda: s.token_logprobs(x, top=-1), lambda: s.token_logprobs(x[:, :3], top=4), lambda: s.token_logprobs(x[:, :0]),
           lambda: s.token_logprobs(x, torch.zeros(4)), lambda: s.token_logprobs(x, torch.zeros(4, dtype=torch.int64)),
           lambda: s.token_logprobs(x, torch.zeros(4, device='cuda')), lambda: s.token_logprobs(x, idx[:3].long()),
           lambda: s.token_logprobs(x, torch.zeros(4, 65, dtype=torch.int64, device='cuda')),
           lambda: s.token_logprobs(x, torch.zeros(4, dtype=torch.bool, device='cuda')),
           lambda: s.token_logprobs(x, widths=torch.zeros(3, dtype=torch.int32, device='cuda')),
           lambda: s.token_logprobs_backward(x, stats), lambda: s.token_logprobs_backward(x, stats, idx.long()),
           lambda: s.token_logprobs_backward(x, stats[:, :2], idx.long(), g), lambda: s.token_logprobs_backward(x, stats, idx.long(), g[:, :1]),
           lambda: s.token_logprobs_backward(x, stats, idx.long(), g, out=x.bfloat16()),
           lambda: s.token_logprobs_backward(x, stats, idx.long(), g, out=x[:, :32]),
           lambda: s.token_logprobs_backward(x[:, :32], stats, idx.long(), g, out=x[:, 1:33]),
           lambda: s.token_logprobs_backward(x[:1].expand(4, 64), stats, idx.long(), g, out=x[:1].expand(4, 64)),
           lambda: s.route_experts(x, 0), lambda: s.route_experts(x, 33), lambda: s.route_experts(x, 4, score='relu'),
           lambda: s.route_experts(x, 4, groups=3), lambda: s.route_experts(x, 4, groups=4, top_groups=5),
           lambda: s.route_experts(x, 17, groups=4, top_groups=1), lambda: s.route_experts(x, 4, group_score='sum'),
           lambda: s.route_experts(x, 4, bias=torch.zeros(63, device='cuda')), lambda: s.route_experts(x, 4, bias=torch.zeros(64)),
           lambda: s.route_experts(torch.zeros(4, 1025, device='cuda'), 4), lambda: s.route_experts_backward(x, idx.float(), g),
           lambda: s.route_experts_backward(x, idx, g[:, :1]), lambda: s.route_experts_backward(x, idx[:2], g),
           lambda: s.route_experts_backward(x, idx[0], g), lambda: s.route_experts_backward(x, idx, g, out=x[:, :-1])]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail('call %d was not refused' % k)
    empty = x[:0]
    r = s.token_logprobs(empty, idx[:0].long(), top=3)
    assert r.logp.shape == (0, 2) and r.top_index.shape == (0, 3)
    assert s.token_logprobs_backward(empty, stats[:0], idx[:0].long(), g[:0]).shape == (0, 64)
    assert s.route_experts(empty, 3).index.shape == (0, 3) and s.route_experts_backward(empty, idx[:0], g[:0]).shape == (0, 64)


def test_calls_for_another_device_than_the_current_one(monkeypatch):
    """With the device reported as another one first, each function calls itself under the tensors' own: the same answer."""
    s = _scores()
    x, tokens = _rows(6, 300, 'bf16'), _tokens(6, 300, 2)
    widths = torch.tensor([300, 200, 100, 3, 0, 299], dtype=torch.int32, device='cuda')
    g, ge, bias = torch.randn(6, 2, device='cuda'), torch.randn(6, device='cuda'), torch.randn(300, device='cuda') * 0.01
    stats = s.token_logprobs(x, tokens, 4, widths).stats
    index = s.route_experts(x, 2).index
    out = torch.empty_like(x)
    how = dict(score='sigmoid', bias=bias, groups=10, top_groups=3, group_score='top2', renormalise=False, scale=1.5)
    calls = [lambda: s.token_logprobs(x, tokens, 4, widths), lambda: s.route_experts(x, 5, **how),
             lambda: (s.token_logprobs_backward(x, stats, tokens, g, ge, widths, out).clone(),),
             lambda: (s.route_experts_backward(x, index, g, 'sigmoid', False, 1.5, out).clone(),)]
    want = [c() for c in calls]
    answers = []
    monkeypatch.setattr(s, '_current', lambda device: answers.pop(0))
    for call, w in zip(calls, want):
        answers[:] = [False, True]
        got = call()
        assert not answers and all(torch.equal(a, b) for a, b in zip(got, w))


def test_calls_on_two_streams_at_once():
    s = _scores()
    xs = [_rows(3, 140001, 'bf16', seed=k) for k in range(4)]
    want = [s.token_logprobs(x, top=20) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(5):
        got = []
        for x, stream in zip(xs, streams):
            with torch.cuda.stream(stream):
                got.append(s.token_logprobs(x, top=20))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a[1:], b[1:]))


def _mixture(s, x, gate, heads, tokens, g):
    """Rows go to two of the heads; their scores, mixed, are read out; back to the gate and the heads."""
    routes = s.route_experts(gate, 2)
    rows = torch.arange(x.shape[0], device='cuda')[:, None]
    chosen = heads[routes.index.long()]                                  # (rows, 2, columns, depth)
    each = (chosen * x[:, None, None, :]).sum(3)
    mixed = (each * routes.weights[:, :, None]).sum(1)
    read = s.token_logprobs(mixed, tokens, top=4)
    d_mixed = s.token_logprobs_backward(mixed, read.stats, tokens, g, torch.full((x.shape[0],), 0.01, device='cuda'))
    d_weights = (each * d_mixed[:, None]).sum(2)
    d_gate = s.route_experts_backward(gate, routes.index, d_weights)
    d_heads = torch.zeros(heads.shape[0], x.shape[0], heads.shape[1], device='cuda')
    d_heads[routes.index.long(), rows] = routes.weights[:, :, None] * d_mixed[:, None]
    return routes.weights, routes.index, read.logp, read.entropy, read.top_logp, read.top_index, d_gate, d_heads


def _mixture_inputs(seed):
    gen = torch.Generator().manual_seed(seed)
    rows, depth, columns, n = 36, 16, 184, 8
    x, gate = torch.randn(rows, depth, generator=gen).cuda(), torch.randn(rows, n, generator=gen).cuda()
    heads = torch.randn(n, columns, depth, generator=gen).cuda()
    tokens = torch.randint(columns, (rows,), generator=gen).cuda()
    return x, gate, heads, tokens, torch.randn(rows, generator=gen).cuda()


def test_a_mixture_of_answering_heads_forward_and_backward():
    s = _scores()
    x, gate, heads, tokens, g = _mixture_inputs(3)
    got = _mixture(s, x, gate, heads, tokens, g)
    # the same in float64 with torch's own gradients, on the CPU; the choice of heads is taken over
    xd, hd = x.double().cpu(), heads.double().cpu()
    gd = gate.double().cpu().requires_grad_()
    index = got[1].long().cpu()
    assert np.array_equal(index.numpy(), ref.route(_np(gate), 2)[1])
    w = torch.softmax(gd, 1).gather(1, index)
    w = w / w.sum(1, keepdim=True)
    each = (hd[index] * xd[:, None, None, :]).sum(3)
    mixed = (each * w[:, :, None]).sum(1)
    lp = torch.log_softmax(mixed, 1)
    logp = lp.gather(1, tokens.cpu()[:, None])[:, 0]
    entropy = -(lp.exp() * lp).sum(1)
    mixed.retain_grad()
    ((logp * g.double().cpu()).sum() + 0.01 * entropy.sum()).backward()
    # products of depth 16 in float32, differences of scores of size 10: some hundred u of 30
    for a, b in ((got[0], w), (got[2], logp), (got[3], entropy), (got[6], gd.grad)):
        assert (a.double().cpu() - b).abs().max() < 1e-4
    rows = torch.arange(len(x))[:, None]
    assert (got[7].double().cpu()[index, rows] - w.detach()[:, :, None] * mixed.grad[:, None]).abs().max() < 1e-4


def test_a_captured_run_replays_with_new_inputs_between_eager_work():
    s = _scores()
    buffers = _mixture_inputs(1)
    big = _rows(2, 140001, 'bf16', seed=1)         # a row that several workgroups share
    masked = _rows(4, 64, 'f32', seed=2)
    _mixture(s, *buffers)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graphs = []
    for _ in range(2):                              # two captured graphs of the same calls, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = _mixture(s, *buffers) + tuple(s.token_logprobs(big, top=9)[1:]) + tuple(
                s.route_experts(masked, 4, bias=buffers[0].flatten()[:64], groups=4, top_groups=2, group_score='top2'))
        graphs.append((graph, out))
    for turn in range(6):
        fresh = _mixture_inputs(10 + turn)
        for b, f in zip(buffers, fresh):
            b.copy_(f)
        big.copy_(_rows(2, 140001, 'bf16', seed=20 + turn))
        masked.copy_(_rows(4, 64, 'f32', seed=30 + turn))
        graph, out = graphs[turn % 2]
        graph.replay()
        torch.cuda.synchronize()
        want = _mixture(s, *buffers) + tuple(s.token_logprobs(big, top=9)[1:]) + tuple(
            s.route_experts(masked, 4, bias=buffers[0].flatten()[:64], groups=4, top_groups=2, group_score='top2'))
        torch.cuda.synchronize()
        for k, (a, b) in enumerate(zip(out, want)):
            assert torch.equal(a, b), (turn, k)
