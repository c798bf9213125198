"""Rows of scores on the GPU at their edges: group sums that cancel, biases of NaN and infinities, what results share with
each other and with autograd, gradients next to their logits, rows that share a wavefront.  Tolerances as in
``test_gpu_scores``, whose checks these tests use."""
import math

import numpy as np
import pytest

from tests import scores_ref as ref
from tests.test_gpu_scores import TYPES, _check_logprobs, _check_route, _np, _rows, _scores, _tokens

torch = pytest.importorskip('torch')
pytestmark = pytest.mark.gpu


# ---- routing in groups by sums ---------------------------------------------------------------

def _alternating(experts, groups, big):
    """One expert of every group pushed up by ``big``, all others down: the two largest of a group cancel."""
    bias = torch.full((experts,), -big, device='cuda')
    bias[::experts // groups] = big
    return bias


def test_route_by_group_sums_that_cancel():
    x = torch.tensor([[-0.29003906, 0.11914062, -0.04101562, -0.13085938]], device='cuda')
    bias = torch.tensor([1e4, -1e4, 1e4, -1e4], device='cuda')
    how = dict(score='sigmoid', groups=2, top_groups=1, group_score='top2', bias=bias)
    assert _check_route(x, 2, **how).index[0].tolist() == [0, 1]        # 0.957744 against 0.957079


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('big', [1e2, 1e3, 1e4, 1e5])
def test_route_by_group_sums_next_to_large_biases(big, score):
    for experts, groups, top_groups in ((64, 8, 4), (128, 4, 1), (48, 16, 5)):
        bias = _alternating(experts, groups, big)
        for k, scale in enumerate((1e-3, 0.05, 1.0)):    # p + p of two groups apart by less and by more than a step of `big`
            gen = torch.Generator().manual_seed(k)
            x = (torch.randn(150, experts, generator=gen) * scale).cuda()
            for b in (bias, -bias, bias + torch.randn(experts, generator=gen).cuda()):
                _check_route(x, 4, bias=b, score=score, groups=groups, top_groups=top_groups, group_score='top2')


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
def test_route_by_group_sums_with_nan_biases(score):
    """An expert whose bias is NaN comes behind all others, and adds nothing to its group."""
    logit = torch.tensor([0.9, 0.5, 0.1, 0.6, 0.7, 0.2], device='cuda').logit()
    x = logit[None].expand(3, 6)
    bias = torch.tensor([0, math.nan, 0, 0, 0, 0], device='cuda')
    how = dict(score=score, groups=2, top_groups=1, group_score='top2')
    _check_route(x, 2, bias=bias, **how)             # sigmoid: 0.9 + 0.1 against 0.6 + 0.7
    gen = torch.Generator().manual_seed(2)
    for experts, groups, top_groups, top in ((64, 8, 4, 8), (256, 8, 2, 6), (24, 3, 1, 2), (512, 32, 5, 16)):
        bias = torch.randn(experts, generator=gen) * 0.05
        bias.view(groups, -1)[:, ::3] = math.nan     # (two or more are left in every group)
        x = _rows(70, experts, 'f32', seed=experts, scale=1.0)
        for group_score in ('top2', 'max'):
            _check_route(x, top, bias=bias.cuda(), score=score, groups=groups, top_groups=top_groups, group_score=group_score)


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
def test_route_by_group_sums_with_experts_shut_out(score):
    """A group with fewer than two experts that are not shut out has a sum of -inf, all such groups alike."""
    gen = torch.Generator().manual_seed(3)
    for experts, groups, top_groups, top in ((64, 8, 4, 8), (16, 4, 1, 2), (256, 8, 2, 6), (60, 20, 7, 5), (8, 8, 3, 3), (1000, 40, 3, 20)):
        per = experts // groups
        x = _rows(40, experts, 'f32', seed=groups, scale=1.0)
        for left in range(per + 1):                  # of group g: g mod (left + 1) experts, so that there are some of every kind
            if left > 6 and left < per:
                continue
            bias = torch.randn(experts, generator=gen) * 0.05
            for g in range(groups):
                out = torch.randperm(per, generator=gen)[min(per, (g * 3 + 1) % (left + 1)):]
                bias[g * per + out] = -math.inf if left % 2 else math.nan
            for group_score in ('top2', 'max'):
                _check_route(x, top, bias=bias.cuda(), score=score, groups=groups, top_groups=top_groups, group_score=group_score)
    x = _rows(9, 64, 'f32')
    for low in (-math.inf, torch.finfo(torch.float32).min):       # everybody; sums past float32
        _check_route(x, 5, bias=torch.full((64,), low, device='cuda'), score=score, groups=8, top_groups=3, group_score='top2')


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
def test_route_by_group_sums_with_a_bias_of_plus_infinity(score):
    """A group that holds one comes before all that hold none, also where its other experts are shut out."""
    x = _rows(30, 64, 'f32', scale=1.0)
    for other in (0.0, -math.inf):
        bias = torch.full((64,), other, device='cuda')
        bias[:48] = 0
        bias[61] = math.inf
        r = _scores().route_experts(x, 3, score=score, bias=bias, groups=4, top_groups=1, group_score='top2')
        assert (r.index[:, 0] == 61).all() and (r.index >= 48).all()


# ---- what results share ----------------------------------------------------------------------

@pytest.mark.parametrize('rows, cols', [(5, 300), (3, 5000), (2, 140001)])
def test_results_are_tensors_of_their_own(rows, cols):
    s = _scores()
    x, tokens = _rows(rows, cols, 'bf16'), _tokens(rows, cols, 2)
    r = s.token_logprobs(x, tokens, top=3)
    # nothing else is kept alive by one of them, and writing one does not mark the others as changed
    assert [part.untyped_storage().nbytes() for part in r] == [part.numel() * 4 for part in r]
    assert [part._is_view() for part in r] == [False] * 5 and all(part.is_contiguous() for part in r)
    weight = torch.ones(rows, device='cuda', requires_grad=True)
    loss = (weight * r.entropy).sum()
    r.logp.mul_(2)
    r.top_index.fill_(0)
    r.stats.zero_()
    loss.backward()
    assert torch.equal(weight.grad, r.entropy)


# ---- autograd --------------------------------------------------------------------------------

def test_logits_that_autograd_would_lose_are_refused():
    s = _scores()
    x = _rows(4, 64, 'f32').requires_grad_()
    for call in (lambda: s.token_logprobs(x, top=2), lambda: s.route_experts(x, 2), lambda: s.token_logprobs(x * 1, top=2)):
        with pytest.raises(ValueError, match='detach'):
            call()
        with torch.no_grad():
            call()
    r, routes = s.token_logprobs(x.detach(), top=2), s.route_experts(x.detach(), 2, bias=torch.zeros(64, device='cuda', requires_grad=True))
    ones = torch.ones(4, 2, device='cuda')
    # the backward forms give the gradient itself, and take the logits as they are
    x.backward(s.token_logprobs_backward(x, r.stats, r.top_index, ones))
    x.backward(s.route_experts_backward(x, routes.index, ones, renormalise=False))
    want = torch.log_softmax(x.double(), 1).gather(1, r.top_index.long()).sum() + torch.softmax(x.double(), 1).gather(1, routes.index.long()).sum()
    (grad,) = torch.autograd.grad(want, x)
    assert (x.grad - grad).abs().max() < 1e-5


def test_a_gradient_written_over_the_logits_is_seen_by_autograd():
    s = _scores()
    for backward in ('logprobs', 'route'):
        leaf = torch.randn(4, 64, device='cuda', requires_grad=True)
        logits = leaf.tanh()                          # keeps what it returned for its own backward pass
        x = logits.detach()
        r, index = s.token_logprobs(x, top=2), s.route_experts(x, 2).index
        ones, before = torch.ones(4, 2, device='cuda'), x._version
        if backward == 'logprobs':
            s.token_logprobs_backward(x, r.stats, r.top_index, ones, out=x)
        else:
            s.route_experts_backward(x, index, ones, out=x)
        after = x._version
        assert after == before + 1
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            logits.sum().backward()


# ---- gradients next to their logits ----------------------------------------------------------

def test_gradients_between_the_rows_of_their_logits():
    """In the columns next to them, in every other row, before and behind them in the same buffer, rows at other distances."""
    s = _scores()
    ones = torch.ones(5, 2, device='cuda')
    for dtype in TYPES.values():
        def buffer():
            return _rows(24, 96, 'f32', seed=7).to(dtype)
        places = [lambda b: (b[:5, :32], b[:5, 32:64]), lambda b: (b[:5, 64:], b[:5, :64]), lambda b: (b[1:10:2], b[:10:2]),
                  lambda b: (b[:10:2], b[1:11:2]), lambda b: (b[:10:2, :48], b[:5, 48:]), lambda b: (b[:5, 48:], b[:10:2, :48]),
                  lambda b: (b[:5], b[5:10]), lambda b: (b[2:3, :40].expand(5, 40), b[:5, 40:80]),
                  lambda b: (b.as_strided((5, 30), (50, 1)), b.as_strided((5, 20), (100, 1), 30)),
                  lambda b: (b.as_strided((5, 20), (50, 1)), b.as_strided((5, 20), (101, 1), 20)),
                  lambda b: (b.as_strided((5, 30), (7, 1), 120), b.as_strided((5, 30), (96, 1), 83))]
        for k, place in enumerate(places):
            b = buffer()
            x, out = place(b)
            out = out[:, :x.shape[1]]
            x = x[:, :out.shape[1]]
            plain = x.contiguous()
            r, index = s.token_logprobs(plain, top=2), s.route_experts(plain, 2).index
            for want, call in ((s.token_logprobs_backward(plain, r.stats, r.top_index, ones),
                                lambda: s.token_logprobs_backward(x, r.stats, r.top_index, ones, out=out)),
                               (s.route_experts_backward(plain, index, ones, renormalise=False),
                                lambda: s.route_experts_backward(x, index, ones, renormalise=False, out=out))):
                assert call() is out and torch.equal(out, want) and torch.equal(x, plain), (dtype, k)


def test_the_routing_gradient_of_rows_without_an_order():
    """Index -1 names no expert: 0 where only chosen logits are read, NaN where a softmax that is not renormalised reads all."""
    s = _scores()
    x = _rows(3, 40, 'f32')
    x[1, 7] = math.nan
    g = torch.ones(3, 4, device='cuda')
    for how in (dict(), dict(score='sigmoid'), dict(score='sigmoid', renormalise=False), dict(renormalise=False)):
        routes = s.route_experts(x, 4, **how)
        assert torch.isnan(routes.weights[1]).all() and (routes.index[1] == -1).all()
        grad = s.route_experts_backward(x, routes.index, g, **how)
        if how == dict(renormalise=False):
            assert torch.isnan(grad[1]).all()
        else:
            assert not grad[1].any()
        assert torch.isfinite(grad[[0, 2]]).all()


def test_a_bias_of_another_type_is_rounded_to_float32_first():
    s = _scores()
    x = _rows(20, 64, 'f32')
    bias = torch.randn(64, dtype=torch.float64, generator=torch.Generator().manual_seed(4)).cuda()
    for b in (bias, bias.bfloat16(), bias.half()):
        got, want = s.route_experts(x, 6, bias=b), s.route_experts(x, 6, bias=b.float())
        assert torch.equal(got.index, want.index) and torch.equal(got.weights, want.weights)


def test_the_stream_is_found_without_torchs_inner_function(monkeypatch):
    s = _scores()
    x = _rows(3, 300, 'f32')
    want = s.token_logprobs(x, top=4)
    stream = torch.cuda.Stream()
    assert s._stream(x.device) == torch.cuda.current_stream().cuda_stream
    monkeypatch.setattr(s, '_raw_stream', None)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        assert s._stream(x.device) == stream.cuda_stream
        got = s.token_logprobs(x, top=4)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))


# ---- rows that share a wavefront, and the longest --------------------------------------------

def _pick(v, keep):
    return None if v is None else v[keep]


@pytest.mark.parametrize('dtype', list(TYPES))
@pytest.mark.parametrize('rows, cols', [(16385, 184), (16386, 256), (16387, 41), (8193, 1000), (8195, 520), (8193, 90)])
def test_rows_that_share_wavefronts_with_some_left_over(rows, cols, dtype):
    """Not a whole number of wavefronts; rows of every width next to each other, down to 0 and to fewer than the alternatives."""
    s = _scores()
    x = _rows(1, cols, dtype).expand(rows, cols).clone()
    x += torch.randn(rows, cols, generator=torch.Generator().manual_seed(rows)).to(x.dtype).cuda()
    x[5::97, ::3] = -math.inf
    x[6::97] = -math.inf
    x[7::97, cols // 2] = math.nan
    widths = torch.randint(0, cols + 1, (rows,), generator=torch.Generator().manual_seed(cols), dtype=torch.int32)
    widths[::5], widths[1::7], widths[2::9], widths[3::11] = 0, 1, 4, cols
    keep = torch.cat([torch.arange(0, 60), torch.arange(rows - 40, rows)]).cuda()
    for n, top, w in ((1, 0, None), (1, 5, None), (20, 8, None), (1, 5, widths.cuda()), (20, 8, widths.cuda()), (20, 0, widths.cuda()), (3, 14, widths.cuda())):
        if top > 8 and rows > 16384:
            continue
        tokens = _tokens(rows, cols, n)
        many = s.token_logprobs(x, tokens, top, w)
        few = _check_logprobs(x[keep], tokens[keep], top, _pick(w, keep))
        err = (cols / 64 + 96) * 2.0 ** -24 * (1 + math.log(cols + 1))
        for a, b in zip(many, few):
            if a is not None and a.dtype == torch.int32:
                assert torch.equal(a[keep], b)
            elif a is not None:
                a, b = _np(a[keep]), _np(b)
                assert np.array_equal(np.isfinite(a), np.isfinite(b)) and np.array_equal(a[~np.isfinite(a)], b[~np.isfinite(b)], equal_nan=True)
                fine = np.isfinite(a)
                # two results of other orders of adding, each off by at most err and 2 u of its value
                assert (np.abs(a[fine] - b[fine]) <= 2 * err + 4 * 2.0 ** -24 * np.abs(b[fine])).all()


def test_rows_of_the_most_columns():
    cols = 1 << 24
    x = torch.randn(2, cols, device='cuda', generator=torch.Generator('cuda').manual_seed(1)).bfloat16()
    tokens = torch.tensor([[0, cols - 1], [cols, 77]], device='cuda')
    x[0, cols - 1] = 9
    widths = torch.tensor([cols, cols - 5], dtype=torch.int32, device='cuda')
    r = _check_logprobs(x, tokens, 5, widths)
    g = torch.ones(2, 2, device='cuda')
    grad = _scores().token_logprobs_backward(x, r.stats, tokens, g, widths=widths)
    p = torch.softmax(x[0].double(), 0)
    want = -2 * p
    want[0] += 1
    want[-1] += 1
    # bfloat16's half step, and the statistics' error times the value
    assert ((grad[0].double() - want).abs() <= want.abs() * (2.0 ** -8 + (cols / 64 + 96) * 2.0 ** -24) + 2.0 ** -134).all()
    assert not grad[1, cols - 5:].any()
    with pytest.raises(ValueError):
        _scores().token_logprobs(x[:1].expand(1, cols).as_strided((1, cols + 1), (cols + 1, 1)), top=1)
