"""Rows of scores without a GPU: the refusals of the C entry points and of the Python functions (every
check comes before anything touches a device), and the float64 restatement against differences."""
import numpy as np
import pytest
import torch

from poseestimation_amd import _ffi, scores
from tests import scores_ref as ref

P = 1 << 20     # an address that nothing reads: every call below is refused before it would


def _logprobs(**kw):
    a = dict(x=P, dtype=_ffi.F32, rows=4, cols=100, stride=100, widths=None, tokens=P, n=1, top=2, logp=P, entropy=P, stats=P,
             tl=P, ti=P, ws=None, ws_bytes=0)
    a.update(kw)
    return _ffi.lib().pd_token_logprobs(*a.values(), None)


def _logprobs_grad(**kw):
    a = dict(x=P, dtype=_ffi.BF16, rows=4, cols=100, stride=100, widths=None, stats=P, tokens=P, n=1, g=P, ge=P, out=2 * P,
             out_stride=100)
    a.update(kw)
    return _ffi.lib().pd_token_logprobs_grad(*a.values(), None)


def _route(**kw):
    a = dict(x=P, dtype=_ffi.F16, rows=4, experts=64, stride=64, bias=None, score=0, groups=4, top_groups=2, gs=0, top=8, renorm=1,
             scale=1.0, weights=P, index=P)
    a.update(kw)
    return _ffi.lib().pd_route_experts(*a.values(), None)


def _route_grad(**kw):
    a = dict(x=P, dtype=_ffi.F32, rows=4, experts=64, stride=64, index=P, g=P, score=1, top=8, renorm=1, scale=1.0, out=2 * P,
             out_stride=64)
    a.update(kw)
    return _ffi.lib().pd_route_experts_grad(*a.values(), None)


BAD = [
    (_logprobs, dict(dtype=_ffi.F64), 'PD_F32'), (_logprobs, dict(dtype=9), 'PD_F32'), (_logprobs, dict(rows=-1), 'rows'),
    (_logprobs, dict(rows=1 << 31), 'rows'), (_logprobs, dict(cols=0), 'columns'), (_logprobs, dict(cols=(1 << 24) + 1), 'columns'),
    (_logprobs, dict(stride=-1), 'stride'), (_logprobs, dict(stride=1 << 62), 'stride'), (_logprobs, dict(x=None), 'logits'),
    (_logprobs, dict(x=P + 2), 'aligned'), (_logprobs, dict(x=P + 1, dtype=_ffi.BF16), 'aligned'),
    (_logprobs, dict(n=-1), 'n_tokens'), (_logprobs, dict(n=65), 'n_tokens'), (_logprobs, dict(tokens=None), 'tokens'),
    (_logprobs, dict(logp=None), 'tokens'), (_logprobs, dict(top=-1), 'top'), (_logprobs, dict(top=65), 'top'),
    (_logprobs, dict(cols=5, top=6), 'top'), (_logprobs, dict(tl=None), 'top_logp'), (_logprobs, dict(ti=None), 'top_logp'),
    (_logprobs, dict(cols=1 << 20, stride=1 << 20), 'workspace'), (_logprobs, dict(cols=1 << 20, ws=P, ws_bytes=16), 'workspace'),
    (_logprobs, dict(cols=1 << 20, ws=P + 8, ws_bytes=1 << 20), 'aligned'),
    (_logprobs_grad, dict(dtype=_ffi.U8), 'PD_F32'), (_logprobs_grad, dict(cols=0), 'columns'),
    (_logprobs_grad, dict(stats=None), 'stats'), (_logprobs_grad, dict(out=None), 'grad'),
    (_logprobs_grad, dict(out=2 * P + 1), 'aligned'), (_logprobs_grad, dict(out_stride=99), 'overlap'),
    (_logprobs_grad, dict(out=P + 2), 'overlaps'), (_logprobs_grad, dict(out=P, out_stride=101), 'overlaps'),
    (_logprobs_grad, dict(out=P, stride=0), 'overlaps'), (_logprobs_grad, dict(tokens=None), 'tokens'),
    (_logprobs_grad, dict(g=None), 'tokens'), (_logprobs_grad, dict(n=65), 'n_tokens'),
    (_route, dict(dtype=_ffi.U8), 'PD_F32'), (_route, dict(experts=0), 'columns'), (_route, dict(experts=1025, groups=1), 'columns'),
    (_route, dict(score=2), 'score'), (_route, dict(top=0), 'top'), (_route, dict(top=33), 'top'),
    (_route, dict(experts=4, groups=1, top_groups=1, top=5), 'top'), (_route, dict(groups=0), 'groups'),
    (_route, dict(groups=5), 'groups'), (_route, dict(experts=1024, groups=128), 'groups'), (_route, dict(top_groups=0), 'top_groups'),
    (_route, dict(top_groups=5), 'top_groups'), (_route, dict(groups=32, top_groups=3), 'fewer'), (_route, dict(gs=2), 'group_score'),
    (_route, dict(weights=None), 'weights'), (_route, dict(index=None), 'weights'), (_route, dict(x=P + 1), 'aligned'),
    (_route_grad, dict(score=-1), 'score'), (_route_grad, dict(top=0), 'top'), (_route_grad, dict(top=65, experts=64), 'top'),
    (_route_grad, dict(index=None), 'index'), (_route_grad, dict(g=None), 'index'), (_route_grad, dict(out=None), 'index'),
    (_route_grad, dict(out_stride=63), 'overlap'), (_route_grad, dict(out=P + 4), 'overlaps'),
]


@pytest.mark.parametrize('call, kw, text', BAD, ids=['%s-%s' % (c.__name__[1:], '-'.join(map(str, k.items()))) for c, k, _ in BAD])
def test_bad_arguments_are_refused(call, kw, text):
    assert call(**kw) == _ffi.PD_E_INVALID
    said = _ffi.lib().pd_last_error(None).decode()
    assert said.startswith('pd_') and text in said, said


@pytest.mark.parametrize('call', [_logprobs, _logprobs_grad, _route, _route_grad])
def test_no_rows_are_no_work(call):
    # (the addresses may be NULL then: torch gives an empty tensor none)
    assert call(rows=0, x=None) == _ffi.PD_OK


def test_a_workspace_is_needed_for_few_long_rows_only():
    need = _ffi.lib().pd_token_logprobs_workspace
    assert need(_ffi.F32, 4, 2048, 64) == need(_ffi.BF16, 4096, 131072, 5) == need(_ffi.F16, 100, 131072, 5) == 0
    assert need(_ffi.F32, 0, 1 << 20, 5) == need(_ffi.F32, 4, (1 << 24) + 1, 5) == need(9, 4, 1 << 20, 5) == 0
    for rows, cols, top in ((1, 131072, 0), (1, 1 << 24, 64), (32, 131072, 5), (1000, 200000, 3)):
        bytes_ = need(_ffi.BF16, rows, cols, top)
        # between two and 256 slices of a row, 12 bytes of statistics and `top` keys of 8 each
        assert 2 * rows * (12 + 8 * top) <= bytes_ <= 256 * rows * (12 + 8 * top) + 16


def test_python_functions_refuse_what_is_not_on_a_gpu_or_misshapen():
    x = torch.zeros(4, 16)
    for fn in (lambda v: scores.token_logprobs(v, top=1), lambda v: scores.route_experts(v, 2),
               lambda v: scores.token_logprobs_backward(v, torch.zeros(4, 3), grad_entropy=torch.zeros(4)),
               lambda v: scores.route_experts_backward(v, torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2))):
        for bad in (x, x[0], x.double(), x.long(), x[None], x.numpy(), None):
            with pytest.raises(ValueError):
                fn(bad)
    assert scores.TokenLogprobs._fields == ('logp', 'entropy', 'top_logp', 'top_index', 'stats')


@pytest.mark.parametrize('dtype', [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64, torch.uint16, torch.uint32])
def test_whole_numbers_of_every_size_are_taken(dtype):
    x = torch.tensor([5, 100, 3], dtype=dtype)
    for to in (torch.int32, torch.int64):
        got = scores._like(x, 'x', to, ((3,),), x.device)
        assert got.dtype == to and got.tolist() == [5, 100, 3]


def test_whole_numbers_past_32_bits_stay_out_of_range():
    x = torch.tensor([1 << 32, -(1 << 32) + 2, (1 << 63) - 1])
    assert scores._like(x, 'x', torch.int32, ((3,),), x.device).tolist() == [0x7fffffff, -1, 0x7fffffff]
    for dtype in (torch.bool, torch.uint64):
        with pytest.raises(ValueError):
            scores._like(x.to(dtype), 'x', torch.int32, ((3,),), x.device)


def test_the_restated_gradients_agree_with_differences():
    rng = np.random.default_rng(5)
    h = 1e-5
    for trial in range(20):
        rows, cols = 3, int(rng.integers(2, 40))
        x = rng.normal(0, 2, (rows, cols))
        d = rng.normal(0, 1, x.shape)
        tokens = rng.integers(-1, cols, (rows, 4))
        tokens[0, 1] = tokens[0, 0]
        widths = rng.integers(1, cols + 1, rows) if trial % 2 else None
        if widths is not None:
            tokens = np.minimum(tokens, widths[:, None] - 1)
        g, ge = rng.normal(0, 1, tokens.shape), rng.normal(0, 1, rows)

        def value(v):
            logp, entropy = ref.logprobs(v, tokens, 0, widths)[:2]
            return (logp * g).sum() + (entropy * ge).sum()
        slope = (value(x + h * d) - value(x - h * d)) / (2 * h)
        # third derivatives are of order one: the difference is good to h^2 and to rounding / h
        assert abs((ref.logprobs_grad(x, tokens, g, ge, widths) * d).sum() - slope) < 1e-7 * (1 + abs(slope)) * cols
        top = int(rng.integers(1, cols + 1))
        for score in ('softmax', 'sigmoid'):
            for renormalise in (False, True):
                index = np.stack([rng.permutation(cols)[:top] for _ in range(rows)])
                g = rng.normal(0, 1, (rows, top))

                def value(v):
                    return sum((2.5 * ref.weights_of(v[r], index[r], score, renormalise) * g[r]).sum() for r in range(rows))
                slope = (value(x + h * d) - value(x - h * d)) / (2 * h)
                got = (ref.route_grad(x, index, g, score, renormalise, 2.5) * d).sum()
                assert abs(got - slope) < 1e-7 * (1 + abs(slope)) * cols
