"""Rows of scores at their edges, without a GPU."""
import pytest
import torch

from poseestimation_amd import _ffi, scores


@pytest.mark.parametrize('call', [lambda x: scores.token_logprobs(x, top=1), lambda x: scores.route_experts(x, 2)])
def test_logits_that_autograd_would_lose_are_refused(call):
    x = torch.zeros(4, 16, requires_grad=True)
    for logits in (x, x * 1):
        with pytest.raises(ValueError, match='detach'):
            call(logits)
    with torch.no_grad(), pytest.raises(ValueError, match='GPU'):
        call(x)
    with pytest.raises(ValueError, match='GPU'):
        call(x.detach())


P = 1 << 20     # an address that nothing reads: every call below is refused before it would


@pytest.mark.parametrize('x, stride, grad, grad_stride', [
    (0, 100, 39, 100), (0, 100, 61, 100), (39, 100, 0, 100), (0, 100, 100, 100), (400, 100, 0, 100), (0, 100, 361, 100),
    (0, 0, 20, 100), (100, 0, 61, 100), (0, 20, 119, 100), (0, 100, 40, 99), (0, 101, 40, 100), (0, 50, 40, 100), (0, 100, 40, 150),
    (0, 100, 0, 200), (200, 100, 0, 99)])
def test_gradients_that_overlap_their_logits_are_refused(x, stride, grad, grad_stride):
    """Five rows of 40 columns, places in columns: a column or more of some row is in the logits and in the gradient."""
    for dtype, size in ((_ffi.F32, 4), (_ffi.BF16, 2)):
        rc = _ffi.lib().pd_token_logprobs_grad(P + x * size, dtype, 5, 40, stride, None, P, P, 1, P, P, P + grad * size, grad_stride, None)
        assert rc == _ffi.PD_E_INVALID and 'overlaps' in _ffi.lib().pd_last_error(None).decode()
        rc = _ffi.lib().pd_route_experts_grad(P + x * size, dtype, 5, 40, stride, P, P, 0, 4, 1, 1.0, P + grad * size, grad_stride, None)
        assert rc == _ffi.PD_E_INVALID and 'overlaps' in _ffi.lib().pd_last_error(None).decode()
