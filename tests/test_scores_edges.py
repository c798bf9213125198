"""Rows of scores at their edges, without a GPU."""
import pytest
import torch

from poseestimation_amd import scores


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
