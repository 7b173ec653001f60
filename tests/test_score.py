"""What token_logprobs refuses, on the CPU (a refused call launches nothing)."""

import pytest
import torch

from linuxformer_amd.score import token_logprobs


@pytest.mark.parametrize("logits,tokens,top", [
    (torch.zeros(8), torch.zeros(8, dtype=torch.int64), 0),
    (torch.zeros(2, 8, dtype=torch.float64), torch.zeros(2, dtype=torch.int64), 0),
    (torch.zeros(2, 0), torch.zeros(2, dtype=torch.int64), 0),
    (torch.zeros(2, 8), torch.zeros(3, dtype=torch.int64), 0),
    (torch.zeros(2, 8), torch.zeros(2), 0),
    (torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64), -1),
    (torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64), 65),
    (torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64), 4),  # nothing wrong, but no GPU
])
def test_token_logprobs_refuses(logits, tokens, top):
    with pytest.raises(ValueError) as e:
        token_logprobs(logits, tokens, top)
    assert ("runs on a GPU" in str(e.value)) == (top == 4), e.value


def test_token_logprobs_refuses_gradients():
    with torch.enable_grad(), pytest.raises(RuntimeError, match="gradients"):
        token_logprobs(torch.zeros(2, 8, requires_grad=True), torch.zeros(2, dtype=torch.int64))


def test_token_logprobs_refuses_tangents():
    with torch.autograd.forward_ad.dual_level():
        x = torch.autograd.forward_ad.make_dual(torch.zeros(2, 8), torch.ones(2, 8))
        with pytest.raises(RuntimeError, match="gradients"):
            token_logprobs(x, torch.zeros(2, dtype=torch.int64))
