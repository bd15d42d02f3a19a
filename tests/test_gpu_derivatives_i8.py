"""Derivatives that the operators do not have are refused, not left out."""
import pytest
import torch
import torch.autograd.forward_ad as forward

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("leaf", [False, True])
@pytest.mark.parametrize("top", [0, 3])
def test_log_probabilities_in_forward_mode(wf, leaf, top):
    x, tok = torch.randn(3, 10, device=DEV), torch.zeros(3, dtype=torch.long, device=DEV)
    with forward.dual_level():
        dual = forward.make_dual(x.clone().requires_grad_(leaf), torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            wf.token_logprobs(dual, tok, top=top)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            wf.token_logprobs(dual, tok, top=top)
        assert forward.unpack_dual(wf.token_logprobs(x, tok, top=top).logprob).tangent is None  # beside other tensors that have one
    assert torch.isfinite(wf.token_logprobs(x, tok, top=top).logprob).all()
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda a: wf.token_logprobs(a, tok).logprob, (x,), (torch.ones_like(x),))
