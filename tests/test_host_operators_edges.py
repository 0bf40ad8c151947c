"""The operators around the Linear where no GPU is needed, at the edges of what they accept."""
import pytest
import torch

from optimus_dl_amd.modules.logprobs import token_logprobs


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1e-30, 1e-10, 1.0, 1e30])
def test_plain_log_probabilities_of_logits_of_any_size(dtype, temperature):
    """Logits that 1 / temperature takes out of fp32, and the lowest value of the type as a mask: what is left is a choice between equals, or certain.
    A probability of 1 / 3 and its logarithm are off by a few last places: 8 of them."""
    low = torch.finfo(dtype).min
    l = torch.tensor([[2.0 ** 100, 2.0 ** 100, 2.0 ** 100, low], [-(2.0 ** 100), low, low, float("-inf")], [2.0 ** 120, -(2.0 ** 120), 0.0, low]], dtype=dtype)
    live = l.clone().requires_grad_(True)
    r = token_logprobs(live, torch.tensor([1, 0, 0]), top_k=2, temperature=temperature)
    third, tol = torch.log(torch.tensor(3.0)).item(), 8 * 2.0 ** -24
    want = torch.tensor([-third, 0.0, 0.0])
    # (at 1e30 the second logits are 1.3e6 or 3.4e8 behind the first)
    assert bool(((r.logprobs - want).abs() <= tol).all()) and abs(r.entropy[0].item() - third) <= tol and not r.entropy[1:].any()
    assert r.top_ids.tolist() == [[0, 1], [0, 1], [0, 2]]
    (r.logprobs.sum() + r.entropy.sum()).backward()
    assert live.grad.isfinite().all() and not live.grad[1:].any()
