"""What else than a backward may look at a call: the tracer of torch.jit, forward-mode differentiation, functorch.  A traced call computes, and what the
operators cannot differentiate or batch is refused, not left out."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from optimus_dl_amd.modules.fp4_linear import FP4Linear, fp4_linear
from optimus_dl_amd.modules.fused import residual_norm
from optimus_dl_amd.modules.logprobs import token_logprobs

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def calls(seed=0):
    """name -> (function of one tensor, that tensor)"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    n = lambda *s: torch.randn(s, device="cuda", generator=g)
    h, w, post, gate = n(6, 256).to(BF16), n(256), n(256), n(1)
    targets = torch.randint(0, 500, (6,), device="cuda", generator=g)
    codes = torch.randint(0, 256, (96, 128), device="cuda", generator=g, dtype=torch.int64).to(torch.uint8)
    scales = (torch.rand((96, 4), device="cuda", generator=g) + 0.5).to(BF16)
    linear = FP4Linear.from_codes(codes, scales, n(96))
    return {
        "residual_norm": (lambda x: residual_norm(x, h, w, 1e-6, post_weight=post, gate=gate, residual_scale=0.5, out_dtype=BF16), n(6, 256)),
        "token_logprobs": (lambda x: tuple(token_logprobs(x, targets, n_vocab=500, temperature=0.7)[:2]), n(6, 512)),
        "token_logprobs_top": (lambda x: tuple(token_logprobs(x, targets, n_vocab=500, top_k=3)), n(6, 512)),
        "fp4_linear": (lambda x: fp4_linear(x, codes, scales), n(6, 256).to(BF16)),
        "FP4Linear": (linear, n(6, 256)),
    }


NAMES = ("residual_norm", "token_logprobs", "token_logprobs_top", "fp4_linear", "FP4Linear")


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", NAMES[:-1])
def test_traced_calls_compute(name, grad):
    f, x = calls()[name]
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(f, (x,), check_trace=False)
        for seed in (1, 2):
            new = torch.randn(x.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(x.dtype)
            want, got = f(new), traced(new)
            want, got = (want, got) if isinstance(want, tuple) else ((want,), (got,))
            assert len(want) == len(got) and all(torch.equal(a, b) for a, b in zip(want, got))


def test_a_module_with_codes_says_that_it_cannot_be_traced():
    m, x = calls()["FP4Linear"]
    for module, given in ((m, x), (m.cpu(), x.cpu())):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(module, (given,), check_trace=False)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(name, grad):
    f, x = calls()[name]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="jvp"):
            f(forward_ad.make_dual(x, torch.ones_like(x)))
    f(x)                                                       # (and nothing of it stays)


@pytest.mark.parametrize("name", NAMES)
def test_functorch_is_refused(name):
    f, x = calls()[name]
    first = lambda t: f(t)[0] if isinstance(f(t), tuple) else f(t)
    with pytest.raises(RuntimeError, match="setup_context"):
        torch.func.vmap(f)(x.unsqueeze(0))
    with pytest.raises(RuntimeError, match="setup_context|no backward"):
        torch.func.grad(lambda t: first(t).float().sum())(x)
