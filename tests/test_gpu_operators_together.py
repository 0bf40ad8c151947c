"""Decoders that use the operators around the Linear as they are meant to be used: training with FP8 Linears, a decode step with 4-bit ones."""
import pytest
import torch

from optimus_dl_amd import native
from optimus_dl_amd.modules.amp import create_fp8_recipe, fp8_autocast, fp8_backward
from optimus_dl_amd.modules.fp4_linear import FP4Linear
from optimus_dl_amd.modules.model import Llama, LlamaConfig, Qwen3, Qwen3Config
from optimus_dl_amd.modules.model_transforms import build_model_transform

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")
SIZES = dict(vocab_size=1024, n_layer=2, n_head=4, n_kv_head=2, n_embd=256, intermediate_size=512)


def model(family="llama", dtype=torch.float32, **kwargs):
    torch.manual_seed(0)
    with CUDA:
        m = Llama(LlamaConfig(**SIZES, **kwargs)) if family == "llama" else Qwen3(Qwen3Config(**SIZES, head_dim=64, **kwargs))
    return m.to(dtype)


def step(m, ids, recipe):
    for p in m.parameters():
        p.grad = None
    with fp8_autocast(CUDA, recipe):
        r = m.score(ids)
        loss = -(r.logprobs.sum() + 0.01 * r.entropy.sum()) / ids.numel()
    with fp8_backward(recipe):
        loss.backward()
    return loss.detach(), {n: p.grad for n, p in m.named_parameters()}


@pytest.mark.parametrize("family", ["llama", "qwen3"])
@pytest.mark.parametrize("kwargs", [dict(post_norms=True, layer_scale=0.5), dict(residual_scale=0.8), dict(post_norms=True)])
def test_training_hands_maxima_from_kernel_to_cast(monkeypatch, family, kwargs):
    """Same bits with the maxima that the producers leave as with a pass over each tensor, and no such pass over the gradient of the logits, the
    norms' outputs or the gradients of what ends a half."""
    m = build_model_transform({"_name": "fp8_linear"}).apply(model(family, **kwargs))
    ids = torch.randint(0, 1024, (4, 32), device=CUDA, generator=torch.Generator(device="cuda").manual_seed(1))
    recipe = create_fp8_recipe("tensorwise", "hybrid")
    recipe.cache_weights = False                           # (both steps pass over the weights)
    passes = []
    monkeypatch.setattr(native, "amax_parts", lambda x, f=native.amax_parts: (passes.append(tuple(x.shape)), f(x))[1])
    loss, grads = step(m, ids, recipe)
    with_parts = list(passes)
    assert all(g is not None and g.isfinite().all() and g.abs().max() > 0 for g in grads.values())
    assert (128, 1024) not in with_parts                   # the head's gradient
    passes.clear()
    monkeypatch.setattr(type(recipe), "take_parts_and_slabs", lambda self, t: (None, None))
    again, regrads = step(m, ids, recipe)
    assert (128, 1024) in passes and len(passes) >= len(with_parts) + 1 + 2 * 2 * 2        # the head; each half's norm and its gradient
    assert torch.equal(loss, again)
    for n, g in grads.items():
        assert torch.equal(g, regrads[n]), n


@pytest.mark.parametrize("recipe", ["delayed", "rowwise", "mxfp8", "blockwise"])
def test_training_under_the_other_recipes(recipe):
    m = build_model_transform({"_name": "fp8_linear"}).apply(model(post_norms=True, layer_scale=0.5, residual_scale=0.9))
    ids = torch.randint(0, 1024, (4, 32), device=CUDA)
    r = create_fp8_recipe(recipe, "hybrid", amax_history_len=4)
    for _ in range(2):
        loss, grads = step(m, ids, r)
        assert loss.isfinite() and all(g is not None and g.isfinite().all() for g in grads.values())


def test_gradients_of_a_stepped_model_without_fp8():
    """bf16 autocast: the loss along its gradient.  With the step chosen so that the loss falls by d, a bf16 network's rounding (a half step of 2^-8 on
    logits of size 1, over 127 tokens) moves it by far less than d = 0.05."""
    m = model(post_norms=True, layer_scale=1.0)
    ids = torch.randint(0, 1024, (4, 32), device=CUDA, generator=torch.Generator(device="cuda").manual_seed(2))

    def loss():
        with torch.autocast("cuda", torch.bfloat16):
            return -m.score(ids).logprobs.sum() / 124

    grads = torch.autograd.grad(loss(), list(m.parameters()))
    norm = sum(g.double().square().sum() for g in grads).item()
    with torch.no_grad():
        ends = []
        for sign in (1, -1):
            for p, g in zip(m.parameters(), grads):
                p.add_(g, alpha=sign * 0.05 / norm)
            ends.append(loss().item())
            for p, g in zip(m.parameters(), grads):
                p.sub_(g, alpha=sign * 0.05 / norm)
    assert abs((ends[0] - ends[1]) / 0.1 - 1) < 0.2


@pytest.mark.parametrize("group", [32, 128])
def test_decode_step_with_4_bit_weights(group):
    """The Linears of the blocks in 4 bits, the head in FP8, norms in one kernel with the stream, the answer with its alternatives; beside it the same
    model with the weights that the codes stand for.  Each of the 24 tensors between two roundings is off by a half step of bf16 (2^-8) at most, on both
    sides."""
    m = model(dtype=torch.bfloat16, post_norms=True, layer_scale=0.5).eval()
    ids = torch.randint(0, 1024, (8, 5), device=CUDA, generator=torch.Generator(device="cuda").manual_seed(3))
    build_model_transform({"_name": "fp4_linear", "group_size": group}).apply(m)
    four = [x for x in m.modules() if isinstance(x, FP4Linear)]
    assert len(four) == 2 * 7 and type(m.lm_head) is torch.nn.Linear
    same = model(dtype=torch.bfloat16, post_norms=True, layer_scale=0.5).eval()
    lookup = dict(m.named_modules())
    for name, lin in same.named_modules():
        if isinstance(lookup.get(name), FP4Linear):
            lin.weight.data = lookup[name].dequantised_weight().bfloat16()
    with torch.no_grad():
        r = m.score(ids, top_k=8)
        logits, other = m(ids)["logits"].float(), same(ids)["logits"].float()
        assert (logits - other).norm() <= 48 * 2.0 ** -8 * other.norm()
        logp = torch.log_softmax(logits.double(), -1)
        assert torch.allclose(r.logprobs[:, :-1].double(), logp[:, :-1].gather(-1, ids[:, 1:, None]).squeeze(-1), atol=1e-5)
        assert torch.equal(r.top_ids[:, :-1], logits[:, :-1].sort(dim=-1, descending=True, stable=True).indices[..., :8])
        # one token of each sequence, as a decode step has it
        one = m.score(ids[:, :1], targets=ids[:, 1:2], top_k=4)
        assert one.logprobs.shape == (8, 1) and one.top_ids.shape == (8, 1, 4) and one.logprobs.isfinite().all()
        # the rest of the model under FP8
        build_model_transform({"_name": "fp8_linear"}).apply(m)
        with fp8_autocast(CUDA, create_fp8_recipe("tensorwise", "hybrid")):
            assert m.score(ids).logprobs.isfinite().all() and len([x for x in m.modules() if isinstance(x, FP4Linear)]) == 14


def test_a_step_of_the_operators_captured_with_its_backward():
    """The public functions and autograd under capture; replays on new data, with eager passes and synchronizations between them, give the eager bits."""
    from optimus_dl_amd.modules.fused import residual_norm
    from optimus_dl_amd.modules.logprobs import token_logprobs

    g = torch.Generator(device="cuda").manual_seed(4)
    n = lambda *s: torch.randn(s, device=CUDA, generator=g)
    x, h, w, wp, gate = n(40, 256).requires_grad_(True), n(40, 256).bfloat16().requires_grad_(True), *(n(256).requires_grad_(True) for _ in range(3))
    head = (n(256, 1003) * 0.05).bfloat16()
    targets = torch.randint(0, 1003, (40,), device=CUDA, generator=g)

    def step():
        y, z = residual_norm(x, h, w, 1e-6, post_weight=wp, gate=gate, residual_scale=0.9, out_dtype=torch.bfloat16)
        r = token_logprobs(z @ head, targets, n_vocab=1000, top_k=3, temperature=0.8)
        loss = r.logprobs.clamp(min=-20).sum() + r.entropy.sum() + r.top_logprobs.sum() + y.sum()
        return loss.detach(), r.top_ids, *torch.autograd.grad(loss, (x, h, w, wp, gate))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        with torch.no_grad():
            for t in (x, h, w):
                t.copy_(n(*t.shape))
            targets.copy_(torch.randint(0, 1003, (40,), device=CUDA, generator=g).clamp(max=999))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in held]
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, eager))


def test_an_unconverted_head_is_offered_nothing():
    """A gradient that no FP8 Linear takes is not kept for one."""
    m = model(post_norms=True)
    head, m.lm_head = m.lm_head, torch.nn.Identity()
    build_model_transform({"_name": "fp8_linear"}).apply(m)
    m.lm_head = head
    ids = torch.randint(0, 1024, (2, 32), device=CUDA)
    recipe = create_fp8_recipe("tensorwise", "hybrid")
    with fp8_autocast(CUDA, recipe):
        loss = -m.score(ids).logprobs.sum()
    with fp8_backward(recipe):
        loss.backward()
        assert not any(t.shape[-1] == 1024 for _, t, *_ in recipe.producer_parts)
    assert all(p.grad.isfinite().all() for p in m.parameters())


@pytest.mark.parametrize("stream", [torch.float32, torch.bfloat16])
def test_nodes_of_either_side_give_the_same_bits(monkeypatch, stream):
    """The autograd node in C++, which graphs without a recipe get, and the one in Python: values, gradients, what is left out, what is refused."""
    from optimus_dl_amd.modules.fused import residual_norm
    from optimus_dl_amd.modules.logprobs import token_logprobs

    g = torch.Generator(device="cuda").manual_seed(5)
    n = lambda *s: torch.randn(s, device=CUDA, generator=g)
    x, h, dy, dz = n(3, 20, 512).to(stream), n(3, 20, 512).bfloat16(), n(3, 20, 512).to(stream), n(3, 20, 512).bfloat16()
    w, wp, gates = n(512), n(512), (None, n(512), n(1), torch.tensor(0.3, device=CUDA))
    logits, targets, dl = n(3, 20, 1003).to(stream), torch.randint(0, 1000, (3, 20), device=CUDA, generator=g), n(3, 20)

    def everything():
        out = []
        for gate in gates:
            for post in (None, wp):
                for frozen in (False, True):
                    leaves = [t.clone().requires_grad_(True) for t in (x, h)] + [None if t is None else t.clone().requires_grad_(not frozen) for t in (w, post, gate)]
                    y, z = residual_norm(leaves[0], leaves[1], leaves[2], 1e-5, post_weight=leaves[3], gate=leaves[4], residual_scale=0.5, out_dtype=torch.bfloat16)
                    asked = [t for t in leaves if t is not None and t.requires_grad]
                    for outs, grads in (((y, z), (dy, dz)), ((y,), (dy,)), ((z,), (dz,))):
                        out += [o.detach() for o in outs] + list(torch.autograd.grad(outs, asked, grads, retain_graph=True))
        for k in (0, 4):
            leaf = logits.clone().requires_grad_(True)
            r = token_logprobs(leaf, targets, n_vocab=1000, top_k=k, temperature=0.5)
            out += [t.detach() for t in r if t is not None]
            out += torch.autograd.grad(r.logprobs, leaf, dl, retain_graph=True) + torch.autograd.grad(r.entropy.sum(), leaf, retain_graph=True)
            if k:
                out += torch.autograd.grad((r.logprobs, r.top_logprobs), leaf, (dl, n(3, 20, 4).fill_(0.25)), retain_graph=True)
        return out, type(y.grad_fn).__name__, type(r.logprobs.grad_fn).__name__

    here, *names = everything()
    monkeypatch.setattr(native, "residual_norm_node", lambda *a: None)
    monkeypatch.setattr(native, "token_logprobs_node", lambda *a: None)
    there, *others = everything()
    assert names != others and len(here) == len(there)
    for a, b in zip(here, there):
        assert a.dtype == b.dtype and torch.equal(a, b)
    monkeypatch.undo()
    leaf = logits.clone().requires_grad_(True)
    r = token_logprobs(leaf, targets, n_vocab=1000)
    leaf.data_ptr(), leaf.detach().add_(1.0)               # changed since it was kept
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.logprobs.sum().backward()
    (first,) = torch.autograd.grad(token_logprobs(logits.requires_grad_(True), targets).entropy.sum(), logits, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        first.sum().backward()
