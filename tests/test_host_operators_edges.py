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


def stepped_llama():
    from optimus_dl_amd.modules.model import Llama, LlamaConfig

    torch.manual_seed(0)
    return Llama(LlamaConfig(vocab_size=50, n_layer=3, n_embd=32, n_head=2, n_kv_head=2, intermediate_size=64, post_norms=True, layer_scale=0.5,
                             residual_scale=0.9))


IDS = torch.arange(14).reshape(2, 7)
# the same fp32 operations, some in another order: a few roundings of values near one
CLOSE = 64 * 2.0 ** -24


def close(model, want, ids=IDS):
    got = model(ids)["logits"]
    torch.testing.assert_close(got, want, rtol=0, atol=CLOSE * float(want.abs().max()))


@pytest.mark.parametrize("kind", ["forward", "forward_pre", "full_backward", "full_backward_pre", "global"])
@pytest.mark.parametrize("name", ["transformer.h.0.ln_1", "transformer.h.1.ln_1", "transformer.h.1.ln_2", "transformer.h.2.post_ln_1", "transformer.h.0.post_ln_2",
                                  "transformer.ln_f", "transformer.h.1"])
def test_hooks_of_stepped_models_run(name, kind):
    model = stepped_llama()
    want, module, seen = model(IDS)["logits"].detach(), model.get_submodule(name), []
    note = lambda m, *args: seen.append(args) if m is module else None
    if kind == "global":
        handle = torch.nn.modules.module.register_module_forward_hook(note)
    else:
        handle = getattr(module, f"register_{kind}_hook")(note)
    try:
        close(model, want)
        model(IDS)["logits"].sum().backward()
    finally:
        handle.remove()
    assert len(seen) == (1 if "backward" in kind else 2)
    if kind in ("forward", "global"):
        (inputs, output) = seen[0]
        assert output.shape == (2, 7, 32) == inputs[0].shape and len(inputs) == 1      # the stream alone, as in a model of plain blocks


def test_what_a_hook_answers_takes_effect():
    model = stepped_llama()
    x = model.embed(IDS)
    for block in model.transformer.h:
        x = 2 * block(x)
    want = model.lm_head(model.transformer.ln_f(x)).detach()
    for block in model.transformer.h:
        block.register_forward_hook(lambda m, args, out: 2 * out)
    close(model, want)


def test_modules_in_the_place_of_norms_and_blocks_are_called():
    from optimus_dl_amd.modules.model.blocks import LlamaBlock, RMSNorm

    class Shifted(RMSNorm):
        def forward(self, x):
            return super().forward(x) + 1.0

    class Doubled(LlamaBlock):
        def forward(self, x):
            return 2 * super().forward(x)

    class Forwards(torch.nn.Module):                       # a wrapper that passes attributes on
        def __init__(self, inner):
            super().__init__()
            self.inner = inner

        def __getattr__(self, name):
            try:
                return super().__getattr__(name)
            except AttributeError:
                return getattr(self.inner, name)

        def forward(self, x):
            return self.inner(x)

    def reference(model, after=1.0):
        x = model.embed(IDS)
        for block in model.transformer.h:
            x = block(x)
        return model.lm_head(model.transformer.ln_f(x)).detach()

    for change in (lambda m: setattr(m.transformer, "ln_f", Shifted(32)), lambda m: setattr(m.transformer.h[1], "ln_1", Shifted(32)),
                   lambda m: setattr(m.transformer.h[1], "ln_2", torch.nn.LayerNorm(32)), lambda m: setattr(m.transformer.h[0], "post_ln_2", Shifted(32)),
                   lambda m: setattr(m.transformer.h[1], "__class__", Doubled), lambda m: setattr(m.transformer.h[2], "forward", lambda x: x + 1.0),
                   lambda m: m.transformer.h.__setitem__(1, Forwards(m.transformer.h[1]))):
        model = stepped_llama()
        plain = reference(model)
        change(model)
        want = reference(model)
        close(model, want)
        if not isinstance(model.transformer.h[1], Forwards):
            assert (want - plain).abs().max() > 0.01


def test_blocks_sharded_in_place(tmp_path):
    """A block that is sharded by itself has its weights whole while it runs, and nobody else then."""
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.fsdp import fully_shard

    model = stepped_llama()
    want = model(IDS)["logits"].detach()
    model(IDS)["logits"].square().sum().backward()
    grads = {n: p.grad for n, p in model.named_parameters()}
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    try:
        mesh = init_device_mesh("cpu", (1,))
        model = stepped_llama()
        for block in model.transformer.h:
            fully_shard(block, mesh=mesh)
        fully_shard(model, mesh=mesh)
        close(model, want)
        model(IDS)["logits"].square().sum().backward()
        for n, p in model.named_parameters():
            torch.testing.assert_close(p.grad.full_tensor(), grads[n], rtol=1e-4, atol=1e-5 * float(grads[n].abs().max()))
    finally:
        dist.destroy_process_group()


def fake_codes(monkeypatch):
    """4-bit weights without a GPU."""
    from optimus_dl_amd.modules import fp4_linear as F4

    def quantise(w, group):
        if w.dtype not in (torch.float32, torch.bfloat16):
            raise F4.native.NativeError(f"weights of {w.dtype}")
        return torch.zeros(w.shape[0], w.shape[1] // 2, dtype=torch.uint8), torch.zeros(w.shape[0], w.shape[1] // group, dtype=torch.bfloat16)

    monkeypatch.setattr(F4.native, "fp4_quantise", quantise)
    return F4.FP4Linear


def test_linears_with_hooks_keep_them(monkeypatch):
    from optimus_dl_amd.modules.model_transforms import build_model_transform

    FP4Linear = fake_codes(monkeypatch)
    net = torch.nn.Sequential(*(torch.nn.Linear(64, 64) for _ in range(5)))
    seen = []
    net[1].register_forward_hook(lambda m, args, out: seen.append(m))
    net[2].register_forward_pre_hook(lambda m, args: seen.append(m))
    net[3].forward = lambda x: seen.append(net[3]) or x
    t = build_model_transform({"_name": "fp4_linear", "group_size": 32})
    t.apply(net)
    assert [isinstance(m, FP4Linear) for m in net] == [True, False, False, False, True] and t.left == ["1", "2", "3"] and t.replaced == 2
    with torch.no_grad():
        net(torch.zeros(1, 64))
    assert seen == [net[1], net[2], net[3]]


@pytest.mark.parametrize("bad", ["not finite", "type", "both"])
def test_a_model_that_is_refused_is_left_whole(monkeypatch, bad):
    from optimus_dl_amd import native
    from optimus_dl_amd.modules.model_transforms import build_model_transform

    fake_codes(monkeypatch)
    net = torch.nn.Sequential(torch.nn.Linear(64, 64), torch.nn.Sequential(torch.nn.Linear(64, 64), torch.nn.Linear(64, 64)), torch.nn.Linear(64, 64))
    if bad == "not finite":
        net[1][1].weight.data[3, 5] = float("inf")
    elif bad == "type":
        net[1][1].half()
    else:
        net[1][1].weight.data[0, 0] = float("nan")
        net[1][0].half()
    before = list(net.modules())
    with pytest.raises((ValueError, native.NativeError)):
        build_model_transform({"_name": "fp4_linear"}).apply(net)
    assert all(a is b for a, b in zip(before, net.modules())) and len(before) == len(list(net.modules()))


def test_a_model_on_the_cpu_is_refused_whole():
    from optimus_dl_amd import native
    from optimus_dl_amd.modules.model_transforms import build_model_transform

    net = torch.nn.Sequential(torch.nn.Linear(64, 64), torch.nn.Linear(64, 64))
    if native.is_built():
        with pytest.raises(native.NativeError, match="GPU"):
            build_model_transform({"_name": "fp4_linear"}).apply(net)
    assert type(net[0]) is type(net[1]) is torch.nn.Linear


def test_which_products_of_a_few_rows_are_cut_into_runs():
    """What the comparisons of few rows of a long K rely on: one launch without partial results up to some 41 000 inputs of many columns, runs beyond."""
    from optimus_dl_amd import native

    if not native.is_built():
        pytest.skip("library not built")
    runs = native.load().odl_fp8_fp4_linear_runs
    for rows, n, k, group in ((16, 1000, 5152, 32), (16, 4100, 5248, 128), (11, 4100, 7200, 32), (16, 100, 4128, 32), (7, 1030, 8256, 64), (4, 1030, 14464, 128),
                              (1, 3001, 32800, 32), (1, 4099, 41024, 64)):
        assert runs(rows, n, k, group) == 0, (rows, n, k, group)
    for rows, n, k, group in ((1, 40, 65568, 32), (2, 300, 131392, 64), (5, 40, 262528, 128)):
        assert runs(rows, n, k, group) > 8, (rows, n, k, group)
