"""The operators around the Linear where no GPU is needed: refusals of the C entries and the wrappers, and the forms that CPU tensors take."""
import pytest
import torch

from optimus_dl_amd import native
from optimus_dl_amd.modules.fp4_linear import E2M1, FP4Linear, dequantise_fp4, fp4_linear
from optimus_dl_amd.modules.fused import residual_norm
from optimus_dl_amd.modules.logprobs import token_logprobs

needs_library = pytest.mark.skipif(not native.is_built(), reason="library not built")
P = 4096                                                   # any aligned address: refused calls never reach it


def refused(name, args, word):
    L = native.load()
    assert getattr(L, name)(*args) != 0, (name, word)
    assert word in L.odl_fp8_last_error().decode(), (word, L.odl_fp8_last_error())


@needs_library
def test_residual_norm_entry_refuses():
    ok = dict(x=P, xd=1, h=P, hd=0, w=P, post=P, gate=P, gs=64, rows=4, cols=64, a=1.0, eps=1e-6, pe=1e-6, y=P, z=P, stats=P, parts=P, stream=None)
    for change, word in ((dict(rows=-1), "negative"), (dict(xd=2), "x_dtype"), (dict(xd=0, hd=1), "h_dtype"), (dict(cols=60, gs=60), "multiple of 8"), (dict(cols=0), "multiple of 8"),
                         (dict(cols=8200), "8192"), (dict(gs=2), "gate"), (dict(w=None), "null"), (dict(y=None), "null"), (dict(x=None), "null"),
                         (dict(x=P + 8), "aligned"), (dict(z=P + 2), "aligned")):
        refused("odl_fp8_residual_norm", tuple({**ok, **change}.values()), word)
    ok = dict(dy=P, dz=P, x=P, xd=1, h=P, hd=0, w=P, post=P, gate=P, gs=1, rows=4, cols=64, a=1.0, stats=P, dx=P, dh=P, parts=P, dw=P, dpost=P, dgate=P, ws=P,
              stream=None)
    for change, word in ((dict(cols=-8), "negative"), (dict(hd=3), "h_dtype"), (dict(cols=12), "multiple of 8"), (dict(gs=63), "gate"), (dict(dx=None), "null"),
                         (dict(ws=None), "workspace"), (dict(dw=None), "dweight"), (dict(post=None), "not there"), (dict(gate=None), "not there"),
                         (dict(dz=P + 4), "aligned"), (dict(ws=P + 4), "aligned")):
        refused("odl_fp8_residual_norm_bwd", tuple({**ok, **change}.values()), word)


@needs_library
def test_token_logprobs_entry_refuses():
    ok = dict(l=P, dt=0, rows=4, stride=100, vocab=100, t=P, ign=-100, it=1.0, k=5, lp=P, H=P, st=P, top=P, ids=P, ws=None, wsb=0, stream=None)
    for change, word in ((dict(rows=-1), "negative"), (dict(dt=2), "dtype"), (dict(vocab=0), "columns"), (dict(vocab=(1 << 24) + 1), "columns"), (dict(rows=1 << 22), "rows"),
                         (dict(k=-1), "top_k"), (dict(k=65), "top_k"), (dict(vocab=4), "top_k"), (dict(it=0.0), "temperature"),
                         (dict(it=float("nan")), "temperature"), (dict(it=float("inf")), "temperature"), (dict(l=None), "null"), (dict(ids=None), "null"),
                         (dict(vocab=1 << 20), "workspace"), (dict(vocab=1 << 20, ws=P, wsb=4), "workspace")):
        refused("odl_fp8_token_logprobs", tuple({**ok, **change}.values()), word)
    assert native.load().odl_fp8_token_logprobs(*{**ok, "rows": 0}.values()) == 0
    ok = dict(l=P, dt=1, rows=4, stride=100, vocab=90, padded=100, t=P, ign=-100, it=1.0, k=5, ids=P, st=P, H=P, a=P, b=P, c=P, dl=P, parts=P, stream=None)
    for change, word in ((dict(vocab=101), "columns"), (dict(dt=-1), "dtype"), (dict(k=91), "top_k"), (dict(ids=None), "null"), (dict(dl=None), "null"), (dict(st=None), "null")):
        refused("odl_fp8_token_logprobs_bwd", tuple({**ok, **change}.values()), word)


@needs_library
def test_fp4_entries_refuse():
    ok = dict(x=P, ldx=128, codes=P, scales=P, group=32, bias=None, bd=0, M=4, N=16, K=128, y=P, ws=None, wsb=0, stream=None)
    for change, word in ((dict(M=-1), "negative"), (dict(group=16), "group"), (dict(bias=P, bd=2), "bias_dtype"), (dict(K=100), "multiple"), (dict(K=0), "multiple"),
                         (dict(x=None), "null"), (dict(scales=None), "null"), (dict(ldx=132), "aligned"), (dict(ldx=64), "aligned"), (dict(codes=P + 8), "aligned"),
                         (dict(x=P + 2), "aligned"), (dict(ldx=(1 << 24) + 8), "2^24"), (dict(N=(1 << 22) + 1), "2^22"), (dict(M=(1 << 20) + 1), "2^20"),
                         (dict(M=32, N=4096, K=14336, ldx=14336), "workspace"), (dict(M=32, N=4096, K=14336, ldx=14336, ws=P, wsb=1 << 20), "workspace")):
        refused("odl_fp8_fp4_linear", tuple({**ok, **change}.values()), word)
    runs = native.load().odl_fp8_fp4_linear_runs
    assert runs(1, 14336, 4096, 128) == runs(24, 2304, 768, 32) == runs(64, 28672, 8192, 64) == runs(0, 4096, 4096, 32) == 0 and 1 < runs(32, 4096, 14336, 32) <= 14
    ok = dict(w=P, src=0, N=16, K=128, group=64, codes=P, scales=P, stream=None)
    for change, word in ((dict(N=-1), "negative"), (dict(src=2), "src_dtype"), (dict(group=0), "group"), (dict(K=96), "multiple"), (dict(codes=None), "null"), (dict(w=P + 4), "aligned")):
        refused("odl_fp8_fp4_quantise", tuple({**ok, **change}.values()), word)


@needs_library
def test_wrappers_refuse_cpu_tensors():
    x, one, ids = torch.zeros(4, 64, dtype=torch.bfloat16), torch.ones(64), torch.zeros(4, dtype=torch.int64)
    calls = {"residual_norm": (x, x, one, 1e-6), "residual_norm_bwd": (x, x, x, x, one, None, None, 1.0, torch.zeros(2, 4)), "token_logprobs": (x, ids, 64),
             "token_logprobs_bwd": (x, ids, 64, 0, 1.0, -100, None, torch.zeros(2, 4), torch.zeros(4), None, None, None),
             "fp4_linear": (x, torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.bfloat16)), "fp4_quantise": (x, 32)}
    for name, args in calls.items():
        with pytest.raises(native.NativeError, match="GPU"):
            getattr(native, name)(*args)


def test_arguments_are_checked():
    x, w = torch.zeros(4, 64), torch.ones(64)
    for args, kwargs in (((x, x[:3], w, 1e-6), {}), ((x, x, w[:63], 1e-6), {}), ((x, x, w, 1e-6), {"post_weight": w[:8]}), ((x, x, w, 1e-6), {"gate": w[:2]}),
                         ((x[0, 0], x[0, 0], w, 1e-6), {})):
        with pytest.raises(ValueError, match="residual_norm"):
            residual_norm(*args, **kwargs)
    t = torch.zeros(4, dtype=torch.int64)
    for args, kwargs in (((x, t[:3]), {}), ((x, t.int()), {}), ((x.long(), t), {}), ((x, t), {"n_vocab": 0}), ((x, t), {"n_vocab": 65}), ((x, t), {"top_k": 65}),
                         ((x, t), {"top_k": -1}), ((x, t), {"n_vocab": 3, "top_k": 4}), ((x, t), {"temperature": 0.0}), ((x, t), {"temperature": float("inf")}),
                         ((x, t), {"temperature": float("nan")}), ((x, t), {"temperature": -1.0}), ((x, t), {"temperature": 1e-31}), ((x, t.unsqueeze(1)), {})):
        with pytest.raises(ValueError, match="token_logprobs"):
            token_logprobs(*args, **kwargs)
    codes, scales, xb = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.bfloat16), x.bfloat16()
    for args in ((x, codes, scales), (xb[:, :32], codes, scales), (xb, codes.int(), scales), (xb, codes, scales.float()), (xb, codes, scales[:7]), (xb, codes, scales[:, :0]),
                 (xb, codes, scales.repeat(1, 2)), (xb, codes, scales, torch.zeros(7))):
        with pytest.raises(ValueError, match="fp4"):
            fp4_linear(*args)
    with pytest.raises(RuntimeError, match="no backward"):
        fp4_linear(xb.requires_grad_(True), codes, scales)
    for bad in ((60, 8), (64, 8, True, 16), (0, 8)):
        with pytest.raises(ValueError, match="FP4Linear"):
            FP4Linear(*bad)


def test_plain_forms_against_differences():
    """The torch operations that CPU tensors take, in 64 bits: gradients against differences."""
    g = torch.Generator().manual_seed(0)
    n = lambda *s: torch.randn(s, generator=g, dtype=torch.float64).requires_grad_(True)
    x, h, w, wp, gate = n(3, 10), n(3, 10), n(10), n(10), n(10)
    f = lambda x, h, w, wp, gate: residual_norm(x, h, w, 1e-3, post_weight=wp, gate=gate, residual_scale=0.7)
    assert torch.autograd.gradcheck(f, (x, h, w, wp, gate)) and torch.autograd.gradcheck(f, (x, h, w, wp, n(1)))
    assert torch.autograd.gradcheck(lambda x, h, w: residual_norm(x, h, w, 1e-3), (x, h, w))
    t = torch.tensor([2, -100, 9])
    assert torch.autograd.gradcheck(lambda l: token_logprobs(l, t, n_vocab=10, top_k=3, temperature=0.7)[:3], (n(3, 12),))


def test_plain_log_probabilities_of_rows_that_are_masked():
    inf = float("inf")
    l = torch.tensor([[0.0, 0, -inf, -inf], [-inf] * 4, [1, inf, 0, 0], [float("nan"), 0, 0, 0], [3, 1, 2, 2]], requires_grad=True)
    r = token_logprobs(l, torch.tensor([1, 0, 0, -100, 7]), top_k=3)
    (grad,) = torch.autograd.grad((r.logprobs[:2].sum() + r.entropy[:2].sum()), l)
    assert grad[:2].isfinite().all() and not grad[1].any()
    ln2 = torch.tensor(2.0).log().item()
    assert abs(r.logprobs[0].item() + ln2) < 1e-6 and abs(r.entropy[0].item() - ln2) < 1e-6 and r.top_ids[0].tolist() == [0, 1, 2] and r.top_logprobs[0, 2] == -inf
    assert r.logprobs[1] == -inf and r.entropy[1] == 0 and r.top_ids[1].tolist() == [0, 1, 2]
    assert r.logprobs[2].isnan() and r.top_ids[2].tolist() == [-1] * 3
    assert r.logprobs[3] == 0 and r.entropy[3] == 0 and r.top_ids[3].tolist() == [-1] * 3 and not r.top_logprobs[3].any()
    assert r.logprobs[4].isnan() and r.entropy[4].isfinite() and r.top_ids[4].tolist() == [0, 2, 3]


def test_fp4_weights_on_the_cpu():
    codes = torch.arange(256).to(torch.uint8).reshape(8, 32)
    scales = torch.full((8, 2), 0.5, dtype=torch.bfloat16)
    w = dequantise_fp4(codes, scales)
    assert w.shape == (8, 64) and w[0, :4].tolist() == [0.0, 0.0, 0.25, 0.0] and w[1, 0].item() == 0.0 and set(w.abs().unique().tolist()) == {v / 2 for v in E2M1}
    x = torch.randn(3, 64).bfloat16()
    assert torch.equal(fp4_linear(x, codes, scales), (x.float() @ w.t()).bfloat16())
    m = FP4Linear.from_codes(codes, scales, torch.ones(8))
    assert m.group_size == 32 and m.in_features == 64 and torch.equal(m(x), (x.float() @ w.t() + 1).bfloat16())
    assert sorted(m.state_dict()) == ["bias", "codes", "scale_bits"] and torch.equal(m.double().scales, scales)


def test_transform_replaces_linears_of_whole_groups(monkeypatch):
    from optimus_dl_amd.modules import fp4_linear as F4
    from optimus_dl_amd.modules.model_transforms import build_model_transform

    fake = lambda w, group: (torch.zeros(w.shape[0], w.shape[1] // 2, dtype=torch.uint8), torch.zeros(w.shape[0], w.shape[1] // group, dtype=torch.bfloat16))
    monkeypatch.setattr(F4.native, "fp4_quantise", fake)
    shared = torch.nn.Linear(64, 64)
    net = torch.nn.ModuleDict({"a": shared, "b": shared, "odd": torch.nn.Linear(40, 8), "lm_head": torch.nn.Linear(64, 8),
                               "inner": torch.nn.Sequential(torch.nn.Linear(128, 8, bias=False), torch.nn.ReLU())})
    t = build_model_transform({"_name": "fp4_linear", "group_size": 64})
    assert t.apply(net) is net and t.replaced == 2 and t.left == ["odd"]
    assert isinstance(net["a"], FP4Linear) and net["a"] is net["b"] and net["a"].bias is not None and type(net["lm_head"]) is torch.nn.Linear
    assert isinstance(net["inner"][0], FP4Linear) and net["inner"][0].group_size == 64
    assert build_model_transform({"_name": "fp4_linear", "enabled": False}).apply(torch.nn.Sequential(torch.nn.Linear(64, 64)))[0].__class__ is torch.nn.Linear
    with pytest.raises(ValueError):
        t.apply(torch.nn.Linear(64, 64))


def small_llama(**kwargs):
    from optimus_dl_amd.modules.model import Llama, LlamaConfig

    torch.manual_seed(0)
    return Llama(LlamaConfig(vocab_size=50, n_layer=2, n_head=2, n_kv_head=1, n_embd=16, intermediate_size=24, **kwargs))


def test_plain_models_are_what_they_were_and_stepped_ones_chain_their_norms():
    ids = torch.arange(12).reshape(2, 6)
    plain = small_llama()
    assert not any("post_ln" in n or "gate" in n for n, _ in plain.named_parameters())
    x = plain.embed(ids)
    for block in plain.transformer.h:
        x = x + block.attn(block.ln_1(x))
        x = x + block.mlp(block.ln_2(x))
    assert torch.equal(plain(ids)["logits"], plain.lm_head(plain.transformer.ln_f(x)))
    m = small_llama(post_norms=True, layer_scale=0.3, residual_scale=0.9)
    assert {"transformer.h.0.post_ln_1.weight", "transformer.h.1.post_ln_2.weight", "transformer.h.0.gate_1", "transformer.h.1.gate_2"} <= set(m.state_dict())
    x = m.embed(ids)
    for block in m.transformer.h:
        alone = block(x)
        x = 0.9 * x + block.gate_1 * block.post_ln_1(block.attn(block.ln_1(x)))
        x = 0.9 * x + block.gate_2 * block.post_ln_2(block.mlp(block.ln_2(x)))
        assert torch.allclose(alone, x, rtol=1e-5, atol=1e-6)
    assert torch.allclose(m(ids)["logits"], m.lm_head(m.transformer.ln_f(x)), rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("kwargs", [dict(post_norms=True), dict(layer_scale=0.5), dict(residual_scale=0.7), dict(post_norms=True, layer_scale=0.3, residual_scale=0.9)])
def test_loss_of_a_stepped_model_against_differences(monkeypatch, kwargs):
    """In 64 bits (the RMSNorm module, which a model begins with, computes in 32 by itself): central differences of size h are off by h^2 times a
    third derivative, and by 1e-16 / h."""
    from optimus_dl_amd.modules.model import blocks

    monkeypatch.setattr(blocks.RMSNorm, "forward", lambda self, x: x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + self.eps) * self.weight)
    m = small_llama(**kwargs).double()
    ids = torch.arange(12).reshape(2, 6) % 50

    def loss():
        r = m.score(ids, top_k=2)
        return -(r.logprobs.sum() + 0.1 * r.entropy.sum() + 0.01 * r.top_logprobs.sum())

    params = list(m.parameters())
    grads = torch.autograd.grad(loss(), params)
    g = torch.Generator().manual_seed(1)
    along = [torch.randn(p.shape, generator=g, dtype=p.dtype) for p in params]
    ends = []
    for sign in (1, -1):
        with torch.no_grad():
            for p, v in zip(params, along):
                p.add_(v, alpha=sign * 1e-5)
            ends.append(loss().item())
            for p, v in zip(params, along):
                p.sub_(v, alpha=sign * 1e-5)
    want = sum((gr * v).sum().item() for gr, v in zip(grads, along))
    assert abs((ends[0] - ends[1]) / 2e-5 - want) < 1e-5 * (1 + abs(want)) and all(gr.abs().max() > 0 for gr in grads)


def test_score_asks_for_the_next_token():
    m = small_llama()
    ids = torch.arange(12).reshape(2, 6)
    with torch.no_grad():
        r = m.score(ids, top_k=3, temperature=0.5)
        logp = torch.log_softmax(m(ids)["logits"] / 0.5, -1)
        assert torch.allclose(r.logprobs[:, :-1], logp[:, :-1].gather(-1, ids[:, 1:, None]).squeeze(-1), atol=1e-5) and not r.logprobs[:, -1].any()
        assert torch.equal(r.top_ids[:, :-1], logp[:, :-1].topk(3).indices) and (r.top_ids[:, -1] == -1).all()
        one = m.score(ids[:, :1], targets=ids[:, 1:2])
        assert torch.allclose(one.logprobs, torch.log_softmax(m(ids[:, :1])["logits"], -1).gather(-1, ids[:, 1:2, None]).squeeze(-1), atol=1e-6)


def test_only_conversions_that_widen_codes_need_no_saturating_mode():
    from optimus_dl_amd.build import check_saturating_conversions

    def found(instruction):
        return len(check_saturating_conversions(f"_Z1kv:\n\t{instruction}\n", "x.s"))

    assert found("v_cvt_scalef32_pk_bf16_fp4 v0, v1, 1.0") == 0
    assert found("v_cvt_scalef32_pk_fp4_bf16 v0, v1, 1.0") == 1
    assert found("v_cvt_scalef32_pk_bf16_fp8 v0, v1, 1.0") == 1
    assert found("v_cvt_scalef32_pk_bf8_f32 v0, v1, v2, 1.0") == 1


@pytest.mark.parametrize("wrapped", [(0,), (1,), (2,), (0, 2), (0, 1, 2)])
def test_blocks_behind_a_wrapper_take_and_give_the_stream_alone(wrapped):
    from optimus_dl_amd.modules.model.families import Llama, LlamaConfig

    class Wrapper(torch.nn.Module):
        def __init__(self, inner):
            super().__init__()
            self.inner = inner

        def forward(self, x):
            return self.inner(x)

    torch.manual_seed(0)
    model = Llama(LlamaConfig(vocab_size=50, n_layer=3, n_embd=32, n_head=2, n_kv_head=2, intermediate_size=64, post_norms=True,
                              layer_scale=0.5, residual_scale=0.9))
    ids = torch.randint(0, 50, (2, 7))
    want = model(ids)["logits"]
    for i in wrapped:
        model.transformer.h[i] = Wrapper(model.transformer.h[i])
    # the same fp32 operations, some in another order: a few roundings of values near one
    torch.testing.assert_close(model(ids)["logits"], want, rtol=0, atol=64 * 2.0 ** -24 * float(want.abs().max()))
