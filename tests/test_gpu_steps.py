"""Decoders that run in steps over a paged cache on the GPU: prompts, single tokens, drafts, 4-bit and FP8 Linears, captured steps."""
import pytest
import torch

from optimus_dl_amd.modules.amp import create_fp8_recipe, fp8_autocast
from optimus_dl_amd.modules.model import GPT2, GPT2Config, Llama, LlamaConfig, Qwen3, Qwen3Config
from optimus_dl_amd.modules.model_transforms import build_model_transform

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")
SIZES = dict(vocab_size=512, n_layer=2, n_head=4, n_embd=256, block_size=256)


def model(family, dtype=torch.bfloat16):
    torch.manual_seed(0)
    with CUDA:
        m = {"llama": lambda: Llama(LlamaConfig(n_kv_head=2, intermediate_size=512, post_norms=True, layer_scale=0.5, **SIZES)),
             "plain": lambda: Llama(LlamaConfig(n_kv_head=4, intermediate_size=512, **SIZES)),
             "qwen3": lambda: Qwen3(Qwen3Config(n_kv_head=2, head_dim=64, intermediate_size=512, **SIZES)),
             "gpt2": lambda: GPT2(GPT2Config(**SIZES))}[family]()
    return m.to(dtype).eval()


def run(m, ids, counts, cache):
    s, at, got = [cache.add() for _ in ids], 0, []
    for n in counts:
        batch = cache.batch(s, [n] * len(s))
        got.append(m.step(ids[:, at:at + n].reshape(-1), cache, batch)["logits"].view(len(s), n, -1))
        at += n
    return torch.cat(got, 1)


@pytest.mark.parametrize("family", ["llama", "plain", "qwen3", "gpt2"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_steps_answer_what_a_forward_does(family, dtype):
    """Beside an fp32 forward of the same weights.  A block rounds some 12 tensors to bf16 on its way (2^-8 each, of their own size); two blocks, head and
    embedding: 26 half steps at most.  An fp32 model rounds what goes into the cache and comes out of attention: 5 a block."""
    m = model(family, dtype)
    exact = model(family, torch.float32)
    exact.load_state_dict({k: v.float() for k, v in m.state_dict().items()})
    ids = torch.randint(0, 512, (3, 80), device=CUDA, generator=torch.Generator(device="cuda").manual_seed(1))
    with torch.no_grad():
        want = exact(ids)["logits"]
        got = run(m, ids, (33, 1, 1, 4, 40, 1), m.new_cache(40, page_size=16)).float()
    assert (got - want).norm() <= (26 if dtype == torch.bfloat16 else 10) * 2.0 ** -8 * want.norm()


def test_an_8_bit_cache():
    """Keys and values are off by half a step of E4M3 at most (2^-4) where they are not tiny; they enter one of two terms of each of the four halves' streams."""
    m = model("llama")
    ids = torch.randint(0, 512, (2, 60), device=CUDA, generator=torch.Generator(device="cuda").manual_seed(2))
    with torch.no_grad():
        want = run(m, ids, (50, 1, 9), m.new_cache(20, page_size=16)).float()
        got = run(m, ids, (50, 1, 9), m.new_cache(20, page_size=16, dtype=torch.float8_e4m3fn)).float()
    assert (got - want).norm() <= 2 * 2.0 ** -4 * want.norm() and not torch.equal(got, want)


def test_with_4_bit_and_8_bit_linears():
    m = model("llama")
    build_model_transform({"_name": "fp4_linear"}).apply(m)
    build_model_transform({"_name": "fp8_linear"}).apply(m)
    ids = torch.randint(0, 512, (4, 33), device=CUDA, generator=torch.Generator(device="cuda").manual_seed(3))
    with torch.no_grad(), fp8_autocast(CUDA, create_fp8_recipe("tensorwise", "hybrid")):
        got = run(m, ids, (16, 1, 16), m.new_cache(40, page_size=16))
    assert got.isfinite().all() and got.shape == (4, 33, 512)


@pytest.mark.parametrize("cache_dtype", [torch.bfloat16, torch.float8_e4m3fn])
def test_drafts_and_single_tokens(cache_dtype):
    """Greedy, several sequences, drafts of different lengths of which some are wrong.  A step over drafts and a step over one token add in other orders, so that near ties may
    be settled differently: every token that was emitted has to be the largest logit, to 8 half steps of bf16, of one forward over all of them."""
    m = model("llama")
    prompts = torch.randint(0, 512, (3, 9), device=CUDA, generator=torch.Generator(device="cuda").manual_seed(4))
    cache = m.new_cache(60, page_size=8, dtype=cache_dtype)
    s = [cache.add() for _ in range(3)]
    first = m.step(prompts.reshape(-1), cache, cache.batch(s, [9] * 3), last_only=True)["logits"].argmax(-1)
    texts = [prompts[i].tolist() + [int(first[i])] for i in range(3)]
    for turn in range(12):
        counts = [1 + (turn + i) % 4 for i in range(3)]
        fed = []
        for i in range(3):
            fed += [texts[i][-1]] + [(texts[i][-1] * 7 + j) % 512 for j in range(counts[i] - 1)]
        rows = torch.tensor(fed + [0, 0], device=CUDA)                                 # (two rows of padding)
        batch = cache.batch(s, counts)
        r = m.verify_step(rows, cache, batch, torch.rand(len(fed) + 2, device=CUDA), temperature=0.0)
        for i, first_row in enumerate(batch.offsets[:-1].tolist()):
            n = int(r.accepted[i])
            texts[i] += r.tokens[first_row:first_row + n + 1].tolist()
            cache.shorten(s[i], len(texts[i]) - 1)
        assert r.tokens[len(fed):].tolist() == [-1, -1]
    for text in texts:
        with torch.no_grad():
            c = m.new_cache(60, page_size=8, dtype=cache_dtype)
            logits = m.step(torch.tensor(text, device=CUDA), c, c.batch([c.add()], [len(text)]))["logits"].float()
        at = torch.arange(8, len(text) - 1, device=CUDA)
        chosen = logits[at].gather(1, torch.tensor(text[9:], device=CUDA).unsqueeze(1)).squeeze(1)
        assert (chosen >= logits[at].amax(1) - 8 * 2.0 ** -8 * logits[at].abs().amax()).all()


def test_drawn_tokens_with_a_drafter():
    """The model drafts for itself: all drafts hold, whatever is drawn."""
    m = model("qwen3")
    cache = m.new_cache(30, page_size=16)
    s = [cache.add(), cache.add()]
    prompt = torch.randint(0, 512, (2, 20), device=CUDA, generator=torch.Generator(device="cuda").manual_seed(5))
    m.step(prompt.reshape(-1), cache, cache.batch(s, [20, 20]))
    rows = torch.randint(0, 512, (8,), device=CUDA, generator=torch.Generator(device="cuda").manual_seed(6))
    batch = cache.batch(s, [4, 4])
    logits = m.step(rows, cache, batch)["logits"]
    for i in s:
        cache.shorten(i, 20)
    r = m.verify_step(rows, cache, cache.batch(s, [4, 4]), torch.rand(8, device=CUDA), draft_logits=logits, temperature=0.8)
    assert r.accepted.tolist() == [3, 3] and (r.tokens >= 0).all() and (r.logprobs <= 0).all()
    assert r.tokens[:3].tolist() == rows[1:4].tolist()


@pytest.mark.parametrize("family", ["llama", "gpt2"])
def test_a_captured_step(family):
    """One decode step of three sequences as a graph: replayed on new tokens and lengths, it answers what the eager step does, bit by bit."""
    m = model(family)
    ids = torch.randint(0, 512, (3, 40), device=CUDA, generator=torch.Generator(device="cuda").manual_seed(7))
    cache = m.new_cache(30, page_size=16)
    s = [cache.add() for _ in range(3)]
    m.step(ids[:, :30].reshape(-1), cache, cache.batch(s, [30] * 3))
    static = cache.batch(s, [1] * 3)._replace(max_new=1)
    token = ids[:, 30].clone()
    want0 = m.step(token, cache, static)["logits"]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.step(token, cache, static)["logits"]
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want0)
    for i in range(31, 38):
        batch = cache.batch(s, [1] * 3)
        for a, b in zip(static[:3], batch[:3]):
            a.copy_(b)
        token.copy_(ids[:, i])
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(m.step(ids[:, i].clone(), cache, batch)["logits"], got)
