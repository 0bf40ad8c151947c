"""The paged cache on the CPU: the operators' plain forms against their definitions, the book-keeping of pages, decoders that run in steps, refusals."""
import ctypes

import pytest
import torch

from optimus_dl_amd import native
from optimus_dl_amd.modules.drafts import verify_drafts
from optimus_dl_amd.modules.model import GPT2, GPT2Config, Llama, LlamaConfig, Qwen3, Qwen3Config
from optimus_dl_amd.modules.paged import PagedBatch, PagedKVCache, append_kv, paged_attention
from tests.paged_helpers import BF16, E4M3, Case, angles, append32, assert_near, attention64, bits


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("norm", [True, False])
def test_append(cache, interleaved, norm):
    c = Case([1, 3, 0, 9], [1, 30, 9, 9], 6, 2, 32, 4, cache, pad=2, seed=1)
    cos, sin = angles(c.width * 4, 8)
    weights = [1 + 0.2 * torch.randn(32) for _ in range(2)] if norm else [None, None]
    want = append32(c, cos, sin, interleaved, *weights)
    q = append_kv(c.q, c.k, c.v, c.keys, c.values, *c.batch(), cos=cos, sin=sin, interleaved=interleaved, q_weight=weights[0], k_weight=weights[1], **c.scales())
    for got, w in zip((q, c.keys, c.values), want):
        assert torch.equal(bits(got), bits(w))


@pytest.mark.parametrize("window,softcap", [(0, 0.0), (7, 0.0), (0, 10.0)])
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_attention(window, softcap, cache):
    c = Case([1, 20, 0, 3], [40, 25, 9, 3], 4, 2, 16, 8, cache, pad=3, seed=2)
    c.pages[0, 2] = -1
    want, far = attention64(c, 0.25, window, softcap)
    got = paged_attention(c.q, c.keys, c.values, *c.batch(), scale=0.25, window=window, softcap=softcap, **c.scales())
    assert_near(got, want, far)


def test_attention_of_odd_values():
    c = Case([4], [20], 2, 1, 16, 8, seed=3)
    page = int(c.pages[0, 2])
    c.values[page, 0, 1, 2], c.values[page, 0, 2, 3], c.keys[page, 0, 4:], c.values[page, 0, 4:] = float("nan"), float("inf"), float("nan"), float("nan")
    want, far = attention64(c, 0.25)
    assert_near(paged_attention(c.q, c.keys, c.values, *c.batch(), scale=0.25), want, far)


def test_pages_are_handed_out_and_come_back():
    cache = PagedKVCache(2, 2, 16, pages=6, page_size=4, max_tokens=16, device="cpu", dtype=torch.float32)
    a, b = cache.add(), cache.add()
    batch = cache.batch([a, b], [5, 4])
    assert cache.free_pages == 3 and batch.offsets.tolist() == [0, 5, 9] and batch.lengths.tolist() == [5, 4] and batch.max_new == 5
    assert len(set(batch.pages[0, :2].tolist() + batch.pages[1, :1].tolist())) == 3 and batch.pages.shape == (2, 4)
    assert batch.positions(11).tolist() == [0, 1, 2, 3, 4, 0, 1, 2, 3, 0, 0]
    batch = cache.batch([b, a], [1, 2])
    assert cache.free_pages == 2 and batch.lengths.tolist() == [5, 7] and batch.positions(3).tolist() == [4, 5, 6]
    assert cache.batch([a, b], [5, 5]).lengths.tolist() == [12, 10] and cache.free_pages == 0
    with pytest.raises(RuntimeError, match="1 pages wanted"):
        cache.batch([b, a], [2, 1])
    assert cache.free_pages == 0 and cache.length(a) == 12 and cache.length(b) == 10
    with pytest.raises(ValueError, match="of 16"):
        cache.batch([a], [10])
    with pytest.raises(ValueError, match="each once"):
        cache.batch([a, a], [1, 1])
    cache.shorten(a, 4)
    assert cache.free_pages == 2 and cache.length(a) == 4
    with pytest.raises(ValueError, match="not 5"):
        cache.shorten(a, 5)
    cache.remove(a)
    assert cache.free_pages == 3
    cache.batch([b], [0])
    with pytest.raises(ValueError, match="power of two"):
        PagedKVCache(1, 1, 16, pages=1, page_size=3, device="cpu")


def models():
    torch.manual_seed(0)
    sizes = dict(vocab_size=100, n_layer=2, n_head=4, n_embd=64)
    yield Llama(LlamaConfig(n_kv_head=2, post_norms=True, layer_scale=0.5, **sizes))
    yield Llama(LlamaConfig(**sizes))
    yield Qwen3(Qwen3Config(n_kv_head=2, head_dim=32, **sizes))
    yield GPT2(GPT2Config(**sizes))


@pytest.mark.parametrize("which", range(4))
def test_steps_answer_what_a_forward_does(which):
    """fp32 both ways.  The orders of sums of up to 64 products and 20 terms differ: 1e-5 of logits of size 1 is far more than they can."""
    m = list(models())[which].eval()
    ids = torch.randint(0, 100, (3, 20))
    full = m(ids)["logits"].detach()
    cache = m.new_cache(40, page_size=4, max_tokens=32)
    s = [cache.add() for _ in range(3)]
    at = 0
    for n in (7, 1, 1, 5, 6):
        got = m.step(ids[:, at:at + n].reshape(-1), cache, cache.batch(s, [n] * 3))["logits"].view(3, n, -1)
        assert torch.allclose(got, full[:, at:at + n], atol=1e-5)
        at += n
    cache.shorten(s[1], 10)                          # taken back and run again, beside a prompt
    t = cache.add()
    got = m.step(torch.cat((ids[1, 10:14], ids[0, :9])), cache, cache.batch([s[1], t], [4, 9]))["logits"]
    assert torch.allclose(got[:4], full[1, 10:14], atol=1e-5) and torch.allclose(got[4:], full[0, :9], atol=1e-5)
    last = m.step(torch.cat((ids[1, 14:16], ids[0, 9:12])), cache, cache.batch([s[1], t], [2, 3]), last_only=True)["logits"]
    assert torch.allclose(last, torch.stack((full[1, 15], full[0, 11])), atol=1e-5)


def test_drafting_does_not_change_what_is_generated():
    """Greedy decoding one token at a time, and with drafts of which some are wrong: the same tokens."""
    m = list(models())[0].eval()
    prompt = torch.randint(0, 100, (6,))

    def start():
        cache = m.new_cache(20, page_size=4, max_tokens=64)
        s = cache.add()
        return cache, s, int(m.step(prompt, cache, cache.batch([s], [6]), last_only=True)["logits"].argmax())

    cache, s, token = start()
    plain = [token]
    for _ in range(15):
        plain.append(int(m.step(torch.tensor([plain[-1]]), cache, cache.batch([s], [1]))["logits"].argmax()))
    cache, s, token = start()
    fast, steps = [token], 0
    while len(fast) < 16:
        guess = [(t + (len(fast) + i) % 3 // 2) % 100 for i, t in enumerate(plain[len(fast):len(fast) + 3])]
        rows = torch.tensor([fast[-1]] + guess)
        r = m.verify_step(rows, cache, cache.batch([s], [len(rows)]), torch.rand(len(rows)), temperature=0.0)
        n = int(r.accepted[0])
        fast += r.tokens[:n + 1].tolist()
        cache.shorten(s, 6 + len(fast) - 1)
        steps += 1
    assert fast[:16] == plain and steps < 12


def test_verify_on_the_cpu():
    x = torch.tensor([[0.0, 1.0, 2.0]] * 3)
    offsets, tokens = torch.tensor([0, 3], dtype=torch.int32), torch.tensor([0, 2, 0])
    p = torch.softmax(x[0].double(), 0)
    r = verify_drafts(x, tokens, offsets, torch.tensor([0.6, 0.2, 0.5]))                  # 0.6 < p(2), 0.2 > p(0): then from tokens 1 and 2
    assert r.accepted.tolist() == [1] and r.tokens.tolist() == [2, 2, -1]
    assert torch.allclose(r.logprobs.double(), torch.tensor([p[2].log(), p[2].log(), 0.0], dtype=torch.float64))
    r = verify_drafts(x, tokens, offsets, torch.tensor([0.6, 0.05, 0.1]))
    assert r.accepted.tolist() == [2] and r.tokens.tolist() == [2, 0, 1]
    with pytest.raises(ValueError, match="n_vocab"):
        verify_drafts(x, tokens, offsets, torch.rand(3), n_vocab=4)
    with pytest.raises(ValueError, match="temperature"):
        verify_drafts(x, tokens, offsets, torch.rand(3), temperature=-1.0)
    with pytest.raises(ValueError, match="tokens"):
        verify_drafts(x, tokens.int(), offsets, torch.rand(3))
    with pytest.raises(ValueError, match="draft_logits"):
        verify_drafts(x, tokens, offsets, torch.rand(3), draft_logits=x[:, :2])
    with pytest.raises(ValueError, match="gradient"):
        verify_drafts(x.requires_grad_(True), tokens, offsets, torch.rand(3))


def test_a_row_of_scores_of_minus_infinity_answers_0():
    q, keys = torch.ones(2, 1, 16), torch.zeros(1, 1, 4, 16)
    keys[0, 0, 0, 3] = -torch.inf
    args = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32), torch.tensor([2], dtype=torch.int32)
    y = paged_attention(q, keys, torch.ones_like(keys), *args)
    assert (y[0] == 0).all() and (y[1] == 1).all()             # (the first token sees that key alone)


def test_steps_that_a_model_has_no_place_for():
    model = GPT2(GPT2Config(vocab_size=32, n_embd=32, n_head=2, n_layer=1, block_size=16))
    cache = model.new_cache(pages=4, page_size=8)
    s = cache.add()
    with pytest.raises(ValueError, match="no last one"):
        model.step(torch.zeros(0, dtype=torch.int64), cache, cache.batch([s], [0]), last_only=True)
    batch = cache.batch([s], [1])                              # rows behind the last sequence, and an offset behind the rows
    late = batch._replace(offsets=torch.tensor([0, 9], dtype=torch.int32))
    assert model.step(torch.zeros(3, dtype=torch.int64), cache, late, last_only=True)["logits"].shape == (1, 32)
    wide = model.new_cache(pages=4, page_size=8, max_tokens=17)
    with pytest.raises(ValueError, match="embeddings of 16"):
        model.step(torch.zeros(1, dtype=torch.int64), wide, wide.batch([wide.add()], [1]))


def test_angles_are_not_made_in_a_capture(monkeypatch):
    cache = PagedKVCache(1, 1, 16, pages=1, page_size=8, device="cpu")
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    cache.device = torch.device("cuda")
    with pytest.raises(RuntimeError, match="before a step is captured"):
        cache.angles(lambda *args: args, 16, 1e4)


def test_refusals_of_arguments():
    c = Case([1, 2], [5, 9], 4, 2, 16, 4, seed=4)
    args = (c.keys, c.values, *c.batch())
    for bad, match in (((c.q[:, :3],) + args, "multiple of the heads"), ((c.q,) + args[:2] + (c.pages.long(),) + args[3:], "int32"),
                       ((c.q, c.keys[:, :, :3], c.values[:, :, :3]) + args[2:], "power of two"), ((c.q, c.keys, c.values[:, :1]) + args[2:], "of one type")):
        with pytest.raises(ValueError, match=match):
            paged_attention(*bad)
    for kwargs in ({"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")}, {"window": -1}, {"softcap": -1.0}, {"max_new": -1}):
        with pytest.raises(ValueError, match="window"):
            paged_attention(c.q, *args, **kwargs)
    with pytest.raises(ValueError, match="scale for each"):
        paged_attention(c.q, *args, key_scale=torch.ones(2), value_scale=torch.ones(2))
    with pytest.raises(ValueError, match="gradient"):
        append_kv(c.q.clone().requires_grad_(True), c.k, c.v, *args)
    with pytest.raises(ValueError, match="cos and sin"):
        append_kv(c.q, c.k, c.v, *args, cos=torch.ones(5, 8), sin=torch.ones(5, 8))
    with pytest.raises(ValueError, match="cos and sin"):
        append_kv(c.q, c.k, c.v, *args, cos=torch.ones(64, 8))
    with pytest.raises(ValueError, match="beside q"):
        append_kv(c.q, c.k[:2], c.v[:2], *args)
    with pytest.raises(ValueError, match="weights"):
        append_kv(c.q, c.k, c.v, *args, q_weight=torch.ones(8))


@pytest.fixture
def L():
    if not native.is_built():
        pytest.skip("library not built")
    return native.load()


def entry(L, **change):
    """odl_fp8_append_kv and odl_fp8_paged_attention with pointers that nothing follows: calls that are refused in front of a launch."""
    cache = native._PagedCache(4096, 4096, None, None, 10, 2, 16, 64)
    cache.key_strides[:] = cache.value_strides[:] = (2048, 1024, 64)
    batch = native._PagedBatch(4096, 4096, 4096, 3, 8, 5, 5)
    args = dict(heads=4, scale=1.0, window=0, softcap=0.0, out=4096, ws=4096, floats=1 << 30, q=4096, strides=(256, 64), positions=80, half=16, interleaved=1)
    for k, v in change.items():
        target = next((o for o in (cache, batch) if hasattr(o, k)), None)
        if target is None:
            args[k] = v
        elif k.endswith("strides"):
            getattr(target, k)[:] = v
        else:
            setattr(target, k, v)
    q, kv = (ctypes.c_int64 * 2)(*args["strides"]), (ctypes.c_int64 * 2)(128, 64)
    refs = ctypes.byref(cache), ctypes.byref(batch)
    attend = lambda: L.odl_fp8_paged_attention(args["q"], q, args["heads"], 8, *refs, args["scale"], args["window"], args["softcap"], args["out"], args["ws"], args["floats"], None)
    append = lambda: L.odl_fp8_append_kv(args["q"], q, 4096, kv, 4096, kv, args["heads"], *refs, 4096, 4096, args["positions"], args["half"], args["interleaved"], None, None,
                                         1e-6, args["out"], None)
    return append, attend


@pytest.mark.parametrize("change,message", [
    (dict(keys=None), b"null"), (dict(e4m3=1), b"null"), (dict(table=None), b"null"), (dict(offsets=None), b"null"), (dict(lengths=None), b"null"), (dict(q=None), b"null"),
    (dict(pages=-1), b"negative"), (dict(rows=-1), b"negative"), (dict(head_dim=24), b"16 to 128"), (dict(head_dim=144), b"16 to 128"), (dict(page_size=12), b"power of two"),
    (dict(width=1 << 30), b"2^30"), (dict(keys=4104), b"aligned"), (dict(key_strides=(2048, 1024, 60)), b"strides"), (dict(value_strides=(2048, -1024, 64)), b"strides"),
    (dict(q=4104), b"aligned"), (dict(strides=(252, 64)), b"multiples of 8"), (dict(out=4104), b"aligned"), (dict(out=None), b"aligned"), (dict(seqs=1 << 21), b"more"),
    (dict(rows=1 << 25), b"more")])
def test_entries_refuse(L, change, message):
    for call in entry(L, **change):
        assert call() in (1, 2) and message in L.odl_fp8_last_error(), L.odl_fp8_last_error()


@pytest.mark.parametrize("change,message", [(dict(heads=5), b"a multiple"), (dict(heads=0), b"a multiple"), (dict(scale=0.0), b"scale"), (dict(scale=float("nan")), b"scale"),
                                            (dict(window=-1), b"window"), (dict(softcap=-2.0), b"softcap"), (dict(softcap=float("nan")), b"softcap"),
                                            (dict(ws=None), b"workspace"), (dict(floats=8), b"workspace"), (dict(ws=4100), b"workspace")])
def test_attention_refuses(L, change, message):
    assert entry(L, **change)[1]() in (1, 2) and message in L.odl_fp8_last_error()


@pytest.mark.parametrize("change,message", [(dict(half=33), b"rotation"), (dict(half=10, interleaved=0), b"rotation"), (dict(half=6), b"rotation"), (dict(positions=79), b"angles"),
                                            (dict(heads=0), b"heads")])
def test_append_refuses(L, change, message):
    assert entry(L, **change)[0]() in (1, 2) and message in L.odl_fp8_last_error()


def test_verify_refuses(L):
    good = dict(logits=4096, stride=10, drafts=None, dstride=0, dtype=0, rows=4, vocab=10, tokens=4096, offsets=4096, seqs=2, u=4096, t=1.0, acc=4096, out=4096, lp=4096, ws=4096,
                floats=1 << 30)
    for change, message in ((dict(vocab=0), b"vocabulary"), (dict(vocab=(1 << 24) + 1), b"vocabulary"), (dict(rows=65536), b"65535"), (dict(seqs=65536), b"65535"),
                            (dict(dtype=2), b"dtype"), (dict(t=-1.0), b"temperature"), (dict(t=float("nan")), b"temperature"), (dict(logits=None), b"null"),
                            (dict(offsets=None), b"null"), (dict(acc=None), b"null"), (dict(stride=-1), b"stride"), (dict(floats=3), b"workspace"), (dict(rows=-1), b"negative")):
        a = {**good, **change}
        assert L.odl_fp8_verify_drafts(*a.values(), None) in (1, 2) and message in L.odl_fp8_last_error(), change
    assert L.odl_fp8_verify_drafts_workspace(4, 2, 0) == -1
    assert native.load().odl_fp8_paged_attention_workspace(4, 1, None, None) == -1
