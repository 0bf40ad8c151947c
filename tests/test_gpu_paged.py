"""A paged cache on the GPU: what goes into it, bit by bit, and attention over it against its definition in 64 bits."""
import math

import pytest
import torch

from optimus_dl_amd import native
from optimus_dl_amd.modules.paged import append_kv, paged_attention
from tests.paged_helpers import BF16, E4M3, Case, angles, append32, assert_near, attention64, bits

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")


def attend(c, scale=None, window=0, softcap=0.0, max_new=None):
    scale = c.dim ** -0.5 if scale is None else scale
    want, far = attention64(c, scale, window, softcap)
    c.to(CUDA)
    got = paged_attention(c.q, c.keys, c.values, *c.batch(), scale=scale, window=window, softcap=softcap, max_new=max_new, **c.scales())
    assert got.dtype == BF16 and got.is_contiguous()
    assert_near(got, want, far)
    return got


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("dim,half,norm", [(128, 64, False), (128, 64, True), (64, 16, False), (96, 48, True), (16, 8, False), (80, 40, False), (48, 0, True), (112, 0, False)])
def test_append_bits(interleaved, cache, dim, half, norm):
    c = Case([1, 3, 0, 17, 1], [1, 40, 9, 17, 33], 6, 2, dim, 16, cache, pad=2, seed=dim)
    cos, sin = angles(c.width * c.page, half) if half else (None, None)
    weights = [1 + 0.2 * torch.randn(dim) for _ in range(2)] if norm else [None, None]
    want = append32(c, cos, sin, interleaved, *weights)
    c.to(CUDA)
    on = [None if t is None else t.to(CUDA) for t in (cos, sin, *weights)]
    q = append_kv(c.q, c.k, c.v, c.keys, c.values, *c.batch(), cos=on[0], sin=on[1], interleaved=interleaved, q_weight=on[2], k_weight=on[3], **c.scales())
    for got, w, name in zip((q, c.keys, c.values), want, ("q", "keys", "values")):
        assert torch.equal(bits(got.cpu()), bits(w)), name


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("dim,heads,kv", [(128, 8, 2), (64, 12, 12), (96, 3, 1), (16, 8, 1)])
def test_attention_of_single_tokens(cache, dim, heads, kv):
    attend(Case([1] * 5, [1, 31, 32, 129, 700], heads, kv, dim, 16, cache, seed=1), max_new=1)


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("dim,heads,kv,page", [(128, 8, 2, 16), (64, 3, 3, 64), (112, 4, 1, 4)])
def test_attention_of_prompts_and_chunks(cache, dim, heads, kv, page):
    attend(Case([100, 1, 33, 0, 70], [100, 200, 65, 12, 300], heads, kv, dim, page, cache, pad=5, seed=2))


@pytest.mark.parametrize("window,softcap", [(1, 0.0), (5, 0.0), (64, 0.0), (1000, 0.0), (0, 5.0), (40, 30.0)])
@pytest.mark.parametrize("new,lengths", [([1, 1, 1], [1, 64, 513]), ([130, 3, 64], [130, 300, 64])])
def test_window_and_softcap(window, softcap, new, lengths):
    attend(Case(new, lengths, 6, 2, 64, 16, seed=3), window=window, softcap=softcap)


@pytest.mark.parametrize("page", [1, 2, 4, 8, 32, 256])
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_page_sizes(page, cache):
    attend(Case([1, 90, 2], [45, 200, 2], 4, 2, 128, page, cache, seed=4))


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 16, 31, 32, 33])
def test_heads_of_a_group(group):
    attend(Case([1, 2, 40], [70, 5, 77], 2 * group, 2, 64, 8, seed=5))
    attend(Case([1, 1], [300, 17], group, 1, 128, 16, seed=6))


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_head_dims(dim, cache):
    attend(Case([1, 150], [260, 170], 4, 2, dim, 16, cache, seed=7))


def test_many_sequences():
    """More than the 64 that are looked at at a time, single tokens and chunks, empty sequences among them."""
    g = torch.Generator().manual_seed(8)
    new = [int(n) for n in torch.randint(0, 3, (150,), generator=g)] + [50, 0, 70] + [1] * 50
    lengths = [n + int(k) for n, k in zip(new, torch.randint(0, 90, (len(new),), generator=g))]
    attend(Case(new, lengths, 4, 2, 64, 16, pad=9, seed=8))
    attend(Case([1] * 130, [1 + 3 * i for i in range(130)], 2, 1, 64, 16, seed=9), max_new=1)


def test_one_long_sequence_beside_short_ones():
    attend(Case([1, 1, 1, 1], [3000, 2, 40, 129], 4, 1, 128, 16, seed=10), max_new=1)
    attend(Case([30, 1, 200], [2500, 2, 200], 4, 1, 128, 16, seed=11))


@pytest.mark.parametrize("most", [0, 1, 2, 7, 40, 1000])
def test_results_do_not_hang_on_the_hint(most):
    attend(Case([40, 1, 3], [500, 90, 3], 8, 2, 64, 16, seed=12), max_new=most)


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("new,lengths", [([1, 1], [100, 70]), ([60, 2], [140, 70])])
def test_pages_that_are_none(cache, new, lengths):
    """Numbers outside of the cache: what lies there is not seen, and a token that sees nothing answers 0."""
    c = Case(new, lengths, 4, 2, 128, 16, cache, seed=13)
    c.pages[0, 1], c.pages[0, 3], c.pages[0, 4] = -1, c.keys.shape[0], 2 ** 31 - 1
    c.pages[1] = -2 ** 31
    got = attend(c)
    assert (got[int(c.offsets[1]):] == 0).all()
    attend(Case(new, lengths, 4, 2, 128, 2, cache, seed=14, width=20))               # lengths beyond the table's reach


def test_lengths_that_hold_less_than_is_new():
    """Rows in front of position 0 see nothing; nothing is read in front of the table."""
    for length in (0, 3, -5, -2 ** 31):
        c = Case([5, 1], [64, 20], 4, 2, 64, 16, seed=15)
        c.length[0] = length
        c.lengths[0] = length
        if length < -2 ** 20:
            c.to(CUDA)
            got = paged_attention(c.q, c.keys, c.values, *c.batch())
            assert got[:5].isfinite().all()
        else:
            got = attend(c)
            assert (got[:5 - max(length, 0)] == 0).all()


@pytest.mark.parametrize("new,lengths", [([1, 4], [50, 70]), ([70, 1], [90, 33]), ([300], [300])])
@pytest.mark.parametrize("odd", ["nan", "inf", "-inf", "mixed"])
def test_what_a_row_does_not_see_does_not_reach_it(new, lengths, odd):
    """NaN and infinities behind the end of sequences, in unused pages and in tokens that only later rows of the same tile see."""
    c = Case(new, lengths, 4, 2, 64, 16, seed=16)
    used = torch.zeros(c.keys.shape[:1] + c.keys.shape[2:3], dtype=torch.bool)
    for s, n in enumerate(lengths):
        for p in range(n):
            used[int(c.pages[s, p // 16]), p % 16] = True
    bad = {"nan": math.nan, "inf": math.inf, "-inf": -math.inf, "mixed": math.nan}[odd]
    for t in (c.keys, c.values):
        t.masked_fill_(~used[:, None, :, None], bad)
    for s, n in enumerate(lengths):
        if new[s] > 2:                             # the value of the second last token, which two rows see; of another one in one head only
            page, slot = int(c.pages[s, (n - 2) // 16]), (n - 2) % 16
            c.values[page, :, slot, ::3] = bad
            if odd == "mixed":
                c.values[page, 0, slot, 1] = math.inf
                c.values[page, 1, slot, 2] = -math.inf
    attend(c)


def test_nan_in_one_query_stays_there():
    c = Case([1, 40], [80, 60], 4, 2, 64, 16, seed=17)
    c.q[0, 1, 3] = math.nan
    c.q[7, 2, 0] = math.nan
    got = attend(c)
    assert got.isnan().any(-1).sum() == 2


def test_scores_far_from_one_another():
    c = Case([1, 33], [500, 200], 4, 2, 64, 16, seed=18, q_scale=200.0)
    attend(c)


def test_strided_operands():
    """Queries, keys and values as parts of one projection; a cache whose tokens of all heads lie together; a table with wider rows."""
    c = Case([40, 1, 3], [100, 31, 3], 6, 2, 64, 16, seed=19)
    want, far = attention64(c, 0.125)
    fused = torch.randn(c.rows, 1 + 6 + 2 + 2, 64).bfloat16()
    fused[:, 1:7], fused[:, 7:9], fused[:, 9:] = c.q, c.k, c.v
    want_append = append32(c)
    c.to(CUDA)
    fused = fused.cuda()
    q, k, v = fused[:, 1:7], fused[:, 7:9], fused[:, 9:]
    pages = torch.cat((c.pages, c.pages), dim=1)[:, :c.width]
    keys, values = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (c.keys, c.values))
    assert not keys.is_contiguous()
    got = paged_attention(q, keys, values, pages, c.offsets, c.lengths, scale=0.125)
    assert_near(got, want, far)
    odd = torch.empty(c.rows * 6 * 64 + 1, dtype=BF16, device=CUDA)[1:].view(c.rows, 6, 64).copy_(q)      # not aligned: copied
    assert torch.equal(paged_attention(odd, keys, values, pages, c.offsets, c.lengths, scale=0.125), got)
    out = append_kv(q, k, v, keys, values, pages, c.offsets, c.lengths)
    for x, w in zip((out, keys, values), want_append):
        assert torch.equal(bits(x.cpu().contiguous()), bits(w))


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_append_edges(cache):
    """Pages that are none, positions outside of the table, tokens of nobody, codes out of range: nothing else changes."""
    c = Case([3, 5, 0, 20, 2], [3, 12, 4, 30, 2], 4, 2, 32, 4, cache, pad=4, seed=20)
    c.pages[1, 2], c.pages[3, 3] = -1, c.keys.shape[0]
    c.length[0] = 1                                # two of three tokens lie in front of position 0
    c.lengths[0] = 1
    c.length[4] = c.width * 4 + 1                  # the second lies behind the table's reach
    c.lengths[4] = c.length[4]
    c.k[3, 0, :4] = torch.tensor([1e4, -1e4, math.inf, math.nan])
    cos, sin = angles(c.width * 4, 16)
    want = append32(c, cos, sin)
    c.to(CUDA)
    q = append_kv(c.q, c.k, c.v, c.keys, c.values, *c.batch(), cos=cos.cuda(), sin=sin.cuda(), **c.scales())
    assert torch.equal(bits(q.cpu()), bits(want[0]))
    for got, w in zip((c.keys, c.values), want[1:]):
        same = (bits(got.cpu()) == bits(w)) | (got.cpu().float().isnan() & w.float().isnan())
        assert same.all()


def test_cache_of_more_than_4_gb():
    """Pages whose offsets pass 2^32 bytes."""
    shape = (34000, 8, 64, 128)                    # 2.2e9 elements
    keys, values = (torch.zeros(shape, dtype=BF16, device=CUDA) for _ in range(2))
    small = Case([1, 80], [90, 100], 16, 8, 128, 64, seed=21)
    want, far = attention64(small, 0.1)
    ids = torch.tensor([33999, 16390, 32768, 33001, 16384, 8191, 1])[:small.keys.shape[0]]
    keys[ids.cuda()], values[ids.cuda()] = small.keys.cuda(), small.values.cuda()
    pages = ids[small.pages.long().clamp(min=0)].int().cuda()
    small.to(CUDA)
    got = paged_attention(small.q, keys, values, pages, small.offsets, small.lengths, scale=0.1)
    assert_near(got, want, far)
    append_kv(small.q, small.k, small.v, keys, values, pages, small.offsets, small.lengths)
    last = int(pages[1, 99 // 64])
    assert torch.equal(keys[last, :, 99 % 64], small.k[80]) and torch.equal(values[last, :, 99 % 64], small.v[80])


def test_the_same_call_answers_the_same_bits():
    c = Case([1] * 20 + [100], [700 + 37 * i for i in range(20)] + [900], 8, 2, 128, 16, seed=22).to(CUDA)
    first = paged_attention(c.q, c.keys, c.values, *c.batch())
    for _ in range(5):
        assert torch.equal(paged_attention(c.q, c.keys, c.values, *c.batch()), first)


def test_on_another_stream_and_two_calls_at_once():
    c, d = Case([1] * 8, [900] * 8, 8, 2, 128, 16, seed=23).to(CUDA), Case([60, 2], [700, 900], 8, 2, 128, 16, seed=24).to(CUDA)
    want = [paged_attention(x.q, x.keys, x.values, *x.batch()) for x in (c, d)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(4):
        for i, (s, x) in enumerate(zip(streams, (c, d))):
            with torch.cuda.stream(s):
                got[i].append(paged_attention(x.q, x.keys, x.values, *x.batch()))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_captured_steps_follow_the_lengths():
    """Two graphs of a step, captured one after the other on one stream and replayed on new lengths, offsets and pages."""
    c = Case([1, 5, 2], [300, 40, 90], 8, 2, 64, 16, seed=25).to(CUDA)
    q = torch.zeros_like(c.q)
    cos, sin = (t.cuda() for t in angles(c.width * 16, 32))

    def step():
        q.copy_(append_kv(c.q, c.k, c.v, c.keys, c.values, *c.batch(), cos=cos, sin=sin))
        return paged_attention(q, c.keys, c.values, *c.batch())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(step())
    for lengths, offsets in (([301, 41, 91], [0, 1, 6, 8]), ([17, 200, 2], [0, 0, 8, 8]), ([320, 320, 320], [0, 3, 4, 7])):
        c.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        c.offsets.copy_(torch.tensor(offsets, dtype=torch.int32))
        c.pages.clamp_(min=0)
        keys, values = c.keys.clone(), c.values.clone()
        for graph, out in zip(graphs, outs):
            c.keys.copy_(keys)
            c.values.copy_(values)
            graph.replay()
            torch.cuda.synchronize()
            replayed, held = out.clone(), c.keys.clone()
            c.keys.copy_(keys)
            c.values.copy_(values)
            assert torch.equal(step(), replayed) and torch.equal(c.keys, held)


def test_nothing_to_do():
    c = Case([], [], 4, 2, 64, 16, pad=3, seed=26).to(CUDA)
    assert (paged_attention(c.q, c.keys, c.values, *c.batch()) == 0).all()
    keys = c.keys.clone()
    assert (append_kv(c.q, c.k, c.v, c.keys, c.values, *c.batch()) == 0).all() and torch.equal(c.keys, keys)
    none = c.q[:0]
    assert paged_attention(none, c.keys, c.values, *c.batch()).shape == (0, 4, 64)
    c = Case([0, 0], [5, 0], 4, 2, 64, 16, seed=27).to(CUDA)
    assert paged_attention(c.q, c.keys, c.values, *c.batch()).numel() == 0


def test_refusals_on_the_gpu():
    c = Case([1, 2], [5, 9], 4, 2, 64, 16, seed=28).to(CUDA)
    args = (c.keys, c.values, *c.batch())
    with pytest.raises(native.NativeError, match="bf16"):
        paged_attention(c.q.float(), *args)
    with pytest.raises(native.NativeError, match="bf16 or float8"):
        paged_attention(c.q, c.keys.float(), c.values.float(), *c.batch())
    with pytest.raises(native.NativeError, match="one GPU"):
        paged_attention(c.q, c.keys, c.values, c.pages.cpu(), c.offsets, c.lengths)
    with pytest.raises(native.NativeError, match="dense"):
        paged_attention(c.q, c.keys.transpose(2, 3).contiguous().transpose(2, 3), c.values, *c.batch())
    with pytest.raises(native.NativeError, match="16 to 128"):
        paged_attention(c.q[..., :24], c.keys[..., :24], c.values[..., :24], *c.batch())
    with pytest.raises(native.NativeError, match="pairs"):
        append_kv(c.q, c.k, c.v, *args, cos=torch.ones(64, 4, device=CUDA), sin=torch.ones(64, 4, device=CUDA), interleaved=False)
    with pytest.raises(ValueError, match="gradient"):
        paged_attention(c.q.clone().requires_grad_(True), *args)
    with pytest.raises(native.NativeError, match="does not see into"):
        import torch.autograd.forward_ad as fwd

        with fwd.dual_level():
            paged_attention(fwd.make_dual(c.q, torch.ones_like(c.q)), *args)


@pytest.mark.parametrize("rows", [2, 40])
def test_a_row_of_scores_of_minus_infinity_answers_0(rows):
    q = torch.ones(rows, 1, 16, dtype=BF16, device="cuda")
    keys = torch.zeros(1, 1, 64, 16, dtype=BF16, device="cuda")
    keys[0, 0, 0, 3] = -torch.inf
    args = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([[0]], [0, rows], [rows]))
    y = paged_attention(q, keys, torch.ones_like(keys), *args)
    assert (y[0] == 0).all() and (y[1:] == 1).all()            # (the first token sees that key alone)


@pytest.mark.parametrize("length", [1, 129, 257, 511, 512])
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_wider_tables_answer_the_same(length, cache):
    """A table of 512 tokens is not cut, wider ones are: a rounding of the weights and one of the result each, of at most half a step, relative to the largest value."""
    g = torch.Generator(device="cuda").manual_seed(length)
    q = torch.randn(1, 8, 64, generator=g, device="cuda").to(BF16)
    keys, values = (torch.randn(32, 2, 16, 64, generator=g, device="cuda").to(cache) for _ in range(2))
    scales = {k: torch.ones(2, device="cuda") for k in ("key_scale", "value_scale")} if cache == E4M3 else {}
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    outs = [paged_attention(q, keys, values, ints([list(range(32)) + [-1] * more]), ints([0, 1]), ints([length]), max_new=1, **scales).double() for more in (0, 1, 40)]
    most = values.double().abs().max()
    for y in outs[1:]:
        assert (y - outs[0]).abs().max() <= 4 * (torch.finfo(BF16).eps / 2 + 2.0 ** -16) * most
