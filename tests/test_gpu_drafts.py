"""Verification of drafts on the GPU against the CPU's form in 64 bits, row by row: whole numbers are equal."""
import math

import pytest
import torch

from optimus_dl_amd.modules.drafts import verify_drafts

pytestmark = pytest.mark.gpu
CUDA = torch.device("cuda")
INF = math.inf


def drafted(rows, vocab, dtype, seed=0, padded=None, agree=0.7, pad=0):
    """Sequences of `rows` rows, logits of a model and of a drafter that mostly agrees with it, drafts drawn from the drafter."""
    g = torch.Generator().manual_seed(seed)
    total = sum(rows) + pad
    x = torch.randn((total, padded or vocab), generator=g) * 2.0
    x[torch.arange(total), torch.randint(0, vocab, (total,), generator=g)] += 6.0
    y = x + (1 - agree) * torch.randn(x.shape, generator=g)
    race = torch.empty((total, vocab)).exponential_(generator=g).log()
    draw = (y[:, :vocab] - race).argmax(1)
    tokens = torch.cat((draw[:1], draw[:-1]))
    offsets = torch.tensor([sum(rows[:i]) for i in range(len(rows) + 1)], dtype=torch.int32)
    return x.to(dtype), tokens, offsets, torch.rand(total, generator=g), y.to(dtype)


def both(x, tokens, offsets, u, y=None, **kwargs):
    want = verify_drafts(x, tokens, offsets, u, draft_logits=y, **kwargs)
    got = verify_drafts(x.cuda(), tokens.cuda(), offsets.cuda(), u.cuda(), draft_logits=None if y is None else y.cuda(), **kwargs)
    assert torch.equal(got.accepted.cpu(), want.accepted)
    assert torch.equal(got.tokens.cpu(), want.tokens)
    # a logarithm and a difference in 64 bits, rounded once: half a step of fp32 on both sides
    assert torch.allclose(got.logprobs.cpu(), want.logprobs, rtol=2.0 ** -22, atol=2.0 ** -40, equal_nan=True)
    return want


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("temperature", [1.0, 0.6, 0.0])
@pytest.mark.parametrize("vocab,padded", [(1, 1), (7, 9), (2048, 2048), (8193, 8200), (50257, 50304)])
def test_against_64_bits(dtype, drafter, temperature, vocab, padded):
    x, tokens, offsets, u, y = drafted([1, 4, 0, 9, 2, 3], vocab, dtype, padded=padded, seed=vocab, pad=2)
    both(x, tokens, offsets, u, y if drafter else None, temperature=temperature, n_vocab=vocab)


def test_many_sequences_are_accepted_in_all_lengths():
    x, tokens, offsets, u, y = drafted([6] * 60, 3000, torch.float32, seed=3, agree=0.9)
    want = both(x, tokens, offsets, u, y)
    assert len(set(want.accepted.tolist())) >= 5
    both(x, tokens, offsets, u, x)                         # the drafter is the model: every draft holds
    assert (verify_drafts(x, tokens, offsets, u, draft_logits=x).accepted == 5).all()


def test_rows_that_have_no_distribution():
    """NaN, +inf and -inf only: the sequence stops there.  In the drafter's row: the token is drawn from the model's."""
    for dtype in (torch.bfloat16, torch.float32):
        x, tokens, offsets, u, y = drafted([3, 3, 3, 3, 3, 3], 500, dtype, seed=5, agree=1.0)
        x[0, 77], x[4, 3], x[6] = math.nan, INF, -INF
        y[9, 5], y[13] = math.nan, -INF
        x[15, 100:] = -INF                           # masked logits weigh nothing
        x[16] = torch.finfo(dtype).min               # and a row of the lowest values is a row like others
        for kwargs in ({}, {"temperature": 0.0}, {"temperature": 1e-30}, {"temperature": 1e30}):
            want = both(x, tokens, offsets, u, y, **kwargs)
            assert want.tokens[0] == -1 and want.logprobs[0].isnan()
        both(x, tokens, offsets, u)


def test_numbers_at_the_ends():
    x, tokens, offsets, u, y = drafted([4] * 8, 300, torch.float32, seed=6)
    for value in (0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan):
        both(x, tokens, offsets, torch.full_like(u, value), y)
        both(x, tokens, offsets, torch.full_like(u, value))


def test_drafts_that_are_no_tokens():
    x, tokens, offsets, u, y = drafted([3, 3, 3], 300, torch.float32, seed=7)
    tokens[1], tokens[4], tokens[7] = -1, 300, 2 ** 40
    both(x, tokens, offsets, u, y, n_vocab=290)
    both(x, tokens, offsets, u, n_vocab=290)
    both(x, tokens, offsets, u, temperature=0.0, n_vocab=290)


def test_equal_distributions_refuse_only_what_is_impossible():
    """p and q the same but for the drafted token, which p does not have: what is left is p."""
    x, tokens, offsets, u, y = drafted([2] * 6, 100, torch.float32, seed=8)
    y = x.clone()
    for s in range(6):
        d = int(tokens[2 * s + 1])
        x[2 * s, d] = -INF
    want = both(x, tokens, offsets, u, y)
    assert (want.accepted == 0).all()
    flat = torch.zeros_like(x)                       # all tokens alike, in both: a draft holds, whatever the number
    assert (both(flat, tokens, offsets, u, flat).accepted == 1).all()


def test_ties_go_to_the_lowest_token():
    x, tokens, offsets, u, _ = drafted([2, 2], 9000, torch.bfloat16, seed=9)
    x[:, 8500] = x[:, 40] = 50.0
    tokens[1], tokens[3] = 8500, 40
    want = both(x, tokens, offsets, u, temperature=0.0)
    assert want.tokens.tolist() == [40, -1, 40, 40] and want.accepted.tolist() == [0, 1]


@pytest.mark.parametrize("vocab", [1 << 20, (1 << 21) + 5])
def test_wide_rows(vocab):
    x, tokens, offsets, u, y = drafted([2, 3], vocab, torch.bfloat16, seed=10)
    both(x, tokens, offsets, u, y)


def test_unaligned_rows_of_views():
    x, tokens, offsets, u, y = drafted([3, 1, 4], 1001, torch.bfloat16, seed=11)
    wide = torch.zeros((8, 2 * 1003 + 1), dtype=torch.bfloat16, device=CUDA)[:, 1:]
    a, b = wide[:, :1001], wide[:, 1003:1003 + 1001]
    a.copy_(x)
    b.copy_(y)
    want = verify_drafts(x, tokens, offsets, u, draft_logits=y)
    got = verify_drafts(a, tokens.cuda(), offsets.cuda(), u.cuda(), draft_logits=b)
    assert torch.equal(got.tokens.cpu(), want.tokens) and torch.equal(got.accepted.cpu(), want.accepted)
    got = verify_drafts(x.cuda().t().contiguous().t(), tokens.cuda(), offsets.cuda(), u.cuda(), draft_logits=y.cuda())         # columns apart: copied
    assert torch.equal(got.tokens.cpu(), want.tokens)


def test_nothing_to_verify():
    x, tokens, offsets, u, y = drafted([0, 0], 50, torch.float32, pad=3)
    want = both(x, tokens, offsets, u, y)
    assert (want.tokens == -1).all() and (want.logprobs == 0).all() and (want.accepted == 0).all()
    r = verify_drafts(x[:0].cuda(), tokens[:0].cuda(), offsets.cuda(), u[:0].cuda())
    assert r.accepted.tolist() == [0, 0] and r.tokens.numel() == 0


def test_captured_and_on_two_streams():
    x, tokens, offsets, u, y = (t.cuda() for t in drafted([5] * 12, 40000, torch.bfloat16, seed=12))
    want = verify_drafts(x, tokens, offsets, u, draft_logits=y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        others = [verify_drafts(x, tokens, offsets, 1 - u, draft_logits=y) for _ in range(3)]
    again = [verify_drafts(x, tokens, offsets, u, draft_logits=y) for _ in range(3)]
    torch.cuda.synchronize()
    for r in again:
        assert all(torch.equal(a, b) for a, b in zip(r, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = verify_drafts(x, tokens, offsets, u, draft_logits=y)
    first = u.clone()
    for numbers, expected in ((1 - first, others[0]), (first, want), (1 - first, others[0])):
        u.copy_(numbers)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, expected))


def test_what_is_emitted_is_distributed_as_the_model():
    """4096 sequences of one draft over 6 tokens.  A frequency's standard deviation is at most sqrt(.25 / 4096) = 0.0079; six of them."""
    n, vocab = 4096, 6
    g = torch.Generator().manual_seed(13)
    p_logits, q_logits = torch.randn(vocab, generator=g), torch.randn(vocab, generator=g)
    x, y = p_logits.repeat(2 * n, 1).cuda(), q_logits.repeat(2 * n, 1).cuda()
    drafts = torch.multinomial(torch.softmax(q_logits, 0), n, True, generator=g)
    tokens = torch.zeros(2 * n, dtype=torch.int64)
    tokens[1::2] = drafts
    r = verify_drafts(x, tokens.cuda(), torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=CUDA), torch.rand(2 * n, generator=g).cuda(), draft_logits=y)
    share = torch.bincount(r.tokens[0::2].cpu(), minlength=vocab).double() / n
    assert (share - torch.softmax(p_logits.double(), 0)).abs().max() < 6 * 0.0079
