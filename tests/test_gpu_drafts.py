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
