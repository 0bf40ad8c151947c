"""What the logits of a head say about given tokens: their log probabilities, with entropy and top alternatives.

The step behind the vocabulary-sized Linear: the loss of training (the negative mean of the log probabilities), the scores
of an evaluation, the answer of a decode step.  The reference leaves it to PyTorch's cross entropy, which is a softmax of the whole
matrix in fp32.  Here the logits are read once in their own type, and the backward reads them once more and writes their gradient;
under an FP8 recipe that gradient hands its maxima to the cast of the head's backward, which then has no pass of its own over it.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import native
from .amp import state as _state
from .calls import no_graph, once_differentiable, untraced, untransformed
from .fused import gradient_is_cast

MAX_TOP = native.LOGPROBS_MAX_TOP


class TokenLogProbs(NamedTuple):
    """logprobs and entropy: fp32, one for each row of logits; top_logprobs fp32 and top_ids int64 [..., top_k], None for top_k = 0."""

    logprobs: torch.Tensor
    entropy: torch.Tensor
    top_logprobs: torch.Tensor | None
    top_ids: torch.Tensor | None


class _TokenLogProbsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: torch.Tensor, targets: torch.Tensor, n_vocab: int, top_k: int, temperature: float, ignore_index: int, recipe):
        rows = logits.reshape(-1, logits.shape[-1])
        targets = targets.reshape(-1)
        logprobs, entropy, stats, top, ids = native.token_logprobs(rows, targets, n_vocab, top_k, temperature, ignore_index,
                                                                   keep_stats=ctx.needs_input_grad[0])
        ctx.save_for_backward(logits, targets, entropy, stats, ids)
        ctx.set_materialize_grads(False)
        ctx.asked, ctx.recipe = (n_vocab, top_k, temperature, ignore_index), recipe if gradient_is_cast(logits, recipe) else None
        lead = logits.shape[:-1]
        if top is None:
            return logprobs.reshape(lead), entropy.reshape(lead), None, None
        ids_out = ids.reshape(*lead, top_k)
        ctx.mark_non_differentiable(ids_out)
        return logprobs.reshape(lead), entropy.reshape(lead), top.reshape(*lead, top_k), ids_out

    @staticmethod
    @once_differentiable
    def backward(ctx, d_logprobs, d_entropy, d_top, _):
        if d_logprobs is None and d_entropy is None and d_top is None:
            return (None,) * 7
        logits, targets, entropy, stats, ids = ctx.saved_tensors
        dlogits, parts = native.token_logprobs_bwd(logits.reshape(-1, logits.shape[-1]), targets, *ctx.asked, ids, stats, entropy, d_logprobs,
                                                   d_entropy, d_top)
        dlogits = dlogits.reshape(logits.shape)
        if ctx.recipe is not None:
            ctx.recipe.offer_parts(dlogits, parts)
        return dlogits, None, None, None, None, None, None


def _plain(logits, targets, n_vocab, top_k, temperature, ignore_index) -> TokenLogProbs:
    x = logits[..., :n_vocab].to(torch.promote_types(logits.dtype, torch.float32))
    kept, known = targets != ignore_index, (targets >= 0) & (targets < n_vocab)
    empty = (x == float("-inf")).all(-1)
    dead = ~kept | empty
    d = torch.where(dead.unsqueeze(-1), torch.zeros_like(x), x)
    logp = torch.log_softmax((d - d.detach().amax(-1, keepdim=True)) / temperature, dim=-1)      # (the quotient of the logits may be out of range)
    lp = logp.gather(-1, torch.where(known, targets, torch.zeros_like(targets)).unsqueeze(-1)).squeeze(-1)
    p = logp.exp()
    entropy = -(p * torch.where(p == 0, torch.zeros_like(p), logp)).sum(-1)
    zero, nowhere, nan = torch.zeros_like(lp.detach()), torch.full_like(lp, float("-inf")), torch.full_like(lp, float("nan"))
    lp = torch.where(empty, nowhere, lp) * torch.where(known | ~kept, zero + 1, nan)      # (a factor: gradients pass it by row)
    lp = torch.where(kept, lp, zero)
    entropy = torch.where(dead, zero, entropy)
    if not top_k:
        return TokenLogProbs(lp, entropy, None, None)
    ids = x.sort(dim=-1, descending=True, stable=True).indices[..., :top_k]
    top = torch.where(empty.unsqueeze(-1), nowhere.unsqueeze(-1), logp.gather(-1, ids))
    sound = ~(x.isnan() | (x == float("inf"))).any(-1)
    ids = torch.where((kept & sound).unsqueeze(-1), ids, torch.full_like(ids, -1))
    top = top * torch.where(sound | ~kept, zero + 1, nan).unsqueeze(-1)
    return TokenLogProbs(lp, entropy, torch.where(kept.unsqueeze(-1), top, torch.zeros_like(top)), ids)


@untraced
def token_logprobs(logits: torch.Tensor, targets: torch.Tensor, *, n_vocab: int | None = None, top_k: int = 0, temperature: float = 1.0,
                   ignore_index: int = -100) -> TokenLogProbs:
    """Log probabilities of ``targets`` (int64, the shape of ``logits`` without its last axis) under ``softmax(logits / temperature)``, the
    entropy of each row in nats, and the log probabilities and ids of its ``top_k`` largest logits (at most 64; ties go to the lowest id).

    n_vocab: columns in use, where the head has more than the vocabulary; the others are not read and get a gradient of zero.
    Rows whose target is ``ignore_index`` are not read: 0, 0, top_logprobs 0 with ids -1, gradient 0.  Another target that is no token
    answers NaN (and a gradient of NaN).  A row of -inf only answers -inf, entropy 0, gradient 0; one with NaN or +inf NaN, ids -1.

    Differentiable in the logits through logprobs, entropy and top_logprobs, once.  bf16 and fp32 logits on the GPU run in one kernel each
    way (rows may lie at any distance and alignment); everything is accumulated in fp32.  CPU tensors run as torch operations."""
    if logits.dim() == 0 or not logits.is_floating_point():
        raise ValueError(f"token_logprobs: logits are {logits.dtype} {tuple(logits.shape)}")
    if targets.dtype != torch.int64 or targets.shape != logits.shape[:-1] or targets.device != logits.device:
        raise ValueError(f"token_logprobs: targets are {targets.dtype} {tuple(targets.shape)} on {targets.device}, expected int64 {tuple(logits.shape[:-1])} "
                         f"on {logits.device}")
    columns = logits.shape[-1]
    n_vocab = columns if n_vocab is None else n_vocab
    if not 1 <= n_vocab <= columns:
        raise ValueError(f"token_logprobs: n_vocab {n_vocab} of {columns} columns")
    if not 0 <= top_k <= min(MAX_TOP, n_vocab):
        raise ValueError(f"token_logprobs: top_k {top_k} (0 to {MAX_TOP}, and to the vocabulary)")
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"token_logprobs: temperature {temperature} (1e-30 to 1e30)")
    if not logits.is_cuda:
        return _plain(logits, targets, n_vocab, top_k, float(temperature), ignore_index)
    if no_graph():
        if logits.dim() == 2:
            logprobs, entropy, _, top, ids = native.token_logprobs(logits, targets, n_vocab, top_k, temperature, ignore_index)
            return TokenLogProbs(logprobs, entropy, top, ids)
        lead = logits.shape[:-1]
        logprobs, entropy, _, top, ids = native.token_logprobs(logits.reshape(-1, columns), targets.reshape(-1), n_vocab, top_k, temperature, ignore_index)
        return TokenLogProbs(logprobs.view(lead), entropy.view(lead), *((None, None) if top is None else (t.view(*lead, top_k) for t in (top, ids))))
    recipe = _state.active_recipe()
    if untransformed() and not gradient_is_cast(logits, recipe):             # nobody to hand maxima to
        r = native.token_logprobs_node(logits, targets, n_vocab, top_k, temperature, ignore_index)
        if r is not None:
            return TokenLogProbs(*r)
    return TokenLogProbs(*_TokenLogProbsFn.apply(logits, targets, n_vocab, top_k, float(temperature), ignore_index, recipe))
