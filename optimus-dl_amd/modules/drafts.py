"""Verification of tokens that something cheaper than the model drafted (a smaller model, a look-up in the prompt).

The model runs once over the drafts of a sequence and says how many of them it would have drawn itself, and what it draws behind them: several tokens for
one pass over its weights.  The step behind the head, as :mod:`.logprobs` is for training and scores.  The reference has no counterpart.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import native
from .calls import untraced, untransformed
from .paged import refuse_transforms


class VerifiedDrafts(NamedTuple):
    """accepted: int32, drafts of each sequence that hold; tokens: int64, the token behind each row, -1 behind the row that stopped; logprobs: fp32,
    the model's log probability of it, 0 where there is none."""

    accepted: torch.Tensor
    tokens: torch.Tensor
    logprobs: torch.Tensor


def _distribution(x):
    """Probabilities of a row in 64 bits; None where it has none."""
    if x.isnan().any() or (x == float("inf")).any() or (x == float("-inf")).all():
        return None
    e = (x - x.max()).exp()
    return e / e.sum()


def _plain(logits, tokens, offsets, uniforms, draft_logits, temperature, n_vocab) -> VerifiedDrafts:
    rows = logits.shape[0]
    accepted = torch.zeros(offsets.numel() - 1, dtype=torch.int32)
    out, logprobs = torch.full((rows,), -1, dtype=torch.int64), torch.zeros(rows, dtype=torch.float32)
    at = offsets.tolist()
    for s in range(len(at) - 1):
        first, end = min(max(at[s], 0), rows), min(at[s + 1], rows)
        for r in range(first, end):
            x = logits[r, :n_vocab].double()
            p = _distribution((x - x.max()) / (temperature or 1.0)) if not x.isnan().any() else None
            if p is None:
                logprobs[r] = float("nan")
                break
            d = int(tokens[r + 1]) if r + 1 < end else -1
            known, q = 0 <= d < n_vocab, None
            if temperature and draft_logits is not None and r + 1 < end:
                y = draft_logits[r, :n_vocab].double()
                q = _distribution((y - y.max()) / temperature) if not y.isnan().any() else None
                of_q = float("nan") if q is None else float(q[d]) if known else 1.0
            else:
                of_q = 1.0
            yes = known and (d == int((x == x.max()).nonzero()[0]) if not temperature else float(uniforms[r]) * of_q < float(p[d]))
            if not yes:
                if not temperature:
                    d = int((x == x.max()).nonzero()[0])
                else:
                    w = p.clone()
                    if q is not None:
                        w = (p - q).clamp(min=0.0)
                    elif known and draft_logits is None:
                        w[d] = 0.0
                    w = w if w.sum() > 0 else p
                    upto = w.cumsum(0)
                    over = ((upto > float(uniforms[end - 1]) * upto[-1]) & (w > 0)).nonzero()
                    d = int(over[0]) if over.numel() else int((w > 0).nonzero()[-1])
            out[r], logprobs[r] = d, float(p[d].log())
            if not yes:
                break
            accepted[s] += 1
    return VerifiedDrafts(accepted, out, logprobs)


@untraced
def verify_drafts(logits: torch.Tensor, tokens: torch.Tensor, offsets: torch.Tensor, uniforms: torch.Tensor, *, draft_logits: torch.Tensor | None = None,
                  temperature: float = 1.0, n_vocab: int | None = None) -> VerifiedDrafts:
    """How many drafted tokens the model accepts, the token behind them, and the log probabilities of all of these.

    Sequence s fed rows ``offsets[s]`` to ``offsets[s + 1]`` (int32) of ``tokens`` (int64) to the model: the last token that is sure, and its drafts.
    ``logits`` [rows, columns] are the model's answer: row r speaks of the token behind ``tokens[r]``.  ``draft_logits`` are the drafter's of the same
    places (a sequence's last row of them is not read), None where drafts were not drawn from a distribution.  ``uniforms``: fp32 numbers from [0, 1),
    one a row, drawn apart from everything else: a row's decides on the draft behind it, the last row's draws the token.

    With p and q the softmax of both over ``temperature``, a draft d holds while ``u * q(d) < p(d)``; behind the first that does not the token is drawn
    from ``max(p - q, 0)``, behind the last draft from p: the lowest token at which the running sum exceeds ``u`` times the whole.  What is emitted is
    then distributed as the model's own tokens would be.  temperature 0: the largest logit (the lowest of them), and drafts that are that.

    n_vocab: columns in use.  A draft that is no token does not hold.  A row with NaN or +inf, or of -inf only, stops its sequence: token -1, logprob
    NaN.  Rows behind the last sequence answer -1 and 0.

    bf16 and fp32 logits on the GPU (rows at any distance and alignment): three launches, sums in 64 bits, so that how a row is cut, by the
    number of rows, settles one draw in some 10^13 otherwise."""
    if logits.is_cuda and untransformed():
        r = native.plain_verify_drafts(logits, tokens, offsets, uniforms, draft_logits, temperature, n_vocab)
        if r is not None:
            return VerifiedDrafts(*r)
    if logits.dim() != 2 or not logits.is_floating_point():
        raise ValueError(f"verify_drafts: logits are {logits.dtype} {tuple(logits.shape)}, expected [rows, columns]")
    rows, columns = logits.shape
    n_vocab = columns if n_vocab is None else n_vocab
    if not 1 <= n_vocab <= columns:
        raise ValueError(f"verify_drafts: n_vocab {n_vocab} of {columns} columns")
    if tokens.dtype != torch.int64 or tokens.shape != (rows,) or uniforms.dtype != torch.float32 or uniforms.shape != (rows,):
        raise ValueError(f"verify_drafts: tokens {tokens.dtype} {tuple(tokens.shape)} and uniforms {uniforms.dtype} {tuple(uniforms.shape)}, expected int64 and fp32 [{rows}]")
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.numel() < 1:
        raise ValueError(f"verify_drafts: offsets {offsets.dtype} {tuple(offsets.shape)}, expected int32 [sequences + 1]")
    if draft_logits is not None and (draft_logits.dim() != 2 or draft_logits.dtype != logits.dtype or draft_logits.shape[0] != rows or draft_logits.shape[1] < n_vocab):
        raise ValueError(f"verify_drafts: draft_logits {draft_logits.dtype} {tuple(draft_logits.shape)} beside logits {logits.dtype} {tuple(logits.shape)}")
    if not (temperature == 0 or 1e-30 <= temperature <= 1e30):
        raise ValueError(f"verify_drafts: temperature {temperature} (0, or 1e-30 to 1e30)")
    if torch.is_grad_enabled() and (logits.requires_grad or (draft_logits is not None and draft_logits.requires_grad)):
        raise ValueError("verify_drafts is for inference; logits want a gradient (torch.no_grad() around the call, or detach them)")
    if not logits.is_cuda:
        return _plain(logits, tokens, offsets, uniforms, draft_logits, float(temperature), n_vocab)
    refuse_transforms("verify_drafts")
    return VerifiedDrafts(*native.verify_drafts(logits, tokens, offsets, uniforms, draft_logits, float(temperature), n_vocab))
