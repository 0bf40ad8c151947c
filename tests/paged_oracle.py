"""Attention over a paged cache from its definition in 64 bits, for some rows of a batch: long contexts, wide ranges of scores, odd values."""
import math

import torch


def attention_rows(c, rows, scale, window=0, softcap=0.0):
    """(answers, how far bf16 weights, fp32 scores and a bf16 answer may be from them) of the given rows of a `paged_helpers.Case` on the CPU, both [len(rows), heads, dim].

    A score is off by 2^-24 of its own size a rounding (16 of them) and by 2^-24 of what is added up a term of its product; a cap of up to 256 puts 5 * 2^-24 of itself on it (the
    rounding of a reciprocal near 1/2, of an exponential and of two sums near 1), and larger ones no more than 16 roundings of the score.  Weights are then off by as much, relative to themselves, and by half
    a step of bf16; sums by 2^-23 a key; the answer by half a step.  Seen values that are not finite come through as they are, whatever their weight."""
    half, group = 2.0 ** -8, c.heads // c.kv
    out, far = (torch.zeros((len(rows), c.heads, c.dim), dtype=torch.float64) for _ in range(2))
    offsets = c.offsets.tolist()
    for i, r in enumerate(rows):
        s = next((s for s in range(len(offsets) - 1) if offsets[s] <= r < offsets[s + 1]), None)
        if s is None:
            continue
        position = c.length[s] - c.new[s] + r - offsets[s]
        at = torch.arange(max(0, position - window + 1) if window else 0, max(0, min(position + 1, c.width * c.page)))
        page = c.pages[s].long()[at // c.page]
        held = (page >= 0) & (page < c.keys.shape[0])
        at, page = at[held], page[held]
        if not at.numel():
            continue
        keys, values = (t[page, :, at % c.page].double() for t in (c.keys, c.values))        # [keys, kv heads, dim]
        if c.key_scale is not None:
            keys, values = keys * c.key_scale.double().view(1, -1, 1), values * c.value_scale.double().view(1, -1, 1)
        for h in range(c.heads):
            q, k, v = c.q[r, h].double(), keys[:, h // group], values[:, h // group]
            x = (k @ q) * scale
            noise = (c.dim + 8) * 2.0 ** -24 * (k.abs() @ q.abs()) * scale
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            top = x[x != -math.inf].amax() if (x != -math.inf).any() else None
            if top is None:                      # no score above -inf
                continue
            noise = noise + 16 * 2.0 ** -24 * x.abs() + (5 * 2.0 ** -24 * softcap if softcap <= 256 else 0.0)
            w = torch.exp(x - top)
            near = x > top - 30                  # (what is further away weighs less than 2^-43 of the row, and no key's noise outweighs that)
            odd = ~v.isfinite()
            fine = torch.where(odd, 0.0, v)
            y, size = (w @ fine) / w.sum(), (w @ fine.abs()) / w.sum()
            y = y + torch.where(odd, v, 0.0).sum(0)
            loose = half + 2.0 * (noise[near].max() if near.any() else 0.0) + at.numel() * 2.0 ** -23
            out[i, h] = y
            far[i, h] = 1.01 * (loose * (size + y.abs()) + half * y.abs()) + 1e-30
    return out, far
