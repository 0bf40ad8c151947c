"""A decode step of a decoder over a paged cache of keys and values, with tokens that a smaller model drafted.

``append_kv``: norm and rotation of new queries and keys, keys and values into their slots of the cache.
``paged_attention``: attention of the new tokens of every sequence over what its pages hold, the new tokens included.
``verify_drafts``: how many drafted tokens the model's logits accept, and the token behind them, from given random numbers.

Everything here is inference.  Sequences have their new tokens at ``offsets[s]`` to ``offsets[s + 1]`` and ``lengths[s]`` tokens in the cache with them.
"""

import torch

own = False

DEVICE = torch.device("cuda")
CACHE = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
LOGITS = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6
THETA = 500000.0


def listed():
    return [
        # One token of one sequence in Qwen3-0.6B, whose queries and keys are normed: latency counts.
        {"name": "append_token", "op": "append", "seqs": 1, "new": 1, "ragged": False, "context": 700, "heads": 16, "kv_heads": 8, "head_dim": 128,
         "page": 16, "cache": "bf16", "norm": True, "halves": False, "rotary": 128, "pad": 0},
        # A decode step of 256 sequences with the heads of Llama-3-8B into an 8-bit cache.
        {"name": "append_decode", "op": "append", "seqs": 256, "new": 1, "ragged": False, "context": 500, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "page": 16, "cache": "e4m3", "norm": False, "halves": True, "rotary": 128, "pad": 0},
        # A step of five prompts and three single tokens, 7254 tokens and 77 rows of padding.
        {"name": "append_prompts", "op": "append", "seqs": 8, "new": 2560, "ragged": True, "context": 2560, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "cache": "bf16", "norm": False, "halves": False, "rotary": 128, "pad": 77},
        # One token of GPT-2 124M behind 500: the smallest call.
        {"name": "attention_token", "op": "attention", "seqs": 1, "new": 1, "ragged": False, "context": 501, "heads": 12, "kv_heads": 12, "head_dim": 64,
         "page": 16, "cache": "bf16", "window": 0, "softcap": 0.0, "pad": 0},
        # A decode step of 64 sequences of up to 8192 tokens, heads of Llama-3-8B: the cache is read once.
        {"name": "attention_decode", "op": "attention", "seqs": 64, "new": 1, "ragged": True, "context": 8192, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 16, "cache": "bf16", "window": 0, "softcap": 0.0, "pad": 0},
        # Four drafted tokens and the one in front of them for each of 32 sequences, an 8-bit cache.
        {"name": "attention_drafts", "op": "attention", "seqs": 32, "new": 5, "ragged": False, "context": 4099, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "cache": "e4m3", "window": 0, "softcap": 0.0, "pad": 0},
        # One token behind 131071: few rows, a long axis.
        {"name": "attention_long", "op": "attention", "seqs": 1, "new": 1, "ragged": False, "context": 131072, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 128, "cache": "bf16", "window": 0, "softcap": 0.0, "pad": 0},
        # Prompts of up to 1000 tokens beside single tokens, heads of 96, a window and capped scores, padded rows.
        {"name": "attention_mixed", "op": "attention", "seqs": 12, "new": 1000, "ragged": True, "context": 4000, "heads": 16, "kv_heads": 4, "head_dim": 96,
         "page": 32, "cache": "bf16", "window": 1500, "softcap": 30.0, "pad": 19},
        # A chunk of 2048 tokens of a long prompt, 14336 before it in the cache: matrix products.
        {"name": "attention_chunk", "op": "attention", "seqs": 1, "new": 2048, "ragged": False, "context": 16384, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page": 64, "cache": "bf16", "window": 0, "softcap": 0.0, "pad": 0},
        # Two drafted tokens of one sequence, found in its prompt: no distribution of a drafter.
        {"name": "verify_one", "op": "verify", "seqs": 1, "rows": 3, "ragged": False, "vocab": 32000, "padded": 32000, "dtype": "bf16", "drafter": False,
         "temperature": 0.8},
        # 0 to 7 drafts of 24 sequences, GPT-2's vocabulary in a head padded to 50304 columns.
        {"name": "verify_ragged", "op": "verify", "seqs": 24, "rows": 8, "ragged": True, "vocab": 50257, "padded": 50304, "dtype": "bf16", "drafter": True,
         "temperature": 1.0},
        # Five drafts of 64 sequences with Qwen3's vocabulary, fp32 logits of both models.
        {"name": "verify_batch", "op": "verify", "seqs": 64, "rows": 6, "ragged": False, "vocab": 151936, "padded": 151936, "dtype": "fp32",
         "drafter": True, "temperature": 0.7},
    ]


def draw(rng):
    def spread(low, high, multiple=1):
        value = int(round(low * (high / low) ** rng.random() / multiple)) * multiple
        return max(low, min(high, value))

    op = rng.choice(("append", "attention", "attention", "verify"))
    if op == "verify":
        dtype, vocab, rows = rng.choice(("bf16", "fp32")), spread(1000, 151936), spread(1, 9)
        most = max(1, 64 * 6 * 151936 // (vocab * rows) // (1 if dtype == "fp32" else 2))
        return {"op": op, "seqs": spread(1, min(256, most)), "rows": rows, "ragged": rng.random() < 0.5, "vocab": vocab,
                "padded": vocab if rng.random() < 0.5 else -(-vocab // 64) * 64, "dtype": dtype, "drafter": rng.random() < 0.6,
                "temperature": rng.choice((0.0, 0.7, 1.0, 1.3))}
    kv_heads, group, head_dim = rng.choice((1, 2, 4, 8, 12)), rng.choice((1, 2, 3, 4, 8)), rng.choice((64, 64, 96, 128, 128, 128, 80, 32))
    case = {"op": op, "ragged": rng.random() < 0.6, "heads": kv_heads * group, "kv_heads": kv_heads, "head_dim": head_dim,
            "page": rng.choice((8, 16, 16, 32, 64, 128)), "cache": rng.choice(("bf16", "bf16", "e4m3")), "pad": rng.choice((0, 0, 3, 40))}
    if op == "append":
        case["new"] = spread(1, 4000)
        case["seqs"] = spread(1, max(1, min(256, 8192 * 48 // (kv_heads * (group + 2)) // case["new"])))
        case["context"] = case["new"] + spread(1, 500)
        case["norm"], case["halves"] = rng.random() < 0.4, rng.random() < 0.5
        case["rotary"] = head_dim // 2 if head_dim % 32 == 0 and rng.random() < 0.2 else head_dim
        return case
    case["new"] = rng.choice((1, 1, spread(2, 8), spread(2, 2048)))
    case["context"] = case["new"] + spread(1, 30000)
    held = case["context"] * kv_heads * head_dim                         # elements of keys of the longest sequence; a pass reads as many values
    pairs = case["new"] * case["context"] * case["heads"]
    case["seqs"] = spread(1, max(1, min(128, 64 * 8192 * 8 * 128 // 2 // held, 2048 * 16384 * 32 // pairs)))
    case["window"] = rng.choice((0, 0, spread(1, 4096)))
    case["softcap"] = rng.choice((0.0, 0.0, 20.0, 50.0))
    return case


def _counts(case):
    """New tokens and lengths of the sequences: by the case alone."""
    new, length = [], []
    for i in range(case["seqs"]):
        part = (0.6180339887 * (i + 1)) % 1.0 if case["ragged"] else 1.0
        new.append(max(1, round(case["new"] * part)) if i % 3 or not case["ragged"] else 1)      # (a third of a ragged batch is single tokens)
        length.append(max(new[-1], round(case["context"] * (part if i % 2 else 1.0))))
    return new, length


def _rows(case):
    """Rows of logits of each sequence: its drafts and one."""
    return [(1 + (3 * i + 1) % case["rows"] if case["ragged"] else case["rows"]) for i in range(case["seqs"])]


class _State:
    """The tensors that a program holds before the call."""


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _cache_state(s, case, gen):
    def normal(*shape, scale=1.0):
        return (torch.randn(shape, device=DEVICE, generator=gen) * scale).bfloat16()

    new, length = _counts(case)
    heads, kv, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    s.offsets, s.lengths = _ints([sum(new[:i]) for i in range(len(new) + 1)]), _ints(length)
    s.used, s.total, s.max_new = sum(new), sum(new) + case["pad"], max(new)
    need = [-(-n // page) for n in length]
    ids = torch.randperm(sum(need) + 3, device=DEVICE, generator=gen)[:sum(need)].int()
    width = max(need)
    s.pages = torch.zeros((len(need), width), dtype=torch.int32, device=DEVICE)
    held = torch.arange(width, device=DEVICE).unsqueeze(0) < _ints(need).unsqueeze(1)
    s.pages[held] = ids
    shape = (sum(need) + 3, kv, page, dim)
    s.key_scale = s.value_scale = None
    if case["cache"] == "e4m3":
        s.key_scale = 0.01 + 0.01 * torch.rand((kv,), device=DEVICE, generator=gen)
        s.value_scale = 0.01 + 0.01 * torch.rand((kv,), device=DEVICE, generator=gen)
        s.keys, s.values = ((torch.randn(shape, device=DEVICE, generator=gen) / 0.015).to(torch.float8_e4m3fn) for _ in range(2))
    else:
        s.keys, s.values = normal(*shape), normal(*shape)
    s.dim = dim
    if case["op"] == "append":
        # queries, keys and values as one projection left them
        fused = normal(s.total, (heads + 2 * kv) * dim)
        s.q, s.k, s.v = (t.unflatten(1, (-1, dim)) for t in fused.split((heads * dim, kv * dim, kv * dim), dim=1))
        half = case["rotary"] // 2
        angle = torch.outer(torch.arange(width * page, device=DEVICE, dtype=torch.float64),
                            THETA ** (-torch.arange(half, device=DEVICE, dtype=torch.float64) / half))
        s.cos, s.sin, s.interleaved = angle.cos().float(), angle.sin().float(), not case["halves"]
        s.q_weight = s.k_weight = None
        if case["norm"]:
            s.q_weight, s.k_weight = (1.0 + 0.1 * torch.randn((dim,), device=DEVICE, generator=gen) for _ in range(2))
    else:
        s.q = normal(s.total, heads, dim, scale=1.5)
        s.scale, s.window, s.softcap = dim ** -0.5, case["window"], case["softcap"]


def _verify_state(s, case, gen):
    rows, vocab, t = _rows(case), case["vocab"], case["temperature"] or 1.0
    s.offsets = _ints([sum(rows[:i]) for i in range(len(rows) + 1)])
    s.total, s.most = sum(rows), max(rows)
    x = torch.randn((s.total, case["padded"]), device=DEVICE, generator=gen) * 2.5
    x[torch.arange(s.total, device=DEVICE), torch.randint(0, vocab, (s.total,), device=DEVICE, generator=gen)] += 9.0
    # a drafter that agrees with the model in most places
    y = x + 0.7 * torch.randn(x.shape, device=DEVICE, generator=gen)
    race = torch.empty((s.total, vocab), device=DEVICE).exponential_(generator=gen).log_()
    drafted = (y[:, :vocab] / t - race).argmax(1)
    drafted = torch.where(torch.rand((s.total,), device=DEVICE, generator=gen) < 0.5, x[:, :vocab].argmax(1), drafted)
    s.tokens = torch.cat((torch.zeros_like(drafted[:1]), drafted[:-1]))
    dtype = LOGITS[case["dtype"]]
    s.logits, s.draft_logits = x.to(dtype), y.to(dtype) if case["drafter"] else None
    s.uniforms = torch.rand((s.total,), device=DEVICE, generator=gen)
    s.vocab, s.temperature = vocab, case["temperature"]


def prepare(case, seed):
    s = _State()
    s.op = case["op"]
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    (_verify_state if s.op == "verify" else _cache_state)(s, case, gen)
    return s


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_append(s):
    from optimus_dl_amd.modules.paged import append_kv

    q = append_kv(s.q, s.k, s.v, s.keys, s.values, s.pages, s.offsets, s.lengths, cos=s.cos, sin=s.sin, interleaved=s.interleaved,
                  q_weight=s.q_weight, k_weight=s.k_weight, eps=EPS, key_scale=s.key_scale, value_scale=s.value_scale)
    return {"q": q, "keys": s.keys, "values": s.values}


def _own_attention(s):
    from optimus_dl_amd.modules.paged import paged_attention

    return paged_attention(s.q, s.keys, s.values, s.pages, s.offsets, s.lengths, max_new=s.max_new, scale=s.scale, window=s.window, softcap=s.softcap,
                           key_scale=s.key_scale, value_scale=s.value_scale)


def _own_verify(s):
    from optimus_dl_amd.modules.drafts import verify_drafts

    r = verify_drafts(s.logits, s.tokens, s.offsets, s.uniforms, draft_logits=s.draft_logits, temperature=s.temperature, n_vocab=s.vocab)
    return {"accepted": r.accepted, "tokens": r.tokens, "logprobs": r.logprobs}


# ------------------------------------------------------------------------------------------------------ the plain forms
def _sequence_of(offsets, total):
    """For every row its sequence, its place there, and whether it has one (rows behind the last sequence have none)."""
    row = torch.arange(total, device=DEVICE)
    seq = torch.searchsorted(offsets[1:].long(), row, right=True)
    live = seq < offsets.numel() - 1
    seq = seq.clamp(max=offsets.numel() - 2)
    return seq, row - offsets.long()[seq], live


def _plain_append(s):
    seq, at, live = _sequence_of(s.offsets, s.total)
    offsets, lengths = s.offsets.long(), s.lengths.long()
    position = torch.where(live, lengths[seq] - (offsets[1:] - offsets[:-1])[seq] + at, torch.zeros_like(at))
    cos, sin = s.cos[position].unsqueeze(1), s.sin[position].unsqueeze(1)
    rotary, half = 2 * cos.shape[-1], cos.shape[-1]

    def turned(x, weight):
        x = x.float()
        if weight is not None:
            x = x * (1.0 / (x.double().square().mean(-1, keepdim=True) + EPS).sqrt()).float() * weight
        a, b = (x[..., 0:rotary:2], x[..., 1:rotary:2]) if s.interleaved else (x[..., :half], x[..., half:rotary])
        a, b = a * cos - b * sin, a * sin + b * cos
        return torch.cat((torch.stack((a, b), -1).flatten(-2) if s.interleaved else torch.cat((a, b), -1), x[..., rotary:]), -1)

    q = torch.where(live.view(-1, 1, 1), turned(s.q, s.q_weight).bfloat16(), torch.zeros((), dtype=torch.bfloat16, device=DEVICE))
    k, v = turned(s.k, s.k_weight), s.v.float()
    page, used = s.keys.shape[2], s.used
    ids, slot = s.pages.long()[seq, position // page][:used], (position % page)[:used]
    for x, cache, scale in ((k, s.keys, s.key_scale), (v, s.values, s.value_scale)):
        x = x[:used]
        if scale is not None:
            x = (x / scale.view(1, -1, 1)).clamp(-448.0, 448.0)
        codes = {1: torch.uint8, 2: torch.int16}[cache.element_size()]
        cache.view(codes)[ids, :, slot] = x.to(cache.dtype).view(codes)
    return {"q": q, "keys": s.keys, "values": s.values}


def _gathered(cache, pages, scale):
    """What the pages of every sequence hold, fp32 [sequences, kv heads, positions, head_dim]."""
    if scale is not None:
        x = cache.view(torch.uint8)[pages.long()].view(cache.dtype).float() * scale.view(1, 1, -1, 1, 1)
    else:
        x = cache[pages.long()].float()
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attention(s):
    heads, dim, kv = s.q.shape[1], s.q.shape[2], s.keys.shape[1]
    offsets, lengths = s.offsets.long(), s.lengths.long()
    j = torch.arange(s.max_new, device=DEVICE)
    row = (offsets[:-1].unsqueeze(1) + j).clamp(max=s.total - 1)
    q = s.q[row].float().transpose(1, 2).reshape(len(lengths), kv, -1, dim)                   # [sequences, kv heads, group * new, head_dim]
    k, v = _gathered(s.keys, s.pages, s.key_scale), _gathered(s.values, s.pages, s.value_scale)
    score = torch.matmul(q, k.transpose(-1, -2)) * s.scale
    if s.softcap:
        score = s.softcap * torch.tanh(score / s.softcap)
    place = torch.arange(k.shape[2], device=DEVICE).view(1, 1, -1)
    position = (lengths - (offsets[1:] - offsets[:-1])).view(-1, 1, 1) + j.view(1, -1, 1)
    seen = (place <= position) & (place < lengths.view(-1, 1, 1))
    if s.window:
        seen &= place > position - s.window
    score = score.unflatten(2, (heads // kv, s.max_new)).masked_fill_(~seen.view(len(lengths), 1, 1, s.max_new, -1), float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    v = torch.where((place < lengths.view(-1, 1, 1)).view(len(lengths), 1, -1, 1), v, torch.zeros((), device=DEVICE))
    out = torch.matmul(p.flatten(2, 3), v).unflatten(2, (heads // kv, s.max_new)) / total
    out = out.flatten(1, 2).transpose(1, 2)                                                   # [sequences, new, heads, head_dim]
    seq, at, live = _sequence_of(s.offsets, s.total)
    out = out[seq, at.clamp(max=s.max_new - 1)]
    return torch.where(live.view(-1, 1, 1), out, torch.zeros((), device=DEVICE)).bfloat16()


def _plain_verify(s):
    seq, _, live = _sequence_of(s.offsets, s.total)
    offsets, count = s.offsets.long(), len(s.offsets) - 1
    row = torch.arange(s.total, device=DEVICE)
    drafted = torch.cat((s.tokens[1:], s.tokens[:1]))                                         # the token behind each row
    last = row == offsets[seq + 1] - 1
    x = s.logits[:, :s.vocab].double()
    p = _softmax(x / (s.temperature or 1.0))
    if s.temperature == 0:
        best = torch.where(x == x.amax(1, keepdim=True), torch.arange(s.vocab, device=DEVICE), s.vocab).amin(1)
        agreed = best == drafted
    else:
        of_p = p.gather(1, drafted.unsqueeze(1)).squeeze(1)
        q = None if s.draft_logits is None else _softmax(s.draft_logits[:, :s.vocab].double() / s.temperature)
        of_q = torch.ones_like(of_p) if q is None else q.gather(1, drafted.unsqueeze(1)).squeeze(1)
        agreed = s.uniforms.double() * of_q < of_p
    # the first row of each sequence that stops: a draft that is not agreed to, or the last row
    stop = torch.full((count,), s.total, device=DEVICE).scatter_reduce(0, seq, torch.where(live & (last | ~agreed), row, s.total), "amin")
    if s.temperature == 0:
        chosen = best[stop]
    else:
        r = p[stop]
        at = torch.arange(s.vocab, device=DEVICE)
        less = (at == drafted[stop].unsqueeze(1)).double() * r if q is None else q[stop]
        r = torch.where(last[stop].unsqueeze(1), r, (r - less).clamp(min=0.0))
        r = torch.where((r.sum(1) > 0).unsqueeze(1), r, p[stop])
        below = r.cumsum(1)
        chosen = (below <= s.uniforms.double()[offsets[1:] - 1].unsqueeze(1) * below[:, -1:]).sum(1)
    tokens = torch.where(row < stop[seq], drafted, torch.where(row == stop[seq], chosen[seq], -1))
    told = tokens >= 0
    logp = p.gather(1, tokens.clamp(min=0).unsqueeze(1)).squeeze(1).log()
    return {"accepted": (stop - offsets[:-1]).int(), "tokens": tokens, "logprobs": torch.where(told, logp, torch.zeros_like(logp)).float()}


def _softmax(x):
    e = (x - x.amax(1, keepdim=True)).exp()
    return e / e.sum(1, keepdim=True)


def run(state):
    if own:
        with torch.no_grad():
            return {"append": _own_append, "attention": _own_attention, "verify": _own_verify}[state.op](state)
    with torch.no_grad():
        return {"append": _plain_append, "attention": _plain_attention, "verify": _plain_verify}[state.op](state)


# ----------------------------------------------------------------------------------------------------- from definitions
def _exact_append(s, case):
    new, length = _counts(case)
    page = s.keys.shape[2]
    q_out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEVICE)
    caches = [s.keys.double(), s.values.double()]
    for i, (n, held) in enumerate(zip(new, length)):
        rows = slice(sum(new[:i]), sum(new[:i]) + n)
        position = torch.arange(held - n, held, device=DEVICE)
        turn = torch.complex(s.cos[position].double(), s.sin[position].double()).unsqueeze(1)

        def rotated(x, weight):
            x = x[rows].double()
            if weight is not None:
                x = torch.nn.functional.rms_norm(x, x.shape[-1:], weight.double(), EPS)
            m = 2 * turn.shape[-1]
            pairs = x[..., :m].unflatten(-1, (-1, 2)) if s.interleaved else x[..., :m].unflatten(-1, (2, -1)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            return torch.cat(((z if s.interleaved else z.transpose(-1, -2)).flatten(-2), x[..., m:]), -1)

        q_out[rows] = rotated(s.q, s.q_weight)
        for cache, x, scale in zip(caches, (rotated(s.k, s.k_weight), s.v[rows].double()), (s.key_scale, s.value_scale)):
            x = x if scale is None else (x / scale.double()[:, None]).clamp(-448.0, 448.0)
            cache[s.pages[i].long()[position // page], :, position % page] = x
    return {"q": q_out, "keys": caches[0], "values": caches[1]}


def _exact_attention(s, case):
    new, length = _counts(case)
    heads, kv = case["heads"], case["kv_heads"]
    out = torch.zeros(s.q.shape, dtype=torch.float64, device=DEVICE)
    for i, (n, held) in enumerate(zip(new, length)):
        first, page = sum(new[:i]), s.keys.shape[2]
        at = torch.arange(held, device=DEVICE)
        ids = s.pages[i].long()[at // page]
        for h in range(kv):
            k, v = (c[:, h].float()[ids, at % page].double() * (1.0 if z is None else z[h].double())
                    for c, z in ((s.keys, s.key_scale), (s.values, s.value_scale)))
            for g in range(h * heads // kv, (h + 1) * heads // kv):
                score = torch.mm(s.q[first:first + n, g].double(), k.t()).mul_(s.scale)
                if s.softcap:
                    score = (score / s.softcap).tanh_().mul_(s.softcap)
                before = torch.arange(held - n, held, device=DEVICE)[:, None] - at                # how far behind the row a key lies
                hidden = (before < 0) | (before >= s.window) if s.window else before < 0
                out[first:first + n, g] = torch.mm(torch.softmax(score.masked_fill(hidden, float("-inf")), -1), v)
    return out


def _exact_verify(s, case):
    logprobs = torch.zeros(s.total, dtype=torch.float64, device=DEVICE)
    rows, t = _rows(case), s.temperature
    for i, n in enumerate(rows):
        first = sum(rows[:i])
        logp = torch.log_softmax(s.logits[first:first + n, :s.vocab].double() / (t or 1.0), 1)
        u = s.uniforms[first:first + n].double().tolist()
        for j in range(n):
            token = int(s.tokens[first + j + 1]) if j + 1 < n else None
            p = logp[j].exp()
            q = torch.zeros_like(p)
            if token is not None and s.draft_logits is not None and t:
                q = torch.softmax(s.draft_logits[first + j, :s.vocab].double() / t, 0)
            elif token is not None:
                q[token] = 1.0
            if not t:
                keep, other = token == int(logp[j].argmax()), int(logp[j].argmax())
            else:
                keep = token is not None and u[j] < float(p[token] / q[token])
                rest = torch.relu(p - q).cumsum(0)
                other = int(torch.searchsorted(rest, u[-1] * rest[-1], right=True))
            logprobs[first + j] = logp[j, token if keep else other]
            if not keep:
                break
    return {"accepted": None, "tokens": None, "logprobs": logprobs}


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "verify": _exact_verify}[s.op](s, case)


def work(case):
    """Bytes of what comes in and goes out, each once, and the operations of the formulas (of products: multiply and add)."""
    if case["op"] == "verify":
        rows, size = sum(_rows(case)), 4 if case["dtype"] == "fp32" else 2
        drafts = rows - case["seqs"] if case["drafter"] and case["temperature"] else 0
        return {"bytes": (rows + drafts) * case["vocab"] * size + rows * 24, "flops": (rows + drafts) * case["vocab"] * 4.0}
    new, length = _counts(case)
    heads, kv, dim, size = case["heads"], case["kv_heads"], case["head_dim"], 2 if case["cache"] == "bf16" else 1
    if case["op"] == "append":
        row = 2 * dim * (2 * heads + 2 * kv) + 2 * kv * dim * size
        return {"bytes": sum(new) * (row + 8 * case["rotary"] // 2), "flops": sum(new) * dim * (heads + kv) * (7.0 if case["norm"] else 3.0)}
    window = case["window"] or 1 << 60
    read = sum(min(m, window + n - 1) for n, m in zip(new, length))
    # pairs of a row and a key that it sees: the row at position p sees min(p + 1, window)
    full = [sum(min(p + 1, window) for p in range(m - n, m)) for n, m in zip(new, length)]
    return {"bytes": 2 * read * kv * dim * size + 4 * sum(new) * heads * dim, "flops": 4.0 * sum(full) * heads * dim}
