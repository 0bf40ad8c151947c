"""What stands around the FP8 Linear of a decoder: the residual stream's norms, the answer of the head, Linears with 4-bit weights.

``residual_norm``: the norm behind a block, its gate and the scaled residual, and the norm in front of the next block.
``token_logprobs``: log probabilities of given tokens from the logits of a head, with entropy and top alternatives.
``fp4_linear``: product with weights held as E2M1 codes, two a byte, with a bf16 scale for each group of 32, 64 or 128.

Training passes are forward and backward for given gradients of the outputs.
"""

import torch

own = False

DEVICE = torch.device("cuda")
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6
IGNORE = -100
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # One token of one sequence in a Llama-3-8B-sized decoder with norms before and after its blocks: latency counts.
        {"name": "norm_token", "op": "residual_norm", "train": False, "rows": 1, "cols": 4096, "stream": "fp32", "branch": "bf16",
         "post": True, "gate": "channel", "scale": 1.0},
        # Evaluation of 16 sequences of 1024 tokens at the width of Qwen3-0.6B, no gate.
        {"name": "norm_eval", "op": "residual_norm", "train": False, "rows": 16384, "cols": 1024, "stream": "fp32", "branch": "bf16",
         "post": True, "gate": "none", "scale": 1.0},
        # Training on sequences of 1004 tokens, everything in bf16, no norm behind the block, one learned gate, scaled residual.
        {"name": "norm_step_ragged", "op": "residual_norm", "train": True, "rows": 4016, "cols": 2048, "stream": "bf16", "branch": "bf16",
         "post": False, "gate": "scalar", "scale": 0.5},
        # Training step of a Llama-3-8B-sized decoder on 8192 tokens: fp32 stream, both norms, a gate for each channel.
        {"name": "norm_step", "op": "residual_norm", "train": True, "rows": 8192, "cols": 4096, "stream": "fp32", "branch": "bf16",
         "post": True, "gate": "channel", "scale": 1.0},
        # A decode step of 16 sequences: the sampled token's log probability and the 20 likeliest others.
        {"name": "logprobs_token", "op": "token_logprobs", "train": False, "rows": 16, "vocab": 32000, "padded": 32000, "dtype": "bf16",
         "top_k": 20, "temperature": 0.7},
        # Scoring of two sequences of 1024 tokens with GPT-2's vocabulary in a head padded to 50304 columns.
        {"name": "logprobs_score", "op": "token_logprobs", "train": False, "rows": 2048, "vocab": 50257, "padded": 50304, "dtype": "bf16",
         "top_k": 5, "temperature": 1.0},
        # Training on one sequence of 1004 tokens, fp32 logits whose rows begin at no 16-byte boundary.
        {"name": "logprobs_step_odd", "op": "token_logprobs", "train": True, "rows": 1004, "vocab": 50257, "padded": 50257, "dtype": "fp32",
         "top_k": 0, "temperature": 1.0},
        # The loss of GPT-2 124M on 8192 tokens and its gradient, with an entropy term.
        {"name": "logprobs_step", "op": "token_logprobs", "train": True, "rows": 8192, "vocab": 50257, "padded": 50304, "dtype": "bf16",
         "top_k": 0, "temperature": 1.0},
        # q, k and v of GPT-2 124M for one token: the smallest product, with a bias.
        {"name": "fp4_token_small", "op": "fp4_linear", "rows": 1, "n_in": 768, "n_out": 2304, "group": 32, "bias": True},
        # The up-projection of Llama-3-8B for one token.
        {"name": "fp4_token", "op": "fp4_linear", "rows": 1, "n_in": 4096, "n_out": 14336, "group": 128, "bias": False},
        # Its down-projection for a decode step of 32 sequences, the finest groups.
        {"name": "fp4_decode_32", "op": "fp4_linear", "rows": 32, "n_in": 14336, "n_out": 4096, "group": 32, "bias": False},
        # The up-projection of a 70B layer for 120 rows: a large batch of single tokens, or short prompts.
        {"name": "fp4_batch_120", "op": "fp4_linear", "rows": 120, "n_in": 8192, "n_out": 28672, "group": 64, "bias": False},
    ]


def draw(rng):
    def spread(low, high, multiple=1):
        value = int(round(low * (high / low) ** rng.random() / multiple)) * multiple
        return max(low, min(high, value))

    op = rng.choice(("residual_norm", "token_logprobs", "fp4_linear"))
    if op == "residual_norm":
        cols = spread(64, 8192, 8)
        stream = rng.choice(("bf16", "fp32"))
        return {"op": op, "train": rng.random() < 0.6, "rows": spread(1, min(16384, 8192 * 4096 // cols)), "cols": cols, "stream": stream,
                "branch": "fp32" if stream == "fp32" and rng.random() < 0.3 else "bf16", "post": rng.random() < 0.6,
                "gate": rng.choice(("none", "scalar", "channel")), "scale": rng.choice((1.0, 0.5, 0.7071))}
    if op == "token_logprobs":
        vocab, train = spread(1000, 131072), rng.random() < 0.5
        dtype = rng.choice(("bf16", "fp32"))
        most = 8192 * 50304 // vocab // (2 if dtype == "fp32" else 1)
        return {"op": op, "train": train, "rows": spread(1, min(8192 if train else 2048, most)), "vocab": vocab,
                "padded": vocab if rng.random() < 0.5 else -(-vocab // 64) * 64, "dtype": dtype,
                "top_k": 0 if train else rng.choice((1, 5, 8, 20, 32)), "temperature": rng.choice((1.0, 1.0, 0.7, 1.5))}
    group = rng.choice((32, 64, 128))
    return {"op": op, "rows": spread(1, 120), "n_in": spread(256, 14336, group), "n_out": spread(100, 28672 // 2), "group": group,
            "bias": rng.random() < 0.5}


class _State:
    """The tensors that a program holds before the call."""


def _norm_state(s, case, gen):
    rows, cols = case["rows"], case["cols"]

    def normal(*shape, dtype=torch.float32, scale=1.0, shift=0.0):
        return (torch.randn(shape, device=DEVICE, generator=gen) * scale + shift).to(dtype)

    stream, branch = DTYPES[case["stream"]], DTYPES[case["branch"]]
    s.x, s.h = normal(rows, cols, dtype=stream), normal(rows, cols, dtype=branch, scale=0.3)
    s.weight = normal(cols, scale=0.1, shift=1.0)
    s.post_weight = normal(cols, scale=0.1, shift=1.0) if case["post"] else None
    s.gate = {"none": None, "scalar": normal(1, scale=0.1, shift=0.5), "channel": normal(cols, scale=0.2, shift=0.5)}[case["gate"]]
    s.scale = case["scale"]
    if case["train"]:
        s.dy, s.dz = normal(rows, cols, dtype=stream, scale=1e-3), normal(rows, cols, dtype=torch.bfloat16, scale=1e-3)
        for t in (s.x, s.h, s.weight, s.post_weight, s.gate):
            if t is not None:
                t.requires_grad_(True)


def _logprobs_state(s, case, gen):
    rows, vocab, padded = case["rows"], case["vocab"], case["padded"]
    logits = torch.randn((rows, padded), device=DEVICE, generator=gen)
    logits.mul_(2.5)
    s.targets = torch.randint(0, vocab, (rows,), device=DEVICE, generator=gen)
    # a model that has learned something: the target stands out in most rows, by different amounts
    at = torch.arange(rows, device=DEVICE)
    logits[at, s.targets] += 12.0 * torch.rand((rows,), device=DEVICE, generator=gen)
    s.logits = logits.to(DTYPES[case["dtype"]])
    s.vocab, s.top_k, s.temperature = vocab, case["top_k"], case["temperature"]
    if case["train"]:
        s.targets[torch.rand((rows,), device=DEVICE, generator=gen) < 0.05] = IGNORE         # prompts and padding
        s.d_logprobs = -(0.5 + torch.rand((rows,), device=DEVICE, generator=gen)) / rows
        s.d_entropy = -1e-2 * (0.5 + torch.rand((rows,), device=DEVICE, generator=gen)) / rows
        s.logits.requires_grad_(True)


def _fp4_state(s, case, gen):
    n, k, group = case["n_out"], case["n_in"], case["group"]
    w = torch.randn((n, k // group, group), device=DEVICE, generator=gen) * 0.02
    s.scales = (w.abs().amax(-1) / 6.0).bfloat16()
    middle = torch.tensor([(a + b) / 2 for a, b in zip(E2M1, E2M1[1:])], device=DEVICE)
    codes = torch.bucketize(w.abs() / s.scales.float().unsqueeze(-1), middle) + 8 * (w < 0)
    codes = codes.to(torch.uint8).reshape(n, k // 2, 2)
    s.codes = codes[..., 0] | (codes[..., 1] << 4)
    s.x = torch.randn((case["rows"], k), device=DEVICE, generator=gen).bfloat16()
    s.bias = torch.randn((n,), device=DEVICE, generator=gen) * 0.1 if case["bias"] else None


def prepare(case, seed):
    s = _State()
    s.op, s.train = case["op"], case.get("train", False)
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    {"residual_norm": _norm_state, "token_logprobs": _logprobs_state, "fp4_linear": _fp4_state}[s.op](s, case, gen)
    return s


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_norm(s):
    from optimus_dl_amd.modules.fused import residual_norm

    def forward():
        return residual_norm(s.x, s.h, s.weight, EPS, post_weight=s.post_weight, gate=s.gate, residual_scale=s.scale,
                             out_dtype=torch.bfloat16)

    if not s.train:
        with torch.no_grad():
            y, z = forward()
        return {"y": y, "z": z}
    y, z = forward()
    names = ["x", "h", "weight"] + [n for n in ("post_weight", "gate") if getattr(s, n) is not None]
    grads = torch.autograd.grad((y, z), [getattr(s, n) for n in names], (s.dy, s.dz))
    return {"y": y.detach(), "z": z.detach(), **{"d" + n: g for n, g in zip(names, grads)}}


def _own_logprobs(s):
    from optimus_dl_amd.modules.logprobs import token_logprobs

    def forward():
        return token_logprobs(s.logits, s.targets, n_vocab=s.vocab, top_k=s.top_k, temperature=s.temperature, ignore_index=IGNORE)

    if not s.train:
        with torch.no_grad():
            r = forward()
        return {"logprobs": r.logprobs, "entropy": r.entropy, "top_logprobs": r.top_logprobs, "top_ids": r.top_ids}
    r = forward()
    (dlogits,) = torch.autograd.grad((r.logprobs, r.entropy), (s.logits,), (s.d_logprobs, s.d_entropy))
    return {"logprobs": r.logprobs.detach(), "entropy": r.entropy.detach(), "dlogits": dlogits}


def _own_fp4(s):
    from optimus_dl_amd.modules.fp4_linear import fp4_linear

    with torch.no_grad():
        return fp4_linear(s.x, s.codes, s.scales, s.bias)


# ------------------------------------------------------------------------------------------------------ the plain forms
def _plain_norm(s):
    with torch.no_grad():
        cols = s.x.shape[1]
        x, h, wn = s.x.float(), s.h.float(), s.weight
        wp = s.post_weight if s.post_weight is not None else torch.ones(cols, device=DEVICE)
        g = s.gate if s.gate is not None else torch.ones(1, device=DEVICE)
        rh = 1.0 / ((h * h).mean(-1, keepdim=True) + EPS).sqrt() if s.post_weight is not None else 1.0
        hh = h * rh
        y = s.scale * x + g * (hh * wp)
        ry = 1.0 / ((y * y).mean(-1, keepdim=True) + EPS).sqrt()
        yh = y * ry
        out = {"y": y.to(s.x.dtype), "z": (yh * wn).bfloat16()}
        if not s.train:
            return out
        dz = s.dz.float()
        t = dz * wn
        e = s.dy.float() + ry * (t - yh * (t * yh).mean(-1, keepdim=True))
        q = e * (g * wp)
        dh = rh * (q - hh * (q * hh).mean(-1, keepdim=True)) if s.post_weight is not None else q
        out.update(dx=(s.scale * e).to(s.x.dtype), dh=dh.to(s.h.dtype), dweight=(dz * yh).sum(0))
        d = (e * hh).sum(0)
        if s.post_weight is not None:
            out["dpost_weight"] = g * d
        if s.gate is not None:
            out["dgate"] = wp * d if s.gate.numel() == cols and cols > 1 else (wp * d).sum().reshape(1)
        return out


def _plain_logprobs(s):
    with torch.no_grad():
        x = s.logits[:, :s.vocab].float()
        kept = s.targets != IGNORE
        target = torch.where(kept, s.targets, torch.zeros_like(s.targets)).unsqueeze(1)
        d = (x - x.max(1, keepdim=True).values) / s.temperature
        e = d.exp()
        total = e.sum(1, keepdim=True)
        log_total = total.log()
        logp = (d.gather(1, target) - log_total).squeeze(1)
        entropy = (log_total - (e * d).sum(1, keepdim=True) / total).squeeze(1)
        out = {"logprobs": torch.where(kept, logp, torch.zeros_like(logp)), "entropy": torch.where(kept, entropy, torch.zeros_like(entropy))}
        if not s.train:
            del e
            top, ids = x.sort(dim=1, descending=True, stable=True)
            ids = ids[:, :s.top_k].contiguous()
            out.update(top_logprobs=d.gather(1, ids) - log_total, top_ids=ids)
            return out
        p = e.div_(total)
        a, b = s.d_logprobs.unsqueeze(1), s.d_entropy.unsqueeze(1)
        grad = -p * (a + b * (d - log_total + entropy.unsqueeze(1)))
        grad.scatter_add_(1, target, a)
        grad = torch.where(kept.unsqueeze(1), grad / s.temperature, torch.zeros_like(a))
        dlogits = torch.zeros_like(s.logits)
        dlogits[:, :s.vocab] = grad.to(s.logits.dtype)
        out["dlogits"] = dlogits
        return out


def _plain_fp4(s):
    n, k = s.codes.shape[0], 2 * s.codes.shape[1]
    codes = torch.stack((s.codes & 15, s.codes >> 4), dim=-1).reshape(n, k)
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=DEVICE)
    w = table[codes.long()].reshape(n, s.scales.shape[1], -1) * s.scales.float().unsqueeze(-1)
    y = s.x.float() @ w.reshape(n, k).t()
    return (y if s.bias is None else y + s.bias).bfloat16()


def run(state):
    if own:
        return {"residual_norm": _own_norm, "token_logprobs": _own_logprobs, "fp4_linear": _own_fp4}[state.op](state)
    return {"residual_norm": _plain_norm, "token_logprobs": _plain_logprobs, "fp4_linear": _plain_fp4}[state.op](state)


# ----------------------------------------------------------------------------------------------------- from definitions
def _exact_norm(s):
    def leaf(t):
        return None if t is None else t.detach().double().requires_grad_(True)

    x, h, w, wp, g = (leaf(t) for t in (s.x, s.h, s.weight, s.post_weight, s.gate))
    cols = (x.shape[1],)
    u = h if wp is None else torch.nn.functional.rms_norm(h, cols, wp, EPS)
    y = s.scale * x + (u if g is None else g * u)
    z = torch.nn.functional.rms_norm(y, cols, w, EPS)
    out = {"y": y.detach(), "z": z.detach()}
    if s.train:
        leaves = {"dx": x, "dh": h, "dweight": w, "dpost_weight": wp, "dgate": g}
        leaves = {n: t for n, t in leaves.items() if t is not None}
        grads = torch.autograd.grad((y, z), list(leaves.values()), (s.dy.double(), s.dz.double()))
        out.update(zip(leaves, grads))
    return out


def _exact_logprobs(s):
    parts = []
    for i in range(0, s.logits.shape[0], 1024):                        # (rows are independent: less memory at once)
        logits = s.logits[i:i + 1024].detach().double().requires_grad_(s.train)
        targets = s.targets[i:i + 1024]
        kept = targets != IGNORE
        logp = torch.log_softmax(logits[:, :s.vocab] / s.temperature, dim=1)
        lp = torch.where(kept, logp.gather(1, targets.clamp(min=0).unsqueeze(1)).squeeze(1), 0.0)
        entropy = torch.where(kept, torch.special.entr(logp.exp()).sum(1), 0.0)
        part = {"logprobs": lp.detach(), "entropy": entropy.detach()}
        if s.train:
            loss = (lp * s.d_logprobs[i:i + 1024]).sum() + (entropy * s.d_entropy[i:i + 1024]).sum()
            part["dlogits"] = torch.autograd.grad(loss, logits)[0]
        else:
            part["top_logprobs"] = logp.topk(s.top_k, dim=1).values
        parts.append(part)
    out = {n: torch.cat([p[n] for p in parts]) for n in parts[0]}
    if not s.train:
        out["top_ids"] = None
    return out


def _exact_fp4(s):
    signs = torch.tensor([1.0, -1.0], dtype=torch.float64, device=DEVICE)
    ys = []
    for codes, scales in zip(s.codes.split(4096), s.scales.split(4096)):
        nibbles = torch.stack((codes.int() % 16, codes.int() // 16), dim=2).flatten(1)
        exponent, mantissa = (nibbles // 2) % 4, nibbles % 2
        value = torch.where(exponent == 0, 0.5 * mantissa, (1.0 + 0.5 * mantissa) * 2.0 ** (exponent - 1)).double()
        w = value * signs[nibbles // 8] * scales.double().repeat_interleave(nibbles.shape[1] // scales.shape[1], dim=1)
        ys.append(torch.mm(s.x.double(), w.t()))
    y = torch.cat(ys, dim=1)
    return y if s.bias is None else y + s.bias.double()


def exact(case, seed):
    s = prepare(case, seed)
    return {"residual_norm": _exact_norm, "token_logprobs": _exact_logprobs, "fp4_linear": _exact_fp4}[s.op](s)


def work(case):
    """Bytes of the tensors that come in and go out, each once, and the operations of the formulas (of products: multiply and add)."""
    rows = case["rows"]
    if case["op"] == "residual_norm":
        stream, branch = (4 if case[n] == "fp32" else 2 for n in ("stream", "branch"))
        each = stream + branch + stream + 2                            # x, h in; y, z out
        if case["train"]:
            each += 2 * stream + 2 + branch                            # dy, dz in; dx, dh out
        return {"bytes": rows * case["cols"] * each, "flops": rows * case["cols"] * (40.0 if case["train"] else 10.0)}
    if case["op"] == "token_logprobs":
        size = 4 if case["dtype"] == "fp32" else 2
        moved = rows * case["vocab"] * size + rows * (8 + 8 + 12 * case["top_k"])
        if case["train"]:
            moved += rows * case["padded"] * size + rows * 8
        return {"bytes": moved, "flops": rows * case["vocab"] * (16.0 if case["train"] else 8.0)}
    n, k = case["n_out"], case["n_in"]
    moved = n * k // 2 + 2 * n * (k // case["group"]) + 2 * rows * (n + k) + (4 * n if case["bias"] else 0)
    return {"bytes": moved, "flops": 2.0 * rows * n * k}

