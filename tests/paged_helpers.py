"""A paged cache and batches over it for tests, and both operators from their definitions in 64 bits, sequence by sequence and head by head."""
import math

import torch

BF16, E4M3 = torch.bfloat16, torch.float8_e4m3fn


class Case:
    """Sequences with `new` new tokens and `lengths` tokens in all, pages in a random order among `spare` unused ones.  Everything on the CPU; `to` moves it."""

    def __init__(self, new, lengths, heads, kv_heads, dim, page, cache=BF16, pad=0, seed=0, spare=3, width=None, q_scale=1.5):
        g = torch.Generator().manual_seed(seed)
        self.new, self.length, self.heads, self.kv, self.dim, self.page = list(new), list(lengths), heads, kv_heads, dim, page
        need = [-(-n // page) for n in lengths]
        ids = torch.randperm(sum(need) + spare, generator=g).int()
        self.width = max(need + [1]) if width is None else width
        self.pages = torch.full((len(need), self.width), -7, dtype=torch.int32)
        at = 0
        for s, n in enumerate(need):
            self.pages[s, :n] = ids[at:at + n][:self.width]
            at += n
        self.offsets = torch.tensor([sum(new[:i]) for i in range(len(need) + 1)], dtype=torch.int32)
        self.lengths = torch.tensor(self.length, dtype=torch.int32)
        self.rows = sum(new) + pad
        shape = (sum(need) + spare, kv_heads, page, dim)
        normal = lambda *s: torch.randn(s, generator=g)
        self.key_scale = self.value_scale = None
        if cache == E4M3:
            self.key_scale, self.value_scale = (0.01 + 0.02 * torch.rand(kv_heads, generator=g) for _ in range(2))
            self.keys, self.values = (normal(*shape).mul_(60.0).clamp_(-448, 448).to(E4M3) for _ in range(2))
        else:
            self.keys, self.values = normal(*shape).to(cache), normal(*shape).to(cache)
        self.q, self.k, self.v = (normal(self.rows, h, dim).mul_(z).bfloat16() for h, z in ((heads, q_scale), (kv_heads, 1.0), (kv_heads, 1.0)))

    def batch(self):
        return self.pages, self.offsets, self.lengths

    def scales(self):
        return {"key_scale": self.key_scale, "value_scale": self.value_scale}

    def to(self, device):
        for name, t in list(vars(self).items()):
            if isinstance(t, torch.Tensor):
                setattr(self, name, t.to(device))
        return self


def bits(t):
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def attention64(c, scale, window=0, softcap=0.0):
    """(answers, how far bf16 weights, fp32 scores and a bf16 answer may be from them), both [rows, heads, dim] in 64 bits."""
    out, far = torch.zeros((c.rows, c.heads, c.dim), dtype=torch.float64), torch.zeros((c.rows, c.heads, c.dim), dtype=torch.float64)
    half, group = 2.0 ** -8, c.heads // c.kv
    for s, (n, length) in enumerate(zip(c.new, c.length)):
        first = int(c.offsets[s])
        for h in range(c.kv):
            places, ks, vs = [], [], []
            for p in range(max(0, min(length, c.width * c.page))):
                page = int(c.pages[s, p // c.page])
                if 0 <= page < c.keys.shape[0]:
                    places.append(p)
                    ks.append(c.keys[page, h, p % c.page].double())
                    vs.append(c.values[page, h, p % c.page].double())
            if not places or n == 0:
                continue
            at, k, v = torch.tensor(places), torch.stack(ks), torch.stack(vs)
            if c.key_scale is not None:
                k, v = k * c.key_scale[h].double(), v * c.value_scale[h].double()
            for g in range(group):
                q = c.q[first:first + n, h * group + g].double()
                x = (q @ k.T) * scale
                noise = (c.dim + 8) * 2.0 ** -24 * ((q.abs() @ k.abs().T) * scale).nan_to_num(0.0, 0.0, 0.0)
                if softcap:
                    x = softcap * torch.tanh(x / softcap)
                    noise = noise + 16 * 2.0 ** -24 * softcap
                position = torch.arange(length - n, length).unsqueeze(1)
                seen = at <= position
                if window:
                    seen &= at > position - window
                x = x.masked_fill(~seen, -math.inf)
                top = x.amax(-1, keepdim=True)
                w = torch.where(seen, torch.exp(x - torch.where(top == -math.inf, 0.0, top)), torch.zeros_like(x))
                total = w.sum(-1, keepdim=True)
                y = torch.zeros((n, c.dim), dtype=torch.float64)
                size = torch.zeros_like(y)
                for j in range(n):
                    if not seen[j].any():
                        continue
                    y[j] = (w[j][seen[j]].unsqueeze(1) * v[seen[j]]).sum(0) / total[j]
                    size[j] = (w[j][seen[j]].unsqueeze(1) * v[seen[j]].abs()).sum(0) / total[j]
                # weights off by half a step of bf16 and by their scores' noise, sums by 2^-24 a term, the answer by half a step
                loose = half + 2.0 * noise.masked_fill(~seen, 0.0).amax(-1, keepdim=True) + len(places) * 2.0 ** -23
                out[first:first + n, h * group + g] = y
                far[first:first + n, h * group + g] = 1.01 * (loose * (size + y.abs()) + half * y.abs()) + 1e-30
    return out, far


def assert_near(got, want, far, what=""):
    got = got.double().cpu()
    assert got.shape == want.shape
    assert torch.equal(got.isnan(), want.isnan()), what
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf]) and not got[~inf & ~want.isnan()].isinf().any(), what
    ok = ((got - want).abs() <= far) | ~want.isfinite()
    assert ok.all(), (what, (~ok).nonzero()[:4].tolist(), got[~ok][:4].tolist(), want[~ok][:4].tolist(), far[~ok][:4].tolist())


def angles(positions, half, theta=10000.0):
    a = torch.outer(torch.arange(positions, dtype=torch.float64), theta ** (-torch.arange(half, dtype=torch.float64) / max(half, 1)))
    return a.cos().float(), a.sin().float()


def append32(c, cos=None, sin=None, interleaved=True, q_weight=None, k_weight=None, eps=1e-6):
    """(queries, keys, values) with every step rounded to fp32 in the order that is promised, one token after the other."""
    q_out = torch.zeros_like(c.q)
    keys, values = c.keys.clone(), c.values.clone()

    def turned(x, weight, p):
        x = x.float()
        if weight is not None:
            x = x * (1.0 / ((x.double() ** 2).mean(-1, keepdim=True) + eps).sqrt()).float()
            x = x * weight
        if cos is None:
            return x
        y, half = x.clone(), cos.shape[1]
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, half + i)
            y[:, a] = x[:, a] * cos[p, i] - x[:, b] * sin[p, i]
            y[:, b] = x[:, a] * sin[p, i] + x[:, b] * cos[p, i]
        return y

    for s, (n, length) in enumerate(zip(c.new, c.length)):
        for j in range(n):
            r, p = int(c.offsets[s]) + j, length - n + j
            if not 0 <= p < c.width * c.page:
                continue
            q_out[r] = turned(c.q[r], q_weight, p).bfloat16()
            page = int(c.pages[s, p // c.page])
            if not 0 <= page < keys.shape[0]:
                continue
            for cache, x, scale in ((keys, turned(c.k[r], k_weight, p), c.key_scale), (values, c.v[r].float(), c.value_scale)):
                if scale is not None:
                    x = (x / scale.unsqueeze(1)).clamp(-448.0, 448.0)
                bits(cache)[page, :, p % c.page] = bits(x.to(cache.dtype))
    return q_out, keys, values
