"""Transformer blocks whose ``nn.Linear`` members carry the names the reference
uses (optimus_dl/modules/model/blocks/attention.py:120-123 ``wq wk wv wo``;
blocks/mlp.py:47-49 ``w1 w2 c_proj``; :101-102,142-144 ``c_fc c_proj``).  Only
what the FP8 Linear path needs is here: plain PyTorch attention (SDPA), RoPE,
RMSNorm / LayerNorm.  These are the callers either side of the Linear, not a
re-implementation of the reference's model zoo."""

from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F

from ..calls import called_as_it_is
from ..fused import plain_class, residual_norm
from ..paged import PagedLayer, append_kv, paged_attention


class RMSNorm(nn.Module):
    def __init__(self, dim: int, eps: float = 1e-5):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        xf = x.float()
        y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + self.eps)
        return (y * self.weight.float()).to(x.dtype)


def _is_its_weight(norm: nn.Module) -> bool:
    """Whether a call of the norm is the norm of its weight and nothing else, which a kernel may do in its place."""
    cls = plain_class(norm)
    return issubclass(cls, RMSNorm) and cls.forward is RMSNorm.forward and called_as_it_is(norm)


def rope_tables(head_dim: int, seq_len: int, theta: float, device) -> tuple[torch.Tensor, torch.Tensor]:
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, device=device, dtype=torch.float32) / head_dim))
    ang = torch.outer(torch.arange(seq_len, device=device, dtype=torch.float32), inv)
    return ang.cos(), ang.sin()


def apply_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    # x: [B, H, T, D]; rotate pairs (even, odd)
    xf = x.float()
    x1, x2 = xf[..., 0::2], xf[..., 1::2]
    c, s = cos[None, None], sin[None, None]
    out = torch.stack((x1 * c - x2 * s, x1 * s + x2 * c), dim=-1).flatten(-2)
    return out.to(x.dtype)


class CausalSelfAttention(nn.Module):
    def __init__(self, n_embd: int, n_head: int, n_kv_head: int | None = None, head_dim: int | None = None,
                 bias: bool = False, use_qk_norm: bool = False, rope: bool = True, rope_theta: float = 10000.0,
                 rmsnorm_eps: float = 1e-5):
        super().__init__()
        assert n_embd % n_head == 0
        self.n_head = n_head
        self.n_kv_head = n_kv_head or n_head
        self.head_dim = head_dim or n_embd // n_head
        self.rope, self.rope_theta = rope, rope_theta
        self.wq = nn.Linear(n_embd, n_head * self.head_dim, bias=bias)
        self.wk = nn.Linear(n_embd, self.n_kv_head * self.head_dim, bias=bias)
        self.wv = nn.Linear(n_embd, self.n_kv_head * self.head_dim, bias=bias)
        self.wo = nn.Linear(n_head * self.head_dim, n_embd, bias=bias)
        self.use_qk_norm = use_qk_norm
        if use_qk_norm:
            self.q_norm = RMSNorm(self.head_dim, eps=rmsnorm_eps)
            self.k_norm = RMSNorm(self.head_dim, eps=rmsnorm_eps)

    def step(self, x: torch.Tensor, layer: PagedLayer) -> torch.Tensor:
        """New tokens [rows, n_embd] of the sequences of a batch, over a cache of those in front of them that they are put into."""
        q, k, v = (w(x).unflatten(-1, (-1, self.head_dim)) for w in (self.wq, self.wk, self.wv))
        norms = {}
        if self.use_qk_norm:
            if _is_its_weight(self.q_norm) and _is_its_weight(self.k_norm) and self.q_norm.eps == self.k_norm.eps:
                norms = {"q_weight": self.q_norm.weight, "k_weight": self.k_norm.weight, "eps": self.q_norm.eps}
            else:
                q, k = self.q_norm(q), self.k_norm(k)
        dtype = q.dtype
        if x.is_cuda:                                  # (what the kernels and the cache hold)
            q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
        cos, sin = layer.cache.angles(rope_tables, self.head_dim, self.rope_theta) if self.rope else (None, None)
        pages, offsets, lengths, max_new = layer.batch
        scales = {"key_scale": layer.key_scale, "value_scale": layer.value_scale}
        q = append_kv(q, k, v, layer.keys, layer.values, pages, offsets, lengths, cos=cos, sin=sin, **norms, **scales)
        y = paged_attention(q, layer.keys, layer.values, pages, offsets, lengths, max_new=max_new, **scales)
        return self.wo(y.to(dtype).flatten(1))

    def forward(self, x: torch.Tensor, layer: PagedLayer | None = None) -> torch.Tensor:
        if layer is not None:
            return self.step(x, layer)
        B, T_, _ = x.shape
        q = self.wq(x).view(B, T_, self.n_head, self.head_dim).transpose(1, 2)
        k = self.wk(x).view(B, T_, self.n_kv_head, self.head_dim).transpose(1, 2)
        v = self.wv(x).view(B, T_, self.n_kv_head, self.head_dim).transpose(1, 2)
        if self.use_qk_norm:
            q, k = self.q_norm(q), self.k_norm(k)
        if self.rope:
            cos, sin = rope_tables(self.head_dim, T_, self.rope_theta, x.device)
            q, k = apply_rope(q, cos, sin), apply_rope(k, cos, sin)
        if self.n_kv_head != self.n_head:
            rep = self.n_head // self.n_kv_head
            k, v = k.repeat_interleave(rep, dim=1), v.repeat_interleave(rep, dim=1)
        y = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        return self.wo(y.transpose(1, 2).reshape(B, T_, self.n_head * self.head_dim))


class SwiGLUMLP(nn.Module):
    def __init__(self, n_embd: int, intermediate_size: int | None = None, multiple_of: int = 256, bias: bool = False):
        super().__init__()
        if intermediate_size is None:
            hidden = int(2 * (4 * n_embd) / 3)
            hidden = multiple_of * ((hidden + multiple_of - 1) // multiple_of)
        else:
            hidden = intermediate_size
        self.w1 = nn.Linear(n_embd, hidden, bias=bias)
        self.w2 = nn.Linear(n_embd, hidden, bias=bias)
        self.c_proj = nn.Linear(hidden, n_embd, bias=bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.c_proj(F.silu(self.w1(x)) * self.w2(x))


class GELUMLP(nn.Module):
    def __init__(self, n_embd: int, intermediate_size: int | None = None, bias: bool = True):
        super().__init__()
        hidden = intermediate_size or 4 * n_embd
        self.c_fc = nn.Linear(n_embd, hidden, bias=bias)
        self.gelu = nn.GELU()
        self.c_proj = nn.Linear(hidden, n_embd, bias=bias)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.c_proj(self.gelu(self.c_fc(x)))


class LlamaBlock(nn.Module):
    """Pre-norm block: x + attn(ln_1(x)); x + mlp(ln_2(x)).

    post_norms, layer_scale, residual_scale (not in the reference): a norm behind each half (``post_ln_1``, ``post_ln_2``), a learned gate for each
    channel of it that begins at ``layer_scale`` (``gate_1``, ``gate_2``) and a factor on the stream that it is added to.  With any of them a
    half ends in ``residual_norm``, one kernel that also is the norm in front of the next half: a model hands the block what the step before
    made of ``ln_1`` (``z``) and the norm that comes behind it (``next_norm``), and gets the stream and that norm of it.  Norms that are more than their
    weight (hooks, another class) are called."""

    def __init__(self, n_embd: int, n_head: int, n_kv_head: int | None, intermediate_size: int | None,
                 use_qk_norm: bool = False, head_dim: int | None = None, eps: float = 1e-5, rope_theta: float = 10000.0,
                 post_norms: bool = False, layer_scale: float | None = None, residual_scale: float = 1.0):
        super().__init__()
        self.ln_1 = RMSNorm(n_embd, eps)
        self.attn = CausalSelfAttention(n_embd, n_head, n_kv_head, head_dim, bias=False, use_qk_norm=use_qk_norm,
                                        rope_theta=rope_theta, rmsnorm_eps=eps)
        self.ln_2 = RMSNorm(n_embd, eps)
        self.mlp = SwiGLUMLP(n_embd, intermediate_size)
        self.residual_scale = residual_scale
        self.stepped = post_norms or layer_scale is not None or residual_scale != 1.0
        self.post_ln_1, self.post_ln_2 = (RMSNorm(n_embd, eps) if post_norms else None for _ in range(2))
        self.gate_1, self.gate_2 = (None if layer_scale is None else nn.Parameter(torch.full((n_embd,), float(layer_scale))) for _ in range(2))

    def takes_steps(self) -> bool:
        """Whether what is in front of the block and behind it may hand each other norms of the stream.  Hooks of a block, and whatever stands in its
        place, have the stream alone: what shards a block's weights while it does not run, say."""
        return self.stepped and type(self).forward is LlamaBlock.forward and called_as_it_is(self)

    def _end(self, x: torch.Tensor, h: torch.Tensor, post: "RMSNorm | None", gate: torch.Tensor | None, norm: RMSNorm | None):
        """The stream behind a half that answered h, and the norm in front of the next half of it."""
        if norm is not None and _is_its_weight(norm) and (post is None or _is_its_weight(post)):
            return residual_norm(x, h, norm.weight, norm.eps, post_weight=None if post is None else post.weight,
                                 post_eps=None if post is None else post.eps, gate=gate, residual_scale=self.residual_scale)
        h = (h if post is None else post(h)).to(x.dtype)
        x = self.residual_scale * x + (h if gate is None else (gate * h).to(x.dtype))
        return x, None if norm is None else norm(x)

    def forward(self, x: torch.Tensor, z: torch.Tensor | None = None, next_norm: RMSNorm | None = None, layer: PagedLayer | None = None):
        over = () if layer is None else (layer,)
        if not self.stepped:
            x = x + self.attn(self.ln_1(x), *over)
            return x + self.mlp(self.ln_2(x))
        x, z = self._end(x, self.attn(self.ln_1(x) if z is None else z, *over), self.post_ln_1, self.gate_1, self.ln_2)
        x, z = self._end(x, self.mlp(z), self.post_ln_2, self.gate_2, next_norm)
        return x if next_norm is None else (x, z)


class Qwen3Block(LlamaBlock):
    def __init__(self, n_embd: int, n_head: int, n_kv_head: int | None, intermediate_size: int | None,
                 head_dim: int | None = None, eps: float = 1e-6, rope_theta: float = 1e6, **step):
        super().__init__(n_embd, n_head, n_kv_head, intermediate_size, use_qk_norm=True, head_dim=head_dim, eps=eps,
                         rope_theta=rope_theta, **step)


class GPT2Block(nn.Module):
    def __init__(self, n_embd: int, n_head: int, bias: bool = True):
        super().__init__()
        self.ln_1 = nn.LayerNorm(n_embd, bias=bias)
        self.attn = CausalSelfAttention(n_embd, n_head, bias=bias, rope=False)
        self.ln_2 = nn.LayerNorm(n_embd, bias=bias)
        self.mlp = GELUMLP(n_embd, bias=bias)

    def forward(self, x: torch.Tensor, layer: PagedLayer | None = None) -> torch.Tensor:
        x = x + self.attn(self.ln_1(x), *(() if layer is None else (layer,)))
        return x + self.mlp(self.ln_2(x))
