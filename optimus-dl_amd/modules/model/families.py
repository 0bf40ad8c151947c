"""Llama / Qwen3 / GPT-2 shaped models (``transformer.{wte,h,ln_f}`` + ``lm_head``
as in optimus_dl/modules/model/{llama2,qwen3,gpt2}.py), random-initialised with
the reference's standard deviations (gpt2.py:167-180: 0.02, and 0.02/sqrt(2*n_layer)
for the residual projections ``c_proj`` / ``wo``).  Not in the reference: norms behind the blocks, gates and a scaled stream
(``post_norms``, ``layer_scale``, ``residual_scale``), ``score``, the log probabilities that a model gives to tokens, and ``step`` and ``verify_step``, new tokens
over a paged cache of those in front of them."""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn

from ..drafts import VerifiedDrafts, verify_drafts
from ..logprobs import TokenLogProbs, token_logprobs
from ..paged import PagedBatch, PagedKVCache
from .blocks import GPT2Block, LlamaBlock, Qwen3Block, RMSNorm


@dataclass
class LlamaConfig:
    vocab_size: int = 32000
    n_layer: int = 2
    n_head: int = 8
    n_kv_head: int | None = None
    n_embd: int = 512
    intermediate_size: int | None = None
    block_size: int = 2048
    rmsnorm_eps: float = 1e-5
    rope_theta: float = 10000.0
    tie_word_embeddings: bool = False
    post_norms: bool = False                # a norm behind each half of a block as well
    layer_scale: float | None = None        # a learned gate for each channel of a half's output, beginning at this
    residual_scale: float = 1.0             # factor on the residual stream where a half's output is added

    def step(self) -> dict:
        return {"post_norms": self.post_norms, "layer_scale": self.layer_scale, "residual_scale": self.residual_scale}


@dataclass
class Qwen3Config(LlamaConfig):
    head_dim: int | None = None
    rmsnorm_eps: float = 1e-6
    rope_theta: float = 1e6
    tie_word_embeddings: bool = True


@dataclass
class GPT2Config:
    vocab_size: int = 50304
    n_layer: int = 2
    n_head: int = 12
    n_embd: int = 768
    block_size: int = 1024
    bias: bool = True
    tie_word_embeddings: bool = True


def _init_weights(model: nn.Module, n_layer: int) -> None:
    for m in model.modules():
        if isinstance(m, nn.Linear):
            nn.init.normal_(m.weight, mean=0.0, std=0.02)
            if m.bias is not None:
                nn.init.zeros_(m.bias)
        elif isinstance(m, nn.Embedding):
            nn.init.normal_(m.weight, mean=0.0, std=0.02)
    for name, p in model.named_parameters():
        if name.endswith("c_proj.weight") or name.endswith("wo.weight"):
            nn.init.normal_(p, mean=0.0, std=0.02 / math.sqrt(2 * n_layer))


class _DecoderLM(nn.Module):
    def _finish(self, cfg) -> None:
        self.lm_head = nn.Linear(cfg.n_embd, cfg.vocab_size, bias=False)
        if cfg.tie_word_embeddings:
            self.transformer.wte.weight = self.lm_head.weight
        _init_weights(self, cfg.n_layer)

    def embed(self, input_ids: torch.Tensor, batch: PagedBatch | None = None) -> torch.Tensor:
        return self.transformer.wte(input_ids)

    def forward(self, input_ids: torch.Tensor, **kwargs) -> dict:
        return {"logits": self.lm_head(self._hidden(input_ids))}

    def _hidden(self, input_ids: torch.Tensor, cache: PagedKVCache | None = None, batch: PagedBatch | None = None) -> torch.Tensor:
        x, z = self.embed(input_ids) if cache is None else self.embed(input_ids, batch), None
        blocks, ln_f = self.transformer.h, self.transformer.ln_f
        stepped = [isinstance(block, LlamaBlock) and block.takes_steps() for block in blocks]      # (a wrapper around a block has the stream alone)
        for i, block in enumerate(blocks):
            over = {} if cache is None else {"layer": cache.layer(i, batch)}
            if not stepped[i]:
                x, z = block(x, **over), None
            elif i + 1 == len(blocks) or stepped[i + 1]:                      # the end of a block and the norm in front of the next in one
                x, z = block(x, z, ln_f if i + 1 == len(blocks) else blocks[i + 1].ln_1, **over)
            else:
                x, z = block(x, z, **over), None
        return ln_f(x) if z is None else z

    def new_cache(self, pages: int, page_size: int = 64, max_tokens: int | None = None, dtype: torch.dtype | None = None, **scales: float) -> PagedKVCache:
        """An empty cache for :meth:`step`, on the model's device.  Sequences of up to ``max_tokens``, by default the configuration's ``block_size``.
        dtype: bf16 by default (on the CPU the weights' own), or float8_e4m3fn, with ``key_scale`` and ``value_scale``."""
        attn, weight = self.transformer.h[0].attn, self.lm_head.weight
        dtype = (torch.bfloat16 if weight.is_cuda else weight.dtype) if dtype is None else dtype
        return PagedKVCache(len(self.transformer.h), attn.n_kv_head, attn.head_dim, pages=pages, page_size=page_size,
                            max_tokens=self.config.block_size if max_tokens is None else max_tokens, dtype=dtype, device=weight.device, **scales)

    @torch.no_grad()
    def step(self, input_ids: torch.Tensor, cache: PagedKVCache, batch: PagedBatch, last_only: bool = False) -> dict:
        """Logits of new tokens [rows] (the sequences of the batch one behind the other), which are put into the cache: single tokens, drafts,
        chunks of prompts.  ``last_only``: of each sequence's last new token alone (of no particular one where it has none)."""
        places = self.transformer["wpe"].num_embeddings if "wpe" in self.transformer else None
        if places is not None and cache.max_tokens > places:
            raise ValueError(f"a cache for sequences of {cache.max_tokens} tokens, and embeddings of {places} positions")
        if last_only and input_ids.shape[0] == 0:
            raise ValueError("a step without tokens has no last one")
        z = self._hidden(input_ids, cache, batch)
        if last_only:
            z = z[(batch.offsets[1:].long() - 1).clamp(min=0, max=z.shape[0] - 1)]
        return {"logits": self.lm_head(z)}

    @torch.no_grad()
    def verify_step(self, input_ids: torch.Tensor, cache: PagedKVCache, batch: PagedBatch, uniforms: torch.Tensor, draft_logits: torch.Tensor | None = None,
                    temperature: float = 1.0) -> VerifiedDrafts:
        """A step over drafts: of each sequence the last token that is sure and what was drafted behind it.  How many drafts hold, and the token behind
        them (see ``verify_drafts``); ``cache.shorten`` takes the others out again."""
        logits = self.step(input_ids, cache, batch)["logits"]
        return verify_drafts(logits, input_ids, batch.offsets, uniforms, draft_logits=draft_logits, temperature=temperature, n_vocab=self.config.vocab_size)

    def score(self, input_ids: torch.Tensor, targets: torch.Tensor | None = None, top_k: int = 0, temperature: float = 1.0,
              ignore_index: int = -100) -> TokenLogProbs:
        """Log probabilities of ``targets`` [batch, tokens], with entropy and ``top_k`` alternatives of every position.  Without targets each
        position is asked for the token behind it, and the last one is ignored.  ``-score(ids).logprobs.sum() / n`` is the loss of training."""
        if targets is None:
            targets = torch.cat((input_ids[:, 1:], torch.full_like(input_ids[:, :1], ignore_index)), dim=1)
        return token_logprobs(self(input_ids)["logits"], targets, n_vocab=self.config.vocab_size, top_k=top_k, temperature=temperature,
                              ignore_index=ignore_index)


class Llama(_DecoderLM):
    def __init__(self, config: LlamaConfig):
        super().__init__()
        self.config = config
        self.transformer = nn.ModuleDict({
            "wte": nn.Embedding(config.vocab_size, config.n_embd),
            "h": nn.ModuleList([LlamaBlock(config.n_embd, config.n_head, config.n_kv_head, config.intermediate_size,
                                           eps=config.rmsnorm_eps, rope_theta=config.rope_theta, **config.step())
                                for _ in range(config.n_layer)]),
            "ln_f": RMSNorm(config.n_embd, config.rmsnorm_eps),
        })
        self._finish(config)


class Qwen3(_DecoderLM):
    def __init__(self, config: Qwen3Config):
        super().__init__()
        self.config = config
        self.transformer = nn.ModuleDict({
            "wte": nn.Embedding(config.vocab_size, config.n_embd),
            "h": nn.ModuleList([Qwen3Block(config.n_embd, config.n_head, config.n_kv_head, config.intermediate_size,
                                           head_dim=config.head_dim, eps=config.rmsnorm_eps,
                                           rope_theta=config.rope_theta, **config.step()) for _ in range(config.n_layer)]),
            "ln_f": RMSNorm(config.n_embd, config.rmsnorm_eps),
        })
        self._finish(config)


class GPT2(_DecoderLM):
    def __init__(self, config: GPT2Config):
        super().__init__()
        self.config = config
        self.transformer = nn.ModuleDict({
            "wte": nn.Embedding(config.vocab_size, config.n_embd),
            "wpe": nn.Embedding(config.block_size, config.n_embd),
            "h": nn.ModuleList([GPT2Block(config.n_embd, config.n_head, config.bias) for _ in range(config.n_layer)]),
            "ln_f": nn.LayerNorm(config.n_embd, bias=config.bias),
        })
        self._finish(config)

    def embed(self, input_ids: torch.Tensor, batch: PagedBatch | None = None) -> torch.Tensor:
        pos = torch.arange(input_ids.shape[1], device=input_ids.device) if batch is None else batch.positions(input_ids.shape[0]).clamp(max=self.config.block_size - 1)
        return self.transformer.wte(input_ids) + self.transformer.wpe(pos)
