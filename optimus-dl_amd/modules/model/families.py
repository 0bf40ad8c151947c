"""Llama / Qwen3 / GPT-2 shaped models (``transformer.{wte,h,ln_f}`` + ``lm_head``
as in optimus_dl/modules/model/{llama2,qwen3,gpt2}.py), random-initialised with
the reference's standard deviations (gpt2.py:167-180: 0.02, and 0.02/sqrt(2*n_layer)
for the residual projections ``c_proj`` / ``wo``).  Not in the reference: norms behind the blocks, gates and a scaled stream
(``post_norms``, ``layer_scale``, ``residual_scale``), and ``score``, the log probabilities that a model gives to tokens."""

from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn

from ..logprobs import TokenLogProbs, token_logprobs
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

    def embed(self, input_ids: torch.Tensor) -> torch.Tensor:
        return self.transformer.wte(input_ids)

    def forward(self, input_ids: torch.Tensor, **kwargs) -> dict:
        x, z = self.embed(input_ids), None
        blocks, ln_f = self.transformer.h, self.transformer.ln_f
        stepped = [isinstance(block, LlamaBlock) and block.takes_steps() for block in blocks]      # (a wrapper around a block has the stream alone)
        for i, block in enumerate(blocks):
            if not stepped[i]:
                x, z = block(x), None
            elif i + 1 == len(blocks) or stepped[i + 1]:                      # the end of a block and the norm in front of the next in one
                x, z = block(x, z, ln_f if i + 1 == len(blocks) else blocks[i + 1].ln_1)
            else:
                x, z = block(x, z), None
        return {"logits": self.lm_head(ln_f(x) if z is None else z)}

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

    def embed(self, input_ids: torch.Tensor) -> torch.Tensor:
        pos = torch.arange(input_ids.shape[1], device=input_ids.device)
        return self.transformer.wte(input_ids) + self.transformer.wpe(pos)
