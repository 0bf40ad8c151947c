"""Model transform that puts :class:`FP4Linear` in the place of ``nn.Linear``, for inference.

Registered as ``"fp4_linear"``.  Like ``"fp8_linear"`` it replaces exact ``torch.nn.Linear`` modules in place and leaves subclasses alone, so the two can be
listed one behind the other: ``[{_name: fp4_linear}, {_name: fp8_linear}]`` gives the Linears of the blocks 4-bit weights and the head, which is
skipped here by default, FP8.  The reference has no counterpart.
"""

from __future__ import annotations

import logging
from dataclasses import dataclass
from typing import Any

import torch.nn as nn

from ..calls import has_hooks
from ..fp4_linear import FP4Linear, check_castable
from . import register_model_transform
from .base import BaseModelTransform
from .config import ModelTransformConfig

logger = logging.getLogger(__name__)


@dataclass
class Fp4LinearTransformConfig(ModelTransformConfig):
    enabled: bool = True
    group_size: int = 32
    skip: tuple = ("lm_head",)          # names of children to leave as they are (a head that is tied to an embedding, say)


@register_model_transform("fp4_linear", Fp4LinearTransformConfig)
class Fp4LinearTransform(BaseModelTransform):
    """nn.Linear -> FP4Linear over the whole module tree; Linears whose inputs are no whole groups, and Linears with hooks (which may look at
    the weight, or make it), stay as they are."""

    def apply(self, model: nn.Module, **kwargs: Any) -> nn.Module:
        self.replaced, self.left = 0, []
        if not self.cfg.enabled:
            return model
        if type(model) is nn.Linear:
            raise ValueError("the fp4_linear transform replaces the Linears inside of a model; this is one: FP4Linear.from_linear")
        places: list[tuple[nn.Module, str, nn.Linear]] = []
        for prefix, parent in list(model.named_modules()):
            for name, child in parent._modules.items():
                if type(child) is not nn.Linear or name in self.cfg.skip:
                    continue
                if child.in_features % self.cfg.group_size or has_hooks(child):
                    self.left.append(f"{prefix}.{name}" if prefix else name)
                    continue
                places.append((parent, name, child))
        for child in {id(child): child for *_, child in places}.values():      # a model is refused before anything of it is replaced
            check_castable(child.weight, self.cfg.group_size)
        made: dict[int, FP4Linear] = {}                 # a module that is used in two places stays one
        for parent, name, child in places:
            if id(child) not in made:
                made[id(child)] = FP4Linear.from_linear(child, self.cfg.group_size)
                self.replaced += 1
            setattr(parent, name, made[id(child)])
        logger.info("Linears with 4-bit weights: %d%s", self.replaced, f"; left as they are: {', '.join(self.left)}" if self.left else "")
        return model
