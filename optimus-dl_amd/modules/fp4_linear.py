"""Linears whose weights are held in 4 bits, for decode steps.

A decode step of a few tokens reads weights and does little else.  :class:`FP8Linear` reads a byte a weight; here a weight is an OCP E2M1 code
(0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives), two a byte, with a bf16 scale for each group of 32, 64 or 128 along the input: 0.56 to 0.52
bytes.  Activations stay bf16 and sums are fp32, so what is lost is lost when the weights are cast, once.  The layout is that
of a checkpoint and is multiplied as it is: codes ``[out, in / 2]``, the even input in the low nibble, scales ``[out, in / group]``.
The reference has no counterpart.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from .. import native
from .calls import untraced, untransformed

GROUPS = native.FP4_GROUPS
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _check_weight(codes: torch.Tensor, scales: torch.Tensor) -> int:
    """-> the group."""
    if codes.dtype != torch.uint8 or scales.dtype != torch.bfloat16 or codes.dim() != 2 or scales.dim() != 2 or codes.shape[0] != scales.shape[0]:
        raise ValueError(f"fp4 weights: codes {codes.dtype} {tuple(codes.shape)} and scales {scales.dtype} {tuple(scales.shape)}, expected uint8 "
                         "[out, in / 2] and bf16 [out, in / group]")
    for group in GROUPS:
        if scales.shape[1] > 0 and scales.shape[1] * group == 2 * codes.shape[1]:
            return group
    raise ValueError(f"fp4 weights: {2 * codes.shape[1]} inputs in {scales.shape[1]} groups (of 32, 64 or 128)")


def quantise_fp4(weight: torch.Tensor, group: int = 32) -> tuple[torch.Tensor, torch.Tensor]:
    """Weights [out, in], bf16 or fp32, finite, as codes and scales: a group's scale is the bf16 nearest to its largest magnitude / 6, a code the
    E2M1 nearest to weight / scale, ties to the even code.  On the GPU.  -> (codes uint8 [out, in / 2], scales bf16 [out, in / group])."""
    check_castable(weight, group)
    return native.fp4_quantise(weight.detach(), group)


def check_castable(weight: torch.Tensor, group: int) -> None:
    """Refuses what :func:`quantise_fp4` refuses."""
    w = weight.detach()
    native.fp4_quantise(w[:0], group)                          # its device, type and shape: none of its rows are as all of them
    if not bool(torch.isfinite(w).all()):
        raise ValueError("quantise_fp4: the weights are not finite")


def dequantise_fp4(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The weights that codes and scales stand for, exactly.  -> fp32 [out, in]."""
    group = _check_weight(codes, scales)
    nibbles = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(1)
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float32, device=codes.device)
    return (table[nibbles.long()].unflatten(1, (-1, group)) * scales.float().unsqueeze(-1)).flatten(1)


class _Fp4LinearFn(torch.autograd.Function):
    """The product where something else than a backward looks at it: a tracer records it, what would differentiate or batch it is refused."""

    @staticmethod
    def forward(ctx, x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, bias: torch.Tensor | None) -> torch.Tensor:
        return native.fp4_linear(x, codes, scales, bias)


@untraced
def fp4_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ weight.T + bias`` for x [..., in] in bf16 and weights as :func:`quantise_fp4` makes them; bias bf16 or fp32 [out] or None.  Accumulated in
    fp32, rounded once.  -> bf16 [..., out].

    Made for up to some hundred rows: the weights are read again for every 16 to 128 of them.  For inference: an input that wants a gradient is refused."""
    if torch.is_grad_enabled() and (x.requires_grad or (bias is not None and bias.requires_grad)):
        raise RuntimeError("fp4_linear has no backward: call it under torch.no_grad()")
    _check_weight(codes, scales)
    if x.dim() == 0 or x.dtype != torch.bfloat16 or x.shape[-1] != 2 * codes.shape[1]:
        raise ValueError(f"fp4_linear: x is {x.dtype} {tuple(x.shape)}, expected bf16 [..., {2 * codes.shape[1]}]")
    if bias is not None and bias.shape != codes.shape[:1]:
        raise ValueError(f"fp4_linear: a bias {tuple(bias.shape)} for {codes.shape[0]} outputs")
    if not x.is_cuda:
        y = x.float() @ dequantise_fp4(codes, scales).t()
        return (y if bias is None else y + bias.float()).bfloat16()
    product = native.fp4_linear if untransformed() else _Fp4LinearFn.apply
    y = product(x if x.dim() == 2 else x.reshape(-1, x.shape[-1]), codes, scales, bias)
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], y.shape[1])


class FP4Linear(nn.Module):
    """``nn.Linear`` with weights in 4 bits, for inference.  Its state is ``codes`` (uint8), ``scale_bits`` (the scales' bf16 patterns as int16, so that a
    cast of the whole model leaves them alone) and the bias.  Computes in bf16: other inputs are converted, and outside of autocast
    the result goes back to their type."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, group_size: int = 32, device=None):
        super().__init__()
        if group_size not in GROUPS or in_features < 1 or in_features % group_size:
            raise ValueError(f"FP4Linear: {in_features} inputs in groups of {group_size} (32, 64 or 128, a divisor of the inputs)")
        self.in_features, self.out_features, self.group_size = in_features, out_features, group_size
        self.register_buffer("codes", torch.zeros((out_features, in_features // 2), dtype=torch.uint8, device=device))
        self.register_buffer("scale_bits", torch.zeros((out_features, in_features // group_size), dtype=torch.int16, device=device))
        self.bias = nn.Parameter(torch.zeros(out_features, device=device), requires_grad=False) if bias else None

    @property
    def scales(self) -> torch.Tensor:
        if torch.jit.is_tracing():                             # (the tracer has no operator for such a view and dies of it)
            raise RuntimeError("an FP4Linear cannot be traced: trace fp4_linear with its codes and scales")
        return self.scale_bits.view(torch.bfloat16)

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor, bias: torch.Tensor | None = None) -> "FP4Linear":
        group = _check_weight(codes, scales)
        m = cls(2 * codes.shape[1], codes.shape[0], bias=False, group_size=group, device="meta")
        m.codes, m.scale_bits = codes, scales.contiguous().view(torch.int16)
        if bias is not None:
            m.bias = nn.Parameter(bias.detach(), requires_grad=False)
        return m

    @classmethod
    def from_linear(cls, linear: nn.Linear, group_size: int = 32) -> "FP4Linear":
        """The weights are cast once; the bias is shared."""
        m = cls.from_codes(*quantise_fp4(linear.weight, group_size), linear.bias)
        return m.train(linear.training)

    def dequantised_weight(self) -> torch.Tensor:
        return dequantise_fp4(self.codes, self.scales)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        y = fp4_linear(x if x.dtype == torch.bfloat16 else x.to(torch.bfloat16), self.codes, self.scales, self.bias)
        return y if x.dtype == torch.bfloat16 or torch.is_autocast_enabled(x.device.type) else y.to(x.dtype)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, group_size={self.group_size}"
