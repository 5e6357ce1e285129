"""Linear layer with bias, activation and residual in the matrix product's epilogue.

    y = act(x W^T + b) + residual

``linear_act`` is the function, ``FusedLinear`` the module: an ``nn.Linear`` (so
that AutoPatcher and MHCRewire take it as one) whose forward is one kernel, and
whose backward is the input's, the weight's and the bias's gradients on the
tensor cores.  bf16 and fp16; outside torch.autocast fp32 operands are refused,
since the tensor cores would round them to fewer bits.
"""

from __future__ import annotations

import torch
from torch import nn

from . import _capi as C

ACTIVATIONS = ("none", "relu", "silu", "gelu")  # gelu: with the error function
_HALF = (torch.float16, torch.bfloat16)


def _check(x, weight, bias, residual, activation) -> int:
    """The activation's code."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    if x.dtype not in _HALF:
        raise ValueError(f"unsupported dtype {x.dtype}; expected float16 or bfloat16")
    if weight.ndim != 2 or 0 in weight.shape:
        raise ValueError(f"weight must be [out, in], got shape {tuple(weight.shape)}")
    if x.ndim < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x must be [..., {weight.shape[1]}], got shape {tuple(x.shape)}")
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None and t.dtype != x.dtype:
            raise ValueError(f"{name} must be {x.dtype} as x is, got {t.dtype}")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"bias must be [{weight.shape[0]}], got shape {tuple(bias.shape)}")
    want = (*x.shape[:-1], weight.shape[0])
    if residual is not None and tuple(residual.shape) != want:
        raise ValueError(f"residual must have the output's shape {want}, got "
                         f"{tuple(residual.shape)}")
    return ACTIVATIONS.index(activation)


def _autocast(*ts):
    """The operands in the type that torch.autocast has set, as nn.Linear casts its own."""
    to = torch.get_autocast_dtype("cuda")
    cast = lambda t: t.is_cuda and t.is_floating_point() and t.dtype != torch.float64  # noqa: E731
    return (t.to(to) if t is not None and cast(t) else t for t in ts)


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
               residual: torch.Tensor | None = None, activation: str = "none") -> torch.Tensor:
    """act(x W^T + bias) + residual.

    x [..., in], weight [out, in], bias [out], residual [..., out], all bf16 or
    all fp16; activation "none", "relu", "silu" or "gelu".  Products and sums are
    fp32, rounded once to y.  The gradients are rounded once to their tensors'
    type; with an activation the pre-activation's gradient, an operand of the
    products on the tensor cores, is rounded to the type too.  The pre-activation
    is kept for the backward in fp32.  Under torch.autocast the operands are cast
    to its type."""
    if torch.is_autocast_enabled("cuda"):
        x, weight, bias, residual = _autocast(x, weight, bias, residual)
    act = _check(x, weight, bias, residual, activation)
    return C.host().linear(x, weight, bias, residual, act)


class FusedLinear(nn.Linear):
    """nn.Linear with an activation, and optionally a residual, in the same kernel.
    MHCRewire calls it with one argument: wrapped, it has no residual."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True,
                 activation: str = "none", device=None, dtype=torch.bfloat16):
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}, got "
                             f"{activation!r}")
        super().__init__(in_features, out_features, bias=bias, device=device, dtype=dtype)
        self.activation = activation

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        return linear_act(x, self.weight, self.bias, residual=residual,
                          activation=self.activation)

    def extra_repr(self) -> str:
        return f"{super().extra_repr()}, activation={self.activation}"
