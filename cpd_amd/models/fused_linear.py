"""Linear layer with bias, activation and residual in the product's epilogue,
backed by the gfx950 kernels in ops/csrc/linear_hip.hip.

The full-speed neighbour of quant/module.py's Quant_Linear: that one rounds
every step of its accumulator to an (exp, man) grid, this one accumulates in
32 bits on the matrix cores and rounds once, after the epilogue.  On CPU the
eager composition of the same formulas runs; on the GPU the kernels are the
only path.
"""
import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import ops

__all__ = ["fused_linear", "FusedLinear"]

_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_ACTS = {None: 0, "relu": 1, "gelu": 2, "silu": 3}


def _check(x, weight, bias, residual):
    """The extension's checks, for the CPU path."""
    if x.dtype not in _TYPES:
        raise TypeError("linear's input must be float32, bfloat16 or "
                        f"float16, got {x.dtype}")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear's input has shape {tuple(x.shape)}, its "
                         f"weight {tuple(weight.shape)}")
    if weight.shape[1] < 1:
        raise ValueError("linear needs one input feature or more")
    for name, v in (("weight", weight), ("bias", bias),
                    ("residual", residual)):
        if v is None:
            continue
        if v.device != x.device:
            raise ValueError(f"{name} is on {v.device}, the input on "
                             f"{x.device}")
        if v.dtype != x.dtype and not (name == "bias"
                                       and v.dtype == torch.float32):
            raise TypeError(f"{name} is {v.dtype}, the input {x.dtype}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise ValueError(f"bias has shape {tuple(bias.shape)}, wanted "
                         f"[{weight.shape[0]}]")
    if residual is not None and \
            residual.shape != x.shape[:-1] + weight.shape[:1]:
        raise ValueError(f"residual has shape {tuple(residual.shape)}, wanted "
                         f"{tuple(x.shape[:-1] + weight.shape[:1])}")


def _eager(x, weight, bias, act, residual):
    _check(x, weight, bias, residual)
    y = F.linear(x.float(), weight.float(),
                 None if bias is None else bias.float())
    y = {0: lambda v: v, 1: F.relu, 2: F.gelu, 3: F.silu}[act](y)
    if residual is not None:
        y = y + residual.float()
    return y.to(x.dtype)


def fused_linear(x, weight, bias=None, activation=None, residual=None):
    """``act(x @ weight.T + bias) + residual`` in one product.

    ``x`` is [..., K], ``weight`` [N, K] and ``residual`` [..., N], all of one
    type (float32, bfloat16 or float16); ``bias`` [N] is of that type or
    float32.  ``activation`` is None, "relu", "gelu" (x times the normal
    distribution's cdf) or "silu".  Sums are 32-bit; the result is rounded
    once.  For the backward pass an activation's argument is kept in ``x``'s
    type; where the products behind gelu and silu are large (over 2^28
    multiplications, or 2^24 weights) and 16-bit, the gradient behind the
    activation is rounded to that type too.  Of float32 operands (the inputs
    and, backward, the incoming gradient) the GPU may leave out what lies below
    2^-133, depending on the sizes.

    Rows may be apart by any stride; the result is contiguous.  Raises
    TypeError and ValueError for types and shapes that do not fit, and on the
    GPU for 2^22 features or more and 2^22 blocks of 128 by 128 or more in
    ``x``, ``weight`` or the result.

    On the GPU gradients are of first order: a graph of them
    (``create_graph=True``) and forward-mode tangents raise RuntimeError.  On
    CPU torch's own operations run, where both work.
    """
    if activation not in _ACTS:
        raise ValueError(f"unknown activation {activation!r}: None, 'relu', "
                         "'gelu' or 'silu'")
    act = _ACTS[activation]
    if not x.is_cuda:
        return _eager(x, weight, bias, act, residual)
    return ops.hip_ext().linear(x, weight, bias, act, residual)


class FusedLinear(nn.Module):
    """``nn.Linear`` (same parameter names and start values) with an
    activation; ``forward(x, residual=None)`` adds the residual behind it.

    ``quantize_model_gemms`` leaves this module as it is: it replaces
    ``nn.Linear``, whose accumulator is what it is about."""

    def __init__(self, in_features, out_features, bias=True, activation=None):
        super().__init__()
        if activation not in _ACTS:
            raise ValueError(f"unknown activation {activation!r}: None, "
                             "'relu', 'gelu' or 'silu'")
        self.in_features = in_features
        self.out_features = out_features
        self.activation = activation
        self.weight = nn.Parameter(torch.empty(out_features, in_features))
        if bias:
            self.bias = nn.Parameter(torch.empty(out_features))
        else:
            self.register_parameter("bias", None)
        self.reset_parameters()

    def reset_parameters(self):
        nn.init.kaiming_uniform_(self.weight, a=math.sqrt(5))
        if self.bias is not None:
            bound = 1.0 / math.sqrt(self.in_features)
            nn.init.uniform_(self.bias, -bound, bound)

    def forward(self, x, residual=None):
        return fused_linear(x, self.weight, self.bias, self.activation,
                            residual)

    def extra_repr(self):
        return (f"in_features={self.in_features}, "
                f"out_features={self.out_features}, "
                f"bias={self.bias is not None}, "
                f"activation={self.activation}")
