"""Layer norm with the residual sum in front of it, backed by the gfx950
kernels in ops/csrc/norm_hip.hip.

The counterpart of fused_bn.py for networks that normalise over features:
``s = x + residual`` and ``y = layer_norm(s)`` are one pass over memory
forward, and one pass (plus the sum of the blocks' shares of the weight's and
the bias's gradients) backward.  Runs in float32, bfloat16 and float16 with
32-bit sums; on CPU the eager composition of the same formulas runs.

On the GPU the kernels are the only path: a type or shape that they do not
take raises, and a missing HIP extension raises.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import ops

__all__ = ["fused_layer_norm", "FusedLayerNorm"]

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check(x, weight, bias, residual):
    """The extension's checks, for the CPU path."""
    if x.dtype not in _TYPES:
        raise TypeError("layer norm's input must be float32, bfloat16 or "
                        f"float16, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("layer norm needs a last axis of one element or more")
    for name, v in (("weight", weight), ("bias", bias)):
        if v is None:
            continue
        if v.device != x.device:
            raise ValueError(f"{name} is on {v.device}, the input on "
                             f"{x.device}")
        if v.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{name} must be {x.dtype} like the input, or "
                            f"float32, got {v.dtype}")
        if v.shape != x.shape[-1:]:
            raise ValueError(f"{name} has shape {tuple(v.shape)}, wanted "
                             f"[{x.shape[-1]}]")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have one type")
    if residual is not None:
        if residual.device != x.device or residual.shape != x.shape:
            raise ValueError("residual must be on the input's device and "
                             "have its shape")
        if residual.dtype != x.dtype:
            raise TypeError(f"residual is {residual.dtype}, the input "
                            f"{x.dtype}")


class _Stored(torch.autograd.Function):
    """A float32 sum as the type it is stored in holds it; gradients go
    through in float32, so that those of both uses are added before they are
    rounded, as in the kernel."""

    @staticmethod
    def forward(ctx, s, dtype):
        return s.to(dtype).float()

    @staticmethod
    def backward(ctx, g):
        return g, None


def _eager(x, weight, bias, eps, residual):
    _check(x, weight, bias, residual)
    s = x.float()
    if residual is not None:
        s = _Stored.apply(s + residual.float(), x.dtype)
    y = F.layer_norm(s, s.shape[-1:],
                     None if weight is None else weight.float(),
                     None if bias is None else bias.float(), eps).to(x.dtype)
    return y if residual is None else (y, s.to(x.dtype))


def fused_layer_norm(x, weight=None, bias=None, eps=1e-5, residual=None):
    """Layer norm over the last axis of ``x`` (any number of axes in front).

    Without ``residual`` returns ``y = (x - mean) / sqrt(var + eps) * weight +
    bias``.  With ``residual`` (``x``'s shape and type) returns ``(y, s)``
    with ``s = x + residual`` in ``x``'s type and ``y`` the norm of that
    ``s``: the two tensors that a pre-norm block goes on with.  Both carry
    gradients.

    ``weight`` and ``bias`` are vectors of ``x``'s type or float32 and may be
    left out; their gradients come in their own type.  Rows of ``x`` may be
    apart by any stride (a slice of a wider tensor is read in place); results
    are contiguous.  Raises TypeError and ValueError for types and shapes that
    do not fit, and on the GPU for 2^31 rows or more, or 2^22 of over 16384
    elements.

    On the GPU gradients are of first order: a graph of them
    (``create_graph=True``) and forward-mode tangents raise RuntimeError.  On
    CPU torch's own operations run, where both work, but for tangents beside a
    ``residual``.
    """
    if not x.is_cuda:
        return _eager(x, weight, bias, eps, residual)
    out = ops.hip_ext().layer_norm(x, weight, bias, eps, residual)
    return out[0] if residual is None else tuple(out)


class FusedLayerNorm(nn.Module):
    """``nn.LayerNorm`` over one axis (same parameter names) whose forward
    takes the residual too: ``norm(x)`` gives ``y``, ``norm(x, residual)``
    gives ``(y, x + residual)``."""

    def __init__(self, num_features, eps=1e-5, affine=True, bias=True):
        super().__init__()
        self.num_features = num_features
        self.eps = eps
        if affine:
            self.weight = nn.Parameter(torch.ones(num_features))
        else:
            self.register_parameter("weight", None)
        if affine and bias:
            self.bias = nn.Parameter(torch.zeros(num_features))
        else:
            self.register_parameter("bias", None)

    def forward(self, x, residual=None):
        if x.shape[-1] != self.num_features:
            raise ValueError(f"the input has {x.shape[-1]} features, wanted "
                             f"{self.num_features}")
        return fused_layer_norm(x, self.weight, self.bias, self.eps, residual)

    def extra_repr(self):
        return (f"{self.num_features}, eps={self.eps}, "
                f"affine={self.weight is not None}, "
                f"bias={self.bias is not None}")
