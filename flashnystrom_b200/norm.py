"""Layer norm over the last dimension, whole or in groups, forward and backward as the library's own kernels."""
import torch
import torch.nn as nn
from torch.autograd import forward_ad as _forward_ad

from . import _C


def layer_norm(x, weight=None, bias=None, eps=1e-5, num_groups=1):
    """Each run of x.shape[-1] / num_groups consecutive elements of the last dimension brought to mean 0 and variance 1, then
    weight and bias (one value for each element of the last dimension) applied:

        y = (x - mean) / sqrt(var + eps) * weight + bias,   var the mean of (x - mean)^2

    num_groups=1 is torch's layer norm over the last dimension; num_groups=heads on a (B, N, heads * head_dim) tensor normalises
    every head's output by itself.  x: CUDA tensor, fp16 / bf16 / fp32, any strides (read in place where rows of the last
    dimension are contiguous and one stride apart, copied otherwise); weight, bias: float32 or of x's dtype, or None.  At most 16384
    elements are normalised together.  Statistics and sums are float32; the gradients of weight and bias are summed in a
    fixed order, so that two calls give the same bits.  There is no second derivative, no forward-mode one, and no CPU path."""
    if not isinstance(x, torch.Tensor):
        raise RuntimeError("layer_norm: x must be a tensor")
    if not torch.compiler.is_compiling():
        if _forward_ad._current_level >= 0:
            _C.refuse_tangents("layer_norm", x, weight, bias)
        if not _C.wants_operators():
            y = _C.native().layer_norm(x, weight, bias, float(eps), int(num_groups))
            if y is not None:
                return y
    from . import _ops
    return _ops.layer_norm_via_ops(x, weight, bias, float(eps), int(num_groups))


class LayerNorm(nn.Module):
    """torch.nn.LayerNorm's last-dimension form (same parameter names, so that its checkpoints load), with groups."""

    def __init__(self, dim, eps=1e-5, elementwise_affine=True, bias=True, num_groups=1, device=None, dtype=None):
        super().__init__()
        if dim <= 0 or num_groups <= 0 or dim % num_groups:
            raise ValueError(f"num_groups ({num_groups}) must divide dim ({dim})")
        self.normalized_shape = (dim,)
        self.eps, self.num_groups, self.elementwise_affine = eps, num_groups, elementwise_affine
        kw = dict(device=device, dtype=dtype)
        self.register_parameter("weight", nn.Parameter(torch.ones(dim, **kw)) if elementwise_affine else None)
        self.register_parameter("bias", nn.Parameter(torch.zeros(dim, **kw)) if elementwise_affine and bias else None)

    def forward(self, x):
        if x.shape[-1] != self.normalized_shape[0]:
            raise RuntimeError(f"the last dimension must be {self.normalized_shape[0]}, got {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps, self.num_groups)

    def extra_repr(self):
        return f"{self.normalized_shape[0]}, eps={self.eps}, num_groups={self.num_groups}, elementwise_affine={self.elementwise_affine}"
