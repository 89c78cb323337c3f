"""Layer norm with a residual sum in front of it, forward and backward (csrc/kernels/layer_norm.cu).

    y = layer_norm(x, weight, bias, eps)                      # over the last dimension
    y, s = layer_norm(x, weight, bias, eps, residual=r)       # s = x + r in the type of x, y = layer norm of s

float32 and bfloat16; weight and bias (each may be None) are float32 or of the type of x. Statistics and
gradients are summed in float32, the gradients of weight and bias in a fixed order: the same bits in every
run. Under autocast x and the residual are cast to its type, as a linear layer casts its input (which leaves float64
alone: that type is refused). Inputs that are not contiguous are copied first. Gradients of gradients, forward-mode
gradients and calls under a tracer (``torch.jit.trace``, ``make_fx``, ``torch.export``) are refused.
"""
import torch

from .._native import native_extension


def layer_norm(x, weight=None, bias=None, eps=1e-5, residual=None):
    """y, or with a `residual` the pair (y, s): see above."""
    out = _ops().layer_norm(x, residual, weight, bias, eps)
    return out[0] if residual is None else tuple(out)


def _ops():
    return native_extension("torch_switchml_train")


class FusedLayerNorm(torch.nn.LayerNorm):
    """``nn.LayerNorm`` over one dimension by :func:`layer_norm`. ``forward(x, residual)`` takes the sum
    in front of it into the kernel and returns the normalised sum only; ``layer_norm`` itself returns the sum too."""

    def __init__(self, normalized_shape, *args, **kwargs):
        super().__init__(normalized_shape, *args, **kwargs)
        if len(self.normalized_shape) != 1:
            raise ValueError("FusedLayerNorm normalises over one dimension, got %s" % (self.normalized_shape,))

    def forward(self, x, residual=None):
        if x.shape[-1:] != self.normalized_shape:
            raise ValueError("FusedLayerNorm over %d features: x has the shape %s" % (self.normalized_shape[0], tuple(x.shape)))
        out = layer_norm(x, self.weight, self.bias, self.eps, residual)
        return out if residual is None else out[0]
