"""Network layers beside the fused 64-wide networks of ``tinycudann``: modules over ``nsr_hip.ops`` for networks that a user builds
from torch layers.  Nothing in this package uses them (no network of the reference normalises: its ``VanillaMLP`` is linear layers
and an activation, models/network_utils.py:100-139)."""
import torch
import torch.nn as nn

from nsr_hip import ops as _ops


class LayerNorm(nn.Module):
    """Layer norm over the last axis (``torch.nn.LayerNorm``'s formula, state-dict keys and defaults for one axis).

    Inputs are float32, float16 or bfloat16 on the GPU; ``weight`` / ``bias`` are float32 unless ``dtype`` names the inputs'
    type.  The output has the input's type.  Differentiable once, in reverse mode."""

    def __init__(self, width, eps=1e-5, elementwise_affine=True, bias=True, device=None, dtype=torch.float32):
        super().__init__()
        if int(width) < 1:
            raise ValueError(f"LayerNorm: width {width}")
        self.width, self.eps = int(width), float(eps)
        new = lambda fill: nn.Parameter(torch.full((self.width,), fill, device=device, dtype=dtype))  # noqa: E731
        self.register_parameter("weight", new(1.0) if elementwise_affine else None)
        self.register_parameter("bias", new(0.0) if elementwise_affine and bias else None)

    def forward(self, x):
        if x.shape[-1:] != (self.width,):
            raise ValueError(f"LayerNorm({self.width}): got an input of shape {tuple(x.shape)}")
        return _ops.layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.width}, eps={self.eps}, elementwise_affine={self.weight is not None}"
