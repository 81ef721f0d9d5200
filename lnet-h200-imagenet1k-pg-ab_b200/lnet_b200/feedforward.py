"""A feed-forward (channel mixing) block for the streams that the temporal mixing writes.

``stream = x + residual``, ``out = down(f(up(norm(stream)))) + stream``: the residual's addition is
inside the norm, bias and activation inside the first product, bias and the second addition inside
the other.  :meth:`B200FeedForward.quantize_` lays the weights out once in 8 bits for serving.
"""

from __future__ import annotations

import torch
from torch import Tensor, nn

from .linear import ACTIVATIONS, linear_act, linear_act_fp8, quantize_rows_fp8
from .norm import RMS_NORM_EPS, residual_rms_norm, residual_rms_norm_fp8


class B200FeedForward(nn.Module):
    """``out = down(f(up(norm(x + residual)))) + (x + residual)`` for bfloat16 streams [..., D].

    The norm's weight is float32, the products' weights and biases bfloat16; all of them train.
    """

    def __init__(self, model_dim: int, hidden_dim: int, *, activation: str = "gelu",
                 eps: float = RMS_NORM_EPS, device=None) -> None:
        super().__init__()
        if model_dim < 1 or hidden_dim < 1:
            raise ValueError(f"model_dim and hidden_dim must be positive, got {model_dim}, "
                             f"{hidden_dim}")
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}, "
                             f"got {activation!r}")
        self.activation = activation
        self.eps = eps
        self.norm_weight = nn.Parameter(torch.ones(model_dim, device=device))
        self.up = nn.Linear(model_dim, hidden_dim, device=device, dtype=torch.bfloat16)
        self.down = nn.Linear(hidden_dim, model_dim, device=device, dtype=torch.bfloat16)
        self._fp8: tuple[Tensor, ...] | None = None

    def forward(self, x: Tensor, residual: Tensor | None = None) -> Tensor:
        if self._fp8 is not None:
            return self._forward_fp8(x, residual)
        y, stream = residual_rms_norm(x, self.norm_weight, residual, self.eps)
        u = linear_act(y, self.up.weight, self.up.bias, activation=self.activation)
        return linear_act(u, self.down.weight, self.down.bias, stream)

    @torch.no_grad()
    def quantize_(self) -> "B200FeedForward":
        """Serve in 8 bits from now on (no gradient) with the weights of this moment; ``train()``
        goes back."""
        self.eval()
        self._fp8 = (*quantize_rows_fp8(self.up.weight), *quantize_rows_fp8(self.down.weight))
        return self

    def train(self, mode: bool = True) -> "B200FeedForward":
        if mode:
            self._fp8 = None
        return super().train(mode)

    def _apply(self, fn, recurse=True):
        self._fp8 = None  # the copies would stay on the old device
        return super()._apply(fn, recurse)

    @torch.no_grad()
    def _forward_fp8(self, x: Tensor, residual: Tensor | None) -> Tensor:
        up, up_scale, down, down_scale = self._fp8
        y, y_scale, stream = residual_rms_norm_fp8(x, self.norm_weight, residual, self.eps)
        u = linear_act_fp8(y, y_scale, up, up_scale, self.up.bias, activation=self.activation)
        u, u_scale = quantize_rows_fp8(u)
        return linear_act_fp8(u, u_scale, down, down_scale, self.down.bias, stream)


__all__ = ["B200FeedForward"]
