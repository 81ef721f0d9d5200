"""A feed-forward (channel mixing) block for the streams that the temporal mixing writes.

``stream = x + residual``, ``out = down(f(up(norm(stream)))) + stream``: the residual's addition is
inside the norm, bias and activation inside the first product, bias and the second addition inside
the other.  :meth:`B200FeedForward.quantize_` lays the weights out once in 8 bits for serving.
"""

from __future__ import annotations

import torch
from torch import Tensor, nn

from ._native import refuse_grad
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
        self._serve_fp8 = False
        self._fp8: tuple[Tensor, ...] | None = None  # 8-bit weights and their scales
        self._fp8_of: tuple = ()  # what they were laid out from

    def forward(self, x: Tensor, residual: Tensor | None = None) -> Tensor:
        if self._serve_fp8:
            refuse_grad("B200FeedForward in 8 bits", x, residual)
            return self._forward_fp8(x, residual)
        y, stream = residual_rms_norm(x, self.norm_weight, residual, self.eps)
        u = linear_act(y, self.up.weight, self.up.bias, activation=self.activation)
        return linear_act(u, self.down.weight, self.down.bias, stream)

    @torch.no_grad()
    def quantize_(self) -> "B200FeedForward":
        """Serve in 8 bits from now on (no gradient); ``train()`` goes back.  The weights are laid out
        here, and again at the next call where they have changed since (``load_state_dict``, ``to``, an
        update in place that autograd counts; after another kind call ``quantize_`` again)."""
        self.eval()
        self._fp8, self._fp8_of = None, ()
        self._fp8_weights()
        self._serve_fp8 = True
        return self

    def _fp8_weights(self) -> tuple[Tensor, ...]:
        """The 8-bit copies, of the weights as they are: those that are held are kept while storage
        and version are the same (the storage is held too, so that its address stays its own)."""
        weights = (self.up.weight, self.down.weight)
        # inference-mode tensors count no versions
        key = [(w.data_ptr(), 0 if w.is_inference() else w._version) for w in weights]
        if self._fp8 is None or key != self._fp8_of[0]:
            self._fp8 = (*quantize_rows_fp8(weights[0]), *quantize_rows_fp8(weights[1]))
            self._fp8_of = (key, [w.detach() for w in weights])
        return self._fp8

    def train(self, mode: bool = True) -> "B200FeedForward":
        if mode:
            self._serve_fp8 = False
            self._fp8, self._fp8_of = None, ()
        return super().train(mode)

    def _apply(self, fn, recurse=True):
        self._fp8, self._fp8_of = None, ()  # they would stay on the old device: the next call lays out new ones
        return super()._apply(fn, recurse)

    @torch.no_grad()
    def _forward_fp8(self, x: Tensor, residual: Tensor | None) -> Tensor:
        up, up_scale, down, down_scale = self._fp8_weights()
        y, y_scale, stream = residual_rms_norm_fp8(x, self.norm_weight, residual, self.eps)
        u = linear_act_fp8(y, y_scale, up, up_scale, self.up.bias, activation=self.activation)
        u, u_scale = quantize_rows_fp8(u)
        return linear_act_fp8(u, u_scale, down, down_scale, self.down.bias, stream)


__all__ = ["B200FeedForward"]
