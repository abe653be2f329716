"""The norms after and before a block, with its gate, residual and residual scale, as one pass.

What stands between two blocks of a ``[B, D, L]`` model, per token over its D channels::

    g = x * gate * sigmoid(gate)                      (x without a gate)
    p = norm(g) * post_weight + post_bias
    residual_out = residual + scale * p
    y = norm(residual_out) * pre_weight + pre_bias    -> the next block's input

``norm`` is ``"rms"`` (``v / sqrt(mean(v^2) + eps)``, without biases) or ``"layer"`` (the mean
taken off first).
PyTorch runs this as about ten passes over the tensors; here each direction reads its inputs and
writes its outputs once. Statistics and sums are fp32; ``y`` is formed from ``residual_out``
before its rounding. Gradients are sums in a fixed order: the same call gives the same bits.

Inputs that are not contiguous are copied first. A backward with ``create_graph`` and an input that
carries a forward-mode tangent are refused. The reference has no counterpart.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from . import load_extension

_EXT = load_extension()

_NORMS = {"rms": False, "layer": True}


def _layer(norm: str) -> bool:
    if norm not in _NORMS:
        raise RuntimeError(f"norm must be 'rms' or 'layer', got {norm!r}.")
    return _NORMS[norm]


def fused_gated_residual_norm(x: torch.Tensor, residual: torch.Tensor, post_weight: torch.Tensor,
                              pre_weight: torch.Tensor, gate: torch.Tensor | None = None,
                              scale: torch.Tensor | None = None,
                              post_bias: torch.Tensor | None = None,
                              pre_bias: torch.Tensor | None = None, norm: str = "rms",
                              eps: float = 1e-5):
    """``(y, residual_out)`` of a block's output ``x [B,D,L]``, its ``gate`` and the residual
    stream ``residual`` (of x's type, or fp32), with ``[D]`` parameters of x's type; one token
    per sequence is ``L = 1``. Differentiable in all tensors."""
    layer = _layer(norm)
    if not layer and (post_bias is not None or pre_bias is not None):
        raise RuntimeError("an rms norm has no bias.")
    if not eps > 0:
        raise RuntimeError(f"eps must be positive, got {eps}.")
    y, rout = _EXT.block_norm(x, residual, gate, post_weight, post_bias, scale, pre_weight,
                              pre_bias, layer, float(eps))
    return y, rout


class FusedGatedResidualNorm1d(nn.Module):
    """``fused_gated_residual_norm`` with its ``[D]`` parameters: both norms' weights (ones), the
    residual scale (``init_scale``) and, with ``use_bias``, both norms' biases (zeros)."""

    def __init__(self, embed_dim: int, norm: str = "rms", eps: float = 1e-5,
                 init_scale: float = 1.0, use_bias: bool = False, dtype=None, device=None):
        super().__init__()
        self.embed_dim, self.norm, self.eps = int(embed_dim), norm, float(eps)
        if not _layer(norm) and use_bias:
            raise ValueError("an rms norm has no bias.")
        if self.embed_dim <= 0:
            raise ValueError("embed_dim must be positive.")
        kw = {"dtype": dtype, "device": device}
        D = self.embed_dim
        self.post_weight = nn.Parameter(torch.ones(D, **kw))
        self.pre_weight = nn.Parameter(torch.ones(D, **kw))
        self.scale = nn.Parameter(torch.full((D,), float(init_scale), **kw))
        if use_bias:
            self.post_bias = nn.Parameter(torch.zeros(D, **kw))
            self.pre_bias = nn.Parameter(torch.zeros(D, **kw))
        else:
            self.register_parameter("post_bias", None)
            self.register_parameter("pre_bias", None)

    def forward(self, x, residual, gate=None):
        def cast(p):
            return None if p is None else p.to(x.dtype)
        return fused_gated_residual_norm(x, residual, cast(self.post_weight),
                                         cast(self.pre_weight), gate, cast(self.scale),
                                         cast(self.post_bias), cast(self.pre_bias), self.norm,
                                         self.eps)
