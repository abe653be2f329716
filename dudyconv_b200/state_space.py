"""Selective state space scan and the short causal conv in front of it, in the op's layout.

Two sequence operators of the dynamic conv's ``[B, D, L]`` layout, for training (forward and
backward), for prompts (a carried state, a batch padded on the right) and for single tokens
(the state updated in place)::

    xe = state in front of x                                     state [B, D, S-1]
    fused_short_conv:     v = bias + sum_{j<S} weight[d,j] xe[t-(S-1)+j];   out = silu(v)

    dt = softplus(delta + delta_bias)
    h[n] = exp(dt A[d,n]) h[n] + dt u B[n]                       state [B, D, N], fp32
    fused_selective_scan: y = sum_n C[n] h[n] + skip u

Tensors of one call share one type (fp32, fp16 or bf16), except ``A``, ``skip``,
``delta_bias`` and the scan's states, which are fp32. Arithmetic is fp32 and each result is
rounded once. ``lengths`` (int32 ``[B]``, on the device) makes a padded batch: positions at and
behind a sequence's length are not read, come out as zeros and carry no gradient, and the final
state is the one at the length (0 gives the initial state back). Gradients are sums in a fixed
order: the same call gives the same bits.

States may grow (``dt A`` above zero): the decays' product over any eight positions, and over any
stretch that a state or its gradient other than zero crosses, has to stay in fp32's range.

Inputs that are not contiguous are copied first; a state that a ``_step`` call updates must be
contiguous. All work goes to the current stream of the inputs' device. The ``_step`` functions
have no backward. A backward with ``create_graph`` is refused, and so is an input that carries a
forward-mode tangent. A call can be captured into a CUDA graph,
its backward too; as for any backward, no eager graph of the same leaves may be alive then (torch
ends the capture otherwise), so drop earlier outputs first.

The scan's blocks wait for their own copies, for 2 s at most. A wait that ran out would leave wrong
results and no exception: ``capi.device_error()`` tells of it, as for the framework's other operators,
and ``capi.device_error_info()`` where it was.

The reference has no counterpart; these stand beside its operators and change none of them.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from . import load_extension

_EXT = load_extension()

_ACTIVATIONS = {"silu": True, None: False}


def _silu(activation) -> bool:
    if activation not in _ACTIVATIONS:
        raise RuntimeError(f"activation must be 'silu' or None, got {activation!r}.")
    return _ACTIVATIONS[activation]


# ---------------------------------------------------------------------------------------
# short causal conv
# ---------------------------------------------------------------------------------------
def fused_short_conv(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                     initial_state: torch.Tensor | None = None,
                     lengths: torch.Tensor | None = None, activation: str | None = "silu",
                     return_final_state: bool = False):
    """Causal depthwise conv of ``x [B,D,L]`` with ``weight [D,S]`` (2 <= S <= 8, tap ``S-1`` on
    the current token), ``bias [D]`` and SiLU (``activation=None``: none).

    ``initial_state [B,D,S-1]`` holds the inputs before position 0 (zeros without it). With
    ``return_final_state`` the result is ``(out, final_state)``, the state for the next chunk or
    for :func:`fused_short_conv_step`. Differentiable in all tensors but ``lengths``."""
    out = _EXT.short_conv(x, weight, bias, initial_state, lengths, _silu(activation),
                          bool(return_final_state))
    return tuple(out) if return_final_state else out[0]


def fused_short_conv_step(x: torch.Tensor, conv_state: torch.Tensor, weight: torch.Tensor,
                          bias: torch.Tensor | None = None,
                          activation: str | None = "silu") -> torch.Tensor:
    """One token of each sequence: ``x [B,D]`` -> ``[B,D]``; ``conv_state [B,D,S-1]`` takes the
    token in, in place."""
    return _EXT.short_conv_step(x, conv_state, weight, bias, _silu(activation))


class FusedShortConv1d(nn.Module):
    """``fused_short_conv`` with its weight ``[D,S]`` and bias ``[D]``."""

    def __init__(self, embed_dim: int, kernel_size: int = 4, use_bias: bool = True,
                 activation: str | None = "silu", dtype=None, device=None):
        super().__init__()
        self.embed_dim, self.kernel_size = int(embed_dim), int(kernel_size)
        self.activation = activation
        _silu(activation)
        if self.embed_dim <= 0:
            raise ValueError("embed_dim must be positive.")
        if not 2 <= self.kernel_size <= 8:
            raise ValueError("kernel_size must be between 2 and 8.")
        kw = {"dtype": dtype, "device": device}
        self.weight = nn.Parameter(torch.empty(self.embed_dim, self.kernel_size, **kw))
        bound = self.kernel_size ** -0.5
        nn.init.uniform_(self.weight, -bound, bound)
        if use_bias:
            self.bias = nn.Parameter(torch.zeros(self.embed_dim, **kw))
        else:
            self.register_parameter("bias", None)

    def _params_as(self, x):
        return (self.weight.to(x.dtype), None if self.bias is None else self.bias.to(x.dtype))

    def forward(self, x, initial_state=None, lengths=None, return_final_state: bool = False):
        w, b = self._params_as(x)
        return fused_short_conv(x, w, b, initial_state, lengths, self.activation,
                                return_final_state)

    @torch.no_grad()
    def step(self, x, conv_state):
        w, b = self._params_as(x)
        return fused_short_conv_step(x, conv_state, w, b, self.activation)


# ---------------------------------------------------------------------------------------
# selective scan
# ---------------------------------------------------------------------------------------
def fused_selective_scan(u: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                         C: torch.Tensor, skip: torch.Tensor | None = None,
                         delta_bias: torch.Tensor | None = None, delta_softplus: bool = True,
                         initial_state: torch.Tensor | None = None,
                         lengths: torch.Tensor | None = None, return_final_state: bool = False):
    """Selective scan of ``u [B,D,L]`` with steps ``delta [B,D,L]``, rates ``A [D,N]`` (fp32,
    1 <= N <= 64), ``B`` and ``C`` ``[B,G,N,L]`` (channel ``d`` reads group ``d // (D // G)``;
    ``[B,N,L]`` for one group), ``skip`` and ``delta_bias`` ``[D]`` (fp32).

    With ``return_final_state`` the result is ``(y, final_state)``, the state ``[B,D,N]`` (fp32)
    for the next chunk or for :func:`fused_selective_scan_step`. Differentiable in all tensors
    but ``lengths``; a forward that will be differentiated keeps the states at every fourth
    position (``B D N L`` bytes)."""
    out = _EXT.selective_scan(u, delta, A, B, C, skip, delta_bias, initial_state, lengths,
                              bool(delta_softplus), bool(return_final_state))
    return tuple(out) if return_final_state else out[0]


def fused_selective_scan_step(u: torch.Tensor, delta: torch.Tensor, A: torch.Tensor,
                              B: torch.Tensor, C: torch.Tensor, state: torch.Tensor,
                              skip: torch.Tensor | None = None,
                              delta_bias: torch.Tensor | None = None,
                              delta_softplus: bool = True) -> torch.Tensor:
    """One token of each sequence: ``u``, ``delta`` ``[B,D]``, ``B``, ``C`` ``[B,G,N]`` (or
    ``[B,N]``) -> ``y [B,D]``; ``state [B,D,N]`` (fp32) is updated in place."""
    return _EXT.selective_scan_step(u, delta, A, B, C, state, skip, delta_bias,
                                    bool(delta_softplus))


class FusedSelectiveScan1d(nn.Module):
    """``fused_selective_scan`` with its fp32 parameters: ``A = -exp(A_log)`` ``[D,N]`` (rates 1
    to N at the start), ``skip`` ``[D]`` and ``delta_bias`` ``[D]`` (steps of ``dt_min`` to
    ``dt_max`` behind the softplus at the start)."""

    def __init__(self, embed_dim: int, state_size: int = 16, dt_min: float = 1e-3,
                 dt_max: float = 1e-1, device=None):
        super().__init__()
        self.embed_dim, self.state_size = int(embed_dim), int(state_size)
        if self.embed_dim <= 0:
            raise ValueError("embed_dim must be positive.")
        if not 1 <= self.state_size <= 64:
            raise ValueError("state_size must be between 1 and 64.")
        if not 0 < dt_min <= dt_max:
            raise ValueError("0 < dt_min <= dt_max is needed.")
        kw = {"dtype": torch.float32, "device": device}
        D, N = self.embed_dim, self.state_size
        self.A_log = nn.Parameter(torch.arange(1, N + 1, **kw).log().repeat(D, 1))
        self.skip = nn.Parameter(torch.ones(D, **kw))
        lo, hi = torch.tensor(dt_min, **kw).log(), torch.tensor(dt_max, **kw).log()
        dt = torch.exp(torch.rand(D, **kw) * (hi - lo) + lo)
        self.delta_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))

    def forward(self, u, delta, B, C, initial_state=None, lengths=None,
                return_final_state: bool = False):
        return fused_selective_scan(u, delta, -self.A_log.float().exp(), B, C, self.skip.float(),
                                    self.delta_bias.float(), True, initial_state, lengths,
                                    return_final_state)

    @torch.no_grad()
    def step(self, u, delta, B, C, state):
        return fused_selective_scan_step(u, delta, -self.A_log.float().exp(), B, C, state,
                                         self.skip.float(), self.delta_bias.float())
