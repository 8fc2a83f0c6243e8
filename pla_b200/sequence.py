"""Sequence operators: causal depthwise convolution, query / key norm with
position rotation, gated delta rule, and the block that chains them.

They are the layers of a delta-rule sequence block, built from the pieces the
library has for images: a depthwise convolution (here along time), a norm
fused to its neighbour (here over a head, with the rotation) and a linearly
updated state.  No reference counterpart (the reference's operator is the
depthwise convolution of data/depthwise_conv_7x7.py:15-29).

* ``causal_depthwise()`` / ``causal_depthwise_step()``
* ``qk_norm_rotate()``
* ``gated_delta_rule()`` / ``gated_delta_rule_step()``
* ``DeltaMixer``: projections, the three operators, output projection

The first form of each runs over whole sequences, has a gradient, and takes
ragged batches: ``cu_seqlens`` is an int32 CUDA vector of N + 1 ascending
token offsets starting at 0 that cuts one batch row into N sequences (rows in
no sequence come back zero).  ``state=`` is what precedes each sequence and
``return_state=True`` also returns what follows it.  The ``_step`` forms
advance every sequence by one token and update ``state`` in place; they have
no gradient.

Dtypes: float32, bfloat16, float16; sums, norms and delta-rule states are
fp32.  Every call runs as ``torch.ops.pla_b200.*`` on the current stream and
can be captured in a CUDA graph.  A CPU tensor raises: there is no fallback.
A second derivative and a forward-mode one raise.  A kernel of the delta rule
whose copies do not arrive within two seconds ends with its results incomplete
(a single token's state unchanged); ``pla_b200.check_faults()`` raises then.
"""
from __future__ import annotations

import torch

from . import _lib


_ops: dict = {}


def _op(name: str, t):
    if not isinstance(t, torch.Tensor) or not (t.is_cuda or t.is_meta):
        raise ValueError(f"{name} requires CUDA inputs")
    if name not in _ops:
        _ops[name] = getattr(_lib.ops(), name).default
    return _ops[name]


def causal_depthwise(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, silu: bool = False,
                     cu_seqlens: torch.Tensor | None = None, state: torch.Tensor | None = None,
                     return_state: bool = False):
    """``y[t] = act(bias + sum_j weight[:, j] * x[t - K + 1 + j])`` for x [B, T, C], weight [C, K] or [C, 1, K].

    K is 2 to 4 taps; ``silu`` applies ``p * sigmoid(p)``.  ``state``
    [N, K - 1, C] holds the inputs before each sequence, oldest first (zeros
    if None).  Returns y, or (y, state after the sequences).  Differentiable
    in x, weight, bias and state.
    """
    y, last = _op("causal_depthwise", x)(x, weight, bias, silu, cu_seqlens, state, return_state)
    return (y, last) if return_state else y


def causal_depthwise_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                          silu: bool = False) -> torch.Tensor:
    """One token of ``causal_depthwise`` for x [N, C]; ``state`` [N, K - 1, C] moves up by one row in place."""
    return _op("causal_depthwise_step", x)(x, state, weight, bias, silu)


def qk_norm_rotate(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor | None = None,
                   k_weight: torch.Tensor | None = None, cos: torch.Tensor | None = None,
                   sin: torch.Tensor | None = None, positions: torch.Tensor | None = None, norm: str = "rms",
                   eps: float = 1e-6, interleaved: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """Norm of every head of q [B, T, Hq, D] and k [B, T, Hk, D], then the rotation of its first features.

    ``norm="rms"``: ``x / sqrt(mean(x^2) + eps) * weight``; ``norm="l2"``:
    ``x / sqrt(sum(x^2) + eps) * weight``; weights [D] or None.  ``cos`` and
    ``sin`` are float32 tables [P, R / 2]: the first R features are rotated in
    pairs (i, i + R / 2), or (2i, 2i + 1) with ``interleaved``, by row
    ``positions`` ([T], [1, T] or [B, T] integers; the token's number if
    None).  A position outside the tables gives NaN in the rotated features; a
    head whose squares overflow float32 (values above about 1e19) gives 0.
    D is at most 256, B at most 65535 (for gradients B * T * heads at most
    2^30).  Differentiable in q, k and the weights.
    """
    if norm not in ("rms", "l2"):
        raise ValueError('norm must be "rms" or "l2"')
    return _op("qk_norm_rotate", q)(q, k, q_weight, k_weight, cos, sin, positions, norm == "l2", eps, interleaved)


def gated_delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                     scale: float | None = None, cu_seqlens: torch.Tensor | None = None,
                     state: torch.Tensor | None = None, return_state: bool = False):
    """Token by token, for every value head: ``S = exp(g) S; u = beta (v - S^T k); S = S + k u^T; o = scale S^T q``.

    q, k [B, T, Hk, Dk], v [B, T, Hv, Dv], g and beta [B, T, Hv] (both of v's
    dtype, or both float32); value head h reads key head ``h // (Hv // Hk)``.
    ``g`` is the log of the decay (0 keeps the state, -inf clears it), ``scale``
    is ``Dk ** -0.5`` if None.  ``state`` is float32 [N, Hv, Dk, Dv] (zeros if
    None).  Dk and Dv are at most 128.  Keys are expected normalised
    (``qk_norm_rotate(..., norm="l2")``): the rule is stable for
    ``beta * |k|^2 <= 2``.  A value that is not finite reaches its sequence's
    outputs from the start of its chunk of 64 tokens on, up to 63 tokens before
    its own (one of v only its own feature); other sequences and heads never.
    Returns o, or (o, state after the sequences).
    Differentiable in q, k, v, g, beta and state; the backward pass computes
    the states again and keeps only the inputs.
    """
    op = _op("gated_delta_rule", q)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    o, last = op(q, k, v, g, beta, scale, cu_seqlens, state, return_state)
    return (o, last) if return_state else o


def gated_delta_rule_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                          state: torch.Tensor, scale: float | None = None) -> torch.Tensor:
    """One token of ``gated_delta_rule``: q, k [N, Hk, Dk], v [N, Hv, Dv], g, beta [N, Hv].

    ``state``, float32 [N, Hv, Dk, Dv], is updated in place.  Dk is at most
    256.  Returns o [N, Hv, Dv].
    """
    op = _op("gated_delta_rule_step", q)
    return op(q, k, v, g, beta, state, q.shape[-1] ** -0.5 if scale is None else scale)


class DeltaMixer(torch.nn.Module):
    """A delta-rule sequence block: projection, short convolution, norms, gated delta rule, output projection.

    ``in_proj`` gives queries and keys (``num_heads`` of ``head_dim``) and
    values (``value_heads`` of ``value_dim``); ``conv`` is the causal
    depthwise convolution with SiLU over all of them; queries and keys are L2
    normalised per head; ``gate_proj`` gives each value head's decay
    ``g = -exp(A_log) softplus(a + dt_bias)`` and ``beta = sigmoid(b)``, in
    fp32; ``out_proj`` maps the heads back.  ``forward`` takes [B, T, dim] (or
    a ragged [1, T, dim] with ``cu_seqlens``); ``step`` takes [N, dim] and a
    state from ``new_state`` or ``forward(..., return_state=True)``, which it
    updates in place.  Under ``torch.autocast`` the operators run in its dtype,
    and so do the convolution's states.  ``head_dim`` and ``value_dim`` are at
    most 128 (``step`` alone takes a ``head_dim`` of 256).
    """

    def __init__(self, dim: int, num_heads: int, head_dim: int = 128, value_heads: int | None = None,
                 value_dim: int | None = None, taps: int = 4):
        super().__init__()
        self.num_heads, self.head_dim = num_heads, head_dim
        self.value_heads = num_heads if value_heads is None else value_heads
        self.value_dim = head_dim if value_dim is None else value_dim
        if self.value_heads % num_heads:
            raise ValueError("value_heads must be a multiple of num_heads")
        self.widths = [num_heads * head_dim, num_heads * head_dim, self.value_heads * self.value_dim]
        channels = sum(self.widths)
        self.in_proj = torch.nn.Linear(dim, channels, bias=False)
        self.gate_proj = torch.nn.Linear(dim, 2 * self.value_heads, bias=False)
        self.conv = torch.nn.Conv1d(channels, channels, taps, groups=channels)
        self.A_log = torch.nn.Parameter(torch.empty(self.value_heads).uniform_(1, 8).log())
        self.dt_bias = torch.nn.Parameter(torch.full((self.value_heads,), -2.0))
        self.out_proj = torch.nn.Linear(self.value_heads * self.value_dim, dim, bias=False)

    def new_state(self, n: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Zero states of n sequences: the convolution's inputs and the delta rule's fp32 state."""
        w = self.in_proj.weight
        dtype = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else w.dtype
        return (torch.zeros(n, self.conv.weight.shape[-1] - 1, sum(self.widths), device=w.device, dtype=dtype),
                torch.zeros(n, self.value_heads, self.head_dim, self.value_dim, device=w.device, dtype=torch.float32))

    def _taps(self, dtype):  # under autocast the projections' results are not of the weights' dtype
        return self.conv.weight.to(dtype), self.conv.bias.to(dtype)

    def _gates(self, x):
        a, b = self.gate_proj(x).float().chunk(2, -1)
        g = -self.A_log.float().exp() * torch.nn.functional.softplus(a + self.dt_bias.float())
        return g, torch.sigmoid(b)

    def _heads(self, h):
        q, k, v = h.split(self.widths, -1)
        heads = (self.num_heads, self.head_dim)
        return q.unflatten(-1, heads), k.unflatten(-1, heads), v.unflatten(-1, (self.value_heads, self.value_dim))

    def forward(self, x: torch.Tensor, cu_seqlens: torch.Tensor | None = None, state=None, return_state: bool = False):
        before = (None, None) if state is None else state
        h = self.in_proj(x)
        h, conv_state = causal_depthwise(h, *self._taps(h.dtype), silu=True, cu_seqlens=cu_seqlens, state=before[0],
                                         return_state=True)
        q, k, v = self._heads(h)
        q, k = qk_norm_rotate(q, k, norm="l2")
        o = gated_delta_rule(q, k, v, *self._gates(x), cu_seqlens=cu_seqlens, state=before[1], return_state=return_state)
        if return_state:
            return self.out_proj(o[0].flatten(-2)), (conv_state, o[1])
        return self.out_proj(o.flatten(-2))

    def _check_delta_state(self, s: torch.Tensor, n: int) -> None:
        # what gated_delta_rule_step would refuse, before the convolution's state has moved on
        shape = (n, self.value_heads, self.head_dim, self.value_dim)
        if s.shape != shape or s.dtype != torch.float32:
            raise ValueError(f"the delta rule's state must be float32 {list(shape)}, got {s.dtype} {list(s.shape)}")
        if n and not (s.is_contiguous() or s[0].is_contiguous() and (n == 1 or s.stride(0) >= s[0].numel())):
            raise ValueError("each sequence's delta rule state must be dense and its own: it is updated in place")
        if s.requires_grad and torch.is_grad_enabled():
            raise ValueError("the delta rule's state is updated in place and must not require grad")

    def step(self, x: torch.Tensor, state: tuple[torch.Tensor, torch.Tensor]) -> torch.Tensor:
        self._check_delta_state(state[1], x.shape[0])
        h = self.in_proj(x)
        h = causal_depthwise_step(h, state[0], *self._taps(h.dtype), silu=True)
        q, k, v = self._heads(h)
        q, k = (t[0] for t in qk_norm_rotate(q[None], k[None], norm="l2"))  # no positions: any number of sequences as one row
        return self.out_proj(gated_delta_rule_step(q, k, v, *self._gates(x), state[1]).flatten(-2))
