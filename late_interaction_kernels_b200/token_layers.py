"""Layers between an encoder's hidden states and the document head: ``layer_norm``, ``linear``, ``gated_feed_forward``.

``maxsim_from_hidden`` projects hidden states inside the scoring kernel; what comes before that projection in a token head - a
layer norm, residual projection layers, a gated block - runs here, forward and backward, so that a head can be written and
trained without leaving the package::

    h = layer_norm(hidden, ln_w, ln_b)
    h = gated_feed_forward(h, w_gate, w_up, w_down, activation="gelu", residual=h)
    scores = maxsim_from_hidden(Q, h, W)

All three take tensors of any number of leading dimensions, with any strides, and compute in ``x``'s type: float32, float16 or
bfloat16; sums, statistics and activations are fp32 and results are rounded once.  Parameters of another type (fp32 master
weights beside bf16 activations, and biases with them) and a residual of another type are brought to ``x``'s - a layer norm reads fp32 weights as they
are - and parameters get gradients of their own type, rounded from fp32 sums.  Gradients are deterministic.  Backward passes keep what they need: the input, in ``x``'s
type the values in front of an activation or, of a gated block, the factors of its gradients, and a row's mean and inverse deviation in fp32 (so the
backward pass of rows far from zero sees them off by a step of their mean; the forward does not).  Everything runs
on the current stream and may be captured into a CUDA graph.  With 16-bit operands ``relu``'s
gradient goes by the sign of the exact sum where that sum is next to nothing beside the lengths of the rows that it is a product of.
(No counterpart in the reference, which starts at the hidden states.)
"""

from __future__ import annotations

from . import _lib, _ops


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension; autograd-aware in ``x``, ``weight`` and ``bias``.

    ``x [..., width]``, ``weight [width]`` or None (1), ``bias [width]`` or None (0).  A row's variance is the mean of the squared
    differences from its mean, both taken in fp32 from the row in registers."""
    return _ops.native_call(_lib.host().layer_norm, x, weight, bias, eps)


def linear(x, weight, bias=None, activation=None, residual=None):
    """``act(x @ weight.T + bias) + residual``; autograd-aware in all four tensors.  Nothing between the product and the result goes through memory,
    but for the shares of a long sum with few rows.

    ``x [..., in]``, ``weight [out, in]``, ``bias [out]`` or None, ``activation`` None, ``"relu"``, ``"silu"``, ``"gelu"`` (with the
    normal distribution), ``"gelu_tanh"`` (its approximation), ``"tanh"`` or ``"sigmoid"``, ``residual [..., out]`` or None."""
    return _ops.native_call(_lib.host().linear, x, weight, bias, activation, residual)


def gated_feed_forward(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, activation="silu", residual=None):
    """``(act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up)) @ w_down.T + b_down + residual``; autograd-aware in all tensors.

    ``x [..., in]``, ``w_gate`` and ``w_up [hidden, in]``, ``w_down [out, hidden]``, biases or None, ``activation`` as for
    ``linear``, ``residual [..., out]`` or None.  Both projections, the activation and the product are one kernel, the second
    projection another.  The product is rounded to ``x``'s type between the two."""
    return _ops.native_call(_lib.host().gated_feed_forward, x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, residual)


__all__ = ["layer_norm", "linear", "gated_feed_forward"]
