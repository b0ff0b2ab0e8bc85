"""Short causal convolution, channel by channel: what stands in front of ``selective_scan`` in a layer.

No counterpart in the reference.  Everything between these calls and the kernels is native code (csrc/torch_recurrent.cpp).
"""
from ._core import native

_ACTIVATIONS = {None: False, "silu": True}


def _act(activation):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}; use None or 'silu'")
    return _ACTIVATIONS[activation]


def causal_conv(x, weight, bias=None, *, activation=None, initial_state=None, cu_seqlens=None, return_state=False):
    """y[:, t] = act(bias + sum_j weight[:, j] * x[:, t - w + 1 + j]), with zeros (or ``initial_state``) before a sequence.

    x: (b, n, c) in float32, bfloat16 or float16; any strides with the channels of a token side by side are taken as they are.
    weight: (c, w) with w of 2, 3 or 4; bias: (c,); both float32 or x's dtype.  activation: None or "silu".
    initial_state: (b, w - 1, c) in x's dtype, the inputs before the first token, oldest first.
    cu_seqlens: (s + 1,) int32 or int64 on the GPU: x is one row (b = 1) of s packed sequences, the i-th of them tokens
    cu_seqlens[i] to cu_seqlens[i + 1]; the states are then (s, w - 1, c).  Outputs of tokens that lie in no sequence are zeros.
    return_state: also return the last w - 1 inputs of each sequence, which a later call or ``causal_conv_step`` goes on from.

    Gradients for x, weight, bias and initial_state (first derivatives).
    """
    return native("causal_conv")(x, weight, bias, _act(activation), initial_state, cu_seqlens, return_state)


def causal_conv_step(state, x, weight, bias=None, *, activation=None, slots=None):
    """``causal_conv`` for one token of every row: x (b, c) -> (b, c); ``state`` is read and updated in place.

    state: (slots, w - 1, c) in x's dtype, contiguous.  slots: (b,) int32 or int64 on the GPU, the state that each row goes by
    (None: row i by state i).  A row whose slot is not one of the state's (-1, say, in a batch that is padded) gets zeros
    and touches none; rows that name the same slot are consecutive tokens of its sequence, in the order of the rows.
    No backward pass: inputs that require grad are refused unless gradients are switched off.
    """
    return native("causal_conv_step")(state, x, weight, bias, _act(activation), slots)
