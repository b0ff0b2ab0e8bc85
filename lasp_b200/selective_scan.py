"""Selective state-space scan: a linear recurrence whose decay, input and read-out depend on the token.

``lightning_attn`` keeps a (d, e) state per head that decays at a fixed rate; here every channel keeps a few states of its own, and
how far a token decays them is an input.  No counterpart in the reference.  Everything between these calls and the kernels is
native code (csrc/torch_recurrent.cpp).
"""
from ._core import native


def selective_scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, *, dt_softplus=False, initial_state=None, cu_seqlens=None,
                   return_state=False):
    """h[t] = exp(dt[t] A) h[t-1] + dt[t] u[t] B[t];  y[t] = (<C[t], h[t]> + D u[t]) * silu(z[t]), channel by channel, where dt is
    softplus(dt + dt_bias) with ``dt_softplus`` and dt + dt_bias without.

    u, dt, z: (b, n, c) in float32, bfloat16 or float16; A: (c, states) float32, 1 to 64 states; B, C: (b, n, states), or
    (b, n, g, states) for g groups of c / g channels each, in u's dtype.  Any strides with the last dimension side by side are taken as
    they are.  D, dt_bias: (c,), float32 or u's dtype; without z there is no gate.  An infinity in A counts as float32's largest number.
    initial_state: (b, c, states) float32, zeros if left out.
    cu_seqlens: (s + 1,) int32 or int64 on the GPU: u is one row (b = 1) of s packed sequences, the i-th of them tokens
    cu_seqlens[i] to cu_seqlens[i + 1]; the states are then (s, c, states).  Outputs of tokens that lie in no sequence are zeros.
    return_state: also return the states behind the last tokens, which a later call or ``selective_scan_step`` goes on from.

    States and sums are float32 whatever the inputs are; y is rounded once.  Gradients for all inputs but cu_seqlens (first
    derivatives); sums are added in a fixed order, so that they repeat to the bit.
    """
    return native("selective_scan")(u, dt, A, B, C, D, z, dt_bias, dt_softplus, initial_state, cu_seqlens, return_state)


def selective_scan_step(state, u, dt, A, B, C, D=None, z=None, dt_bias=None, *, dt_softplus=False, slots=None):
    """``selective_scan`` for one token of every row: u, dt, z (b, c), B, C (b, [g,] states) -> (b, c); ``state`` is read and updated in
    place.

    state: (slots, c, states) float32, contiguous.  slots: (b,) int32 or int64 on the GPU, the state that each row goes by
    (None: row i by state i).  A row whose slot is not one of the state's (-1, say, in a batch that is padded) gets zeros
    and touches none; rows that name the same slot are consecutive tokens of its sequence, in the order of the rows.
    No backward pass: inputs that require grad are refused unless gradients are switched off.
    """
    return native("selective_scan_step")(state, u, dt, A, B, C, D, z, dt_bias, dt_softplus, slots)
