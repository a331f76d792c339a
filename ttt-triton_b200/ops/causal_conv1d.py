"""Short causal convolution along the sequence on the sm_100a kernels: the local mixing in
front of a scan (``ops.selective_scan``), one filter of 2 to 4 taps per channel.

    p[t] = bias + sum_k weight[:, k] x[t - K + 1 + k];   y = p or silu(p)

    y = causal_conv1d(x, weight, bias, activation="silu")
    y, state = causal_conv1d(x, weight, bias, initial_state=state, return_final_state=True)
    y = causal_conv1d_step(x_t, state, weight, bias, activation="silu")

x: [B, L, D] in fp32, bf16 or fp16 (a view of a wider projection is read in place); weight:
[D, K]; bias: [D] or None; states: the K - 1 rows before (after) a sequence, oldest first,
[B, K - 1, D] in x's dtype. ``cu_seqlens`` packs sequences into one row as in
``ops.selective_scan``. Differentiable in x, weight, bias and the initial state.
"""

from __future__ import annotations

import torch

import _scan_core as core


class CausalConv1d(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, init, seq, call):
        act, sizes, nseq, want_final = call
        y, fin, nbytes = core.causal_conv_forward(x, w, b, act, init, seq, nseq, want_final, sizes, True)
        ctx.call = act, sizes, nbytes
        ctx.save_for_backward(x, w, b, init, seq)
        if not want_final:
            return y
        ctx.set_materialize_grads(False)
        return y, fin

    @staticmethod
    @core.first_order
    def backward(ctx, dy, dfin=None):
        x, w, b, init, seq = ctx.saved_tensors
        act, sizes, nbytes = ctx.call
        if dy is None or dy.dtype is not x.dtype or not dy.is_contiguous():
            dy = core._upstream(dy, x)
        if dfin is not None:
            dfin = core._upstream(dfin, x)
        dx, dw, db, dinit = core.causal_conv_backward(x, w, b, act, init, seq, dy, dfin,
                                                      init is not None and ctx.needs_input_grad[3], sizes, nbytes)
        return dx, dw, db if b is not None else None, dinit, None, None


def causal_conv1d(x, weight, bias=None, activation=None, initial_state=None, cu_seqlens=None,
                  return_final_state=False):
    act = core._act_code(activation)
    seq = nseq = None
    if cu_seqlens is not None:
        nseq, cu = core.packed(cu_seqlens, x)
    sizes = core.check_conv(x, weight, bias, initial_state, nseq)
    if cu_seqlens is not None:
        core.require_cuda(x, cu)
        seq = core.sequence_index(cu, sizes[1])
    else:
        nseq = sizes[0]
    # casts and copies, if any, are autograd's
    x, w, b = core._rows(x), core._f32(weight), core._f32(bias)
    init = initial_state.contiguous() if initial_state is not None else None
    if core.training(x, w, b, init):
        return CausalConv1d.apply(x, w, b, init, seq, (act, sizes, nseq, bool(return_final_state)))
    y, fin, _ = core.causal_conv_forward(x, w, b, act, init, seq, nseq, bool(return_final_state), sizes, False)
    return (y, fin) if return_final_state else y


def causal_conv1d_step(x, conv_state, weight, bias=None, activation=None, state_indices=None):
    """One new token for every row: x [B, D]; conv_state [B, K - 1, D] is shifted in place and the
    output [B, D] returned. ``state_indices`` chooses slots as in ``selective_scan_step``. No
    gradient."""
    return core.causal_conv_step(x, conv_state, weight, bias, activation, state_indices)
