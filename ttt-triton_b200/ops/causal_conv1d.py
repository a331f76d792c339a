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
from torch.autograd.function import once_differentiable

import _scan_core as core


class CausalConv1d(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, init, act, seq, nseq, want_final):
        ctx.set_materialize_grads(False)
        ctx.param_dtypes = (weight.dtype, bias.dtype if bias is not None else None)
        x, w, b = core._rows(x), core._f32(weight), core._f32(bias)
        init = init.contiguous() if init is not None else None
        y, fin = core.causal_conv_forward(x, w, b, act, init, seq, nseq, want_final)
        ctx.act = act
        ctx.save_for_backward(x, w, b, init, seq)
        return y, fin

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfin):
        x, w, b, init, seq = ctx.saved_tensors
        dy = torch.zeros(x.shape, device=x.device, dtype=x.dtype) if dy is None else dy.to(x.dtype).contiguous()
        dfin = dfin.to(x.dtype).contiguous() if dfin is not None else None
        dx, dw, db, dinit = core.causal_conv_backward(x, w, b, ctx.act, init, seq, dy, dfin, ctx.needs_input_grad[3])
        dtypes = ctx.param_dtypes
        return (dx, dw.to(dtypes[0]), db.to(dtypes[1]) if dtypes[1] is not None else None, dinit, None, None, None,
                None)


def causal_conv1d(x, weight, bias=None, activation=None, initial_state=None, cu_seqlens=None,
                  return_final_state=False):
    act = core._act_code(activation)
    if x.dim() != 3:
        raise ValueError(f"x must be [B, L, D], got shape {tuple(x.shape)}")
    nseq, cu = core.packed(cu_seqlens, x)
    core.check_conv(x, weight, bias, initial_state, nseq)
    seq = None
    if cu is not None:
        core.require_cuda(x, cu)
        seq = core.sequence_index(cu, x.shape[1])
    if core.training(x, weight, bias, initial_state):
        y, fin = CausalConv1d.apply(x, weight, bias, initial_state, act, seq, nseq, bool(return_final_state))
    else:
        init = initial_state.contiguous() if initial_state is not None else None
        y, fin = core.causal_conv_forward(core._rows(x), core._f32(weight), core._f32(bias), act, init, seq, nseq,
                                          bool(return_final_state))
    return (y, fin) if return_final_state else y


def causal_conv1d_step(x, conv_state, weight, bias=None, activation=None, state_indices=None):
    """One new token for every row: x [B, D]; conv_state [B, K - 1, D] is shifted in place and the
    output [B, D] returned. ``state_indices`` chooses slots as in ``selective_scan_step``. No
    gradient."""
    return core.causal_conv_step(x, conv_state, weight, bias, activation, state_indices)
