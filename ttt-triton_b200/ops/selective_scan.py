"""Selective state space scan on the sm_100a kernels: a layer scan like ``ops.ttt_linear``
whose state decays at an input-dependent rate.

    dt = softplus(delta + delta_bias)                 (or without the softplus)
    h[t] = exp(dt A) h[t-1] + dt u B[t]               per channel, N states
    y = <h, C[t]> + D u;   out = y * silu(z)

    out = selective_scan(u, delta, A, B, C, D, z, delta_bias, delta_softplus=True)
    out, state = selective_scan(..., initial_state=state, return_final_state=True)
    out = selective_scan_step(state, u_t, delta_t, A, B_t, C_t, D, z_t, delta_bias, True)

u, delta, z: [B, L, D] in one of fp32, bf16, fp16; A: [D, N], N <= 128; B, C: [B, L, N], or
[B, L, G, N] with each row shared by D / G adjacent channels; D, delta_bias: [D]; states:
fp32 [B, D, N]. Views of wider projections are read in place when their last dimension is
contiguous. ``cu_seqlens`` (S + 1 ascending int32 offsets on the device, the first 0) packs S
sequences into one row, B = 1: each starts from its initial state (zero without one), states are
[S, D, N], and tokens past the last offset give zeros. Differentiable in every tensor but
cu_seqlens, through the final state too; each gradient has its input's dtype.
"""

from __future__ import annotations

import torch

import _scan_core as core


def _layouts(u, delta, A, B, C, D, z, delta_bias):
    """The inputs as the kernels read them."""
    return (core._rows(u), core._rows(delta), core._f32(A), core._rows(B), core._rows(C), core._f32(D),
            core._rows(z) if z is not None else None, core._f32(delta_bias))


class SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, delta_bias, init, softplus, seq, nseq, want_final):
        ctx.param_dtypes = (A.dtype, D.dtype if D is not None else None,
                            delta_bias.dtype if delta_bias is not None else None,
                            init.dtype if init is not None else None)
        args, init = _layouts(u, delta, A, B, C, D, z, delta_bias), core._f32(init)
        out, fin, saved = core.selective_scan_forward(*args, softplus, init, seq, nseq, want_final, True)
        ctx.softplus = softplus
        ctx.save_for_backward(*args, init, seq, saved)
        if not want_final:
            return out
        ctx.set_materialize_grads(False)
        return out, fin

    @staticmethod
    @core.first_order
    def backward(ctx, dout, dfin=None):
        *args, init, seq, saved = ctx.saved_tensors
        dout, dfin = core._upstream(dout, args[0]), core._f32(dfin)
        du, ddelta, dA, dB, dC, dD, dz, dbias, dinit = core.selective_scan_backward(
            *args, ctx.softplus, init, seq, saved, dout, dfin, ctx.needs_input_grad[8])
        as_, dtypes = core._as, ctx.param_dtypes
        return (du, ddelta, as_(dA, dtypes[0]), dB, dC, as_(dD, dtypes[1]) if dtypes[1] is not None else None, dz,
                as_(dbias, dtypes[2]) if dtypes[2] is not None else None,
                as_(dinit, dtypes[3]) if dinit is not None else None, None, None, None, None)


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=False, initial_state=None,
                   cu_seqlens=None, return_final_state=False):
    if B.dim() == 3:
        B = B.unsqueeze(2)
    if C.dim() == 3:
        C = C.unsqueeze(2)
    if u.dim() != 3:
        raise ValueError(f"u must be [B, L, D], got shape {tuple(u.shape)}")
    nseq, cu = core.packed(cu_seqlens, u) if cu_seqlens is not None else (u.shape[0], None)
    core.check_scan(u, delta, A, B, C, D, z, delta_bias, initial_state, nseq)
    seq = None
    if cu is not None:
        core.require_cuda(u, cu)
        seq = core.sequence_index(cu, u.shape[1])
    if core.training(u, delta, A, B, C, D, z, delta_bias, initial_state):
        return SelectiveScan.apply(u, delta, A, B, C, D, z, delta_bias, initial_state, bool(delta_softplus), seq, nseq,
                                   bool(return_final_state))
    out, fin, _ = core.selective_scan_forward(*_layouts(u, delta, A, B, C, D, z, delta_bias), bool(delta_softplus),
                                              core._f32(initial_state), seq, nseq, bool(return_final_state), False)
    return (out, fin) if return_final_state else out


def selective_scan_step(state, u, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=False,
                        state_indices=None):
    """One new token for every row: u, delta, z [B, D], B, C [B, N] or [B, G, N]; the fp32 state
    [B, D, N] is updated in place and the output [B, D] returned. With ``state_indices`` (int32
    [B]) row i uses slot state_indices[i] of a state [slots, D, N]: a negative index leaves the
    row out (its output is zero); one past the last slot, or equal to an earlier row's, is not
    stepped and its output is NaN. No gradient."""
    return core.selective_scan_step(state, u, delta, A, B.unsqueeze(1) if B.dim() == 2 else B,
                                    C.unsqueeze(1) if C.dim() == 2 else C, D, z, delta_bias, delta_softplus,
                                    state_indices)
