"""Functional host side of the selective scan and its causal convolution: shape checks,
allocation, C-ABI launches, as ``_core`` has them for the TTT scans.

Activations may be strided views (a slice of a wider projection) as long as their last
dimension is contiguous; others are copied. Nothing here synchronises the device.
"""

from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from _lib import DTYPE_CODES, check, dtype_code, lib, require_cuda

MAX_STATES = 128


# These calls are short: the host's work is most of the time of a single token, and of a small
# training call, whose backward runs in a thread of autograd's with cold caches. Addresses go to
# ctypes as plain integers, and the current device and stream are asked for without wrapping them.
_current_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _on_device(fn):
    """Runs a function with its first argument's device current, as ``_core._on_tensor_device``."""

    @functools.wraps(fn)
    def wrapper(t, *args):
        dev = t.get_device()
        if dev < 0 or dev == _current_device():
            return fn(t, *args)
        with torch.cuda.device(dev):
            return fn(t, *args)

    return wrapper


def ptr(t):
    return t.data_ptr() if t is not None else None


def stream_of(t):
    return _current_stream(t.device.index)


def _rows(t):
    """t with a contiguous last dimension."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check_devices(tensors):
    """All of them on one CUDA device."""
    try:
        dev = tensors[0].get_device()
        for t in tensors:
            if t is not None and t.get_device() != dev or dev < 0:
                break
        else:
            return
    except AttributeError:
        pass
    require_cuda(*(t for t in tensors if t is not None))


def _strides(*values):
    return (ctypes.c_longlong * len(values))(*values)


_Strides2 = ctypes.c_longlong * 2


def _f32(t):
    if t is None:
        return None
    return t if t.dtype is torch.float32 and t.is_contiguous() else t.to(torch.float32).contiguous()


def _as(t, dtype):
    return t if t.dtype is dtype else t.to(dtype)


def _upstream(grad, ref):
    """An output's gradient, of the type of ref and contiguous; zero where there is none."""
    if grad is None:
        return torch.zeros(ref.shape, device=ref.device, dtype=ref.dtype)
    return grad if grad.dtype is ref.dtype and grad.is_contiguous() else grad.to(ref.dtype).contiguous()


def first_order(backward):
    """A backward whose gradients have none themselves: ``once_differentiable``, whose wrapping is
    left out where no graph is recorded."""
    guarded = once_differentiable(backward)

    @functools.wraps(backward)
    def wrapper(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return wrapper


def _same(ref, **tensors):
    for name, t in tensors.items():
        if t is not None and t.dtype != ref.dtype:
            raise ValueError(f"{name} must have dtype {ref.dtype}, got {t.dtype}")


def _real(name, t):
    """Parameters and states of other types are used in fp32, which would drop a complex one's
    imaginary part."""
    if isinstance(t, torch.Tensor) and t.dtype is not torch.float32 and t.is_complex():
        raise TypeError(f"{name} must be real, got {t.dtype}")


def _shaped(name, t, shape):
    if t is not None and t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")


@_on_device
def sequence_index(cu_seqlens, T):
    """Each token's sequence, int32 [T], from S + 1 ascending offsets; -1 outside of all."""
    seq = torch.empty(T, device=cu_seqlens.device, dtype=torch.int32)
    if T:
        check(lib.ttt_sequence_index(T, cu_seqlens.numel() - 1, ptr(cu_seqlens), ptr(seq), stream_of(seq)),
              "ttt_sequence_index")
    return seq


def training(*tensors):
    """Whether a call has a gradient to prepare for. (Inside an autograd function's forward both
    the mode and the inputs' flags say something else.)"""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def packed(cu_seqlens, x):
    """(number of sequences, checked int32 offsets) of a row of packed sequences."""
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2 or cu_seqlens.is_floating_point():
        raise ValueError("cu_seqlens must hold the S + 1 >= 2 offsets of S packed sequences")
    if x.shape[0] != 1:
        raise ValueError(f"packed sequences lie in one row: expected a batch of 1, got {x.shape[0]}")
    return cu_seqlens.numel() - 1, cu_seqlens.to(torch.int32).contiguous()


# --------------------------------------------------------------------------- selective scan
def check_scan(u, delta, A, B, C, D, z, delta_bias, init, nseq):
    _real("A", A), _real("D", D), _real("delta_bias", delta_bias), _real("initial_state", init)
    _check_devices((u, delta, A, B, C, D, z, delta_bias, init))
    dtype_code(u)
    if u.dim() != 3:
        raise ValueError(f"u must be [B, L, D], got shape {tuple(u.shape)}")
    rows, L, W = u.shape
    if A.dim() != 2 or A.shape[0] != W or A.shape[1] < 1:
        raise ValueError(f"A must be [{W}, N], got {tuple(A.shape)}")
    N = A.shape[1]
    if N > MAX_STATES:
        raise ValueError(f"{N} states per channel: at most {MAX_STATES} are supported")
    if W < 1:
        raise ValueError("the scan needs at least one channel")
    _shaped("delta", delta, u.shape)
    _shaped("z", z, u.shape)
    if B.dim() != 4 or tuple(B.shape[:2]) != (rows, L) or B.shape[3] != N or B.shape[2] < 1 or W % B.shape[2]:
        raise ValueError(f"B must be [{rows}, {L}, {N}] or [{rows}, {L}, G, {N}] with G dividing {W}, "
                         f"got {tuple(B.shape)}")
    _shaped("C", C, B.shape)
    _shaped("D", D, (W,))
    _shaped("delta_bias", delta_bias, (W,))
    _shaped("initial_state", init, (nseq, W, N))
    _same(u, delta=delta, B=B, C=C, z=z)


def _scan_args(u, delta, A, B, C, D, z, delta_bias, softplus):
    rows, L, W = u.shape
    st = _strides(u.stride(0), u.stride(1), delta.stride(0), delta.stride(1), B.stride(0), B.stride(1), B.stride(2),
                  C.stride(0), C.stride(1), C.stride(2), *(z.stride()[:2] if z is not None else (0, 0)))
    return (rows, L, W, B.shape[2], A.shape[1], ptr(u), ptr(delta), ptr(B), ptr(C), ptr(z), dtype_code(u), st, ptr(A),
            ptr(D), ptr(delta_bias), int(softplus))


@_on_device
def selective_scan_forward(u, delta, A, B, C, D, z, delta_bias, softplus, init, seq, nseq, want_final, for_backward):
    """Returns (out [B, L, D] in u's dtype, final state fp32 or None, saved states or None).
    u, delta, B, C, z with contiguous last dimensions; A, D, delta_bias, init fp32 contiguous."""
    rows, L, W = u.shape
    N = A.shape[1]
    dev = u.device
    out = torch.empty(rows, L, W, device=dev, dtype=u.dtype)
    fin = saved = None
    if want_final:
        if seq is None and L:
            fin = torch.empty(nseq, W, N, device=dev, dtype=torch.float32)
        else:  # sequences without a token keep their initial state
            fin = init.clone() if init is not None else torch.zeros(nseq, W, N, device=dev, dtype=torch.float32)
    if rows * L == 0:
        return out, fin, torch.empty(0, device=dev) if for_backward else None
    args = _scan_args(u, delta, A, B, C, D, z, delta_bias, softplus)
    if for_backward:
        saved = torch.empty(lib.ttt_selective_scan_saved_bytes(rows, L, W, N) // 4, device=dev, dtype=torch.float32)
    nbytes = lib.ttt_selective_scan_fwd_scratch_bytes(rows, L, W, args[3], N)
    scratch = torch.empty(nbytes, device=dev, dtype=torch.uint8) if nbytes else None
    check(lib.ttt_selective_scan_fwd(*args, ptr(seq), ptr(init), ptr(fin), ptr(out), ptr(saved), ptr(scratch), nbytes,
                                     stream_of(u)), "ttt_selective_scan_fwd")
    return out, fin, saved


@_on_device
def selective_scan_backward(u, delta, A, B, C, D, z, delta_bias, softplus, init, seq, saved, dout, dfin, want_dinit):
    """Returns (du, ddelta, dA, dB, dC, dD, dz or None, ddelta_bias, dinit or None); the
    gradients of A, D, delta_bias and the state in fp32, the others in u's dtype."""
    rows, L, W = u.shape
    G, N = B.shape[2], A.shape[1]
    dev, dt = u.device, u.dtype
    du, ddelta = torch.empty_like(dout), torch.empty_like(dout)
    dz = torch.empty_like(dout) if z is not None else None
    dB = torch.empty(rows, L, G, N, device=dev, dtype=dt)
    dC = torch.empty_like(dB)
    dinit = None
    if want_dinit:
        dinit = dfin.clone() if dfin is not None else torch.zeros(init.shape, device=dev, dtype=torch.float32)
    if rows * L == 0:
        zeros = torch.zeros(W * (N + 2), device=dev, dtype=torch.float32)
        return du, ddelta, zeros[:W * N].view(W, N), dB, dC, zeros[-2 * W:-W], dz, zeros[-W:], dinit
    dparams = torch.empty(W * (N + 2), device=dev, dtype=torch.float32)
    nbytes = lib.ttt_selective_scan_bwd_scratch_bytes(rows, L, W, G, N)
    scratch = torch.empty(nbytes, device=dev, dtype=torch.uint8)
    check(lib.ttt_selective_scan_bwd(*_scan_args(u, delta, A, B, C, D, z, delta_bias, softplus), ptr(seq), ptr(init),
                                     ptr(saved), ptr(dout), ptr(dfin), ptr(du), ptr(ddelta), ptr(dB), ptr(dC), ptr(dz),
                                     ptr(dinit), ptr(dparams), ptr(scratch), nbytes, stream_of(u)),
          "ttt_selective_scan_bwd")
    dA, dD, dbias = (dparams.as_strided((W, N), (N, 1)), dparams.as_strided((W,), (1,), W * N),
                     dparams.as_strided((W,), (1,), W * (N + 1)))
    return du, ddelta, dA, dB, dC, dD, dz, dbias, dinit


def _check_step(state, index, rows, inputs, shape):
    """The carried state and the slots of a single-token call."""
    size, stride = state.shape, state.stride()
    if len(size) != 3 or size[1:] != shape:
        raise ValueError(f"the state must be [slots, {shape[0]}, {shape[1]}], got {tuple(size)}")
    # the stride of a dimension of one says nothing
    if stride[2] != 1 and shape[1] > 1 or stride[1] != shape[1] and shape[0] > 1:
        raise ValueError("the state is updated in place: each slot must be contiguous")
    if size[0] > 1 and stride[0] < shape[0] * shape[1]:
        raise ValueError("the state's slots must not overlap")
    if index is None:
        if size[0] != rows:
            raise ValueError(f"{rows} rows need a state of {rows} slots or state_indices, got {state.shape[0]} slots")
    elif index.dim() != 1 or index.numel() != rows or index.dtype != torch.int32 or not index.is_contiguous():
        raise ValueError(f"state_indices must be contiguous int32 [{rows}]")
    if torch.is_grad_enabled() and any([t.requires_grad for t in inputs if t is not None]):
        raise RuntimeError("the single-token step has no gradient: call it under torch.no_grad()")


@_on_device
def selective_scan_step(state, u, delta, A, B, C, D, z, delta_bias, softplus, index):
    """One token per row: out [B, D]; state [slots, D, N] fp32 updated in place."""
    _real("A", A), _real("D", D), _real("delta_bias", delta_bias)
    _check_devices((u, state, delta, A, B, C, D, z, delta_bias, index))
    shape = u.shape
    if len(shape) != 2:
        raise ValueError(f"u must be [B, D], got shape {tuple(shape)}")
    rows, W = shape
    if A.dim() != 2 or A.shape[0] != W or not 1 <= A.shape[1] <= MAX_STATES:
        raise ValueError(f"A must be [{W}, N] with N from 1 to {MAX_STATES}, got {tuple(A.shape)}")
    N = A.shape[1]
    bs = B.shape
    if len(bs) != 3 or bs[0] != rows or bs[2] != N or bs[1] < 1 or W % bs[1]:
        raise ValueError(f"B must be [{rows}, {N}] or [{rows}, G, {N}] with G dividing {W}, got {tuple(bs)}")
    _shaped("delta", delta, shape)
    _shaped("z", z, shape)
    _shaped("C", C, bs)
    _shaped("D", D, (W,))
    _shaped("delta_bias", delta_bias, (W,))
    dt = u.dtype
    if delta.dtype != dt or B.dtype != dt or C.dtype != dt or (z is not None and z.dtype != dt):
        _same(u, delta=delta, B=B, C=C, z=z)
    if state.dtype != torch.float32:
        raise ValueError(f"the state must be float32, got {state.dtype}")
    _check_step(state, index, rows, (state, u, delta, A, B, C, D, z, delta_bias), (W, N))
    u, delta, B, C = _rows(u), _rows(delta), _rows(B), _rows(C)
    z = _rows(z) if z is not None else None
    out = torch.empty(shape, device=u.device, dtype=dt)
    if rows == 0:
        return out
    A, D, delta_bias = _f32(A), _f32(D), _f32(delta_bias)
    bt, ct = B.stride(), C.stride()
    st = _strides(u.stride(0), delta.stride(0), bt[0], bt[1], ct[0], ct[1], z.stride(0) if z is not None else 0,
                  state.stride(0))
    check(lib.ttt_selective_scan_step(rows, W, bs[1], N, state.shape[0], ptr(u), ptr(delta), ptr(B), ptr(C), ptr(z),
                                      dtype_code(u), st, ptr(A), ptr(D), ptr(delta_bias), int(softplus), ptr(index),
                                      ptr(state), ptr(out), stream_of(u)), "ttt_selective_scan_step")
    increment_version(state)  # for autograd, as torch's own in-place operations do
    return out


# --------------------------------------------------------------------------- causal convolution
def _act_code(activation):
    if activation not in (None, "silu"):
        raise ValueError(f"activation must be None or 'silu', got {activation!r}")
    return int(activation == "silu")


def _check_taps(weight, bias, W):
    shape = weight.shape
    if len(shape) != 2 or shape[0] != W or not 2 <= shape[1] <= 4:
        raise ValueError(f"weight must be [{W}, K] with 2 to 4 taps, got {tuple(shape)}")
    _shaped("bias", bias, (W,))
    return shape[1]


def _conv_sizes(x, weight, bias, init, nseq):
    """(rows, L, D, K, type code) of a call, or what is wrong with it. nseq: packed sequences, or None."""
    if x.dim() != 3:
        raise ValueError(f"x must be [B, L, D], got shape {tuple(x.shape)}")
    _real("weight", weight), _real("bias", bias)
    _check_devices((x, weight, bias, init))
    dt, shape = dtype_code(x), x.shape
    if shape[2] < 1:
        raise ValueError(f"x must be [B, L, D], got shape {tuple(shape)}")
    K = _check_taps(weight, bias, shape[2])
    _shaped("initial_state", init, (shape[0] if nseq is None else nseq, K - 1, shape[2]))
    _same(x, initial_state=init)
    return (*shape, K, dt)


def check_conv(x, weight, bias, init, nseq):
    """The same; a call with nothing but plain parameters is seen to be right at a glance."""
    f32 = torch.float32
    if init is None and weight.dtype is f32 and (bias is None or bias.dtype is f32):
        dev, size, taps = x.get_device(), x.shape, weight.shape
        if (dev >= 0 and weight.get_device() == dev and len(size) == 3 and len(taps) == 2 and size[2] == taps[0] > 0
                and 2 <= taps[1] <= 4 and (bias is None or bias.get_device() == dev and bias.shape == taps[:1])
                and x.dtype in DTYPE_CODES):
            return (*size, taps[1], DTYPE_CODES[x.dtype])
    return _conv_sizes(x, weight, bias, init, nseq)


def causal_conv_forward(x, w, b, act, init, seq, nseq, want_final, sizes, for_backward):
    """Returns (y [B, L, D], final state [sequences, K - 1, D] or None), both in x's dtype, and the
    bytes of scratch of the backward (0 without one)."""
    dev = x.get_device()
    if dev != _current_device():
        with torch.cuda.device(dev):
            return causal_conv_forward(x, w, b, act, init, seq, nseq, want_final, sizes, for_backward)
    rows, L, W, K, dt = sizes
    y = torch.empty_like(x) if x.is_contiguous() else x.new_empty((rows, L, W))
    fin = None
    if want_final:
        if seq is None and L:
            fin = x.new_empty((nseq, K - 1, W))
        else:
            fin = init.clone() if init is not None else x.new_zeros((nseq, K - 1, W))
    if rows * L == 0:
        return y, fin, 0
    st = x.stride()
    rc = lib.ttt_causal_conv_fwd(rows, L, W, K, x.data_ptr(), dt, _Strides2(st[0], st[1]), w.data_ptr(), ptr(b), act,
                                 ptr(seq), ptr(init), ptr(fin), y.data_ptr(), _current_stream(dev))
    if rc:
        check(rc, "ttt_causal_conv_fwd")
    return y, fin, lib.ttt_causal_conv_bwd_scratch_bytes(*sizes) if for_backward else 0


def causal_conv_backward(x, w, b, act, init, seq, dy, dfin, want_dinit, sizes, nbytes):
    """Returns (dx, dw fp32, db fp32, dinit or None); dy of x's dtype and contiguous, nbytes as the
    forward gave them."""
    dev = x.get_device()
    if dev != _current_device():
        with torch.cuda.device(dev):
            return causal_conv_backward(x, w, b, act, init, seq, dy, dfin, want_dinit, sizes, nbytes)
    rows, L, W, K, dt = sizes
    dx = torch.empty_like(dy)
    dinit = None
    if want_dinit:
        dinit = dfin.clone() if dfin is not None else torch.zeros_like(init)
    if rows * L == 0:
        return dx, torch.zeros_like(w), w.new_zeros(W), dinit
    dparams, scratch = w.new_empty(W * (K + 1)), w.new_empty(nbytes // 4)
    st = x.stride()
    rc = lib.ttt_causal_conv_bwd(rows, L, W, K, x.data_ptr(), dt, _Strides2(st[0], st[1]), w.data_ptr(), ptr(b), act,
                                 ptr(seq), ptr(init), dy.data_ptr(), ptr(dfin), dx.data_ptr(), ptr(dinit),
                                 dparams.data_ptr(), scratch.data_ptr(), nbytes, _current_stream(dev))
    if rc:
        check(rc, "ttt_causal_conv_bwd")
    return dx, dparams.as_strided((W, K), (K, 1)), dparams.as_strided((W,), (1,), W * K), dinit


@_on_device
def causal_conv_step(x, state, weight, bias, activation, index):
    """One token per row: y [B, D]; state [slots, K - 1, D] shifted in place."""
    _real("weight", weight), _real("bias", bias)
    _check_devices((x, state, weight, bias, index))
    act = _act_code(activation)
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"x must be [B, D], got shape {tuple(x.shape)}")
    rows, W = x.shape
    K = _check_taps(weight, bias, W)
    _same(x, conv_state=state)
    _check_step(state, index, rows, (x, state, weight, bias), (K - 1, W))
    y = torch.empty(rows, W, device=x.device, dtype=x.dtype)
    if rows == 0:
        return y
    x, w, b = _rows(x), _f32(weight), _f32(bias)
    check(lib.ttt_causal_conv_step(rows, W, K, state.shape[0], ptr(x), dtype_code(x),
                                   _strides(x.stride(0), state.stride(0)), ptr(w), ptr(b), act, ptr(index), ptr(state),
                                   ptr(y), stream_of(x)), "ttt_causal_conv_step")
    increment_version(state)  # for autograd, as torch's own in-place operations do
    return y
