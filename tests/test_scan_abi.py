"""CPU: the selective scan's and the causal convolution's entry points refuse bad arguments on
the host, before any CUDA call, and their sizes are what the header says."""

import ctypes

import pytest
import torch

import _lib
import ops

FAKE = ctypes.c_void_p(0x1000)  # never dereferenced: every call below fails its host checks first
lib = _lib.lib


def strides(n):
    return (ctypes.c_longlong * n)()


def message():
    return lib.ttt_last_error().decode()


def scan_fwd(rows=1, L=8, D=8, G=1, N=4, dt=0, u=FAKE, A=FAKE, out=FAKE, st=strides(12), seq=None, scratch=None, n=0):
    return lib.ttt_selective_scan_fwd(rows, L, D, G, N, u, FAKE, FAKE, FAKE, None, dt, st, A, None, None, 1, seq, None,
                                      None, out, None, scratch, n, None)


def scan_bwd(D=8, G=1, N=4, z=None, dz=None, saved=FAKE, scratch=None, n=0):
    return lib.ttt_selective_scan_bwd(1, 8, D, G, N, FAKE, FAKE, FAKE, FAKE, z, 0, strides(12), FAKE, None, None, 1,
                                      None, None, saved, FAKE, None, FAKE, FAKE, FAKE, FAKE, dz, None, FAKE, scratch, n,
                                      None)


def test_scan_refusals():
    assert scan_fwd(rows=0) == -2 and scan_fwd(L=0) == -2 and scan_fwd(D=0) == -2 and scan_fwd(N=0) == -2
    assert scan_fwd(N=129) == -2 and "at most 128" in message()
    assert scan_fwd(D=9, G=2) == -2 and "groups" in message()
    assert scan_fwd(rows=1 << 16, L=1 << 15) == -2 and "tokens" in message()
    assert scan_fwd(dt=3) == -3
    assert scan_fwd(u=None) == -1 and scan_fwd(A=None) == -1 and scan_fwd(out=None) == -1 and scan_fwd(st=None) == -1
    assert scan_fwd(rows=2, seq=FAKE) == -2 and "one row" in message()
    # few channels and a long axis are split, which takes scratch
    need = lib.ttt_selective_scan_fwd_scratch_bytes(1, 1 << 14, 8, 1, 4)
    assert need > 0
    assert scan_fwd(L=1 << 14) == -5 and str(need) in message()
    assert scan_fwd(L=1 << 14, scratch=FAKE, n=need - 1) == -5


def test_scan_backward_refusals():
    assert scan_bwd(saved=None) == -1
    assert scan_bwd(z=FAKE) == -1 and scan_bwd(dz=FAKE) == -1 and "together" in message()
    need = lib.ttt_selective_scan_bwd_scratch_bytes(1, 8, 8, 1, 4)
    assert need >= 4 * (2 * 8 * 4 + 8 * 6)  # partials of dB, dC and of dA, dD, dbias
    assert scan_bwd() == -5 and scan_bwd(scratch=FAKE, n=need - 1) == -5


def test_scan_sizes():
    assert lib.ttt_selective_scan_saved_bytes(2, 9, 6, 16) == 2 * 3 * 6 * 16 * 4  # a state every 4 tokens
    assert lib.ttt_selective_scan_saved_bytes(1, 1, 6, 100) == 6 * 100 * 4
    assert lib.ttt_selective_scan_saved_bytes(1, 1, 6, 129) == 0
    assert lib.ttt_selective_scan_fwd_scratch_bytes(1, 1, 6, 1, 16) == 0


def test_step_refusals():
    def step(rows=2, D=8, N=4, slots=2, index=None, state=FAKE):
        return lib.ttt_selective_scan_step(rows, D, 1, N, slots, FAKE, FAKE, FAKE, FAKE, None, 0, strides(8), FAKE, None,
                                           None, 1, index, state, FAKE, None)

    assert step(state=None) == -1 and step(slots=1) == -2 and step(slots=0, index=FAKE) == -2 and step(N=200) == -2

    def conv(K=4, slots=2, state=FAKE):
        return lib.ttt_causal_conv_step(2, 8, K, slots, FAKE, 0, strides(2), FAKE, None, 0, None, state, FAKE, None)

    assert conv(K=1) == -2 and conv(K=5) == -2 and conv(slots=1) == -2 and conv(state=None) == -1


def test_conv_refusals():
    def fwd(rows=1, L=8, D=8, K=4, dt=0, x=FAKE, act=0, seq=None, y=FAKE):
        return lib.ttt_causal_conv_fwd(rows, L, D, K, x, dt, strides(2), FAKE, None, act, seq, None, None, y, None)

    assert fwd(K=1) == -2 and fwd(K=5) == -2 and "2 to 4" in message()
    assert fwd(L=0) == -2 and fwd(D=0) == -2 and fwd(dt=9) == -3 and fwd(act=2) == -2
    assert fwd(x=None) == -1 and fwd(y=None) == -1 and fwd(rows=2, seq=FAKE) == -2
    need = lib.ttt_causal_conv_bwd_scratch_bytes(1, 8, 8, 4, 0)
    assert need >= 4 * 8 * 5
    rc = lib.ttt_causal_conv_bwd(1, 8, 8, 4, FAKE, 0, strides(2), FAKE, None, 0, None, None, FAKE, None, FAKE, None,
                                 FAKE, FAKE, 16, None)
    assert rc == -5
    assert lib.ttt_sequence_index(4, 0, FAKE, FAKE, None) == -2 and lib.ttt_sequence_index(4, 1, None, FAKE, None) == -1


def test_python_layer_refuses_before_the_device():
    x = torch.zeros(1, 4, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.causal_conv1d(x, torch.zeros(8, 4))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.selective_scan(x, x, torch.zeros(8, 4), torch.zeros(1, 4, 4), torch.zeros(1, 4, 4))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.selective_scan_step(torch.zeros(1, 8, 4), x[:, 0], x[:, 0], torch.zeros(8, 4), torch.zeros(1, 4),
                                torch.zeros(1, 4))
    with pytest.raises(ValueError, match="silu"):
        ops.causal_conv1d(x, torch.zeros(8, 4), activation="relu")
    with pytest.raises(ValueError, match=r"\[B, L, D\]"):
        ops.causal_conv1d(x[0], torch.zeros(8, 4))
    with pytest.raises(ValueError, match="one row"):
        ops.causal_conv1d(torch.zeros(2, 4, 8), torch.zeros(8, 4), cu_seqlens=torch.tensor([0, 4]))
    with pytest.raises(ValueError, match="cu_seqlens"):
        ops.causal_conv1d(x, torch.zeros(8, 4), cu_seqlens=torch.tensor([0]))
