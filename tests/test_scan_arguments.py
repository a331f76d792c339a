"""CPU: the argument checks of the selective scan and the causal convolution that come before
any use of the device."""

import pytest
import torch

import _scan_core as core
import ops


@pytest.mark.parametrize("dtype", [torch.complex64, torch.complex128])
def test_complex_parameters_are_refused(dtype):
    """A cast to fp32 would drop their imaginary part and compute another operator."""
    x, A, B = torch.zeros(1, 4, 8), torch.zeros(8, 4), torch.zeros(1, 4, 4)
    bad = lambda *shape: torch.ones(*shape, dtype=dtype)  # noqa: E731
    for kw, name in ((dict(A=bad(8, 4)), "A"), (dict(D=bad(8)), "D"), (dict(delta_bias=bad(8)), "delta_bias"),
                     (dict(initial_state=bad(1, 8, 4)), "initial_state")):
        with pytest.raises(TypeError, match=f"{name} must be real"):
            ops.selective_scan(x, x, kw.pop("A", A), B, B, **kw)
    for kw, name in ((dict(A=bad(8, 4)), "A"), (dict(D=bad(8)), "D"), (dict(delta_bias=bad(8)), "delta_bias")):
        with pytest.raises(TypeError, match=f"{name} must be real"):
            ops.selective_scan_step(torch.zeros(1, 8, 4), x[:, 0], x[:, 0], kw.pop("A", A), B[:, 0], B[:, 0], **kw)
    for w, b, name in ((bad(8, 3), None, "weight"), (torch.ones(8, 3), bad(8), "bias")):
        with pytest.raises(TypeError, match=f"{name} must be real"):
            ops.causal_conv1d(x, w, b)
        with pytest.raises(TypeError, match=f"{name} must be real"):
            ops.causal_conv1d_step(x[:, 0], torch.zeros(1, 2, 8), w, b)


def test_state_layouts():
    """Slots must be contiguous and apart; a dimension of one may have any stride."""
    check = lambda state, shape: core._check_step(state, None, state.shape[0], (), shape)  # noqa: E731
    wide = torch.zeros(3, 4, 8)
    check(wide[:, 1:2], (1, 8))                           # one row of a longer window
    check(torch.zeros(3, 8, 2)[:, :, :1].transpose(1, 2).transpose(1, 2)[:, :1], (1, 1))
    check(torch.zeros(3, 8, 1), (8, 1))
    check(torch.zeros(8, 3, 1).as_strided((3, 1, 8), (8, 3, 1)), (1, 8))
    check(wide[:, 1:3], (2, 8))
    check(torch.zeros(6, 4, 8)[::2], (4, 8))
    for state, shape in ((wide[:, ::2], (2, 8)), (wide[..., :4], (4, 4)), (wide.transpose(1, 2), (8, 4)),
                         (torch.zeros(3, 8, 2)[:, :, :1], (8, 1)), (torch.zeros(1, 1, 8).expand(3, 1, 8), (1, 8)),
                         (torch.zeros(3, 1, 16)[..., ::2], (1, 8))):
        with pytest.raises(ValueError):
            check(state, shape)


def test_shapes_that_are_no_batches():
    for x in (torch.zeros(()), torch.zeros(8), torch.zeros(2, 3, 4, 8)):
        with pytest.raises(ValueError, match=r"\[B, L, D\]"):
            ops.causal_conv1d(x, torch.zeros(8, 3))
        with pytest.raises(ValueError, match=r"\[B, L, D\]"):
            ops.selective_scan(x, x, torch.zeros(8, 4), torch.zeros(1, 4, 4), torch.zeros(1, 4, 4))
