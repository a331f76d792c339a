"""GPU: what a caller of the selective scan and the causal convolution may rely on beside their
values at ordinary inputs."""

import pytest
import torch

import ops
import scan_reference as R
from test_selective_scan_gpu import call, make

pytestmark = pytest.mark.gpu
DEV = "cuda"


def on_device(t):
    return {k: v.to(DEV) for k, v in t.items()}


# ------------------------------------------------------------------------------ in-place steps
@pytest.mark.parametrize("seqs", [None, [0, 5, 9]])
def test_a_step_on_a_saved_state_is_seen_by_autograd(seqs):
    """A state that a differentiable call has saved and a step then changed: its backward raises,
    as after any in-place operation of torch, for both operators."""
    t = on_device(make(1 if seqs else 2, 9, 8, 4, 1, torch.float32, 3, 2))
    cu = torch.tensor(seqs, device=DEV, dtype=torch.int32) if seqs else None
    state = t["init"]
    t["u"].requires_grad_(True)
    y, _ = call(t, cu=cu)
    tok = lambda k: t[k][:1, 0].detach().expand(2, *t[k].shape[2:])  # noqa: E731
    before = state._version
    ops.selective_scan_step(state, tok("u"), tok("delta"), t["A"], tok("B"), tok("C"))
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()

    x, w, rows = t["u"].detach().requires_grad_(True), torch.randn(8, 3, device=DEV), torch.randn(2, 2, 8, device=DEV)
    y = ops.causal_conv1d(x, w, activation="silu", initial_state=rows, cu_seqlens=cu)
    before = rows._version
    ops.causal_conv1d_step(x[:1, 0].detach().expand(2, 8), rows, w)
    assert rows._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_steps_in_inference_mode():
    """States made in inference mode count no changes; steps on them work."""
    with torch.inference_mode():
        t = on_device(make(2, 1, 8, 4, 1, torch.float32, 3, 2))
        tok = lambda k: t[k][:, 0]  # noqa: E731
        state, want = t["init"].clone(), t["init"].clone()
        ops.selective_scan_step(state, tok("u"), tok("delta"), t["A"], tok("B"), tok("C"))
        _, fin = ops.selective_scan(t["u"], t["delta"], t["A"], t["B"], t["C"], initial_state=want,
                                    return_final_state=True)
        assert R.rel(state, fin) <= 2.0**-20
        rows = torch.zeros(2, 2, 8, device=DEV)
        ops.causal_conv1d_step(tok("u"), rows, torch.ones(8, 3, device=DEV))
        assert torch.equal(rows[:, 1], tok("u"))


def test_a_step_on_one_row_of_a_longer_window():
    """A two-tap filter's state as a slice of a wider one: that row is updated, the others are not."""
    wide, x, w = (torch.randn(*s, device=DEV) for s in ((3, 4, 24), (3, 24), (24, 2)))
    want, before = wide[:, 1:2].clone(), wide.clone()
    y = ops.causal_conv1d_step(x, want, w)
    assert torch.equal(ops.causal_conv1d_step(x, wide[:, 1:2], w), y)
    assert torch.equal(wide[:, 1:2], want)
    assert torch.equal(wide[:, [0, 2, 3]], before[:, [0, 2, 3]])
