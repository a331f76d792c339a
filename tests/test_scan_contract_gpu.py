"""GPU: what a caller of the selective scan and the causal convolution may rely on beside their
values at ordinary inputs."""

import math

import pytest
import torch

import ops
import scan_reference as R
from forecaster import SelectiveScanLayer
from test_selective_scan_gpu import call, make

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


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


# ------------------------------------------------------------------------------ non-finite values
def nonfinite_gradients(dtype, N, G, tensor, value, at, L=60):
    """Gradients of a dense call with one non-finite value at token `at`, and of the same call
    without it, on the device and from the 64-bit form."""
    got = {}
    for bad in (False, True):
        t = make(1, L, 20, N, G, dtype, 12)
        dy = torch.randn(1, L, 20, generator=torch.Generator().manual_seed(5)).to(dtype)
        if bad:
            (dy if tensor == "dy" else t[tensor])[0, at, 3] = value
        leaves = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
        ref = {k: v.double().requires_grad_(True) for k, v in t.items()}
        y = call(leaves, final=False)
        ry, _ = R.selective_scan(*(ref[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")), True)
        got[bad] = ([g.cpu() for g in torch.autograd.grad(y, [leaves[k] for k in ("B", "C")], dy.to(DEV))],
                    torch.autograd.grad(ry, [ref[k] for k in ("B", "C")], dy.double()))
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,G", [(3, 1), (8, 1), (16, 2), (32, 1), (40, 1), (100, 1)])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("at", [0, 22, 25])
def test_a_nonfinite_token_stays_out_of_its_neighbours_sums(dtype, N, G, value, at):
    """dB and dC of the tokens that a non-finite input does not enter equal those without it: u
    enters dB at its own token and dC from there on; dy enters dC at its own token and dB up
    to there. Where an infinite product is the only one of its sum, the sum is that infinity."""
    for tensor in ("u", "dy"):
        runs = nonfinite_gradients(dtype, N, G, tensor, value, at)
        (dB0, dC0), _ = runs[False]
        (dB, dC), (rB, rC) = runs[True]
        t = torch.arange(60)
        cleanB, cleanC = (t != at, t < at) if tensor == "u" else (t > at, t != at)
        assert torch.equal(dB[:, cleanB], dB0[:, cleanB]) and torch.equal(dC[:, cleanC], dC0[:, cleanC])
        own = 0 if G == 1 else 3 // (20 // G)  # the group of channel 3
        for g, r, clean in ((dB, rB, cleanB), (dC, rC, cleanC)):
            assert not bool(torch.isfinite(g[0, at, own]).any())
            if math.isinf(value):
                r = r.to(dtype).float()
                assert torch.equal(g[0, at, own].float().sign(), r[0, at, own].sign())
                assert torch.equal(g[0, at].isnan(), r[0, at].isnan())


# ------------------------------------------------------------------------------ precision
def test_bf16_sums_over_channels_round_as_fp32_ones():
    """dB and dC of bf16 inputs beside the 64-bit values rounded once. A value falls to the other
    side of a rounding border with the probability of its error over the step, 2^-8 of the value
    at least. The recurrence's and the sums' fp32 errors of some 2^-22 of the terms, ten times that
    of a sum in which random signs cancel, give 0.1 %; 0.5 % are allowed (summands rounded to 11
    bits: 9 %)."""
    t = make(4, 100, 64, 16, 1, torch.bfloat16, 31)
    leaves = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    ref = {k: v.double().requires_grad_(True) for k, v in t.items()}
    dy = torch.randn(4, 100, 64, generator=torch.Generator().manual_seed(5)).bfloat16()
    y = call(leaves, final=False)
    ry, _ = R.selective_scan(*(ref[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")), True)
    got = torch.autograd.grad(y, [leaves["B"], leaves["C"]], dy.to(DEV))
    want = torch.autograd.grad(ry, [ref["B"], ref["C"]], dy.double())
    for g, w in zip(got, want):
        assert float((g.cpu() != w.bfloat16()).double().mean()) <= 5e-3


# ------------------------------------------------------------------------------ long sums
@pytest.mark.parametrize("N", [1, 8, 16])
def test_sums_over_long_rows(N):
    """dD = sum u dy and dbias = sum ddelta over 256 rows of 20000 equal tokens, which are not split
    (the rows fill the device), against 64-bit sums of the same fp32 terms. Adding n terms of one
    sign one after another is off by n / 2 half steps of 2^-24 at worst, and equal terms come near
    that. A thread's sums are of at most 32 terms, 20000 / 32 of which are added in turn, and the
    rows' sum is of 16 and 16: 16 + 313 + 16."""
    B, L, D = 256, 20000, 4
    full = lambda *s, v: torch.full(s, v, device=DEV)  # noqa: E731
    t = {"u": full(B, L, D, v=1 / 3), "delta": full(B, L, D, v=0.05), "A": -torch.arange(1, N + 1, device=DEV).expand(D, N).float(),
         "B": full(B, L, 1, N, v=0.7), "C": full(B, L, 1, N, v=0.3), "D": full(D, v=1.0), "bias": full(D, v=0.0)}
    leaves = {k: t[k].requires_grad_(True) for k in ("delta", "D", "bias")}
    y = call(t, softplus=False, final=False)
    dy = full(B, L, D, v=0.1)
    ddelta, dD, dbias = torch.autograd.grad(y, list(leaves.values()), dy)
    for got, terms in ((dD, t["u"].double() * dy.double()), (dbias, ddelta.double())):
        want = terms.sum((0, 1))
        assert float(((got.double() - want) / want).abs().max()) <= (16 + 313 + 16) * 2.0**-24


# ------------------------------------------------------------------------------ autograd
def test_gradients_of_a_graph_and_of_casts():
    """With create_graph the gradients are the same and have none themselves (torch's once_differentiable
    says so where the upstream gradient has one); parameters in 16 bits and transposed inputs
    get gradients of their own type and order."""
    t = on_device(make(2, 12, 8, 4, 1, torch.float32, 3))
    x, A = t["u"].requires_grad_(True), t["A"].requires_grad_(True)
    w = torch.randn(8, 3, device=DEV).bfloat16().requires_grad_(True)
    b = torch.randn(8, device=DEV).half().requires_grad_(True)
    xt = t["z"].transpose(1, 2).contiguous().transpose(1, 2).requires_grad_(True)
    for f, leaves in ((lambda: call(t, final=False), [x, A]),
                      (lambda: ops.causal_conv1d(x, w, b, "silu"), [x, w, b]),
                      (lambda: ops.causal_conv1d(xt, w, b, "silu"), [xt, w, b])):
        y = f()
        dy = torch.randn_like(y)
        plain = torch.autograd.grad(y, leaves, dy)
        graph = torch.autograd.grad(f(), leaves, dy.clone().requires_grad_(True), create_graph=True)
        assert all(torch.equal(p, g) and p.dtype == v.dtype for p, g, v in zip(plain, graph, leaves))
        with pytest.raises(RuntimeError, match="differentiate twice"):
            graph[0].float().sum().backward()
    want = torch.autograd.grad(ops.causal_conv1d(xt.detach().contiguous().requires_grad_(True), w, b, "silu"), [w, b], dy)
    assert all(torch.equal(p, q) for p, q in zip(plain[1:], want))


def test_an_output_or_a_final_state_alone():
    """Gradients where only one of the two outputs has one."""
    t = on_device(make(2, 12, 8, 4, 1, torch.float32, 3, 2))
    leaves = {k: v.requires_grad_(True) for k, v in t.items()}
    both = lambda: call(leaves)  # noqa: E731
    conv_init = torch.randn(2, 2, 8, device=DEV, requires_grad=True)
    w = torch.randn(8, 3, device=DEV, requires_grad=True)
    conv = lambda: ops.causal_conv1d(leaves["u"], w, None, "silu", conv_init, None, True)  # noqa: E731
    for f, ins in ((both, list(leaves.values())), (conv, [leaves["u"], w, conv_init])):
        y, fin = f()
        dy, df = torch.randn_like(y), torch.randn_like(fin)
        sums = torch.autograd.grad([y, fin], ins, [dy, df])
        alone = (torch.autograd.grad(f()[i], ins, g, allow_unused=True) for i, g in enumerate((dy, df)))
        for s, p, q in zip(sums, *alone):
            p, q = (torch.zeros_like(s) if v is None else v for v in (p, q))
            assert R.rel(p + q, s) <= 2.0**-20


# ------------------------------------------------------------------------------ the layer
def test_the_layer_asks_for_states_only_where_they_are_wanted(monkeypatch):
    asked = []
    for name in ("causal_conv1d", "selective_scan"):
        f = getattr(ops, name)
        monkeypatch.setattr(ops, name, lambda *a, f=f: asked.append(a[-1]) or f(*a))
    torch.manual_seed(0)
    m = SelectiveScanLayer(16, act_dtype=torch.float32).to(DEV)
    h = torch.randn(2, 9, 16, device=DEV)
    out = m(h)
    again, (rows, state) = m(h, return_state=True)
    assert asked == [False, False, True, True]
    assert torch.equal(out, again) and rows.shape == (2, 3, 32) and state.shape == (2, 32, 16)
