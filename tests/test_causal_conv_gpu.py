"""GPU: the causal convolution and its single-token step against a plain 64-bit form.

Tolerances (relative L2): K + 1 fp32 operations and the sigmoid's few steps, 16 * 2^-24, and
for gradients summed over M tokens M * 2^-24 of the terms' size, where random signs make the
sum up to sqrt(M) smaller: 2^-24 * (16 + 4 sqrt(M)). 16-bit outputs are rounded once more.
"""

import math

import pytest
import torch

import ops
import scan_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def tol(dtype, M):
    t = 2.0**-24 * (16 + 4 * math.sqrt(M))
    return t if dtype == torch.float32 else t + torch.finfo(dtype).eps / 2


def make(B, L, D, K, dtype, seed, nseq=None, bias=True):
    g = torch.Generator().manual_seed(seed)
    t = {"x": torch.randn(B, L, D, generator=g).to(dtype), "w": torch.randn(D, K, generator=g) * 0.5}
    if bias:
        t["b"] = torch.randn(D, generator=g) * 0.2
    if nseq is not None:
        t["init"] = torch.randn(nseq, K - 1, D, generator=g).to(dtype)
    return t


def call(t, act, cu=None, final=True):
    return ops.causal_conv1d(t["x"], t["w"], t.get("b"), act, t.get("init"), cu, final)


def check(t, dtype, act, cu=None):
    B, L, D = t["x"].shape
    dev = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    ref = {k: v.double().requires_grad_(True) for k, v in t.items()}
    y, fin = call(dev, act, torch.tensor(cu, device=DEV, dtype=torch.int32) if cu is not None else None)
    ry, rfin = R.causal_conv1d(ref["x"], ref["w"], ref.get("b"), act == "silu", ref.get("init"), cu)
    assert y.dtype == dtype and fin.dtype == dtype
    assert R.rel(y, ry) <= tol(dtype, 1)
    assert R.rel(fin, rfin) == 0  # rows are copied
    g = torch.Generator().manual_seed(L + D)
    dy, dfin = torch.randn(y.shape, generator=g).to(dtype), torch.randn(fin.shape, generator=g).to(dtype)
    names = list(t)
    got = torch.autograd.grad([y, fin], [dev[k] for k in names], [dy.to(DEV), dfin.to(DEV)], allow_unused=True)
    want = torch.autograd.grad([ry, rfin], [ref[k] for k in names], [dy.double(), dfin.double()], allow_unused=True)
    for k, a, b in zip(names, got, want):
        assert a.dtype == t[k].dtype
        err = R.rel(a, b if b is not None else torch.zeros_like(ref[k]))
        assert err <= tol(a.dtype, B * L), f"d{k}: {err:.2e}"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [2, 3, 4])
@pytest.mark.parametrize("B,L,D,act", [(1, 1, 1, "silu"), (2, 2, 5, None), (3, 3, 8, "silu"), (2, 19, 33, "silu"),
                                       (1, 150, 64, None), (2, 131, 260, "silu")])
def test_outputs_and_gradients(dtype, K, B, L, D, act):
    check(make(B, L, D, K, dtype, L * D + K, B), dtype, act)
    check(make(B, L, D, K, dtype, L * D + K + 1, None, bias=False), dtype, act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [2, 3, 4])
@pytest.mark.parametrize("D,cu", [(40, [0, 7, 7, 8, 40, 61]), (9, [0, 1, 2, 3, 3]), (16, [0, 0, 15, 17, 18, 33, 33]),
                                  (24, [0, 16, 32, 150])])
@pytest.mark.parametrize("init,behind", [(True, 0), (False, 0), (True, 20)])
def test_packed_sequences(dtype, K, D, cu, init, behind):
    """Empty sequences, ones shorter than the filter, cuts at and beside the runs' ends, tokens
    behind the last one (zero outputs, zero gradients)."""
    check(make(1, cu[-1] + behind, D, K, dtype, cu[-1] + D + K, len(cu) - 1 if init else None), dtype, "silu", cu)


def test_rows_behind_the_last_sequence_stay_out():
    t = {k: v.to(DEV) for k, v in make(1, 40, 24, 4, torch.float32, 3, 2).items()}
    t["x"][:, 30:] = float("nan")
    leaves = {k: v.requires_grad_(True) for k, v in t.items()}
    y, fin = call(leaves, "silu", torch.tensor([0, 11, 30], device=DEV, dtype=torch.int32))
    assert float(y[:, 30:].detach().abs().max()) == 0 and bool(torch.isfinite(fin).all())
    dy = torch.randn(y.shape, device=DEV)
    dy[:, 30:] = float("nan")
    for g in torch.autograd.grad([y, fin], list(leaves.values()), [dy, torch.ones_like(fin)]):
        assert bool(torch.isfinite(g).all())


def test_empty_inputs():
    for B, L in ((0, 5), (2, 0)):
        t = {k: v.to(DEV).requires_grad_(True) for k, v in make(B, L, 6, 4, torch.float32, 1, B).items()}
        y, fin = call(t, "silu")
        assert y.shape == (B, L, 6) and torch.equal(fin, t["init"])
        for (k, v), g in zip(t.items(), torch.autograd.grad([y, fin], list(t.values()),
                                                            [torch.ones_like(y), torch.ones_like(fin)])):
            assert g.shape == v.shape


@pytest.mark.parametrize("offset", [0, 1, 8])
def test_views_of_a_wider_projection(offset):
    t = {k: v.to(DEV) for k, v in make(2, 77, 64, 4, torch.bfloat16, 7).items()}
    wide = torch.randn(2, 77, 64 + 24, device=DEV, dtype=torch.bfloat16)
    wide[..., offset:offset + 64] = t["x"]
    leaves = [t["x"].requires_grad_(True), wide[..., offset:offset + 64].detach().requires_grad_(True)]
    ys = [call({**t, "x": x}, "silu", final=False) for x in leaves]
    assert torch.equal(ys[0], ys[1])
    dy = torch.randn_like(ys[0])
    assert torch.equal(*(torch.autograd.grad(y, x, dy)[0] for y, x in zip(ys, leaves)))


def test_gradients_against_differences():
    """Central differences of the kernel's forward along each gradient: the loss is smooth to the
    scale of the step, error about eps^2 + 2^-22 / eps: 5e-3 at 1e-2."""
    t = {k: v.to(DEV) for k, v in make(2, 35, 12, 4, torch.float32, 21, 2).items()}
    w = torch.randn(2, 35, 12, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))

    def loss(v):
        return (call(v, "silu", final=False).double() * w).sum()

    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    loss(leaves).backward()
    for k in t:
        grad = leaves[k].grad
        d, eps = grad / grad.norm(), 1e-2
        num = (loss({**t, k: t[k] + eps * d}) - loss({**t, k: t[k] - eps * d})) / (2 * eps)
        assert abs(float(num) - float(grad.double().norm())) <= 5e-3 * float(grad.norm()), k


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("K", [2, 3, 4])
def test_step_continues_a_prompt(dtype, K):
    B, L, P, D = 3, 9, 2, 37
    t = make(B, L, D, K, dtype, K, B)
    ry, rfin = R.causal_conv1d(t["x"].double(), t["w"].double(), t["b"].double(), True, t["init"].double())
    dev = {k: v.to(DEV) for k, v in t.items()}
    y, state = call({**dev, "x": dev["x"][:, :P]}, "silu")
    ys = [y]
    for i in range(P, L):
        ys.append(ops.causal_conv1d_step(dev["x"][:, i], state, dev["w"], dev["b"], "silu")[:, None])
    assert R.rel(torch.cat(ys, 1), ry) <= tol(dtype, 1)
    assert R.rel(state, rfin) == 0


def test_step_slots():
    B, D, K, S = 6, 150, 4, 9
    t = {k: v.to(DEV) for k, v in make(B, 1, D, K, torch.bfloat16, 2).items()}
    state = torch.randn(S, K - 1, D, device=DEV).to(torch.bfloat16)
    idx = torch.tensor([7, -1, 2, S, 2, 0], device=DEV, dtype=torch.int32)
    got = state.clone()
    y = ops.causal_conv1d_step(t["x"][:, 0], got, t["w"], t["b"], "silu", idx)
    good = torch.tensor([0, 2, 5], device=DEV)
    slots = idx[good].long()
    sub = state[slots].clone()
    yr = ops.causal_conv1d_step(t["x"][good, 0], sub, t["w"], t["b"], "silu")
    want = state.clone()
    want[slots] = sub
    assert torch.equal(got, want) and torch.equal(y[good], yr)
    assert float(y[1].abs().max()) == 0 and bool(y[3].isnan().all()) and bool(y[4].isnan().all())


def test_captured_and_replayed():
    t = {k: v.to(DEV) for k, v in make(2, 100, 64, 4, torch.bfloat16, 4, 2).items()}
    dy = torch.randn(2, 100, 64, device=DEV).to(torch.bfloat16)

    def train():
        leaves = {k: x.detach().requires_grad_(True) for k, x in t.items()}
        y = call(leaves, "silu", final=False)
        return (y, *torch.autograd.grad(y, list(leaves.values()), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = train()
    for k, v in make(2, 100, 64, 4, torch.bfloat16, 5, 2).items():
        t[k].copy_(v)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, train()))
