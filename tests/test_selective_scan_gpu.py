"""GPU: the selective scan and its single-token step against a plain 64-bit form.

Tolerances (relative L2). fp32: a step's decay is off by the exponential's 2^-22 and its
argument's rounding, and the errors of up to L steps add, so L * 2^-21 for values carried by the
recurrence; sums over D channels, N states or M = B * L tokens add (D + N) * 2^-23 resp.
M * 2^-24 of their terms' size, which random signs make up to sqrt of the count larger than the
sum: 8 * 2^-24 * (L + D + N) covers both at these sizes. 16-bit outputs are rounded once, half a
step of their type, on top. dB and dC of bf16 inputs are sums of products whose two factors
are rounded to tensor-core operands of 11 bits: 2^-10 of a product's size more.
"""

import pytest
import torch

import ops
import scan_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def tol32(L, D, N):
    return L * 2.0**-21 + 8 * 2.0**-24 * (L + D + N)


def tol(dtype, L, D, N, product=False):
    base = tol32(L, D, N)
    if dtype == torch.float32:
        return base
    return torch.finfo(dtype).eps / 2 + base + (2.0**-10 if product and dtype == torch.bfloat16 else 0)


def make(B, L, D, N, G, dtype, seed, nseq=None, z=True, skip=True, bias=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, k=1.0: torch.randn(*s, generator=g) * k  # noqa: E731
    t = {"u": r(B, L, D).to(dtype), "delta": r(B, L, D, k=0.5).to(dtype),
         "A": -torch.arange(1, N + 1).float() * (1 + 0.2 * torch.rand(D, N, generator=g)),
         "B": r(B, L, G, N, k=0.7).to(dtype), "C": r(B, L, G, N, k=0.7).to(dtype)}
    if skip:
        t["D"] = 1 + r(D, k=0.2)
    if z:
        t["z"] = r(B, L, D).to(dtype)
    if bias:
        t["bias"] = r(D) - 2.0
    if nseq is not None:
        t["init"] = r(nseq, D, N, k=0.5)
    return t


def call(t, softplus=True, cu=None, final=True):
    return ops.selective_scan(t["u"], t["delta"], t["A"], t["B"], t["C"], t.get("D"), t.get("z"), t.get("bias"),
                              softplus, initial_state=t.get("init"), cu_seqlens=cu, return_final_state=final)


def check(t, dtype, softplus=True, cu=None, seed=0):
    """Outputs, final states and every gradient (through both) against the 64-bit form."""
    B, L, D = t["u"].shape
    N = t["A"].shape[1]
    dev = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    ref = {k: v.double().requires_grad_(True) for k, v in t.items()}
    cud = torch.tensor(cu, device=DEV, dtype=torch.int32) if cu is not None else None
    y, fin = call(dev, softplus, cud)
    ry, rfin = R.selective_scan(ref["u"], ref["delta"], ref["A"], ref["B"], ref["C"], ref.get("D"), ref.get("z"),
                                ref.get("bias"), softplus, ref.get("init"), cu)
    assert y.dtype == dtype and fin.dtype == torch.float32
    assert R.rel(y, ry) <= tol(dtype, L, D, N)
    assert R.rel(fin, rfin) <= tol32(L, D, N)
    g = torch.Generator().manual_seed(seed + 77)
    dy, dfin = torch.randn(y.shape, generator=g).to(dtype), torch.randn(fin.shape, generator=g)
    names = list(t)
    got = torch.autograd.grad([y, fin], [dev[k] for k in names], [dy.to(DEV), dfin.to(DEV)])
    want = torch.autograd.grad([ry, rfin], [ref[k] for k in names], [dy.double(), dfin.double()])
    for k, a, b in zip(names, got, want):
        assert a.dtype == t[k].dtype, k
        err = R.rel(a, b)
        assert err <= tol(a.dtype, L, D, N, k in ("B", "C")), f"d{k}: {err:.2e}"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,L,D,N,G", [
    (1, 1, 1, 1, 1), (2, 3, 5, 1, 1), (2, 17, 33, 4, 1), (1, 40, 130, 5, 2), (3, 65, 40, 8, 1), (2, 70, 66, 16, 1),
    (1, 129, 34, 16, 2), (2, 50, 24, 20, 3), (1, 33, 70, 32, 1), (2, 19, 9, 40, 1), (1, 37, 36, 64, 1),
    (1, 21, 10, 100, 1), (1, 11, 34, 128, 2)])
def test_outputs_and_gradients(dtype, B, L, D, N, G):
    check(make(B, L, D, N, G, dtype, seed=L * D + N, nseq=B), dtype, seed=N)


@pytest.mark.parametrize("z,skip,bias,softplus", [(False, True, True, True), (True, False, True, True),
                                                  (True, True, False, False), (False, False, False, True)])
def test_optional_inputs(z, skip, bias, softplus):
    t = make(2, 21, 37, 16, 1, torch.float32, 5, None, z, skip, bias)
    if not softplus:
        t["delta"] = t["delta"].abs()
    check(t, torch.float32, softplus)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,N,cu", [
    (40, 16, [0, 7, 7, 8, 40, 61]), (9, 8, [0, 1, 2, 3, 3]), (33, 4, [0, 0, 31, 33, 33]), (20, 40, [0, 16, 32, 50]),
    (70, 16, [0, 16, 48, 49, 60])])
@pytest.mark.parametrize("init,behind", [(True, 0), (False, 0), (True, 9)])
def test_packed_sequences(dtype, D, N, cu, init, behind):
    """Empty and one-token sequences, cuts at and inside tiles, tokens behind the last one."""
    check(make(1, cu[-1] + behind, D, N, 1, dtype, cu[-1] + D, len(cu) - 1 if init else None), dtype, cu=cu)


@pytest.mark.parametrize("cu", [None, [0, 100, 101, 700, 900]])
def test_split_time_axis(cu):
    """Few channels and a long axis: pieces, joined by the states that enter them; one sequence
    spans several pieces and several lie in one."""
    check(make(1, 900, 6, 16, 1, torch.float32, 3, len(cu) - 1 if cu else 1), torch.float32, cu=cu)
    check(make(2, 515, 5, 40, 1, torch.bfloat16, 4, 2), torch.bfloat16)


def test_rows_behind_the_last_sequence_stay_out():
    """NaN in tokens of no sequence reaches nothing, and their outputs and gradients are zero."""
    t = make(1, 50, 20, 16, 1, torch.float32, 8, 2)
    cu = torch.tensor([0, 13, 41], device=DEV, dtype=torch.int32)
    for k in ("u", "delta", "z", "B", "C"):
        t[k][:, 41:] = float("nan")
    dev = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    y, fin = call(dev, cu=cu)
    assert float(y[:, 41:].abs().max().detach()) == 0 and bool(torch.isfinite(fin).all())
    dy = torch.randn(y.shape, device=DEV)
    dy[:, 41:] = float("nan")
    for k, g in zip(dev, torch.autograd.grad([y, fin], list(dev.values()), [dy, torch.randn_like(fin)])):
        assert bool(torch.isfinite(g).all()), k
        if g.dim() >= 3 and g.shape[1] == 50:
            assert float(g[:, 41:].abs().max()) == 0, k


def test_empty_inputs():
    for B, L in ((0, 5), (2, 0)):
        t = {k: v.to(DEV).requires_grad_(True) for k, v in make(B, L, 6, 4, 1, torch.float32, 1, B).items()}
        y, fin = call(t)
        assert y.shape == (B, L, 6)
        assert torch.equal(fin, t["init"])
        grads = torch.autograd.grad([y, fin], list(t.values()), [torch.ones_like(y), torch.ones_like(fin)])
        for (k, v), g in zip(t.items(), grads):
            assert g.shape == v.shape and (k == "init" or float(g.abs().sum()) == 0)
    t = {k: v.to(DEV) for k, v in make(1, 0, 6, 4, 1, torch.float32, 1, 3).items()}
    y, fin = call(t, cu=torch.zeros(4, device=DEV, dtype=torch.int32))
    assert torch.equal(fin, t["init"])


def test_views_of_a_wider_projection():
    """u, z, delta, B and C as slices at odd offsets of one matrix, and a transposed u."""
    B, L, D, N = 2, 30, 24, 10
    t = make(B, L, D, N, 1, torch.bfloat16, 9)
    wide = torch.randn(B, L, 3 * D + 2 * N + 1, device=DEV, dtype=torch.bfloat16)
    at, v = 1, {}
    for k, n in (("u", D), ("delta", D), ("z", D), ("B", N), ("C", N)):
        wide[..., at:at + n] = t[k].reshape(B, L, n).to(DEV)
        v[k] = wide[..., at:at + n]
        at += n
    rest = {k: t[k].to(DEV) for k in ("A", "D", "bias")}
    y0, f0 = call({k: x.to(DEV) for k, x in t.items()})
    y1, f1 = call({**v, **rest})
    assert torch.equal(y0, y1) and torch.equal(f0, f1)
    ut = t["u"].to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    y2, _ = call({**v, **rest, "u": ut})
    assert torch.equal(y0, y2)


def test_decays_at_the_ends():
    """Step sizes that keep or forget everything, and decays that underflow."""
    t = make(1, 40, 8, 16, 1, torch.float32, 11, 1, bias=False)
    t["delta"] = torch.full_like(t["delta"], -100.0)   # softplus 0: the state stays
    dev = {k: v.to(DEV) for k, v in t.items()}
    _, fin = call(dev)
    assert torch.equal(fin, dev["init"])
    t["delta"] = torch.full_like(t["delta"], 1e4)      # the state is forgotten at once
    check(t, torch.float32)


def test_gradients_against_differences():
    """Directional derivatives of a fp32 loss by central differences of the kernel's own forward.
    The difference's own error is about eps^2 + 2^-22 / eps of the loss's scale: 5e-3 at 1e-2."""
    t = {k: v.to(DEV) for k, v in make(2, 33, 12, 16, 1, torch.float32, 21, 2).items()}
    g = torch.Generator(device=DEV).manual_seed(3)
    w = None

    def loss(v):
        nonlocal w
        y, fin = call(v)
        if w is None:
            w = torch.randn(y.shape, generator=g, device=DEV), torch.randn(fin.shape, generator=g, device=DEV)
        return (y.double() * w[0]).sum() + (fin.double() * w[1]).sum()

    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    loss(leaves).backward()
    for k in t:
        grad = leaves[k].grad
        d = grad / grad.norm()
        eps = 1e-2
        num = (loss({**t, k: t[k] + eps * d}) - loss({**t, k: t[k] - eps * d})) / (2 * eps)
        assert abs(float(num) - float(grad.double().norm())) <= 5e-3 * float(grad.norm()), k


def test_results_repeat():
    t = {k: v.to(DEV).requires_grad_(True) for k, v in make(2, 200, 96, 16, 1, torch.bfloat16, 31).items()}
    once = torch.autograd.grad(call(t, final=False).float().square().sum(), list(t.values()))
    for _ in range(2):
        again = torch.autograd.grad(call(t, final=False).float().square().sum(), list(t.values()))
        assert all(torch.equal(a, b) for a, b in zip(once, again))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,D,N,G", [(1, 1, 1, 1), (3, 40, 16, 1), (5, 130, 8, 2), (2, 33, 5, 1), (4, 66, 40, 3),
                                     (2, 17, 64, 1), (3, 12, 128, 1)])
def test_step_continues_a_scan(dtype, B, D, N, G):
    """Steps after a prompt equal the scan over the whole sequence."""
    L, P = 6, 3
    t = make(B, L, D, N, G, dtype, D + N, B)
    ry, rfin = R.selective_scan(*(t[k].double() for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")), True,
                                t["init"].double())
    dev = {k: v.to(DEV) for k, v in t.items()}
    y, state = call({**dev, **{k: dev[k][:, :P] for k in ("u", "delta", "B", "C", "z")}})
    ys = [y]
    for i in range(P, L):
        s = {k: dev[k][:, i] for k in ("u", "delta", "B", "C", "z")}
        ys.append(ops.selective_scan_step(state, s["u"], s["delta"], dev["A"], s["B"], s["C"], dev["D"], s["z"],
                                          dev["bias"], True)[:, None])
    assert R.rel(torch.cat(ys, 1), ry) <= tol(dtype, L, D, N)
    assert R.rel(state, rfin) <= tol32(L, D, N)


def test_step_slots():
    """Slots in any order, rows left out, one past the end, one used twice."""
    B, D, N, S = 6, 40, 16, 9
    t = {k: v.to(DEV)[:, 0] if v.dim() > 2 else v.to(DEV)
         for k, v in make(B, 1, D, N, 1, torch.float32, 2).items()}
    state = torch.randn(S, D, N, device=DEV)
    idx = torch.tensor([7, -1, 2, S, 2, 0], device=DEV, dtype=torch.int32)
    step = lambda st, ix, rows: ops.selective_scan_step(  # noqa: E731
        st, t["u"][rows], t["delta"][rows], t["A"], t["B"][rows], t["C"][rows], t["D"], t["z"][rows], t["bias"], True, ix)
    got = state.clone()
    y = step(got, idx, slice(None))
    want = state.clone()
    good = torch.tensor([0, 2, 5], device=DEV)
    slots = idx[good].long()
    sub = state[slots].clone()
    yr = step(sub, None, good)
    want[slots] = sub
    assert torch.equal(got, want) and torch.equal(y[good], yr)
    assert float(y[1].abs().max()) == 0
    assert bool(y[3].isnan().all()) and bool(y[4].isnan().all())
    # a strided state: every other slot of a larger one
    wide = torch.randn(2 * B, D, N, device=DEV)
    ref = wide.clone()
    part = wide[::2]
    yr = step(part, None, slice(None))
    sub = ref[::2].contiguous()
    assert torch.equal(step(sub, None, slice(None)), yr) and torch.equal(sub, part) and torch.equal(ref[1::2], wide[1::2])


def test_captured_and_replayed():
    """Forward, backward and a step in CUDA graphs, replayed on new inputs, beside each other."""
    t = {k: v.to(DEV) for k, v in make(1, 600, 16, 16, 1, torch.bfloat16, 41, 1).items()}
    dy = torch.randn(1, 600, 16, device=DEV).to(torch.bfloat16)
    names = list(t)

    def train(v):
        leaves = {k: x.detach().requires_grad_(True) for k, x in v.items()}
        y, fin = call(leaves)
        return (y, fin, *torch.autograd.grad([y, fin], [leaves[k] for k in names], [dy, torch.ones_like(fin)]))

    state = t["init"].clone()
    step = lambda st: ops.selective_scan_step(st, *(t[k][:, 0] for k in ("u", "delta")), t["A"],  # noqa: E731
                                              t["B"][:, 0], t["C"][:, 0], t["D"], t["z"][:, 0], t["bias"], True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train(t), step(state)
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        outs = train(t)
    with torch.cuda.graph(g2):
        sy = step(state)
    new = make(1, 600, 16, 16, 1, torch.bfloat16, 42, 1)
    for k in names:
        t[k].copy_(new[k])
    state.copy_(t["init"])
    want_state = state.clone()
    with torch.no_grad():
        want_y = step(want_state)
    for _ in range(2):
        state.copy_(t["init"])
        other = torch.cuda.Stream()
        other.wait_stream(torch.cuda.current_stream())
        g1.replay()
        with torch.cuda.stream(other):
            g2.replay()
        torch.cuda.current_stream().wait_stream(other)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, train(t)))
        assert torch.equal(sy, want_y) and torch.equal(state, want_state)


def test_two_streams_at_once():
    ts = [{k: v.to(DEV) for k, v in make(1, 700, 24, 16, 1, torch.float32, s, 1).items()} for s in (1, 2)]
    want = [call(t) for t in ts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ts]
    got = []
    for t, s in zip(ts, streams):
        with torch.cuda.stream(s):
            got.append([call(t) for _ in range(4)])
    torch.cuda.synchronize()
    for w, gs in zip(want, got):
        assert all(torch.equal(a, b) for g in gs for a, b in zip(w, g))


def test_refusals():
    t = {k: v.to(DEV) for k, v in make(2, 6, 8, 4, 1, torch.bfloat16, 1).items()}
    good = lambda **kw: {**t, **kw}  # noqa: E731
    for bad in (good(delta=t["delta"][:, :5]), good(A=t["A"][:4]), good(B=t["B"][..., :3]), good(C=t["C"].float()),
                good(D=t["D"][:3]), good(z=t["z"][:1]), good(bias=t["bias"][:2]), good(init=torch.zeros(3, 8, 4, device=DEV)),
                good(B=t["B"].expand(2, 6, 3, 4))):
        with pytest.raises(ValueError):
            call(bad)
    with pytest.raises(ValueError, match="at most 128"):
        call(good(A=torch.zeros(8, 129, device=DEV), B=t["B"][..., :1].expand(2, 6, 1, 129),
                  C=t["C"][..., :1].expand(2, 6, 1, 129)))
    with pytest.raises(TypeError):
        call({k: v.double() for k, v in t.items()})
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        call(good(A=t["A"].cpu()))
    with pytest.raises(ValueError, match="one row"):
        call(t, cu=torch.tensor([0, 6], device=DEV, dtype=torch.int32))
    s = {k: v[:, 0] if v.dim() > 2 else v for k, v in t.items()}
    step = lambda st, ix=None, **kw: ops.selective_scan_step(  # noqa: E731
        st, kw.get("u", s["u"]), s["delta"], s["A"], s["B"], s["C"], s["D"], s["z"], s["bias"], True, ix)
    state = torch.zeros(2, 8, 4, device=DEV)
    for st, ix in ((state.bfloat16(), None), (state[:1], None), (state[..., :3], None), (state.transpose(1, 2), None),
                   (state[:1].expand(2, 8, 4), None), (state, torch.zeros(3, device=DEV, dtype=torch.int32)),
                   (state, torch.zeros(2, device=DEV, dtype=torch.int64))):
        with pytest.raises(ValueError):
            step(st, ix)
    with pytest.raises(RuntimeError, match="no gradient"):
        step(state, u=s["u"].clone().requires_grad_(True))
    assert float(state.abs().max()) == 0


def test_bad_sequence_offsets_stay_in_bounds():
    """Offsets out of order, negative or past the end give some result, and touch nothing else."""
    t = {k: v.to(DEV) for k, v in make(1, 70, 12, 16, 1, torch.float32, 6, 4).items()}
    for cu in ([0, 50, 20, 60, 70], [-5, 10, 10, 200, 300], [70, 60, 30, 10, 0], [5, 9, 12, 40, 41]):
        cud = torch.tensor(cu, device=DEV, dtype=torch.int32)
        leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
        y, fin = call(leaves, cu=cud)
        torch.autograd.grad([y, fin], list(leaves.values()), [torch.ones_like(y), torch.ones_like(fin)])
        ops.causal_conv1d(t["u"], torch.ones(12, 4, device=DEV), cu_seqlens=cud)
    torch.cuda.synchronize()


def test_a_nan_stays_in_its_sequence():
    """A NaN in one packed sequence reaches no output or gradient of the others' tokens."""
    t = make(1, 60, 20, 16, 1, torch.bfloat16, 12, 4)
    t["u"][0, 23, 3] = float("nan")
    leaves = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    cu = torch.tensor([0, 21, 26, 41, 60], device=DEV, dtype=torch.int32)
    y, fin = call(leaves, cu=cu)
    g = torch.autograd.grad([y, fin], [leaves[k] for k in ("u", "delta", "B", "C", "z", "init")],
                            [torch.ones_like(y), torch.ones_like(fin)])
    keep = torch.cat([torch.arange(21), torch.arange(26, 60)]).to(DEV)
    for v in (y, *g[:5]):
        assert bool(torch.isfinite(v[:, keep]).all())
    assert bool(torch.isfinite(fin[[0, 2, 3]]).all()) and bool(torch.isfinite(g[5][[0, 2, 3]]).all())
    assert bool(fin[1].isnan().any())


def test_another_stream_than_the_tensors_own():
    t = {k: v.to(DEV) for k, v in make(2, 300, 24, 16, 1, torch.float32, 17, 2).items()}
    want = call(t)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = call(t)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_parameters_in_16_bits_and_shared_leaves():
    """A, D and the bias in bf16 get bf16 gradients; one tensor as both B and C, and an expanded
    u, add their gradients."""
    t = {k: v.to(DEV) for k, v in make(2, 40, 16, 16, 1, torch.float32, 19).items()}
    for k in ("A", "D", "bias"):
        t[k] = t[k].bfloat16()
    u = t["u"][:1].clone().requires_grad_(True)
    bc = t["B"].clone().requires_grad_(True)
    A = t["A"].requires_grad_(True)
    y = call({**t, "u": u.expand(2, 40, 16), "B": bc, "C": bc, "A": A}, final=False)
    dy = torch.randn_like(y)
    got = torch.autograd.grad(y, [u, bc, A], dy)
    ud, bd, Ad = (x.detach().double().cpu().requires_grad_(True) for x in (u, bc, A))
    c = {k: v.detach().double().cpu() for k, v in t.items()}
    ry, _ = R.selective_scan(ud.expand(2, 40, 16), c["delta"], Ad, bd, bd, c["D"], c["z"], c["bias"], True)
    want = torch.autograd.grad(ry, [ud, bd, Ad], dy.double().cpu())
    for a, b in zip(got, want):
        assert R.rel(a, b) <= tol(a.dtype, 40, 16, 16)


def test_no_states_are_kept_without_a_gradient(monkeypatch):
    """Under no_grad, parameters that require gradients or not, the forward keeps no states."""
    import _scan_core as core

    asked = []
    real = core.selective_scan_forward
    monkeypatch.setattr(core, "selective_scan_forward", lambda *a: asked.append(a[-1]) or real(*a))
    t = {k: v.to(DEV) for k, v in make(1, 20, 8, 4, 1, torch.float32, 1).items()}
    t["A"].requires_grad_(True)
    with torch.no_grad():
        y0, _ = call(t)
    y1, _ = call(t)
    assert asked == [False, True] and not y0.requires_grad and y1.requires_grad and torch.equal(y0, y1)


def test_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    t = {k: v.to("cuda:1") for k, v in make(1, 300, 8, 16, 1, torch.float32, 1, 1).items()}
    y, fin = call(t)
    ry, rfin = call({k: v.to("cuda:0") for k, v in t.items()})
    assert torch.equal(y.cpu(), ry.cpu()) and torch.equal(fin.cpu(), rfin.cpu())
