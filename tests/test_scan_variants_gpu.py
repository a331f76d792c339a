"""GPU: forms of the selective scan's and the causal convolution's kernels that sizes choose and the
small tests do not reach: four rows a CTA in the single-token step, several channel tiles of
every shape, the split time axis of every shape, long runs of the convolution, and what
offsets out of order leave alone.

Tolerances (relative L2). Step sizes are at least softplus(-4) = 0.018 and decays at least 1 here,
so that a state remembers some 55 steps; with 2^-22 of a step's decay (the exponential unit's 2
steps of 2^-23, its argument's rounding below that) a recurrence is off by 128 * 2^-22 = 2^-15
at worst, and a gradient, which has two, by 2^-14. Sums add less at these sizes. 16-bit results
are rounded once, half a step of their type, on top.
"""

import pytest
import torch

import _scan_core as core
import ops
import scan_reference as R
from _lib import check, lib
from test_causal_conv_gpu import tol as conv_tol
from test_selective_scan_gpu import call, make

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def tol(dtype, gradient=False):
    half = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    return half + (2.0**-14 if gradient else 2.0**-15)


def compare(B, L, D, N, G, dtype, cu=None, seed=0):
    nseq = len(cu) - 1 if cu else B
    t = make(B, L, D, N, G, dtype, seed, nseq)
    t["bias"], t["delta"] = t["bias"].clamp(min=-2.5), t["delta"].clamp(min=-1.5)
    dev = {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}
    ref = {k: v.double().requires_grad_(True) for k, v in t.items()}
    y, fin = call(dev, cu=torch.tensor(cu, device=DEV, dtype=torch.int32) if cu else None)
    ry, rfin = R.selective_scan(*(ref[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")), True, ref["init"], cu)
    g = torch.Generator().manual_seed(seed + 1)
    dy, dfin = torch.randn(y.shape, generator=g).to(dtype), torch.randn(fin.shape, generator=g)
    got = torch.autograd.grad([y, fin], list(dev.values()), [dy.to(DEV), dfin.to(DEV)])
    want = torch.autograd.grad([ry, rfin], list(ref.values()), [dy.double(), dfin.double()])
    assert R.rel(y, ry) <= tol(dtype) and R.rel(fin, rfin) <= tol(F32)
    for k, a, b in zip(t, got, want):
        assert R.rel(a, b) <= tol(a.dtype, True), (k, R.rel(a, b))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("D,N,G", [(300, 3, 1), (515, 4, 1), (290, 8, 1), (300, 7, 2), (140, 16, 1), (75, 32, 1),
                                   (70, 40, 1), (132, 64, 2), (70, 128, 1)])
def test_several_channel_tiles(dtype, D, N, G):
    """Every shape with full and partial tiles: sums of dB and dC over warps and tiles."""
    compare(2, 23, D, N, G, dtype, seed=D + N)


SPLITS = [(F32, 3, 1), (BF16, 4, 2), (F16, 8, 1), (F32, 8, 2), (F16, 16, 2), (BF16, 16, 1), (F32, 32, 1), (F16, 40, 1),
          (F32, 40, 2), (BF16, 64, 1), (F32, 100, 1), (F16, 128, 2)]


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("dtype,N,G", SPLITS)
def test_split_time_axis(dtype, N, G, packed):
    """Pieces of every shape, groups and types; sequences that span pieces, lie in one, are empty
    and end where a piece does."""
    B, L, D = 1 if packed else 2, 515, 6
    # both directions are split: the backward whole has one tile's dB and dC and dA, dD, dbias
    assert lib.ttt_selective_scan_fwd_scratch_bytes(B, L, D, G, N) > 0
    assert lib.ttt_selective_scan_bwd_scratch_bytes(B, L, D, G, N) > 4 * (2 * B * L * G * N + B * D * (N + 2))
    compare(B, L, D, N, G, dtype, [0, 3, 128, 128, 300, 470] if packed else None, seed=N)


# ------------------------------------------------------------------------------ single token
def step_inputs(rows, D, N, G, dtype, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    return dict(u=r(rows, D).to(dtype), delta=r(rows, D).to(dtype), A=-torch.rand(D, N, device=DEV, generator=g) - 0.1,
                B=r(rows, G, N).to(dtype), C=r(rows, G, N).to(dtype), D=r(D), z=r(rows, D).to(dtype), delta_bias=r(D))


def step(state, t, rows=slice(None), index=None):
    per_row = {k: t[k][rows] if k in ("u", "delta", "B", "C", "z") else t[k] for k in t}
    return ops.selective_scan_step(state, **per_row, delta_softplus=True, state_indices=index)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,D,N,G", [(257, 1100, 16, 1), (310, 1500, 4, 2), (131, 700, 40, 1), (75, 300, 128, 3)])
def test_steps_of_a_large_batch(dtype, rows, D, N, G):
    """Four rows a CTA, the last ones not four: against 64 bits, and bit for bit against calls of few
    rows, which have one a CTA; with slots, rows left out, bad and repeated ones too."""
    t = step_inputs(rows, D, N, G, dtype)
    few = max(1, 2000 // -(-D // 16) // 4)
    state0 = torch.randn(rows, D, N, device=DEV)
    state, want = state0.clone(), state0.clone()
    y = step(state, t)
    ys = [step(want[i:i + few], t, slice(i, i + few)) for i in range(0, rows, few)]
    assert torch.equal(y, torch.cat(ys)) and torch.equal(state, want)
    d = {k: v.double() for k, v in t.items()}
    wide = lambda v: v.repeat_interleave(D // G, 1)  # noqa: E731
    dt = torch.logaddexp(d["delta"] + d["delta_bias"], torch.zeros((), device=DEV, dtype=torch.float64))
    h = torch.exp(dt[..., None] * d["A"]) * state0.double() + (dt * d["u"])[..., None] * wide(d["B"])
    ry = ((h * wide(d["C"])).sum(-1) + d["D"] * d["u"]) * d["z"] * torch.sigmoid(d["z"])
    assert R.rel(state, h) <= 2.0**-20 and R.rel(y, ry) <= 2.0**-20 + (torch.finfo(dtype).eps / 2 if dtype != F32 else 0)

    slots = rows + 30
    index = torch.randperm(slots, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))[:rows].int()
    index[5], index[6], index[8], index[rows - 1] = -1, slots, -7, 2**31 - 1
    index[14], index[13] = index[12].clone(), index[3].clone()  # inside a group of four, and across groups
    index[rows - 2] = index[0].clone()
    cache = torch.randn(slots, D, N, device=DEV)
    before = cache.clone()
    y = step(cache, t, index=index)
    out, nans = [5, 8], [6, rows - 1, 13, 14, rows - 2]
    good = torch.tensor([i for i in range(rows) if i not in out + nans], device=DEV)
    mine = before[index[good].long()]
    ys = torch.cat([step(mine[i:i + few], t, good[i:i + few]) for i in range(0, len(good), few)])
    assert torch.equal(y[good], ys)
    assert float(y[out].float().abs().max()) == 0 and bool(y[nans].isnan().all())
    before[index[good].long()] = mine
    assert torch.equal(cache, before)


# ------------------------------------------------------------------------------ convolution
def conv_reference(x, w, b, init, cu):
    """64 bits, a sequence at a time, whole sequences at once."""
    K, ys, fins = w.shape[1], [], []
    spans = [(i, 0, x.shape[1], i) for i in range(x.shape[0])] if cu is None else \
        [(0, cu[i], cu[i + 1], i) for i in range(len(cu) - 1)]
    for r, t0, t1, i in spans:
        rows = torch.cat([init[i], x[r, t0:t1]])
        p = b + sum(w[:, k] * rows[k:k + t1 - t0] for k in range(K))
        ys.append(p * torch.sigmoid(p))
        fins.append(rows[t1 - t0:])
    y = torch.stack(ys) if cu is None else torch.cat(ys)[None]
    return torch.nn.functional.pad(y, (0, 0, 0, x.shape[1] - y.shape[1])), torch.stack(fins)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,L,D,K,cu", [
    (16, 700, 4164, 4, None), (8, 700, 4164, 3, None), (4, 700, 4164, 2, None), (16, 700, 1031, 4, None),
    (8, 700, 1031, 2, None), (1, 9300, 4164, 4, [0, 129, 131, 131, 1500, 9000]), (1, 9300, 1031, 3, [0, 127, 128, 9299])])
def test_long_runs_of_the_convolution(dtype, B, L, D, K, cu):
    """Runs of 32, 64 and 128 tokens, vectors of channels and single ones."""
    g = torch.Generator(device=DEV).manual_seed(L + D + K)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    nseq = len(cu) - 1 if cu else B
    t = [r(B, L, D).to(dtype), r(D, K) * 0.5, r(D) * 0.2, r(nseq, K - 1, D).to(dtype)]
    dy, dfin = r(B, L, D).to(dtype), r(nseq, K - 1, D).to(dtype)
    ins = [v.clone().requires_grad_(True) for v in t]
    ref = [v.double().requires_grad_(True) for v in t]
    y, fin = ops.causal_conv1d(ins[0], ins[1], ins[2], "silu", ins[3],
                               torch.tensor(cu, device=DEV, dtype=torch.int32) if cu else None, True)
    ry, rfin = conv_reference(*ref, cu)
    rel = lambda a, b: float(((a.double() - b).norm() / b.norm()).detach())  # noqa: E731
    assert rel(y, ry) <= conv_tol(dtype, 1) and torch.equal(fin.double(), rfin)
    got = torch.autograd.grad([y, fin], ins, [dy, dfin])
    want = torch.autograd.grad([ry, rfin], ref, [dy.double(), dfin.double()])
    for name, a, b in zip(("x", "w", "b", "init"), got, want):
        assert rel(a, b) <= conv_tol(a.dtype, B * L), (name, rel(a, b))


# ------------------------------------------------------------------------------ offsets out of order
class Guarded:
    """Buffers with margins that nothing may write to."""

    def __init__(self):
        self.all = []

    def __call__(self, n, dtype=F32):
        whole = torch.full((n + 4096,), 7.5, device=DEV, dtype=dtype)
        self.all.append((whole, n))
        return whole[2048:2048 + n].data_ptr()

    def check(self):
        for whole, n in self.all:
            assert bool((whole[:2048] == 7.5).all()) and bool((whole[2048 + n:] == 7.5).all())


@pytest.mark.parametrize("N", [4, 16, 40])
@pytest.mark.parametrize("L", [70, 515])
@pytest.mark.parametrize("cu", [[0, 50, 20, 60, 70], [-5, 10, 10, 200, 300], [70, 60, 30, 10, 0], [5, 9, 12, 40, 41],
                                [-2**31, 2**31 - 1, 0, -1, 2**31 - 1]])
def test_offsets_out_of_order_stay_in_bounds(N, L, cu):
    """Each token's sequence is one of those or none, and no kernel writes beside its buffers."""
    D, S, K = 12, 4, 4
    seq = core.sequence_index(torch.tensor(cu, device=DEV, dtype=torch.int32), L)
    assert int(seq.min()) >= -1 and int(seq.max()) < S
    t = {k: v.to(DEV) for k, v in make(1, L, D, N, 1, F32, 6, S).items()}
    dy, fin = torch.randn(1, L, D, device=DEV), torch.randn(S, D, N, device=DEV)
    buf, p, st = Guarded(), core.ptr, torch.cuda.current_stream().cuda_stream
    args = core._scan_args(t["u"], t["delta"], t["A"], t["B"], t["C"], t["D"], t["z"], t["bias"], True)
    saved = buf(lib.ttt_selective_scan_saved_bytes(1, L, D, N) // 4)
    n = lib.ttt_selective_scan_fwd_scratch_bytes(1, L, D, 1, N)
    check(lib.ttt_selective_scan_fwd(*args, p(seq), p(t["init"]), buf(S * D * N), buf(L * D), saved, buf(n // 4), n, st),
          "fwd")
    n = lib.ttt_selective_scan_bwd_scratch_bytes(1, L, D, 1, N)
    check(lib.ttt_selective_scan_bwd(*args, p(seq), p(t["init"]), saved, p(dy), p(fin), buf(L * D), buf(L * D), buf(L * N),
                                     buf(L * N), buf(L * D), buf(S * D * N), buf(D * (N + 2)), buf(n // 4), n, st), "bwd")
    w, rows = torch.randn(D, K, device=DEV), torch.randn(S, K - 1, D, device=DEV)
    strides = core._strides(L * D, D)
    check(lib.ttt_causal_conv_fwd(1, L, D, K, p(t["u"]), 0, strides, p(w), None, 1, p(seq), p(rows), buf(S * (K - 1) * D),
                                  buf(L * D), st), "conv fwd")
    n = lib.ttt_causal_conv_bwd_scratch_bytes(1, L, D, K, 0)
    check(lib.ttt_causal_conv_bwd(1, L, D, K, p(t["u"]), 0, strides, p(w), None, 1, p(seq), p(rows), p(dy), p(rows),
                                  buf(L * D), buf(S * (K - 1) * D), buf(D * (K + 1)), buf(n // 4), n, st), "conv bwd")
    buf.check()


# ------------------------------------------------------------------------------ long memory
def test_decays_of_a_long_memory_are_centred():
    """A state set at the first token and kept for 4000 steps of random size. Each decay is off by at
    most about 2^-23 either way: 4 * 4000^0.5 * 2^-24 in all if the errors are centred, beside
    0.15 * 2^-24 a step for what is left of the unit's cut-off (0.3 without the correction) and
    the rounding of A log2(e), 2^-25 of the exponent of 62 * log2(e)."""
    L, D, N = 4000, 64, 4
    g = torch.Generator().manual_seed(4)
    delta = (0.001 + 0.029 * torch.rand(1, L, D, generator=g)).to(DEV)
    zero = torch.zeros(1, L, D, device=DEV)
    A, BC = torch.full((D, N), -1.0, device=DEV), torch.zeros(1, L, N, device=DEV)
    init = torch.ones(1, D, N, device=DEV)
    _, fin = ops.selective_scan(zero, delta, A, BC, BC, initial_state=init, return_final_state=True)
    want = torch.exp(-delta.double().sum(1))[0][:, None].expand(D, N)
    off = (fin[0].double() - want) / want
    assert float(off.abs().max()) <= (0.15 * L + 4 * L**0.5 + 62 * 1.4427 / 2) * 2.0**-24
