"""The selective scan and its short causal convolution: cases, inputs and plain forms.

``own`` chooses what ``run`` calls: the plain torch form of each operator, or this package's
``ops``. A case's ``op`` is "conv" or "scan"; its ``mode`` is

  step    one new token for every sequence, the carried state updated in place (serving),
  prompt  whole sequences, outputs and final states, no gradients (serving); ``seqs`` > 0 packs
          that many sequences of different lengths into one row of L tokens,
  train   the forward pass and every gradient.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token for a handful of sequences: the smallest call, latency alone
        dict(name="conv step 8x512", op="conv", mode="step", B=8, L=1, D=512, K=4, dtype="bf16", silu=True, seqs=0),
        # prompts of different lengths packed together, odd width and total
        dict(name="conv packed 5003x1537", op="conv", mode="prompt", B=1, L=5003, D=1537, K=3, dtype="fp16", silu=True,
             seqs=7),
        # fp32 training of a small model, short odd sequences, two taps, no activation
        dict(name="conv train fp32 3x1001", op="conv", mode="train", B=3, L=1001, D=384, K=2, dtype="fp32", silu=False,
             seqs=0),
        # a forecaster layer: 336 steps, width 256 expanded twice
        dict(name="conv train 32x336x512", op="conv", mode="train", B=32, L=336, D=512, K=4, dtype="bf16", silu=True,
             seqs=0),
        # long training sequences (the 32 x 4096 benchmark batch, width 512 expanded twice)
        dict(name="conv train 32x4096x1024", op="conv", mode="train", B=32, L=4096, D=1024, K=4, dtype="bf16",
             silu=True, seqs=0),
        # one token for one sequence: latency alone
        dict(name="scan step 1x512", op="scan", mode="step", B=1, L=1, D=512, N=16, G=1, dtype="bf16", z=True, seqs=0),
        # one token for a large serving batch: the fp32 states stream through
        dict(name="scan step 256x1536", op="scan", mode="step", B=256, L=1, D=1536, N=16, G=1, dtype="bf16", z=True,
             seqs=0),
        # one long prompt: few channels, a long axis
        dict(name="scan prompt 1x8192x1024", op="scan", mode="prompt", B=1, L=8192, D=1024, N=16, G=1, dtype="bf16",
             z=True, seqs=0),
        # prompts of different lengths packed together, two groups, a wider odd state
        dict(name="scan packed 6007x768 N40", op="scan", mode="prompt", B=1, L=6007, D=768, N=40, G=2, dtype="fp16",
             z=True, seqs=11),
        # fp32 training of a small model, odd sizes, no gate
        dict(name="scan train fp32 2x777", op="scan", mode="train", B=2, L=777, D=200, N=8, G=1, dtype="fp32", z=False,
             seqs=0),
        # a forecaster layer
        dict(name="scan train 32x336x512", op="scan", mode="train", B=32, L=336, D=512, N=16, G=1, dtype="bf16", z=True,
             seqs=0),
        # long training sequences (the 16 x 2048 benchmark batch, width 768 expanded twice)
        dict(name="scan train 16x2048x1536", op="scan", mode="train", B=16, L=2048, D=1536, N=16, G=1, dtype="bf16",
             z=True, seqs=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("conv", "scan"))
    mode = rng.choice(("step", "prompt", "train"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    D = _log(rng, 64, 2048)
    if mode == "step":
        B, L = _log(rng, 1, 512), 1
    else:
        L = _log(rng, 1, 8192)
        B = _log(rng, 1, 64)
    seqs = 0
    if mode == "prompt" and rng.random() < 0.5:
        B, seqs = 1, rng.randint(1, 24)
    case = dict(op=op, mode=mode, B=B, L=L, D=D, dtype=dtype, seqs=seqs)
    if op == "conv":
        case.update(K=rng.choice((2, 3, 4)), silu=rng.random() < 0.7)
        most = 32 * 4096 * 1024
        size = D
    else:
        N = rng.choice((rng.randint(1, 64), 16, 16))
        G = rng.choice((1, 1, 2))
        case.update(N=N, G=G, z=rng.random() < 0.7, D=(D + G - 1) // G * G)
        most = 16 * 2048 * 1536 * 16
        size = case["D"] * N
    if mode != "step":  # no larger than the largest listed case
        case["B"] = max(1, min(B, most // (L * size)))
        case["L"] = max(1, min(L, most // (case["B"] * size)))
    return case


# ------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c = dict(case)
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    B, L, D = c["B"], c["L"], c["D"]
    train, step = c["mode"] == "train", c["mode"] == "step"
    rows = (B,) if step else (B, L)

    def normal(*shape, scale=1.0, dtype=dt):
        return torch.randn(*shape, generator=gen, device=dev).mul_(scale).to(dtype)

    s = {"case": c}
    nseq = c["seqs"] or B
    if c["seqs"]:  # sequences of different lengths that fill the row
        cuts = torch.randint(0, L + 1, (c["seqs"] - 1,), generator=gen, device=dev).sort().values
        ends = torch.tensor([0, L], device=dev)
        s["cu"] = torch.cat([ends[:1], cuts, ends[1:]]).to(torch.int32)
    if c["op"] == "conv":
        K = c["K"]
        s["x"] = normal(*rows, D)
        s["w"] = normal(D, K, scale=1 / math.sqrt(K), dtype=torch.float32)
        s["b"] = normal(D, scale=0.1, dtype=torch.float32)
        if not train:
            s["state"] = normal(nseq, K - 1, D)
        leaves = ("x", "w", "b")
    else:
        N, G = c["N"], c["G"]
        s["u"] = normal(*rows, D, scale=0.7)
        s["delta"] = normal(*rows, D, scale=0.5)
        # step sizes of 0.001 to 0.1 through the softplus, decays -(1 .. N) a little off
        r = torch.rand(D, generator=gen, device=dev) * math.log(100.0) + math.log(1e-3)
        r = torch.exp(r)
        s["bias"] = r + torch.log(-torch.expm1(-r))
        s["A"] = -torch.arange(1, N + 1, device=dev).float() * (1 + 0.1 * torch.rand(D, N, generator=gen, device=dev))
        s["B"] = normal(*rows, G, N, scale=0.7)
        s["C"] = normal(*rows, G, N, scale=0.7)
        s["D"] = 1 + normal(D, scale=0.1, dtype=torch.float32)
        s["z"] = normal(*rows, D) if c["z"] else None
        if not train:
            s["state"] = normal(nseq, D, N, scale=0.5, dtype=torch.float32)
        leaves = ("u", "delta", "A", "B", "C", "D", "z", "bias")
    if train:
        s["dout"] = normal(*rows, D)
        s["leaves"] = [k for k in leaves if s[k] is not None]
        for k in s["leaves"]:
            s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------- what is run
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ttt-triton_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import ops

    return ops


def _run_own(s):
    ops, c = _ops(), s["case"]
    act = "silu" if c.get("silu") else None
    if c["op"] == "conv":
        if c["mode"] == "step":
            return {"y": ops.causal_conv1d_step(s["x"], s["state"], s["w"], s["b"], activation=act), "state": s["state"]}
        if c["mode"] == "prompt":
            y, fin = ops.causal_conv1d(s["x"], s["w"], s["b"], activation=act, initial_state=s["state"],
                                       cu_seqlens=s.get("cu"), return_final_state=True)
            return {"y": y, "state": fin}
        y = ops.causal_conv1d(s["x"], s["w"], s["b"], activation=act)
    else:
        args = (s["u"], s["delta"], s["A"], s["B"], s["C"])
        kw = dict(D=s["D"], z=s["z"], delta_bias=s["bias"], delta_softplus=True)
        if c["mode"] == "step":
            return {"y": ops.selective_scan_step(s["state"], *args, **kw), "state": s["state"]}
        if c["mode"] == "prompt":
            y, fin = ops.selective_scan(*args, **kw, initial_state=s["state"], cu_seqlens=s.get("cu"),
                                        return_final_state=True)
            return {"y": y, "state": fin}
        y = ops.selective_scan(*args, **kw)
    grads = torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dout"])
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(s["leaves"], grads)}}


# ------------------------------------------------------------------------------- plain forms
def _run_plain(s):
    with torch.no_grad():
        return (_plain_conv if s["case"]["op"] == "conv" else _plain_scan)(s)


def _silu_grad(p):
    g = torch.sigmoid(p)
    return g * (1 + p * (1 - g))


def _sequences(s, L):
    """For packed rows: each token's sequence, its sequence's first token, and whether it is that."""
    cu = s["cu"].long()
    t = torch.arange(L, device=cu.device)
    seq = torch.searchsorted(cu, t, right=True) - 1
    return t, seq, cu[seq]


def _plain_conv(s):
    c = s["case"]
    dt, K = DTYPES[c["dtype"]], c["K"]
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    if c["mode"] == "step":
        win = torch.cat([s["state"].float(), x[:, None]], 1)  # [B, K, D]
        p = (win * w.t()).sum(1) + b
        s["state"].copy_(win[:, 1:])
        return {"y": (p * torch.sigmoid(p) if c["silu"] else p).to(dt), "state": s["state"]}
    B, L, D = x.shape
    head = s["state"].float() if c["mode"] == "prompt" and not c["seqs"] else x.new_zeros(B, K - 1, D)
    full = torch.cat([head, x], 1)
    win = full.unfold(1, K, 1)  # [B, L, D, K], oldest row first
    if c["seqs"]:  # rows before a sequence's start are its initial state's
        t, seq, start = _sequences(s, L)
        k = torch.arange(K, device=x.device)
        row = t[:, None] - (K - 1) + k - start[:, None]  # place within the sequence, negative before it
        init = s["state"].float()[seq[:, None], (row + K - 1).clamp(0, K - 2)]  # [L, K, D]
        win = torch.where((row >= 0)[None, :, None, :], win, init.permute(0, 2, 1)[None])
    p = (win * w).sum(-1) + b
    y = (p * torch.sigmoid(p) if c["silu"] else p).to(dt)
    if c["mode"] == "prompt":
        if c["seqs"]:
            cu = s["cu"].long()
            row = cu[1:, None] - (K - 1) + torch.arange(K - 1, device=x.device) - cu[:-1, None]  # [S, K-1]
            rows = x[0][(row + cu[:-1, None]).clamp(0, L - 1)]
            n = cu[1:] - cu[:-1]
            old = (torch.arange(K - 1, device=x.device) + n[:, None]).clamp(max=K - 2)
            kept = s["state"].float().gather(1, old[:, :, None].expand(-1, -1, D))
            fin = torch.where((row >= 0)[:, :, None], rows, kept)
        else:
            fin = full[:, L:]
        return {"y": y, "state": fin.to(dt)}
    dp = s["dout"].float() * (_silu_grad(p) if c["silu"] else 1.0)
    after = torch.cat([dp, dp.new_zeros(B, K - 1, D)], 1).unfold(1, K, 1)  # dp[t .. t + K - 1]
    dx = (after * w.flip(1)).sum(-1)
    dw = (win * dp[..., None]).sum((0, 1))
    return {"y": y, "dx": dx.to(dt), "dw": dw, "db": dp.sum((0, 1))}


def _linear_scan(a, x):
    """h[t] = a[t] h[t-1] + x[t] along dimension 1 for all t at once, by doubling: after the step
    of width w, x[t] holds the sum over the last 2w inputs and a[t] the product of their decays."""
    w, L = 1, x.shape[1]
    while w < L:
        x = torch.cat([x[:, :w], torch.addcmul(x[:, w:], a[:, w:], x[:, :-w])], 1)
        a = torch.cat([a[:, :w], a[:, w:] * a[:, :-w]], 1)
        w *= 2
    return x


def _per_channel(v, D):
    """[..., G, N] -> [..., D, N]: each group's row for its channels."""
    G = v.shape[-2]
    return v.float().unsqueeze(-2).expand(*v.shape[:-1], D // G, v.shape[-1]).reshape(*v.shape[:-2], D, v.shape[-1])


def _plain_scan(s):
    c = s["case"]
    dt_out, D = DTYPES[c["dtype"]], c["D"]
    u, A = s["u"].float(), s["A"].float()
    raw = s["delta"].float() + s["bias"].float()
    dt = torch.clamp(raw, min=0) + torch.log1p(torch.exp(-raw.abs()))
    Bd, Cd = _per_channel(s["B"], D), _per_channel(s["C"], D)
    z = s["z"].float() if s["z"] is not None else None
    gate = z * torch.sigmoid(z) if z is not None else None
    a = torch.exp(dt[..., None] * A)  # [.., D, N]
    x = (dt * u)[..., None] * Bd
    if c["mode"] == "step":
        h = a * s["state"] + x
        s["state"].copy_(h)
    else:
        if c["mode"] == "prompt" and c["seqs"]:
            t, seq, start = _sequences(s, c["L"])
            first = (t == start)[None, :, None, None]
            x = torch.where(first, x + a * s["state"][seq][None], x)
            a = torch.where(first, torch.zeros_like(a), a)
        elif c["mode"] == "prompt":
            x[:, 0] += a[:, 0] * s["state"]
        h = _linear_scan(a, x)
    y0 = (h * Cd).sum(-1) + s["D"].float() * u
    y = (y0 * gate if gate is not None else y0).to(dt_out)
    if c["mode"] == "step":
        return {"y": y, "state": s["state"]}
    if c["mode"] == "prompt":
        if c["seqs"]:
            cu = s["cu"].long()
            some = (cu[1:] > cu[:-1])[:, None, None]
            return {"y": y, "state": torch.where(some, h[0][(cu[1:] - 1).clamp(min=0)], s["state"])}
        return {"y": y, "state": h[:, -1].contiguous()}
    dout = s["dout"].float()
    dy = dout * gate if gate is not None else dout
    # the reverse recurrence g[t] = C dy + a[t + 1] g[t + 1], run forward on flipped time
    nxt = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1).flip(1)
    g = _linear_scan(nxt, (Cd * dy[..., None]).flip(1)).flip(1)
    del nxt
    groups = (*u.shape[:2], c["G"], D // c["G"], c["N"])
    dC = (h * dy[..., None]).reshape(groups).sum(3)
    dB = (g * (dt * u)[..., None]).reshape(groups).sum(3)
    s1 = (g * Bd).sum(-1)
    q = g * a * torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    ddt = u * s1 + (q * A).sum(-1)
    draw_ = ddt * torch.sigmoid(raw)
    out = {"y": y, "du": (dt * s1 + s["D"].float() * dy).to(dt_out), "ddelta": draw_.to(dt_out),
           "dA": (q * dt[..., None]).sum((0, 1)), "dB": dB.to(dt_out), "dC": dC.to(dt_out), "dD": (u * dy).sum((0, 1))}
    if z is not None:
        out["dz"] = (dout * y0 * _silu_grad(z)).to(dt_out)
    out["dbias"] = draw_.sum((0, 1))
    return out


# ------------------------------------------------------------------------------- exact values
def exact(case, seed):
    """The definitions, token by token, in 64 bits."""
    s = prepare(case, seed)
    with torch.no_grad():
        return (_exact_conv if case["op"] == "conv" else _exact_scan)(s)


def _spans(s):
    """(row, first token, end, index of its state) of every sequence."""
    c = s["case"]
    if c["seqs"]:
        cu = s["cu"].tolist()
        return [(0, cu[i], cu[i + 1], i) for i in range(len(cu) - 1)]
    return [(i, 0, c["L"], i) for i in range(c["B"])]


def _exact_conv(s):
    c = s["case"]
    K, dt = c["K"], DTYPES[c["dtype"]]
    w, b = s["w"].double(), s["b"].double()
    x = s["x"].double()
    if c["mode"] == "step":
        x = x[:, None]
    state = s["state"].double() if "state" in s else x.new_zeros(c["B"], K - 1, c["D"])
    train = c["mode"] == "train"
    y, dx = torch.empty_like(x), torch.zeros_like(x)
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    fin = state.clone()
    spans = _spans(s) if c["seqs"] else [(slice(None), 0, c["L"], slice(None))]  # a dense batch goes at once
    for r, t0, t1, i in spans:
        n = t1 - t0
        if n == 0:
            continue
        rows = torch.cat([state[i], x[r, t0:t1]], -2)  # the sequence with its state in front
        p = b.expand_as(x[r, t0:t1]).clone()
        for k in range(K):
            p += w[:, k] * rows[..., k:k + n, :]
        sig = 1 / (1 + torch.exp(-p))
        y[r, t0:t1] = p * sig if c["silu"] else p
        fin[i] = rows[..., n:, :]
        if train:
            dp = s["dout"].double()[r, t0:t1]
            if c["silu"]:
                dp = dp * (sig + p * sig * (1 - sig))
            db += dp.sum((0, 1))
            for k in range(K):
                dw[:, k] += (dp * rows[..., k:k + n, :]).sum((0, 1))
                back = K - 1 - k  # x[t - back] meets tap k
                if n > back:
                    dx[r, t0:t1 - back] += w[:, k] * dp[..., back:, :]
    if train:
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    return {"y": y[:, 0] if c["mode"] == "step" else y, "state": fin.to(dt).double()}


def _exact_scan(s):
    c = s["case"]
    D, N = c["D"], c["N"]
    per = D // c["G"]
    f = {k: s[k].double() if s[k] is not None else None for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")}
    if c["mode"] == "step":
        f.update({k: f[k][:, None] for k in ("u", "delta", "B", "C", "z") if f[k] is not None})
    if c["mode"] == "train" and c["B"] * c["L"] * D * N * 8 > 40e9:
        return None
    u, A = f["u"], f["A"]
    raw = f["delta"] + f["bias"]
    dt = torch.where(raw > 30, raw, torch.log1p(torch.exp(raw.clamp(max=30))))
    sig = 1 / (1 + torch.exp(-f["z"])) if f["z"] is not None else None
    state = s["state"].double() if "state" in s else u.new_zeros(c["B"], D, N)
    train = c["mode"] == "train"
    y0, fin = torch.empty_like(u), state.clone()
    spans = _spans(s) if c["seqs"] else [(slice(None), 0, c["L"], slice(None))]
    hs = u.new_empty(c["L"], c["B"], D, N) if train else None
    wide = lambda v: v.repeat_interleave(per, -2)  # noqa: E731
    for r, t0, t1, i in spans:
        h = state[i]
        for t in range(t0, t1):
            d = dt[r, t][..., None]
            h = torch.exp(d * A) * h + d * u[r, t][..., None] * wide(f["B"][r, t])
            y0[r, t] = (h * wide(f["C"][r, t])).sum(-1)
            if train:
                hs[t] = h
        fin[i] = h
    y0 += f["D"] * u
    y = y0 * f["z"] * sig if sig is not None else y0
    if not train:
        return {"y": y[:, 0] if c["mode"] == "step" else y, "state": fin}
    dout = s["dout"].double()
    dy = dout * f["z"] * sig if sig is not None else dout
    dz = dout * y0 * (sig + f["z"] * sig * (1 - sig)) if sig is not None else None
    du, ddt = f["D"] * dy, torch.zeros_like(u)
    dB, dC, dA = torch.empty_like(f["B"]), torch.empty_like(f["C"]), torch.zeros_like(A)
    carry = torch.zeros_like(state)  # a[t + 1] g[t + 1]
    for t in range(c["L"] - 1, -1, -1):
        d, ut, Bt = dt[:, t][..., None], u[:, t], wide(f["B"][:, t])
        g = carry + wide(f["C"][:, t]) * dy[:, t][..., None]
        dC[:, t] = (hs[t] * dy[:, t][..., None]).reshape(-1, c["G"], per, N).sum(2)
        dB[:, t] = (g * d * ut[..., None]).reshape(-1, c["G"], per, N).sum(2)
        s1 = (g * Bt).sum(-1)
        carry = g * torch.exp(d * A)
        q = carry * hs[t - 1] if t else torch.zeros_like(carry)
        du[:, t] += dt[:, t] * s1
        ddt[:, t] = ut * s1 + (q * A).sum(-1)
        dA += (q * d).sum(0)
    draw_ = ddt / (1 + torch.exp(-raw))
    out = {"y": y, "du": du, "ddelta": draw_, "dA": dA, "dB": dB, "dC": dC, "dD": (u * dy).sum((0, 1))}
    if dz is not None:
        out["dz"] = dz
    out["dbias"] = draw_.sum((0, 1))
    return out


# ------------------------------------------------------------------------------- work
def work(case):
    c = case
    B, L, D = c["B"], c["L"], c["D"]
    e = 4 if c["dtype"] == "fp32" else 2
    tok = B * L * D
    nseq = c["seqs"] or B
    if c["op"] == "conv":
        K = c["K"]
        state = 0 if c["mode"] == "train" else 2 * nseq * (K - 1) * D * e
        flops = tok * (2 * K + (4 if c["silu"] else 0))
        if c["mode"] == "train":  # x and dout in, y and dx out
            return {"bytes": 4 * tok * e + 2 * D * (K + 1) * 4, "flops": 4 * flops}
        return {"bytes": 2 * tok * e + state + D * (K + 1) * 4, "flops": flops}
    N, G = c["N"], c["G"]
    rows = 2 * B * L * G * N * e  # B and C
    params = D * (N + 2) * 4
    per = 4 if c["z"] else 3  # u, delta, (z,) y
    flops = tok * N * 7
    if c["mode"] == "train":  # u, delta, z, dout in; y and the gradients of u, delta, z out; B, C and theirs
        return {"bytes": (2 * per) * tok * e + 2 * rows + 2 * params, "flops": tok * N * 27}
    return {"bytes": per * tok * e + rows + params + 2 * nseq * D * N * 4, "flops": flops}
