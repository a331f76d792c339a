"""Plain 64-bit forms of the selective scan and the causal convolution, token by token, for the
tests: differentiable by autograd, one sequence at a time."""

import torch


def sequences(x, cu):
    """(row, first token, end, state index) of each sequence."""
    if cu is None:
        return [(b, 0, x.shape[1], b) for b in range(x.shape[0])]
    return [(0, cu[i], cu[i + 1], i) for i in range(len(cu) - 1)]


def selective_scan(u, delta, A, B, C, D=None, z=None, bias=None, softplus=False, init=None, cu=None):
    """B, C: [B, L, G, N]. Returns (out, final states). Tokens of no sequence give zeros."""
    rows, L, W = u.shape
    per = W // B.shape[2]
    dt = delta + (bias if bias is not None else 0.0)
    if softplus:
        dt = torch.logaddexp(dt, torch.zeros_like(dt))
    outs = [[torch.zeros(W, dtype=u.dtype, device=u.device) for _ in range(L)] for _ in range(rows)]
    finals = []
    for b, t0, t1, i in sequences(u, cu):
        h = init[i] if init is not None else torch.zeros(W, A.shape[1], dtype=u.dtype, device=u.device)
        for t in range(t0, t1):
            Bt, Ct = B[b, t].repeat_interleave(per, 0), C[b, t].repeat_interleave(per, 0)
            h = torch.exp(dt[b, t][:, None] * A) * h + (dt[b, t] * u[b, t])[:, None] * Bt
            y = (h * Ct).sum(-1)
            if D is not None:
                y = y + D * u[b, t]
            if z is not None:
                y = y * z[b, t] * torch.sigmoid(z[b, t])
            outs[b][t] = y
        finals.append(h)
    out = torch.stack([torch.stack(r) if r else u.new_zeros(0, W) for r in outs])
    return out, torch.stack(finals)


def causal_conv1d(x, w, b=None, silu=False, init=None, cu=None):
    rows, L, W = x.shape
    K = w.shape[1]
    outs = [[torch.zeros(W, dtype=x.dtype, device=x.device) for _ in range(L)] for _ in range(rows)]
    finals = []
    for r, t0, t1, i in sequences(x, cu):
        head = init[i] if init is not None else x.new_zeros(K - 1, W)
        full = torch.cat([head, x[r, t0:t1]])
        for t in range(t1 - t0):
            p = (full[t:t + K].t() * w).sum(-1)
            if b is not None:
                p = p + b
            outs[r][t0 + t] = p * torch.sigmoid(p) if silu else p
        finals.append(full[t1 - t0:])
    return torch.stack([torch.stack(r) if r else x.new_zeros(0, W) for r in outs]), torch.stack(finals)


def rel(got, ref):
    """Relative L2 distance; both empty or both zero count as none."""
    got, ref = got.detach().double().cpu(), ref.detach().double().cpu()
    assert got.shape == ref.shape, (got.shape, ref.shape)
    assert torch.equal(torch.isfinite(got), torch.isfinite(ref))
    d, n = float((got - ref).norm()), float(ref.norm())
    return d / n if n else d
