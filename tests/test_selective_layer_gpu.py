"""GPU: the forecaster's selective scan layer, convolution and scan together as a model uses
them: gradients against the 64-bit composition, prompts continued token by token, packed
prompts, and a captured training step.

Tolerance (relative L2): the layer's five matrix products and its scan in fp32, each a sum of at
most K terms of random signs off by K^0.5 * 2^-24, through one another; 5 * 64^0.5 * 2^-24 *
(a factor of 8 for the chain's conditioning) = 2e-5 with TF32 products off. In bf16 every stage
rounds once to 2^-9 on average: 8 stages in a row, 8 * 2^-8 at worst.
"""

import pytest
import torch

import scan_reference as R
from forecaster import GraphedTrainStep, SelectiveScanLayer, TTTForecaster, make_optimizer, train_step

pytestmark = pytest.mark.gpu
DEV = "cuda"


def layer(act_dtype, seed=0, dim=32, **kw):
    torch.manual_seed(seed)
    return SelectiveScanLayer(dim, act_dtype=act_dtype, **kw).to(DEV)


def reference(m, p, h, cu=None):
    """The layer in 64 bits from its parameters p."""
    x, z = (h @ p["in_proj.weight"].t()).chunk(2, -1)
    x, _ = R.causal_conv1d(x, p["conv_weight"], p["conv_bias"], True, None, cu)
    d, B, C = (x @ p["x_proj.weight"].t()).split([m.dt_rank, m.state_size, m.state_size], -1)
    y, _ = R.selective_scan(x, d @ p["dt_proj.weight"].t(), -torch.exp(p["A_log"]), B.unsqueeze(2), C.unsqueeze(2),
                            p["D"], z, p["dt_proj.bias"], True, None, cu)
    return y @ p["out_proj.weight"].t()


@pytest.mark.parametrize("act_dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 8 * 2.0**-8)])
@pytest.mark.parametrize("cu", [None, [0, 9, 10, 37]])
def test_layer_matches_the_composition(act_dtype, tol, cu):
    m = layer(act_dtype)
    B, L = (1, cu[-1]) if cu else (2, 33)
    h = torch.randn(B, L, 32, device=DEV, requires_grad=True)
    dy = torch.randn(B, L, 32, device=DEV)
    out = m(h, cu_seqlens=torch.tensor(cu, device=DEV, dtype=torch.int32) if cu else None)
    got = torch.autograd.grad(out, [h, *m.parameters()], dy.to(out.dtype))
    p = {k: v.detach().double().requires_grad_(True) for k, v in m.named_parameters()}
    hd = h.detach().double().requires_grad_(True)
    ref = reference(m, p, hd, cu)
    want = torch.autograd.grad(ref, [hd, *p.values()], dy.to(out.dtype).double())
    assert R.rel(out, ref) <= tol
    for name, a, b in zip(["hidden", *p], got, want):
        assert R.rel(a, b) <= tol, (name, R.rel(a, b))


def test_prompt_then_single_tokens():
    m = layer(torch.float32, 1)
    h = torch.randn(3, 20, 32, device=DEV)
    with torch.no_grad():
        whole = m(h)
        out, state = m(h[:, :12], return_state=True)
        outs = [out]
        for t in range(12, 16):
            outs.append(m.step(h[:, t], state)[:, None])
        more, _ = m(h[:, 16:], state=state, return_state=True)  # and a chunk after them
        assert R.rel(torch.cat([*outs, more], 1), whole) <= 2e-5
        # the same from a cache of slots, rows in another order, one row without a sequence
        slots = m.new_state(7)
        for s, v in zip(slots, m(h[:, :12], return_state=True)[1]):
            s[torch.tensor([5, 0, 2], device=DEV)] = v
        idx = torch.tensor([2, -1, 5, 0], device=DEV, dtype=torch.int32)
        rows = torch.stack([h[2, 12], torch.full_like(h[0, 12], float("nan")), h[0, 12], h[1, 12]])
        y = m.step(rows, slots, idx)
        assert R.rel(y[[2, 3, 0]], whole[:, 12]) <= 2e-5 and float(y[1].abs().max()) == 0


@pytest.mark.parametrize("act_dtype", [torch.float32, torch.bfloat16])
def test_forecaster_trains_on_it(act_dtype):
    torch.manual_seed(0)
    model = TTTForecaster(7, 7, 24, 48, model_dim=32, num_layers=2, act_dtype=act_dtype,
                          ssm_layer="selective_scan").to(DEV)
    x, y = torch.randn(4, 48, 7, device=DEV), torch.randn(4, 24, 7, device=DEV)
    opt = make_optimizer(model)
    before = [p.detach().clone() for p in model.parameters()]
    assert bool(torch.isfinite(train_step(model, opt, x, y)))
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in model.parameters())
    assert any(not torch.equal(a, b) for a, b in zip(before, model.parameters()))


def test_captured_training_step_equals_the_ordinary_one():
    def make():
        torch.manual_seed(0)
        m = TTTForecaster(7, 7, 24, 48, model_dim=32, num_layers=2, ssm_layer="selective_scan").to(DEV)
        return m, make_optimizer(m, capturable=True)

    g = torch.Generator(device=DEV).manual_seed(1)
    data = [(torch.randn(4, 48, 7, device=DEV, generator=g), torch.randn(4, 24, 7, device=DEV, generator=g))
            for _ in range(3)]
    a, opt_a = make()
    graphed = GraphedTrainStep(a, opt_a, *data[0], warmup=2)
    b, opt_b = make()
    for _ in range(2):
        train_step(b, opt_b, *data[0])
    for x, y in data:
        la, lb = graphed(x, y).clone(), train_step(b, opt_b, x, y)
        assert torch.equal(la, lb)
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
