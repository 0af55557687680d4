"""Calls of the layer and of the 8-bit operators as a user may make them,
besides the values of test_gpu_int8.py: graphed steps, shared plans, hooks,
unusual types and buffers."""

import numpy as np
import pytest
import torch

import _int8_ref as ref
from tlora_b200 import MultiLoRALinear, _lib, ops
from tlora_b200.graphs import GraphedTrainStep

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, dt, seed, scale=1.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * scale).to(dt)


def layer(d_in, d_out, ranks, dt, seed=0, bias=True):
    torch.manual_seed(seed)
    m = MultiLoRALinear(d_in, d_out, ranks, bias=bias)
    with torch.no_grad():
        if bias:
            m.base.bias.normal_(0, 0.1)
        for i, ad in enumerate(m.adapters.values()):
            ad.B.normal_(0, 0.05)
            ad.scaling = 0.5 + 0.25 * i
    return m.cuda().to(dt)


def step(m, x, ids, dy, plan=None):
    for ad in m.adapters.values():
        ad.A.grad = ad.B.grad = None
    xg = x.detach().clone().requires_grad_(True)
    y = m(xg, ids, plan=plan)
    y.backward(dy)
    return (y.detach(), xg.grad, [a.A.grad for a in m.adapters.values()], [a.B.grad for a in m.adapters.values()])


IDS = torch.cat([torch.full((n,), a, dtype=torch.int64) for a, n in ((0, 64), (1, 128), (2, 70))])
RANKS = {0: 4, 1: 72, 2: 16}


# ------------------------------------------------------------------ graphed steps

@pytest.mark.parametrize("dt, dy_dt", [(BF, F32), (FP, F32), (FP, BF), (F32, BF)])
@pytest.mark.parametrize("eight", [False, True])
def test_graphed_step_casts_the_upstream_gradient(dt, dy_dt, eight):
    # as autograd does: the gradient takes the output's type
    m = layer(256, 192, RANKS, dt)
    if eight:
        m.quantize_base()
        m.save_input = "int8"
    x, dy = randn((len(IDS), 256), dt, 1), randn((len(IDS), 192), dy_dt, 2, 0.1)
    want = step(m, x, IDS, dy.to(dt))
    g = GraphedTrainStep(m, x, IDS, dy, lr=0.0)
    for given in (None, dy):
        y = g(x, given)
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(g.dx, want[1])
        for ad, da, db in zip(m.adapters.values(), want[2], want[3]):
            assert torch.equal(ad.A.grad, da) and torch.equal(ad.B.grad, db)
    assert _lib.device_error() == 0


def test_graphed_step_refuses_other_gradients():
    m = layer(256, 192, RANKS, BF)
    x, rows = randn((len(IDS), 256), BF, 1), len(IDS)
    for bad in (torch.zeros(rows, 191, device="cuda", dtype=BF), torch.zeros(rows - 1, 192, device="cuda", dtype=BF),
                torch.zeros(rows + 1, 192, device="cuda", dtype=BF), torch.zeros(192, device="cuda", dtype=BF)):
        with pytest.raises(ValueError, match="dy"):
            GraphedTrainStep(m, x, IDS, bad, lr=0.0)
    with pytest.raises(RuntimeError, match="dy"):
        GraphedTrainStep(m, x, IDS, torch.zeros(rows, 192, dtype=BF), lr=0.0)
