"""Calls of the layer and of the 8-bit operators as a user may make them,
besides the values of test_gpu_int8.py: graphed steps, shared plans, hooks,
unusual types and buffers."""

import ctypes

import numpy as np
import pytest
import torch

import _int8_ref as ref
import _saved_ref as saved
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


def test_graphed_step_keeps_the_modules_hooks():
    """Hooks and an overridden forward do in a graphed step what they do in an
    eager one."""
    class Doubled(MultiLoRALinear):
        def forward(self, x, adapter_ids, **kw):
            return 2 * super().forward(x + self.shift, adapter_ids, **kw)

    def make():
        torch.manual_seed(0)
        m = Doubled(256, 192, RANKS)
        with torch.no_grad():
            for ad in m.adapters.values():
                ad.B.normal_(0, 0.05)
        m = m.cuda().bfloat16()
        m.shift = torch.nn.Parameter(torch.full((256,), 0.25, device="cuda", dtype=BF))
        m.seen = torch.zeros(3, device="cuda")

        def forward_hook(mod, args, out):
            mod.seen[0] += out.detach().float().abs().sum()
            return out * 0.5

        def backward_hook(mod, gi, go):
            mod.seen[1] += go[0].float().abs().sum()

        def after(p):
            m.seen[2] += p.grad.float().abs().sum()
        m.register_forward_hook(forward_hook)
        m.register_full_backward_hook(backward_hook)
        m.adapters["0"].A.register_hook(lambda g: g * 3)
        m.adapters["1"].B.register_hook(lambda g: g.clamp(-0.5, 0.5))
        m.adapters["2"].A.register_post_accumulate_grad_hook(after)
        return m

    x, dy = randn((len(IDS), 256), BF, 1), randn((len(IDS), 192), BF, 2, 0.1)
    eager, m = make(), make()
    alive = m(x.clone().requires_grad_(True), IDS)  # an eager graph of the same leaves
    g = GraphedTrainStep(m, x, IDS, dy, lr=0.0)
    for k in range(2):
        eager.seen.zero_()
        m.seen.zero_()
        eager.shift.grad = None
        want = step(eager, x, IDS, dy)
        m.shift.grad.zero_()
        y = g(x, dy)
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(g.dx, want[1]) and torch.equal(m.seen, eager.seen)
        assert torch.equal(m.shift.grad, eager.shift.grad) and bool((m.seen > 0).all())
        for ad, da, db in zip(m.adapters.values(), want[2], want[3]):
            assert torch.equal(ad.A.grad, da) and torch.equal(ad.B.grad, db)
        x, dy = randn((len(IDS), 256), BF, 3), randn((len(IDS), 192), BF, 4, 0.1)
    assert alive.requires_grad
    # the module has its own parameters back
    assert all(p.is_leaf and p.requires_grad for ad in m.adapters.values() for p in ad.parameters())


def test_graphed_step_of_frozen_parts():
    m = layer(256, 192, RANKS, BF).quantize_base()
    m.save_input = "int8"
    x, dy = randn((len(IDS), 256), BF, 1), randn((len(IDS), 192), BF, 2, 0.1)
    want = step(m, x, IDS, dy)
    for ad in m.adapters.values():
        ad.A.requires_grad_(False)
        ad.A.grad = None
    g = GraphedTrainStep(m, x, IDS, dy, lr=0.0, need_dx=False)
    assert torch.equal(g(), want[0]) and g.dx is None
    for ad, db in zip(m.adapters.values(), want[3]):
        assert ad.A.grad is None and torch.equal(ad.B.grad, db)


# ------------------------------------------------------------------ plans

@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("dt", [BF, F32])
def test_layers_share_a_resident_plan(dt, eight):
    # one shape and one packed size, other scalings or ranks
    layers = [layer(256, 192, r, dt, seed=i) for i, r in enumerate((RANKS, RANKS, {0: 72, 1: 3, 2: 64}))]
    for ad in layers[1].adapters.values():
        ad.scaling *= 3
    x, dy = randn((len(IDS), 256), dt, 1), randn((len(IDS), 192), dt, 2, 0.1)
    for m in layers:
        if eight:
            m.quantize_base()
            m.save_input = "int8"
    want = [step(m, x, IDS, dy) for m in layers]
    plan = layers[0].route(IDS)
    for m in layers:
        m.make_resident(plan)
    for _ in range(2):
        for m, (y, dx, dA, dB) in zip(layers, want):
            got = step(m, x, IDS, dy, plan)
            assert torch.equal(got[0], y) and torch.equal(got[1], dx)
            for a, b in zip(got[2] + got[3], dA + dB):
                assert torch.equal(a, b)
    layers[0].adapters["1"].scaling *= 2  # no longer what was uploaded
    assert torch.equal(step(layers[0], x, IDS, dy, plan)[0], step(layers[0], x, IDS, dy)[0])
    assert _lib.device_error() == 0


def test_a_plan_that_changes_between_calls():
    m = layer(256, 192, RANKS, BF).quantize_base()
    x, dy = randn((len(IDS), 256), BF, 1), randn((len(IDS), 192), BF, 2, 0.1)
    plan = m.route(IDS)
    for ids in (IDS, IDS.flip(0).contiguous(), IDS):
        new = m.route(ids)
        plan.seg_start, plan.seg_adapter, plan.perm = new.seg_start, new.seg_adapter, new.perm
        for a, b in zip(step(m, x, ids, dy, plan), step(m, x, ids, dy)):
            assert all(torch.equal(u, v) for u, v in zip(a, b)) if isinstance(a, list) else torch.equal(a, b)


@pytest.mark.parametrize("eight", [False, True])
def test_a_plan_that_changes_before_the_backward(eight):
    """The gradients are those of the forward that was made."""
    m = layer(256, 192, RANKS, BF)
    if eight:
        m.quantize_base()
        m.save_input = "int8"
    x, dy = randn((len(IDS), 256), BF, 1), randn((len(IDS), 192), BF, 2, 0.1)
    mixed = IDS[torch.randperm(len(IDS), generator=torch.Generator().manual_seed(3))]
    for ids in (IDS, mixed):
        want = step(m, x, ids, dy)
        plan, other = m.route(ids), m.route(torch.full_like(ids, 2))
        for ad in m.adapters.values():
            ad.A.grad = ad.B.grad = None
        xg = x.clone().requires_grad_(True)
        y = m(xg, ids, plan=plan)
        plan.seg_start, plan.seg_adapter, plan.perm, plan.active = (other.seg_start, other.seg_adapter, other.perm,
                                                                    other.active)
        y.backward(dy)
        assert torch.equal(xg.grad, want[1])
        for ad, a, b in zip(m.adapters.values(), want[2], want[3]):
            assert torch.equal(ad.A.grad, a) and torch.equal(ad.B.grad, b)


# ------------------------------------------------------------------ buffers of a native caller

def odd(t):
    """A copy of t that starts one element past a 256-byte boundary."""
    if t is None:
        return None
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    out = buf[1:].view(t.shape)
    out.copy_(t)
    assert out.data_ptr() % 16 == t.element_size()
    return out


def native_step(m, x, ids, dy, where, save8=True):
    """One forward and backward through the C entry points; ``where`` places
    every tensor of the caller's that has the layer's type."""
    dt, (rows, d_in), d_out = x.dtype, x.shape, dy.shape[1]
    pk, plan, b8 = m._pack(), m.route(ids), m.base.rows8
    pk.sync()
    st = pk.state(plan, m.impl, b8, save8)
    call = ops._Call(rows, d_in, d_out, ops.mlora_dtype(dt), st)
    A, B, bias = where(pk.A_pack), where(pk.B_pack), where(m.base.bias.detach())
    x, dy = where(x), where(dy)
    y, dx = where(torch.zeros(rows, d_out, device="cuda", dtype=dt)), where(torch.zeros_like(x))
    dA, dB = where(torch.zeros_like(A)), where(torch.zeros_like(B))
    z = where(torch.zeros(max(1, call.zbytes // x.element_size()), device="cuda", dtype=dt))
    ws = torch.empty(call.wbytes, dtype=torch.uint8, device="cuda")
    r8, g8 = ops._new_rows8(rows, d_in, x.device), ops._Scratch8(rows, d_out, x.device)
    q8 = ops._q8_struct(b8, r8, g8)
    s, p, r = ops._stream(x.device), ctypes.byref(call.prob), ctypes.byref(call.route)
    ptr = ops._ptr
    _lib.call("mlora_forward_q8", p, r, ctypes.byref(q8), ptr(x), None, ptr(bias), ptr(A), ptr(B), ptr(y), ptr(z),
              ptr(ws), call.wbytes, s)
    scratch = torch.empty(max(1, call.scratch8()), dtype=torch.uint8, device="cuda")
    q8.scratch, q8.scratch_bytes = scratch.data_ptr(), call.scratch8()
    if not save8:
        q8.Xq = q8.x_scale = None
    _lib.call("mlora_backward_q8", p, r, ctypes.byref(q8), ptr(dy), None if save8 else ptr(x), None, ptr(A), ptr(B),
              ptr(z), ptr(dx), ptr(dA), ptr(dB), ptr(ws), call.wbytes, s)
    torch.cuda.synchronize()
    act = plan.active
    return (y, dx, [dA[o:o + k] if act[i] else None for i, (o, k) in enumerate(pk.table.spans())],
            [dB[:, o:o + k] if act[i] else None for i, (o, k) in enumerate(pk.table.spans())])


def check(m, w, x, ids, dy, got, base8=True, save8=True):
    ads = [(a.A.detach(), a.B.detach(), a.scaling) for a in m.adapters.values()]
    slot = torch.full_like(ids, -1).cuda()
    for i, k in enumerate(m.adapters):
        slot[ids.cuda() == int(k)] = i
    y, dx, dA, dB = ref.lora(x, slot, w, m.base.bias, ads, dy, base8, save8)
    ref.assert_within(got[0], *y, what="y")
    ref.assert_within(got[1], *dx, what="dx")
    for i in range(len(ads)):
        if dA[i] is None:
            assert got[2][i] is None and got[3][i] is None
            continue
        ref.assert_within(got[2][i], *dA[i], what=f"dA{i}")
        ref.assert_within(got[3][i], *dB[i], what=f"dB{i}")
    assert _lib.device_error() == 0


@pytest.mark.parametrize("save8", [False, True])
@pytest.mark.parametrize("rows", [5, 262])
@pytest.mark.parametrize("dt", [F32, BF, FP])
def test_buffers_aligned_to_their_elements_only(dt, rows, save8):
    m = layer(256, 192, RANKS, dt)
    w = m.base.weight.detach().clone()
    m.quantize_base()
    ids = IDS[torch.linspace(0, len(IDS) - 1, rows).long()]
    x, dy = randn((rows, 256), dt, 1), randn((rows, 192), dt, 2, 0.1)
    for where in (odd, lambda t: t.clone()):
        check(m, w, x, ids, dy, native_step(m, x, ids, dy, where, save8), save8=save8)


# ------------------------------------------------------------------ product

@pytest.mark.parametrize("rows", [4, 300])
def test_copied_input_lives_until_the_launch(rows):
    # with filled new memory a copy of x that is released early would be overwritten by y's
    w8 = ops.quantize_rows(randn((256, 256), BF, 2))  # y is as large as the copy
    x = randn((256, rows), BF, 1).t()
    want = ops.int8_linear(x.contiguous(), w8)
    torch.cuda.synchronize()
    was = torch.are_deterministic_algorithms_enabled()
    torch.use_deterministic_algorithms(True)
    try:
        torch.cuda.empty_cache()
        got = [ops.int8_linear(x, w8) for _ in range(3)]
    finally:
        torch.use_deterministic_algorithms(was)
    assert all(torch.equal(y, want) for y in got)


def test_more_rows_than_one_launch_of_the_float32_expand():
    rows = 64 * 65535 + 300  # blocks of 64 rows; a grid holds 65,535 in its second dimension
    m = layer(16, 16, {0: 4, 1: 8}, F32).quantize_base()
    ids = torch.cat([torch.zeros(rows - 200, dtype=torch.int64), torch.ones(200, dtype=torch.int64)])
    x, dy = randn((rows, 16), F32, 1), randn((rows, 16), F32, 2)
    y, dx, dA, dB = step(m, x, ids, dy)
    for lo in (0, rows // 2, 64 * 65535 - 150, rows - 300):
        part = slice(lo, lo + 300)
        yp, dxp, _, _ = step(m, x[part], ids[part], dy[part])
        assert torch.equal(y[part], yp) and torch.equal(dx[part], dxp)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("rows", [3, 40])
@pytest.mark.parametrize("dt", [BF, F32])
def test_more_outputs_than_a_contraction_may_have(dt, rows):
    # d_out is no contraction of the forward, only of dx
    d_in, d_out = 80, _lib.Q8_MAX_K + 200
    x, w = randn((rows, d_in), dt, 1), randn((d_out, d_in), dt, 2, 0.1)
    b = randn((d_out,), dt, 3)
    w8 = ops.quantize_rows(w)
    ref.assert_within(ops.int8_linear(x, w8, b), *ref.linear(x, w, b), what="y")
    prob = _lib.Problem(rows, d_in, d_out, ops.mlora_dtype(dt), _lib.IMPL_SIMT)
    y, r8 = torch.empty(rows, d_out, device="cuda", dtype=dt), ops.quantize_rows(x)
    _lib.call("mlora_q8_linear", ctypes.byref(prob), None, 0, r8.q.data_ptr(), r8.scale.data_ptr(), w8.q.data_ptr(),
              w8.scale.data_ptr(), b.data_ptr(), y.data_ptr(), ops._stream(x.device))
    ref.assert_within(y, *ref.linear(x, w, b), what="y")
    with pytest.raises(NotImplementedError, match="contraction"):
        ops.int8_linear(x.requires_grad_(True), w8, b)
    m = layer(d_in, d_out, {0: 8}, dt)
    x, ids = x.detach(), torch.zeros(rows, dtype=torch.int64)
    w = m.base.weight.detach().clone()
    m.quantize_base()
    # without dx the layer trains its adapters
    dy = randn((rows, d_out), dt, 4, 0.1)
    y = m(x, ids)
    y.backward(dy)
    ad = m.adapters["0"]
    slot = torch.zeros(rows, dtype=torch.int64, device="cuda")
    (yw, by), _, dA, dB = ref.lora(x, slot, w, m.base.bias, [(ad.A.detach(), ad.B.detach(), ad.scaling)], dy, True, False)
    ref.assert_within(y, yw, by, what="y")
    ref.assert_within(ad.A.grad, *dA[0], what="dA")
    ref.assert_within(ad.B.grad, *dB[0], what="dB")
    with pytest.raises(NotImplementedError, match="contraction"):
        m(x.requires_grad_(True), ids)


@pytest.mark.parametrize("rows", [5, 40, 300])
@pytest.mark.parametrize("dt", [BF, F32])
def test_one_cta(dt, rows):
    """max_ctas = 1 leaves no pair of SMs: the CUDA-core product."""
    x, w, b = randn((rows, 200), dt, 1), randn((136, 200), dt, 2, 0.1), randn((136,), dt, 3)
    dy = randn((rows, 136), dt, 4, 0.1)
    w8 = ops.quantize_rows(w)
    prob = _lib.Problem(rows, 200, 136, ops.mlora_dtype(dt), _lib.IMPL_AUTO, 1)
    y, dx = torch.empty(rows, 136, device="cuda", dtype=dt), torch.empty_like(x)
    r8, g8 = ops._Scratch8(rows, 200, x.device), ops._Scratch8(rows, 136, x.device)
    s = ops._stream(x.device)
    _lib.call("mlora_q8_linear", ctypes.byref(prob), x.data_ptr(), 200, *r8.ptrs, w8.q.data_ptr(), w8.scale.data_ptr(),
              b.data_ptr(), y.data_ptr(), s)
    _lib.call("mlora_q8_linear_dx", ctypes.byref(prob), dy.data_ptr(), *g8.ptrs, w8.q.data_ptr(), w8.scale.data_ptr(),
              dx.data_ptr(), s)
    ref.assert_within(y, *ref.linear(x, w, b), what="y")
    ref.assert_within(dx, *ref.linear_dx(dy, w), what="dx")


def test_second_derivatives_are_refused():
    w8 = ops.quantize_rows(randn((48, 64), BF, 2))
    x = randn((5, 64), BF, 1).requires_grad_(True)
    dy = randn((5, 48), BF, 3).requires_grad_(True)
    dx, = torch.autograd.grad(ops.int8_linear(x, w8), x, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="not have been used"):  # not a zero
        torch.autograd.grad(dx.float().sum(), dy, retain_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.float().sum().backward()


# ------------------------------------------------------------------ values that are not finite

@pytest.mark.parametrize("base8", [False, True])
@pytest.mark.parametrize("dt", [BF, FP, F32])
def test_infinite_upstream_gradients(dt, base8):
    m = layer(256, 192, RANKS, dt)
    if base8:
        m.quantize_base()
    m.save_input = "int8"
    x, dy = randn((len(IDS), 256), dt, 1), randn((len(IDS), 192), dt, 2, 0.1)
    _, dx0, dA0, dB0 = step(m, x, IDS, dy)
    dy[100, 7] = float("inf")  # a row of adapter 1, in a tile with all three
    _, dx, dA, dB = step(m, x, IDS, dy)
    rest = [i for i in range(len(IDS)) if i != 100]
    assert torch.equal(dx[rest], dx0[rest]) and not torch.isfinite(dx[100]).any()
    for i in (0, 2):
        assert torch.equal(dA[i], dA0[i]) and torch.equal(dB[i], dB0[i])
    # dA = dZ^T (s q(x)): dZ of the row is infinite with the signs of B's row 7
    q, _ = ref.quantize(x[100:101])
    want = torch.sign(m.adapters["1"].B.detach()[7].double())[:, None] * q * float("inf")
    assert bool((q == 0).any()) and torch.equal(torch.isnan(dA[1]), torch.isnan(want))
    keep = ~torch.isnan(want)
    assert torch.equal(dA[1].double()[keep], want[keep])
    # dB = dY^T Z: only column 7 of dY is infinite
    others = [k for k in range(192) if k != 7]
    assert torch.equal(dB[1][others], dB0[1][others]) and not torch.isfinite(dB[1][7]).any()


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("rows", [4, 16])
def test_infinite_inputs_of_a_few_rows(dt, rows):
    m = layer(256, 192, {0: 8, 1: 64}, dt).quantize_base()
    ids = torch.arange(rows) % 2
    x = randn((rows, 256), dt, 1)
    with torch.no_grad():
        clean = m(x, ids)
        x[1, 9], x[2, 0] = float("-inf"), float("nan")
        y = m(x, ids)
    rest = [i for i in range(rows) if i not in (1, 2)]
    assert torch.equal(y[rest], clean[rest]) and torch.isnan(y[[1, 2]]).all()


ODD = torch.cat([torch.full((n,), a, dtype=torch.int64) for a, n in ((0, 50), (1, 1), (2, 330), (-1, 9), (3, 70), (4, 300))])


@pytest.mark.parametrize("base8, save8", [(True, False), (True, True), (False, True)])
@pytest.mark.parametrize("impl, dt, d_in, d_out", [("auto", BF, 264, 200), ("auto", FP, 264, 200), ("auto", F32, 264, 200),
                                                   ("simt", BF, 264, 200), ("simt", F32, 264, 200),
                                                   ("auto", BF, 100, 75)])
def test_bad_rows_reach_no_other_adapter(impl, dt, d_in, d_out, base8, save8):
    """Segments that end inside a slice of rows that the reductions take at a
    time: what is not finite in one segment's rows stays out of the others'."""
    m = layer(d_in, d_out, {0: 4, 1: 72, 2: 16, 3: 300, 4: 8}, dt)
    m.impl = impl
    if base8:
        m.quantize_base()
    m.save_input = "int8" if save8 else "full"
    rows = len(ODD)
    x, dy = randn((rows, d_in), dt, 1), randn((rows, d_out), dt, 2, 0.1)
    clean = step(m, x, ODD, dy)
    for row in (0, 49, 50, 51, 380, 381, 389, 390, 459, 460, rows - 1):
        owner = int(ODD[row])
        rest = [i for i in range(rows) if i != row]
        for bad_x in (True, False):
            xs, ds = x.clone(), dy.clone()
            (xs if bad_x else ds)[row, 3:6] = torch.tensor([float("inf"), float("nan"), float("-inf")])
            y, dx, dA, dB = step(m, xs, ODD, ds)
            assert torch.equal(y[rest], clean[0][rest]) and torch.equal(dx[rest], clean[1][rest])
            for i in range(5):
                if i != owner:
                    assert torch.equal(dA[i], clean[2][i]) and torch.equal(dB[i], clean[3][i]), (row, bad_x, i)
            if owner >= 0:
                assert not torch.isfinite(dA[owner]).all() and not torch.isfinite(dB[owner]).all()
    assert _lib.device_error() == 0


def test_graphed_step_outlives_what_it_captured():
    """The graph's kernels keep reading the weights they were captured with,
    wherever the module's own go afterwards."""
    for change in (lambda m: m.quantize_base(), lambda m: m.cpu(), lambda m: m.half()):
        m = layer(1024, 1024, RANKS, BF)
        x, dy = randn((len(IDS), 1024), BF, 1), randn((len(IDS), 1024), BF, 2, 0.1)
        g = GraphedTrainStep(m, x, IDS, dy, lr=0.0)
        want = g(x, dy).clone(), g.dx.clone()
        held = {t.untyped_storage().data_ptr() for t in g._kept}
        pk = m._pack()
        assert {pk.A_pack.data_ptr(), pk.B_pack.data_ptr(), m.base.weight.data_ptr(), m.base.bias.data_ptr()} <= held
        change(m)
        m._pack().sync()
        torch.cuda.empty_cache()
        y = g(x, dy)
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(g.dx, want[1])


# ------------------------------------------------------------------ bits kept

@pytest.mark.parametrize("base8", [False, True])
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("counts, ranks", [((1, 64, 200), (4, 16, 64)), ((40, 8, 0), (130, 1, 8)),
                                           ((6000, 90, 4100), (8, 33, 100))])
def test_dA_from_saved_rows_is_rounded_once(counts, ranks, dt, base8):
    m = layer(264, 192, dict(enumerate(ranks)), dt)
    if base8:
        m.quantize_base()
    m.save_input = "int8"
    ids = torch.cat([torch.full((n,), i, dtype=torch.int64) for i, n in enumerate(counts)])
    x, dy = randn((len(ids), 264), dt, 1), randn((len(ids), 192), dt, 2, 0.1)
    dA = step(m, x, ids, dy)[2]
    for i, ad in enumerate(m.adapters.values()):
        mine = (ids == i).cuda()
        if counts[i]:
            ref.assert_within(dA[i], *saved.dA_saved(x[mine], ad.B.detach(), ad.scaling, dy[mine]), what=f"dA{i}")
