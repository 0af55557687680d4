"""8-bit operators against their float64 definitions: the row quantizer
exactly, the products and the layer within elementwise bounds of the
arithmetic (tests/_int8_ref.py)."""

import numpy as np
import pytest
import torch

import _int8_ref as ref
from tlora_b200 import MultiLoRALinear, _lib, ops
from tlora_b200.graphs import GraphedTrainStep
from tlora_b200.multi_lora_linear import IndependentLoRALinear

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(shape, dt, seed, scale=1.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * scale).to(dt)


def ints(r8):
    return r8.q[:, :r8.cols].double()


def assert_rows8(r8, x, col_scale=None):
    q, s = ref.quantize(x, col_scale)
    assert torch.equal(torch.isnan(r8.scale), torch.isnan(s))
    keep = ~torch.isnan(s)
    assert torch.equal(r8.scale[keep].double(), s[keep])
    assert torch.equal(ints(r8), q)
    assert not r8.q[:, r8.cols:].any()


# ------------------------------------------------------------------ rows

@pytest.mark.parametrize("dt", [BF, FP, F32])
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 7), (2, 8), (5, 16), (33, 17), (9, 255), (7, 1000), (64, 1024),
                                         (5, 4096), (3, 11008), (2, 16384), (2, 20000), (2, 16390), (300, 64),
                                         # rows enough to fill the GPU: other splits of a row over threads
                                         (1200, 4096), (700, 8200), (600, 11008), (400, 14000), (300, 24000),
                                         (200, 40000), (40, 70000), (5000, 520), (9000, 40)])
def test_rows_are_exact(dt, rows, cols):
    x = randn((rows, cols), dt, rows * 7 + cols)
    assert_rows8(ops.quantize_rows(x), x)
    cs = torch.rand(cols, generator=gen(1), device="cuda") * 0.1
    assert_rows8(ops.quantize_rows(x, cs), x, cs)


@pytest.mark.parametrize("dt", [BF, FP, F32])
def test_rows_next_to_a_border(dt):
    # every quotient is within a step of k + 1/2 of some scale
    k = torch.arange(-127, 127, device="cuda", dtype=torch.float64) + 0.5
    tops = torch.tensor([127.0, 254.0, 1.0, 3.1416, 0.9999, 100.5, 6.1e-5, 127.0 * 2 ** -10], device="cuda",
                        dtype=torch.float64).to(dt).double()
    mid = (k[None, :] * tops[:, None] / 127).to(dt)
    up = torch.nextafter(mid.float(), torch.full_like(mid, 9e9).float()).to(dt) if dt == F32 else mid
    dn = torch.nextafter(mid.float(), torch.full_like(mid, -9e9).float()).to(dt) if dt == F32 else mid
    x = torch.cat([tops.to(dt)[:, None], mid, up, dn], 1).contiguous()
    x = torch.where(x.abs() > x[:, :1].abs(), x[:, :1], x)
    assert_rows8(ops.quantize_rows(x), x)


@pytest.mark.parametrize("dt", [BF, FP, F32])
def test_rows_of_zeros_infinities_and_tiny_values(dt):
    info = torch.finfo(dt)
    x = randn((8, 40), dt, 3)
    x[0] = 0
    x[1, 3] = float("inf")
    x[2, 39] = float("-inf")
    x[3, 0] = float("nan")
    x[4] = randn((40,), F32, 4).sign().to(dt) * (info.smallest_normal * info.eps)  # the smallest subnormal
    x[5] = (randn((40,), F32, 5) * 100 * info.smallest_normal).to(dt)
    x[6] = (randn((40,), F32, 6).clamp(-1, 1) * info.max).to(dt)
    r8 = ops.quantize_rows(x)
    assert_rows8(r8, x)
    back = ops.dequantize_rows(r8, dt)
    assert torch.isnan(back[1:4]).all() and torch.isfinite(back[[0, 4, 5, 6, 7]]).all()
    assert not back[0].any()


@pytest.mark.parametrize("dt", [BF, FP, F32])
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 100), (17, 64), (2, 4097), (0, 8)])
def test_rows_read_back(dt, rows, cols):
    x = randn((rows, cols), dt, 11)
    r8 = ops.quantize_rows(x)
    for out in (dt, F32):
        want = (r8.scale[:, None] * r8.q[:, :cols].float()).to(out)
        assert torch.equal(ops.dequantize_rows(r8, out), want)


def test_rows_of_views():
    x = randn((20, 256), BF, 5)
    for v in (x[:, :100], x[3:9, 8:72], x[::2], x.t(), x[:, ::2], x[:1].expand(6, 256), x[5:5]):
        assert_rows8(ops.quantize_rows(v), v.contiguous())


# ------------------------------------------------------------------ product

@pytest.mark.parametrize("dt", [BF, FP, F32])
@pytest.mark.parametrize("rows, d_in, d_out, bias", [
    (1, 64, 64, True), (1, 1, 1, True), (2, 4096, 129, False), (7, 1000, 1531, True), (16, 256, 4096, True),
    (17, 2048, 260, False), (33, 100, 72, True), (64, 512, 512, False), (128, 128, 256, True),
    (255, 333, 777, True), (256, 4096, 256, False), (300, 1040, 520, True), (513, 72, 1288, True),
    (1500, 640, 2056, True), (20, 520, 2100, True), (100, 200, 300, False), (128, 4096, 520, True),
    (129, 264, 520, True), (5000, 136, 1288, True), (300, 4112, 3, True)])
def test_product(dt, rows, d_in, d_out, bias):
    x, w = randn((rows, d_in), dt, 1), randn((d_out, d_in), dt, 2, d_in ** -0.5)
    b = randn((d_out,), dt, 3) if bias else None
    dy = randn((rows, d_out), dt, 4, 0.1)
    w8 = ops.quantize_rows(w)
    xg = x.clone().requires_grad_(True)
    y = ops.int8_linear(xg, w8, b)
    y.backward(dy)
    ref.assert_within(y, *ref.linear(x, w, b), what="y")
    ref.assert_within(xg.grad, *ref.linear_dx(dy, w), what="dx")
    # rows quantized once give the same bits
    assert torch.equal(ops.int8_linear(ops.quantize_rows(x), w8, b, dtype=dt), y)
    assert _lib.device_error() == 0


def test_product_of_extreme_integers():
    # the longest sums of the largest products: a 32-bit accumulator holds them
    d = _lib.Q8_MAX_K
    x = torch.full((3, d), 2.0, device="cuda", dtype=BF)
    x[1] = -2.0
    x[2, ::2] = -2.0
    w8 = ops.quantize_rows(torch.full((5, d), 0.5, device="cuda", dtype=BF))
    y = ops.int8_linear(x, w8)
    assert torch.equal(y, torch.tensor([[1.0 * d], [-1.0 * d], [0.0]], device="cuda").expand(3, 5).to(BF))
    with pytest.raises(NotImplementedError):
        ops.int8_linear(torch.ones(1, d + 16, device="cuda", dtype=BF),
                        ops.quantize_rows(torch.ones(1, d + 16, device="cuda", dtype=BF)))


@pytest.mark.parametrize("rows", [5, 300])
def test_bad_rows_stay_apart(rows):
    x, w = randn((rows, 192), BF, 1), randn((160, 192), BF, 2, 0.1)
    w8 = ops.quantize_rows(w)
    good = ops.int8_linear(x, w8)
    x[1, 7], x[3, 0] = float("nan"), float("inf")
    x[4] = 0
    y = ops.int8_linear(x, w8)
    assert torch.isnan(y[[1, 3]]).all() and not y[4].any()
    rest = [i for i in range(rows) if i not in (1, 3, 4)]
    assert torch.equal(y[rest], good[rest])


@pytest.mark.parametrize("dt", [BF, F32])
def test_product_of_views_and_no_rows(dt):
    w8 = ops.quantize_rows(randn((48, 96), dt, 2))
    big = randn((40, 200), dt, 1)
    for v in (big[:, :96], big[:, 7:103], big[::3, 96:192], randn((96, 9), dt, 5).t(), big[:1, :96].expand(4, 96)):
        assert torch.equal(ops.int8_linear(v, w8), ops.int8_linear(v.contiguous(), w8))
    x = torch.empty(0, 96, device="cuda", dtype=dt, requires_grad=True)
    y = ops.int8_linear(x, w8)
    assert y.shape == (0, 48)
    y.backward(torch.empty_like(y))
    assert x.grad.shape == (0, 96)
    # the upstream gradient may be any view
    x = randn((6, 96), dt, 7).requires_grad_(True)
    dy = randn((48, 6), dt, 8)
    g1, = torch.autograd.grad(ops.int8_linear(x, w8), x, dy.t())
    g2, = torch.autograd.grad(ops.int8_linear(x, w8), x, dy.t().contiguous())
    assert torch.equal(g1, g2)
    y = ops.int8_linear(x, w8)
    g1, = torch.autograd.grad(y.sum(), x)
    g2, = torch.autograd.grad(ops.int8_linear(x, w8), x, torch.ones(6, 48, device="cuda", dtype=dt))
    assert torch.equal(g1, g2)


def test_product_refusals():
    x, w8 = randn((4, 64), BF, 1), ops.quantize_rows(randn((32, 64), BF, 2))
    with pytest.raises(ValueError, match="features"):
        ops.int8_linear(randn((4, 32), BF, 1), w8)
    with pytest.raises(ValueError, match="shaped"):
        ops.int8_linear(randn((2, 2, 64), BF, 1), w8)
    with pytest.raises(ValueError, match="bias"):
        ops.int8_linear(x, w8, torch.zeros(32, device="cuda"))
    with pytest.raises(ValueError, match="bias"):
        ops.int8_linear(x, w8, torch.zeros(31, device="cuda", dtype=BF))
    with pytest.raises(NotImplementedError, match="frozen"):
        ops.int8_linear(x, w8, torch.zeros(32, device="cuda", dtype=BF, requires_grad=True))
    with pytest.raises(ValueError, match="type of y"):
        ops.int8_linear(ops.quantize_rows(x), w8)
    with pytest.raises(ValueError, match="dtype"):
        ops.int8_linear(x, w8, dtype=F32)
    with pytest.raises(NotImplementedError):
        ops.int8_linear(x.double(), w8)
    with pytest.raises(NotImplementedError):
        ops.quantize_rows(x.to(torch.int32))
    with pytest.raises(ValueError):
        ops.quantize_rows(x[0])
    with pytest.raises(ValueError, match="col_scale"):
        ops.quantize_rows(x, torch.ones(63, device="cuda"))
    with pytest.raises(RuntimeError, match="weight on"):
        ops.int8_linear(x.cpu(), w8)


# ------------------------------------------------------------------ layer

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


def step(m, x, ids, dy, plan=None, add_base=True):
    for ad in m.adapters.values():
        ad.A.grad = ad.B.grad = None
    xg = x.detach().clone().requires_grad_(True)
    y = m(xg, ids, plan=plan, add_base=add_base)
    y.backward(dy)
    return (y.detach(), xg.grad, [a.A.grad for a in m.adapters.values()], [a.B.grad for a in m.adapters.values()])


def check_layer(m, w, x, ids, dy, base8, save8, got=None):
    got = got or step(m, x, ids, dy)
    ads = [(a.A.detach(), a.B.detach(), a.scaling) for a in m.adapters.values()]
    b = m.base.bias
    keys = [int(k) for k in m.adapters]
    slot = torch.full_like(ids, -1).cuda()
    for i, k in enumerate(keys):
        slot[ids.cuda() == k] = i
    y, dx, dA, dB = ref.lora(x, slot, w, b, ads, dy, base8, save8)
    ref.assert_within(got[0], *y, what="y")
    ref.assert_within(got[1], *dx, what="dx")
    for i in range(len(ads)):
        if dA[i] is None:
            assert got[2][i] is None and got[3][i] is None
            continue
        ref.assert_within(got[2][i], *dA[i], what=f"dA{i}")
        ref.assert_within(got[3][i], *dB[i], what=f"dB{i}")
    assert _lib.device_error() == 0


def grouped(*runs):
    return torch.cat([torch.full((n,), a, dtype=torch.int64) for a, n in runs])


LAYERS = {
    # name: d_in, d_out, ranks by id, ids
    "one_row": (64, 64, {0: 4}, grouped((0, 1))),
    "one_job": (512, 256, {3: 16}, grouped((3, 300))),
    "no_job": (256, 192, {0: 8}, grouped((-1, 70))),
    "four_jobs": (1024, 1024, {0: 4, 1: 8, 2: 16, 3: 32}, grouped((0, 64), (1, 128), (2, 192), (3, 256))),
    "ranks": (264, 392, {0: 1, 1: 63, 2: 64, 3: 65, 4: 130, 5: 300}, grouped((0, 9), (1, 250), (2, 1), (3, 256), (4, 77),
                                                                     (5, 40))),
    "empty_and_unknown": (128, 256, {0: 8, 1: 16, 2: 4}, grouped((2, 30), (9, 300), (0, 3))),
    "tokens": (2048, 1536, {i: [8, 16, 32, 64][i % 4] for i in range(16)}, torch.arange(16)),
    "two_tokens_each": (768, 520, {i: 8 for i in range(8)}, torch.arange(8).repeat(2)),
    "unaligned": (100, 75, {0: 3, 1: 20}, grouped((0, 40), (1, 35))),
    # several tiles per pair of SMs, with fewer and with more k-blocks than a tile's expand waits for
    "many_tiles_short": (264, 2312, {0: 24, 1: 64, 2: 100}, grouped((0, 2100), (-1, 300), (1, 1200), (2, 1500))),
    "many_tiles": (2048, 2312, {i: 16 for i in range(9)}, torch.arange(9).repeat_interleave(563)),
    # long contractions over many tiles, forward and backward
    "long_rows": (8200, 3000, {0: 16, 1: 130}, grouped((0, 2500), (-1, 500), (1, 2700))),
    "long_columns": (2560, 8448, {i: 8 for i in range(4)}, torch.arange(4).repeat_interleave(1700)),
    # sums over rows long enough to be split
    "long_jobs": (520, 72, {0: 100, 1: 8}, grouped((0, 6000), (1, 4500))),
    "wide": (72, 2056, {0: 24, 1: 64}, grouped((0, 400), (1, 200))),
}


@pytest.mark.parametrize("base8, save8", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("dt", [BF, FP, F32])
@pytest.mark.parametrize("name", list(LAYERS))
def test_layer(name, dt, base8, save8):
    d_in, d_out, ranks, ids = LAYERS[name]
    m = layer(d_in, d_out, ranks, dt)
    w = m.base.weight.detach().clone()
    if base8:
        m.quantize_base()
    m.save_input = "int8" if save8 else "full"
    x, dy = randn((len(ids), d_in), dt, 1), randn((len(ids), d_out), dt, 2, 0.1)
    check_layer(m, w, x, ids, dy, base8, save8)
    # rows in any order: sorted by adapter inside, answered in the caller's order
    p = torch.randperm(len(ids), generator=torch.Generator().manual_seed(1))
    check_layer(m, w, x[p].contiguous(), ids[p], dy[p].contiguous(), base8, save8)


@pytest.mark.parametrize("dt", [BF, F32])
def test_layer_parts(dt):
    d_in, d_out, ranks, ids = LAYERS["four_jobs"]
    m = layer(d_in, d_out, ranks, dt, bias=False)
    w = m.base.weight.detach().clone()
    x, dy = randn((len(ids), d_in), dt, 1), randn((len(ids), d_out), dt, 2, 0.1)
    delta = step(m, x, ids, dy, add_base=False)
    m.quantize_base()
    full = step(m, x, ids, dy)
    check_layer(m, w, x, ids, dy, True, False, full)
    # the adapters alone do not see the backbone's type
    for a, b in zip(delta[2] + delta[3] + [delta[0], delta[1]],
                    (lambda s: s[2] + s[3] + [s[0], s[1]])(step(m, x, ids, dy, add_base=False))):
        assert torch.equal(a, b)
    # what is not asked for is not computed: inputs without gradients, frozen adapters
    m.save_input = "int8"
    saved = step(m, x, ids, dy)
    y = m(x, ids)
    assert torch.equal(y, full[0])
    for ad in m.adapters.values():
        ad.A.grad = ad.B.grad = None
        ad.A.requires_grad_(False)
    xg = x.clone().requires_grad_(True)
    m(xg, ids).backward(dy)
    assert torch.equal(xg.grad, full[1])
    assert all(a.A.grad is None for a in m.adapters.values())
    for a, g in zip(m.adapters.values(), saved[3]):
        assert torch.equal(a.B.grad, g)
    with torch.no_grad():
        assert torch.equal(m(x, ids), full[0])
    # and back
    m.dequantize_base()
    assert m.base.weight.dtype == dt
    ref.assert_within(m.base.weight, *(lambda q, s: (q * s[:, None], (q * s[:, None]).abs() *
                                                     (ref.half_step(dt) + ref.U) + ref.tiny(dt)))(*ref.quantize(w)))


def test_plain_linear_base_is_the_layer_without_jobs():
    m = layer(512, 384, {0: 8}, BF).quantize_base()
    x = randn((70, 512), BF, 1)
    assert torch.equal(m(x, torch.full((70,), -1)), m.base(x))
    assert torch.equal(m.base(x.view(7, 10, 512)).view(70, 384), m.base(x))


def test_independent_layer_in_8_bits():
    torch.manual_seed(0)
    one = IndependentLoRALinear(256, 192, 16).cuda().bfloat16()
    with torch.no_grad():
        one.adapter.B.normal_(0, 0.05)
    m = MultiLoRALinear(256, 192, {0: 16}).cuda().bfloat16()
    with torch.no_grad():
        m.base.weight.copy_(one.base.weight)
        m.base.bias.copy_(one.base.bias)
        m.adapters["0"].A.copy_(one.adapter.A)
        m.adapters["0"].B.copy_(one.adapter.B)
    m.adapters["0"].scaling = one.adapter.scaling
    one.quantize_base()
    m.quantize_base()
    one.save_input = m.save_input = "int8"
    x, dy = randn((40, 256), BF, 1), randn((40, 192), BF, 2)
    want = step(m, x, torch.zeros(40, dtype=torch.int64), dy)
    xg = x.clone().requires_grad_(True)
    y = one(xg.view(4, 10, 256))
    y.backward(dy.view(4, 10, 192))
    assert torch.equal(y.view(40, 192), want[0]) and torch.equal(xg.grad, want[1])
    assert torch.equal(one.adapter.A.grad, want[2][0]) and torch.equal(one.adapter.B.grad, want[3][0])


@pytest.mark.parametrize("dt", [BF, F32])
def test_bad_rows_reach_only_their_adapter(dt):
    d_in, d_out, ranks, ids = LAYERS["four_jobs"]
    m = layer(d_in, d_out, ranks, dt).quantize_base()
    m.save_input = "int8"
    x, dy = randn((len(ids), d_in), dt, 1), randn((len(ids), d_out), dt, 2, 0.1)
    clean = step(m, x, ids, dy)
    x[70, 5] = float("inf")  # a row of adapter 1, in a tile with rows of adapters 0 and 2
    y, dx, dA, dB = step(m, x, ids, dy)
    rest = [i for i in range(len(ids)) if i != 70]
    assert not torch.isfinite(y[70]).any()
    assert torch.equal(y[rest], clean[0][rest]) and torch.equal(dx, clean[1])
    assert torch.isnan(dA[1]).all()
    for i in (0, 2, 3):
        assert torch.equal(dA[i], clean[2][i])


def test_gradients_against_differences():
    """Central differences of L = <C, y>.  In A and B the layer is linear but
    for the product of the two, so the differences are exact up to U; the
    analytic dA reads x in 8 bits, half a step of the row's scale per element:
    |dA - FD| <= sum_i |dz_i| s_i / 2.  In x, both the differences (through
    8-bit x) and the gradient (through 8-bit dy) carry half a step per
    element."""
    d_in, d_out, ids = 256, 192, grouped((0, 40), (1, 50))
    m = layer(d_in, d_out, {0: 8, 1: 16}, F32)
    m.quantize_base()
    m.save_input = "int8"
    w8 = ints(m.base.rows8) * m.base.rows8.scale.double()[:, None]
    x, c = randn((90, d_in), F32, 1), randn((90, d_out), F32, 2)
    _, dx, dA, dB = step(m, x, ids, c)
    c64 = c.double()

    def loss(xx):
        with torch.no_grad():
            return float((m(xx, ids).double() * c64).sum())

    for i, ad in enumerate(m.adapters.values()):
        mine = (ids == i).cuda()
        dz = (ad.scaling * (c64[mine] @ ad.B.detach().double())).abs()
        sx = ops.quantize_rows(x).scale.double()[mine]
        for p, g, e in ((ad.A, dA[i], (dz * sx[:, None] / 2).sum(0)[:, None].expand(-1, d_in)),
                        (ad.B, dB[i], torch.zeros(d_out, ad.rank, device="cuda", dtype=torch.float64))):
            v = torch.randn(p.shape, generator=gen(9), device="cuda")
            h = 0.25
            old = p.detach().clone()
            with torch.no_grad():
                p.copy_(old + h * v)
                up = loss(x)
                p.copy_(old - h * v)
                dn = loss(x)
                p.copy_(old)
            fd, got = (up - dn) / (2 * h), float((g.double() * v.double()).sum())
            noise = float((e * v.double().abs()).sum())
            # float32 y's: U per operation and term of the sums
            y_abs = (x.double().abs() @ w8.abs().t() + 1).abs()
            noise += float(400 * ref.U * (y_abs * c64.abs()).sum()) / h
            assert abs(fd - got) <= noise, (i, fd, got, noise)
    # x: v along the sign of the gradient, so that the derivative is the sum of its magnitudes
    v = torch.sign(dx)
    h = 4.0
    fd = (loss(x + h * v) - loss(x - h * v)) / (2 * h)
    got = float((dx.double() * v.double()).sum())
    cw = (c64 @ w8).abs()
    s_up, s_dn = (ops.quantize_rows(x + t * h * v).scale.double()[:, None] for t in (1, -1))
    noise = float((cw * (s_up + s_dn) / 2).sum()) / (2 * h)
    r8 = m.base.rows8
    sg = ops.quantize_rows(c, r8.scale).scale.double()[:, None]
    noise += float((sg / 2 * ints(r8).abs().sum(0)).sum())
    noise *= 1.01
    assert abs(fd - got) <= noise and noise < 0.2 * abs(got), (fd, got, noise)


# ------------------------------------------------------------------ together, streams, graphs

@pytest.mark.parametrize("dt", [BF, FP])
def test_training_steps_in_a_graph(dt):
    d_in, d_out, ranks, ids = LAYERS["four_jobs"]
    eager = layer(d_in, d_out, ranks, dt).quantize_base()
    graphed = layer(d_in, d_out, ranks, dt).quantize_base()
    eager.save_input = graphed.save_input = "int8"
    xs = [randn((len(ids), d_in), dt, 10 + i) for i in range(3)]
    dys = [randn((len(ids), d_out), dt, 20 + i, 0.1) for i in range(3)]
    keep = eager(xs[0].clone().requires_grad_(True), ids)  # an eager graph of the same kind lives on
    lr = 0.5
    start = [p.detach().clone() for p in graphed.parameters()]
    g = GraphedTrainStep(graphed, xs[0], ids, dys[0], lr)
    with torch.no_grad():  # the warm-up stepped too: start again from the same weights
        for p, s in zip(graphed.parameters(), start):
            p.copy_(s)
    for x, dy in zip(xs, dys):
        y, dx, dA, dB = step(eager, x, ids, dy)
        eager.sgd_step(lr)
        yg = g(x, dy)
        assert torch.equal(yg, y) and torch.equal(g.dx, dx)
        for a, b in zip(graphed.parameters(), eager.parameters()):
            assert torch.equal(a, b)
    assert keep.shape == (len(ids), d_out)


def test_product_in_a_graph():
    w8 = ops.quantize_rows(randn((1024, 512), BF, 1))
    for rows in (1, 16, 200):
        x = randn((rows, 512), BF, 2)
        ops.int8_linear(x, w8)
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):  # two captured calls, replayed in turn and overlapping on two streams
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                y = ops.int8_linear(x, w8)
            graphs.append((g, y))
        streams = [torch.cuda.Stream() for _ in graphs]
        for k in range(3):
            x.copy_(randn((rows, 512), BF, 30 + k))
            want = ops.int8_linear(x, w8)
            torch.cuda.synchronize()
            for s, (g, _) in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(y, want) for _, y in graphs)


def test_calls_on_two_streams_at_once():
    d_in, d_out, ranks, ids = LAYERS["four_jobs"]
    m = layer(d_in, d_out, ranks, BF).quantize_base()
    m.save_input = "int8"
    data = [(randn((len(ids), d_in), BF, 40 + i), randn((len(ids), d_out), BF, 50 + i)) for i in range(2)]
    want = [step(m, x, ids, dy)[:2] for x, dy in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    for _ in range(5):
        got = []
        for s, (x, dy) in zip(streams, data):
            with torch.cuda.stream(s):
                xg = x.detach().clone().requires_grad_(True)
                y = m(xg, ids)
                got.append((y, torch.autograd.grad(y, xg, dy)[0]))
        torch.cuda.synchronize()
        for (y, dx), (yw, dxw) in zip(got, want):
            assert torch.equal(y, yw) and torch.equal(dx, dxw)


def test_repeated_steps_give_the_same_bits():
    d_in, d_out, ranks, ids = LAYERS["ranks"]
    m = layer(d_in, d_out, ranks, BF).quantize_base()
    m.save_input = "int8"
    x, dy = randn((len(ids), d_in), BF, 1), randn((len(ids), d_out), BF, 2)
    first = step(m, x, ids, dy)
    for _ in range(3):
        again = step(m, x, ids, dy)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
        for a, b in zip(first[2] + first[3], again[2] + again[3]):
            assert torch.equal(a, b)


def test_saved_rows_are_the_smaller_ones():
    m = layer(4096, 256, {0: 8}, BF)
    ids = torch.zeros(2048, dtype=torch.int64)

    def held(how):
        m.save_input = how
        x = randn((2048, 4096), BF, 1)
        y = m(x, ids)
        del x
        torch.cuda.synchronize()
        size = torch.cuda.memory_allocated()
        del y
        return size

    held("full")
    full, eight = held("full"), held("int8")
    assert full - eight >= 2048 * (4096 - 8)


def test_loading_an_8bit_checkpoint():
    a = layer(100, 64, {0: 8}, BF, seed=1).quantize_base()
    b = layer(100, 64, {0: 8}, BF, seed=2).quantize_base()
    b.load_state_dict(a.state_dict())
    x = randn((5, 100), BF, 1)
    ids = torch.zeros(5, dtype=torch.int64)
    assert torch.equal(a(x, ids), b(x, ids))
    c = b.cpu().cuda()
    assert torch.equal(c(x, ids), a(x, ids))
    assert np.isfinite(float(c(x, ids).detach().float().sum()))


# ------------------------------------------------------------------ edges of the layer

@pytest.mark.parametrize("dt", [BF, F32])
def test_layer_without_rows(dt):
    m = layer(64, 96, {0: 8}, dt).quantize_base()
    for how in ("full", "int8"):
        m.save_input = how
        x = torch.empty(0, 64, device="cuda", dtype=dt, requires_grad=True)
        y = m(x, torch.empty(0, dtype=torch.int64))
        y.backward(torch.empty_like(y))
        assert y.shape == (0, 96) and x.grad.shape == (0, 64)
        assert m.adapters["0"].A.grad is None and m.adapters["0"].B.grad is None


@pytest.mark.parametrize("base8", [False, True])
@pytest.mark.parametrize("dt", [BF, F32])
def test_cuda_core_kernels_on_request(dt, base8):
    d_in, d_out, ranks, ids = LAYERS["ranks"]
    m = layer(d_in, d_out, ranks, dt)
    m.impl = "simt"
    m.save_input = "int8"
    w = m.base.weight.detach().clone()
    if base8:
        m.quantize_base()
    x, dy = randn((len(ids), d_in), dt, 1), randn((len(ids), d_out), dt, 2, 0.1)
    check_layer(m, w, x, ids, dy, base8, True)


@pytest.mark.parametrize("dt", [BF, F32])
def test_delta_with_saved_inputs(dt):
    d_in, d_out, ranks, ids = LAYERS["four_jobs"]
    m = layer(d_in, d_out, ranks, dt)
    x, dy = randn((len(ids), d_in), dt, 1), randn((len(ids), d_out), dt, 2, 0.1)
    plain = step(m, x, ids, dy, add_base=False)
    m.save_input = "int8"
    with_base = step(m, x, ids, dy)
    delta = step(m, x, ids, dy, add_base=False)
    assert torch.equal(delta[0], plain[0])
    if dt == BF:  # (float32: other kernels of the low-rank terms, other roundings)
        assert torch.equal(delta[1], plain[1])
    for a, b in zip(delta[2] + delta[3], with_base[2] + with_base[3]):
        assert torch.equal(a, b)


def test_layer_refusals():
    m = layer(64, 96, {0: 8}, BF).quantize_base()
    ids = torch.zeros(4, dtype=torch.int64)
    x = randn((4, 64), BF, 1)
    with pytest.raises(ValueError, match="features"):
        m(randn((4, 72), BF, 1), ids)
    with pytest.raises(RuntimeError, match="dtype"):
        m(x.half(), ids)
    with pytest.raises(RuntimeError, match="CUDA"):
        m(x.cpu(), ids)
    with pytest.raises(ValueError, match="plan"):
        m(x, ids, plan=m.route(torch.zeros(5, dtype=torch.int64)))
    m.impl = "tc"
    odd = layer(100, 96, {0: 8}, BF).quantize_base()
    odd.impl = "tc"  # 16-bit rows of 100 columns are not a tensor-core operand
    with pytest.raises(NotImplementedError):
        odd(randn((4, 100), BF, 1), ids)


def test_copies_of_an_8bit_layer():
    import copy

    m = layer(128, 96, {0: 8}, BF).quantize_base()
    x, ids = randn((40, 128), BF, 1), torch.zeros(40, dtype=torch.int64)
    want = m(x, ids)
    twin = copy.deepcopy(m)
    assert torch.equal(twin(x, ids), want)
    with torch.no_grad():
        m.base.weight_q8.zero_()
    assert torch.equal(twin(x, ids), want)
    plan = twin.route(ids)
    twin(x, ids, plan=plan)
    again = copy.deepcopy(plan)  # a plan that has been used
    assert torch.equal(twin(x, ids, plan=again), want)


@pytest.mark.parametrize("eight", [False, True])
def test_capture_while_an_eager_graph_of_the_adapters_lives(eight):
    d_in, d_out, ranks, ids = LAYERS["four_jobs"]
    m = layer(d_in, d_out, ranks, BF)
    if eight:
        m.quantize_base()
        m.save_input = "int8"
    x, dy = randn((len(ids), d_in), BF, 1), randn((len(ids), d_out), BF, 2, 0.1)
    alive = m(x.clone().requires_grad_(True), ids)  # its nodes for the adapters are not released
    g = GraphedTrainStep(m, x, ids, dy, lr=0.0)
    y = g(x, dy)
    torch.cuda.synchronize()
    assert torch.equal(y, alive.detach())
    alive.backward(dy)
    assert m.adapters["0"].A.grad is not None


@pytest.mark.parametrize("dt", [BF, FP, F32])
def test_fused_sgd_of_the_native_call(dt):
    """MLORA_FUSED_SGD: the gradients of the call, and the weights that the
    separate step would give, bit by bit."""
    import ctypes

    d_in, d_out, ranks, ids = LAYERS["long_jobs"]
    m = layer(d_in, d_out, ranks, dt).quantize_base()
    m.save_input = "int8"
    x, dy = randn((len(ids), d_in), dt, 1), randn((len(ids), d_out), dt, 2, 0.1)
    want = step(m, x, ids, dy)
    pk = m._pack()
    plan = m.route(ids)
    st = pk.state(plan, "auto", m.base.rows8, True)
    r8 = ops._new_rows8(len(ids), d_in, x.device)
    y, z, _, _ = ops.forward_raw(x, None, m.base.bias, st, rows8=r8)
    call = ops._Call(len(ids), d_in, d_out, ops.mlora_dtype(dt), st)
    call.prob.flags, call.prob.lr = _lib.FUSED_SGD, 0.5
    ws = torch.empty(call.wbytes, dtype=torch.uint8, device="cuda")
    g8 = ops._Scratch8(len(ids), d_out, x.device)
    q8 = ops._q8_struct(m.base.rows8, r8, g8)
    scratch = torch.empty(max(1, call.scratch8()), dtype=torch.uint8, device="cuda")
    q8.scratch, q8.scratch_bytes = scratch.data_ptr(), call.scratch8()
    dx, dA, dB = torch.empty_like(x), torch.empty_like(pk.A_pack), torch.empty_like(pk.B_pack)
    old = [p.detach().clone() for p in pk.params()]
    _lib.call("mlora_backward_q8", ctypes.byref(call.prob), ctypes.byref(call.route), ctypes.byref(q8),
              dy.data_ptr(), None, None, pk.A_pack.data_ptr(), pk.B_pack.data_ptr(), z.data_ptr(), dx.data_ptr(),
              dA.data_ptr(), dB.data_ptr(), ws.data_ptr(), call.wbytes, ops._stream(x.device))
    torch.cuda.synchronize()
    assert torch.equal(dx, want[1])
    for i, (o, r) in enumerate(pk.table.spans()):
        assert torch.equal(dA[o:o + r], want[2][i]) and torch.equal(dB[:, o:o + r], want[3][i])
        for p, was, g in ((pk.params()[2 * i], old[2 * i], want[2][i]), (pk.params()[2 * i + 1], old[2 * i + 1],
                                                                       want[3][i])):
            ref_p = was.clone()
            ops.sgd_step_([(ref_p, g.contiguous())], 0.5)
            assert torch.equal(p, ref_p)
    # too little scratch is refused before anything runs
    if dt != F32:
        q8.scratch_bytes -= 1
        with pytest.raises(_lib.MloraError):
            _lib.call("mlora_backward_q8", ctypes.byref(call.prob), ctypes.byref(call.route), ctypes.byref(q8),
                      dy.data_ptr(), None, None, pk.A_pack.data_ptr(), pk.B_pack.data_ptr(), z.data_ptr(),
                      dx.data_ptr(), dA.data_ptr(), dB.data_ptr(), ws.data_ptr(), call.wbytes, ops._stream(x.device))


# ------------------------------------------------------------------ large

def test_offsets_past_32_bits():
    rows, cols = 70000, 32768  # 2.3e9 elements
    x = torch.empty(rows, cols, device="cuda", dtype=BF).normal_(generator=gen(1))
    r8 = ops.quantize_rows(x)
    back = ops.dequantize_rows(r8, BF)
    for s in (slice(0, 3), slice(rows - 3, rows), slice(65534, 65539)):
        part = ops.quantize_rows(x[s].contiguous())
        assert torch.equal(r8.q[s], part.q) and torch.equal(r8.scale[s], part.scale)
        assert torch.equal(back[s], ops.dequantize_rows(part, BF))
    del x, back
    # a product that reads and writes past them
    w8 = ops.quantize_rows(randn((40000, 32768), BF, 2))
    y = ops.int8_linear(r8, w8, dtype=BF)
    assert y.numel() > 2 ** 31
    for s in (slice(0, 2), slice(rows - 2, rows), slice(53700, 53702)):
        part = ops.Int8Rows(r8.q[s].contiguous(), r8.scale[s].contiguous(), cols)
        acc = ints(part) @ ints(w8).t()
        want = acc * part.scale.double()[:, None] * w8.scale.double()
        ref.assert_within(y[s], want, 1.01 * (3 * ref.U + ref.half_step(BF)) * want.abs() + ref.tiny(BF), "y")
    assert _lib.device_error() == 0
