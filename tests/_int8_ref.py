"""The 8-bit operators in float64, from their definitions, with elementwise
bounds of what the kernels' arithmetic may add.

Half a step of a type is ``torch.finfo(t).eps / 2``; U is half a step of
float32, the type of the accumulators, scales and products."""

import torch

U = 2.0 ** -24


def half_step(dt):
    return torch.finfo(dt).eps / 2


def quantize(x, col_scale=None):
    """(integers, scales) of the rows of x as float64 tensors (the scale is a
    float32 number); rows with an infinity or a NaN give (0, NaN)."""
    if col_scale is not None:
        x = x.float() * col_scale
    x = x.double()
    top = x.abs().amax(1) if x.shape[1] else x.new_zeros(x.shape[0])
    s = (top / torch.full_like(top, 127.0)).float().double()
    bad = ~torch.isfinite(x).all(1)
    d = torch.where((s > 0) & ~bad, s, torch.ones_like(s))[:, None]
    q = torch.where(bad[:, None], torch.zeros_like(x), x / d).round().clamp(-127, 127)
    q = torch.where((s > 0)[:, None], q, torch.zeros_like(q))
    return q, torch.where(bad, torch.full_like(s, float("nan")), s)


def linear(x, w, bias):
    """(y, bound): the product rounds float(acc) and multiplies twice (3 U of
    the product), adds the bias (U of what is added), then rounds to the type."""
    q, s = quantize(x)
    wq, ws = quantize(w)
    y = (q @ wq.t()) * s[:, None] * ws
    b = 3 * U * y.abs()
    if bias is not None:
        y = y + bias.double()
        b = b + 2 * U * y.abs()
    h = half_step(x.dtype)
    return y, 1.01 * (b + h * y.abs()) + tiny(x.dtype)


def linear_dx(dy, w):
    wq, ws = quantize(w)
    g, sg = quantize(dy, ws.float())
    dx = (g @ wq) * sg[:, None]
    return dx, 1.01 * (2 * U + half_step(dy.dtype)) * dx.abs() + tiny(dy.dtype)


def tiny(dt):
    """Half the spacing of the type's subnormal numbers."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def lora(x, ids, w, bias, ads, dy, base8, save8):
    """Values and elementwise bounds of y, dx, dA, dB of the multi-LoRA linear.

    ads: list of (A, B, scale).  The low-rank intermediates are rounded to the
    type once (h of their value, and of the accumulated products, n U of the
    sum of magnitudes for n terms; 2 U per term on the tensor cores, whose
    accumulation may truncate); 8-bit rows read back for dA are rounded to the
    type once (h)."""
    dt, h = x.dtype, half_step(x.dtype)
    d_in, d_out, rows = w.shape[1], w.shape[0], x.shape[0]
    xd, dyd = x.double(), dy.double()
    if base8:
        y, by = linear(x, w, bias)
        dx, bdx = linear_dx(dy, w)
    else:
        wd = w.double()
        y, dx = xd @ wd.t(), dyd @ wd
        by = 2 * d_in * U * (xd.abs() @ wd.abs().t())
        bdx = 2 * d_out * U * (dyd.abs() @ wd.abs())
        if bias is not None:
            y = y + bias.double()
    by, bdx = by.clone(), bdx.clone()
    if save8:
        q, s = quantize(x)
        kept = q * s[:, None]
    else:
        kept = xd
    dA, dB = [], []
    for i, (A, B, c) in enumerate(ads):
        m = ids == i
        A, B = A.double(), B.double()
        z, za = c * (xd[m] @ A.t()), abs(c) * (xd[m].abs() @ A.abs().t())
        ez = h * z.abs() + 2 * (d_in + 2) * U * za + tiny(dt)
        y[m] += z @ B.t()
        by[m] += ez @ B.abs().t() + 2 * (z.shape[1] + 64) * U * (z.abs() @ B.abs().t())
        g, ga = c * (dyd[m] @ B), abs(c) * (dyd[m].abs() @ B.abs())
        eg = h * g.abs() + 2 * (d_out + 2) * U * ga + tiny(dt)
        dx[m] += g @ A
        bdx[m] += eg @ A.abs() + 2 * (z.shape[1] + 64) * U * (g.abs() @ A.abs())
        if not bool(m.any()):
            dA.append(None)
            dB.append(None)
            continue
        n = 2 * (int(m.sum()) + 256)
        va, vb = g.t() @ kept[m], dyd[m].t() @ z
        ea = eg.t() @ kept[m].abs() + (n * U + (h if save8 else 0.0)) * (g.abs().t() @ kept[m].abs())
        eb = dyd[m].abs().t() @ ez + n * U * (dyd[m].abs().t() @ z.abs())
        dA.append((va, 1.01 * (ea + h * va.abs()) + tiny(dt)))
        dB.append((vb, 1.01 * (eb + h * vb.abs()) + tiny(dt)))
    return (y, 1.01 * (by + (h + U) * y.abs()) + tiny(dt)), (dx, 1.01 * (bdx + h * dx.abs()) + tiny(dt)), dA, dB


def assert_within(got, want, bound, what=""):
    """Elementwise |got - want| <= bound; NaN exactly where want has NaN."""
    got = got.detach().double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places"
    d = torch.where(nan, torch.zeros_like(want), (got - want).abs())
    b = torch.where(nan, torch.ones_like(bound), bound)
    over = d - b
    if over.numel():
        k = int(over.argmax())
        assert float(over.flatten()[k]) <= 0, (
            f"{what}: off by {float(d.flatten()[k]):.4g} where {float(b.flatten()[k]):.4g} is allowed "
            f"(index {k}, value {float(want.flatten()[k]):.6g})")
