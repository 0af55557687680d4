"""dA of the multi-LoRA linear from inputs saved in 8 bits, in float64, with the
error of the tensor-core kernels alone: dZ is never rounded to the layer's
type on this way.

    dA = sum_i w[i, :]^T q[i, :],   w = s_x c (dY B)

w is a float32 value held as two bf16 numbers: the first leaves at most 2^-8 of
it (half a step of bf16), the second at most 2^-8 of that, so 2^-16 in all.
The integers are exact.  One rounding to the layer's type at the end."""

import torch

import _int8_ref as ref

U = ref.U


def dA_saved(x, B, c, dy):
    """(dA, bound) of one adapter's rows: x [n, d_in], dy [n, d_out], B [d_out, r]."""
    q, s = ref.quantize(x)
    B, dyd, n, d_out = B.double(), dy.double(), x.shape[0], dy.shape[1]
    w = s[:, None] * c * (dyd @ B)
    wa = s[:, None] * abs(c) * (dyd.abs() @ B.abs())
    v = w.t() @ q
    # dZ: d_out products whose float32 sum may be truncated term by term (2 U
    # each), then two float32 products; the sums of n rows, high and low parts
    # apart, in slices of 64 rows (2 U a term), and their addition in parts
    ew = 2 ** -16 * w.abs() + 2 * (d_out + 3) * U * wa
    bound = ew.t() @ q.abs() + 2.02 * (n + 256) * U * (w.abs().t() @ q.abs())
    return v, 1.01 * (bound + ref.half_step(x.dtype) * v.abs()) + ref.tiny(x.dtype)


def dA_high_only(x, B, c, dy):
    """dA as it would be without the low parts, rounded to the type."""
    q, s = ref.quantize(x)
    w = (s[:, None] * c * (dy.double() @ B.double())).float()
    return (w.bfloat16().double().t() @ q).to(x.dtype)


def dA_both(x, B, c, dy):
    """dA of high and low parts, rounded to the type."""
    q, s = ref.quantize(x)
    w = (s[:, None] * c * (dy.double() @ B.double())).float()
    hi = w.bfloat16()
    lo = (w - hi.float()).bfloat16()
    return ((hi.double() + lo.double()).t() @ q).to(x.dtype)
