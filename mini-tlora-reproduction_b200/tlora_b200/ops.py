"""Functional layer over the C ABI: routing, the fused forward/backward
autograd function and the isolated SGD step.

Reference call sites this mirrors:
  * boolean-mask routing          tlora/multi_lora_linear.py:111-116
  * contiguous packing (spans)    phase3_nano_batch.py:43-71, phase5c_fused_triton.py:338-377
  * fused kernel + autograd       phase5c_fused_triton.py:545-577, phase5d_triton_training.py:196-325
  * per-adapter SGD               phase5d_triton_training.py:554-559, phase3_nano_batch.py:90-107
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass, field
from typing import List, Optional, Sequence

import numpy as np
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import BF16, F16, F32, RANK_CHUNK, TILE_ROWS

_DTYPES = {torch.float32: F32, torch.bfloat16: BF16, torch.float16: F16}
_IMPLS = {"auto": _lib.IMPL_AUTO, "simt": _lib.IMPL_SIMT, "tc": _lib.IMPL_TC, "tc1": _lib.IMPL_TC_1SM,
          "tc2": _lib.IMPL_TC_2SM, "tcw": _lib.IMPL_TC_WIDE}


def mlora_dtype(dt: torch.dtype) -> int:
    if dt not in _DTYPES:
        raise NotImplementedError(f"dtype {dt} is not supported (float32, bfloat16 or float16)")
    return _DTYPES[dt]


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream(device):
    """The current stream of a CUDA device (no other: it is where the calls'
    pointers are checked to be a GPU's)."""
    if not isinstance(device, torch.device):
        device = torch.device(device)
    if device.type != "cuda":
        raise ValueError(f"expected a CUDA device, not {device}")
    index = device.index
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if index is None else index)


class _on:
    """``torch.cuda.device(device)`` that costs nothing where the device is
    the current one already."""

    __slots__ = ("device", "guard")

    def __init__(self, device: torch.device):
        self.device, self.guard = device, None

    def __enter__(self):
        if torch.cuda.current_device() != self.device.index:
            self.guard = torch.cuda.device(self.device)
            self.guard.__enter__()

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _no_tangents(*tensors) -> None:
    """Forward-mode derivatives are not computed: a tensor that carries one is
    refused, so that none is lost unseen."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("forward-mode derivatives (jvp) are not computed")


# ---------------------------------------------------------------------------
# adapter table: ranks, packed offsets, scaling
# ---------------------------------------------------------------------------

@dataclass
class AdapterTable:
    """Packed layout of a set of adapters: adapter ``ids[i]`` (slot i) owns
    rows [pack_off[i], pack_off[i] + rank[i]) of A_pack and the same columns
    of B_pack; every offset is a multiple of RANK_CHUNK."""

    ids: List[int]
    rank: np.ndarray      # int32 [n]
    pack_off: np.ndarray  # int32 [n]
    r_pack: int
    _dev_keys: dict = field(default_factory=dict, repr=False)
    _cuts: Optional[tuple] = field(default=None, init=False, repr=False)

    @staticmethod
    def build(ids: Sequence[int], ranks: Sequence[int]) -> "AdapterTable":
        rank = np.asarray(list(ranks), dtype=np.int32)
        pad = (rank + RANK_CHUNK - 1) // RANK_CHUNK * RANK_CHUNK
        off = np.zeros(len(rank), dtype=np.int32)
        if len(rank):
            off[1:] = np.cumsum(pad)[:-1]
        return AdapterTable(list(int(i) for i in ids), rank, off, int(pad.sum()))

    @property
    def n(self) -> int:
        return len(self.ids)

    def layout(self) -> bytes:
        """The ranks and packed offsets, as a key."""
        return self.rank.tobytes() + self.pack_off.tobytes()

    def _cut(self) -> tuple:
        """(layout, spans, pieces, their places), computed once per layout."""
        key = self.layout()
        if self._cuts is None or self._cuts[0] != key:
            spans = [(int(o), int(r)) for o, r in zip(self.pack_off, self.rank)]
            pieces, place, end = [], [0] * self.n, 0
            for i in sorted(range(self.n), key=lambda i: spans[i]):
                o, r = spans[i]
                place[i] = len(pieces) + 1
                pieces += [o - end, r]
                end = o + r
            self._cuts = (key, spans, pieces + [self.r_pack - end], place)
        return self._cuts

    def spans(self) -> list:
        """(first packed row, rank) of every slot, as plain integers."""
        return self._cut()[1]

    def pieces(self) -> tuple:
        """Lengths that cut the packed ranks into gaps and adapters, and the
        place of every slot's among them."""
        return self._cut()[2:]

    def slot_of(self) -> dict:
        return {a: i for i, a in enumerate(self.ids)}

    def device_keys(self, device: torch.device):
        """(sorted adapter ids int64, slot of each int32) on ``device``."""
        key = str(device)
        if key not in self._dev_keys:
            order = np.argsort(np.asarray(self.ids, dtype=np.int64), kind="stable")
            keys = torch.tensor(np.asarray(self.ids, dtype=np.int64)[order], device=device)
            slots = torch.tensor(order.astype(np.int32), device=device)
            self._dev_keys[key] = (keys, slots)
        return self._dev_keys[key]


# ---------------------------------------------------------------------------
# routing: per-row ids -> contiguous segments (+ optional permutation)
# ---------------------------------------------------------------------------

@dataclass
class RoutePlan:
    rows: int
    seg_start: np.ndarray    # int32 [n_seg + 1]
    seg_adapter: np.ndarray  # int32 [n_seg], slot or -1
    perm: Optional[torch.Tensor] = None  # int32 [rows] on device: sorted position -> source row
    active: np.ndarray = None            # bool [n_adapters]: adapter owns >= 1 row
    # workspaces that already hold this plan on the device (make_resident),
    # keyed by all that its tables hold; calls with such a key upload nothing
    resident: dict = field(default_factory=dict)
    # the C descriptions of calls made with this plan, by all that they hold
    # (its segments among it: a plan that changes gets new ones)
    calls: dict = field(default_factory=dict, init=False, repr=False)

    def __getstate__(self):
        return {**self.__dict__, "calls": {}}  # C structures are neither copied nor pickled

    @property
    def n_seg(self) -> int:
        return len(self.seg_adapter)


def _segments_from_runs(starts: np.ndarray, slots: np.ndarray, rows: int, n: int) -> RoutePlan:
    order = np.argsort(starts, kind="stable")
    starts, slots = starts[order], slots[order]
    seg_start = np.append(starts, rows).astype(np.int32)
    seg_adapter = slots.astype(np.int32)
    active = np.zeros(n, dtype=bool)
    active[seg_adapter[seg_adapter >= 0]] = True
    return RoutePlan(rows, seg_start, seg_adapter, None, active)


def _segments_from_counts(counts: np.ndarray, n: int, rows: int, perm: torch.Tensor) -> RoutePlan:
    # sorted order: slot 0..n-1, then rows with unknown ids
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
    keep = [s for s in range(n + 1) if counts[s] > 0]
    seg_start = np.array([starts[s] for s in keep] + [rows], dtype=np.int32)
    seg_adapter = np.array([s if s < n else -1 for s in keep], dtype=np.int32)
    active = counts[:n] > 0
    return RoutePlan(rows, seg_start, seg_adapter, perm, active)


def _use_runs(n_runs: int, run_slots: np.ndarray, rows: int) -> bool:
    n_tiles = max(1, (rows + TILE_ROWS - 1) // TILE_ROWS)
    grouped = n_runs == len(np.unique(run_slots))  # every adapter appears in one run
    return grouped or n_runs <= n_tiles


def route(ids: torch.Tensor, table: AdapterTable, device: torch.device) -> RoutePlan:
    """Segments for per-row adapter ids.  Ids already grouped (each adapter in
    one contiguous run, the packed layout of the reference's phase3-6 scripts)
    are used in place; interleaved ids are stably sorted by adapter, and the
    plan carries the permutation that gathers X (and dY) into adapter order
    and that the kernels use to write Y (and dX) back in the caller's order."""
    rows = int(ids.shape[0])
    n = table.n
    if rows == 0:
        return RoutePlan(0, np.zeros(1, np.int32), np.zeros(0, np.int32), None, np.zeros(n, bool))
    if ids.device.type != "cuda":
        # host ids: routing is host logic on an O(rows) integer array.  Fast
        # path: runs of equal raw id (one vectorised pass), mapped to slots.
        slot_of = table.slot_of()
        v = ids.detach().numpy().astype(np.int64, copy=False)
        head = np.empty(rows, dtype=bool)
        head[0] = True
        np.not_equal(v[1:], v[:-1], out=head[1:])
        starts = np.flatnonzero(head)
        if len(starts) <= max(64, 2 * n + 2, rows // TILE_ROWS + 1):
            rs = np.array([slot_of.get(int(a), -1) for a in v[starts]], dtype=np.int32)
            keep = np.ones(len(rs), dtype=bool)
            keep[1:] = rs[1:] != rs[:-1]  # adjacent runs that map to one slot merge
            starts, rs = starts[keep], rs[keep]
            if _use_runs(len(starts), rs, rows):
                return _segments_from_runs(starts, rs, rows, n)
        uniq, inv = np.unique(v, return_inverse=True)
        slots = np.array([slot_of.get(int(u), -1) for u in uniq], dtype=np.int32)[inv]
        key = np.where(slots < 0, n, slots)
        order = np.argsort(key, kind="stable").astype(np.int32)
        counts = np.bincount(key, minlength=n + 1)
        perm = torch.from_numpy(order).to(device)
        return _segments_from_counts(counts, n, rows, perm)

    ids64 = ids if ids.dtype == torch.int64 else ids.to(torch.int64)
    ids64 = ids64.contiguous()
    keys, slots_d = table.device_keys(ids.device)
    n_tiles = (rows + TILE_ROWS - 1) // TILE_ROWS
    max_runs = max(64, 2 * n + 2, n_tiles)
    out = torch.empty(2 + 2 * max_runs, dtype=torch.int32, device=ids.device)
    st = _stream(ids.device)
    _lib.call("mlora_route_runs", _ptr(ids64), rows, _ptr(keys), _ptr(slots_d), n, max_runs, _ptr(out), st)
    h = out.cpu().numpy()
    n_runs = int(h[0])
    if n_runs <= max_runs:
        starts = h[2:2 + 2 * n_runs:2].astype(np.int64)
        rs = h[3:3 + 2 * n_runs:2].astype(np.int32)
        if _use_runs(n_runs, rs, rows):
            return _segments_from_runs(starts, rs, rows, n)
    perm = torch.empty(rows, dtype=torch.int32, device=ids.device)
    counts = torch.empty(n + 1, dtype=torch.int32, device=ids.device)
    ws = torch.empty(max(1, _lib.lib().mlora_route_sort_workspace_bytes(rows, n)), dtype=torch.uint8,
                     device=ids.device)
    _lib.call("mlora_route_sort", _ptr(ids64), rows, _ptr(keys), _ptr(slots_d), n, _ptr(perm), _ptr(counts),
              _ptr(ws), st)
    return _segments_from_counts(counts.cpu().numpy().astype(np.int64), n, rows, perm)


def gather_rows(src: torch.Tensor, perm: torch.Tensor) -> torch.Tensor:
    dst = torch.empty_like(src)
    _lib.call("mlora_gather_rows", _ptr(src), _ptr(perm), src.shape[0], src.shape[1], mlora_dtype(src.dtype),
              _ptr(dst), _stream(src.device))
    return dst


def scatter_rows(src: torch.Tensor, perm: torch.Tensor) -> torch.Tensor:
    dst = torch.empty_like(src)
    _lib.call("mlora_scatter_rows", _ptr(src), _ptr(perm), src.shape[0], src.shape[1], mlora_dtype(src.dtype),
              _ptr(dst), _stream(src.device))
    return dst


# ---------------------------------------------------------------------------
# 8-bit rows
# ---------------------------------------------------------------------------

@dataclass
class Int8Rows:
    """A matrix [rows, cols] in 8 bits: int8 ``q`` [rows, ld] and one float
    ``scale`` [rows]; element (i, k) stands for ``scale[i] * q[i, k]``.  ``ld``
    is ``cols`` rounded up to 16 and the bytes past ``cols`` are zero.  Rows are
    tokens of an activation, or output channels of a weight."""

    q: torch.Tensor
    scale: torch.Tensor
    cols: int

    def __post_init__(self):
        q, s = self.q, self.scale
        if q.dim() != 2 or q.dtype != torch.int8 or q.shape[1] != q8_ld(self.cols) or not q.is_contiguous():
            raise ValueError(f"Int8Rows.q must be a contiguous int8 matrix [rows, {q8_ld(self.cols)}]")
        if s.dim() != 1 or s.dtype != torch.float32 or s.shape[0] != q.shape[0] or not s.is_contiguous():
            raise ValueError("Int8Rows.scale must be a contiguous float32 vector, one element per row")
        if s.device != q.device:
            raise ValueError(f"Int8Rows: q on {q.device} but scale on {s.device}")

    @property
    def rows(self) -> int:
        return self.q.shape[0]

    @property
    def shape(self):
        return (self.q.shape[0], self.cols)

    @property
    def device(self) -> torch.device:
        return self.q.device


def q8_ld(cols: int) -> int:
    """Bytes between the rows of an 8-bit matrix of ``cols`` columns."""
    return (int(cols) + 15) // 16 * 16


def _wrap8(q: torch.Tensor, scale: torch.Tensor, cols: int) -> Int8Rows:
    """Int8Rows of tensors made here: the layout is right by construction."""
    r = Int8Rows.__new__(Int8Rows)
    r.q, r.scale, r.cols = q, scale, cols
    return r


def _new_rows8(rows: int, cols: int, device) -> Int8Rows:
    return _wrap8(torch.empty((rows, q8_ld(cols)), dtype=torch.int8, device=device),
                  torch.empty(rows, dtype=torch.float32, device=device), cols)


class _Scratch8:
    """8-bit rows that live for one call: one buffer, the scales after the rows."""

    __slots__ = ("buf", "ptrs")

    def __init__(self, rows: int, cols: int, device):
        n = rows * q8_ld(cols)
        self.buf = torch.empty(n + 4 * rows, dtype=torch.uint8, device=device)
        p = self.buf.data_ptr()
        self.ptrs = (p, p + n)


def _ptrs8(m):
    if m is None:
        return None, None
    return m.ptrs if isinstance(m, _Scratch8) else (m.q.data_ptr(), m.scale.data_ptr())


def _q8_struct(base8: Optional[Int8Rows], rows8, grad8=None):
    return _lib.Q8(*_ptrs8(base8), *_ptrs8(rows8), *_ptrs8(grad8))


def _check_cuda(t: torch.Tensor, what: str) -> None:
    if t.device.type != "cuda":
        raise RuntimeError(f"{what} computes on CUDA devices only (sm_100a); there is no CPU path")


def _row_major(x: torch.Tensor):
    """(x, elements between rows): rows with unit column stride are read in
    place, anything else is copied."""
    if x.is_contiguous():
        return x, x.shape[1]
    ld, one = x.stride()
    if x.shape[0] <= 1 or x.shape[1] <= 1 or one != 1 or ld < x.shape[1]:
        return x.contiguous(), x.shape[1]
    return x, ld


def quantize_rows(x: torch.Tensor, col_scale: Optional[torch.Tensor] = None) -> Int8Rows:
    """8-bit rows of ``x`` [rows, cols] (float32, bfloat16 or float16):
    ``scale[i] = float32(max_k |x[i, k]| / 127)`` and
    ``q[i, k] = round(x[i, k] / scale[i])``, ties to even, the quotient rounded
    exactly.  With ``col_scale`` (float32 [cols]) ``x`` is multiplied by it
    first, in float32.  A row of zeros has scale 0; a row with an infinity or a
    NaN has scale NaN and zeros.  Differentiable use goes through
    :func:`int8_linear` and ``MultiLoRALinear``."""
    _check_cuda(x, "quantize_rows")
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError("quantize_rows expects x shaped [rows, cols] with at least one column")
    dt = mlora_dtype(x.dtype)
    if col_scale is not None and (col_scale.dtype != torch.float32 or col_scale.shape != (x.shape[1],) or
                                  col_scale.device != x.device):
        raise ValueError("col_scale must be a float32 vector on x's device, one element per column")
    with _on(x.device):
        x, ld = _row_major(x.detach())
        cs = col_scale.detach().contiguous() if col_scale is not None else None
        out = _new_rows8(x.shape[0], x.shape[1], x.device)
        _lib.call("mlora_q8_quantize", _ptr(x), x.shape[0], x.shape[1], ld, dt, _ptr(cs), _ptr(out.q),
                  _ptr(out.scale), _stream(x.device))
    return out


def dequantize_rows(rows8: Int8Rows, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The matrix [rows, cols] that 8-bit rows stand for, rounded once to ``dtype``."""
    _check_cuda(rows8.q, "dequantize_rows")
    dt = mlora_dtype(dtype)
    with _on(rows8.device):
        out = torch.empty(rows8.rows, rows8.cols, dtype=dtype, device=rows8.device)
        _lib.call("mlora_q8_dequantize", _ptr(rows8.q), _ptr(rows8.scale), rows8.rows, rows8.cols, dt, _ptr(out),
                  _stream(rows8.device))
    return out


class Int8LinearFunction(torch.autograd.Function):
    """y = x W^T + b with x and W in 8 bits; dx through the 8-bit rows of
    dy * (W's scales), no gradient of W or b (both frozen)."""

    @staticmethod
    def forward(ctx, x, wq, w_scale, bias, d_in):
        ctx.save_for_backward(wq, w_scale)
        ctx.d_in = d_in
        return _int8_product(x, _wrap8(wq, w_scale, d_in), bias, x.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        wq, w_scale = ctx.saved_tensors
        rows, d_out, d_in = dy.shape[0], wq.shape[0], ctx.d_in
        dev = dy.device
        with _on(dev):
            dy = dy.contiguous()
            g8 = _Scratch8(rows, d_out, dev)
            dx = torch.empty((rows, d_in), dtype=dy.dtype, device=dev)
            prob = _lib.Problem(rows, d_in, d_out, mlora_dtype(dy.dtype), _lib.IMPL_AUTO)
            _lib.call("mlora_q8_linear_dx", ctypes.byref(prob), _ptr(dy), *g8.ptrs, _ptr(wq), _ptr(w_scale),
                      _ptr(dx), _stream(dev))
        return dx, None, None, None, None


def _int8_product(x, weight: Int8Rows, bias, dtype):
    q = weight.q
    dev = q.device
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _int8_product(x, weight, bias, dtype)
    rows, d_in, d_out = x.shape[0], weight.cols, q.shape[0]
    if isinstance(x, Int8Rows):
        src, ld, (xq, xs) = None, 0, _ptrs8(x)
    else:
        # rows and their 8-bit form stay alive until the launch: y must not take their memory
        src, ld = _row_major(x.detach() if x.requires_grad else x)
        kept = _Scratch8(rows, d_in, dev)
        xq, xs = kept.ptrs
    y = torch.empty((rows, d_out), dtype=dtype, device=dev)
    prob = _lib.Problem(rows, d_in, d_out, _DTYPES[dtype], _lib.IMPL_AUTO)
    _lib.call("mlora_q8_linear", ctypes.byref(prob), _ptr(src), ld, xq, xs, q.data_ptr(), weight.scale.data_ptr(),
              _ptr(bias), y.data_ptr(), _stream(dev))
    return y


def _check_dx8(weight: Int8Rows) -> None:
    """Before a forward whose input wants a gradient."""
    if weight.q.shape[0] > _lib.Q8_MAX_K:
        raise NotImplementedError(f"the input's gradient is a contraction over {weight.q.shape[0]} outputs: an 8-bit "
                                  f"product sums up to {_lib.Q8_MAX_K}")


def int8_linear(x, weight: Int8Rows, bias: Optional[torch.Tensor] = None,
                dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Matrix product in 8-bit integers with a scale per token and per output
    channel: ``y[i, j] = s_x[i] s_w[j] sum_k q_x[i, k] q_w[j, k] + bias[j]``.

    ``x`` is a tensor [rows, in_features] (float32, bfloat16 or float16; its
    rows are quantized as by :func:`quantize_rows`, and the gradient flows back
    to it) or an :class:`Int8Rows` (rows quantized once for several products;
    then ``dtype``, or the bias's type, is the type of ``y``).  ``weight`` holds the
    8-bit rows of W [out_features, in_features] (``quantize_rows(W)``) and is
    frozen, like the backbone of ``MultiLoRALinear``.  Sums run over at most
    131,072 terms: in_features, and out_features where x wants a gradient."""
    if not isinstance(weight, Int8Rows):
        raise TypeError("int8_linear expects weight as Int8Rows (quantize_rows(W))")
    if forward_ad._current_level >= 0:
        _no_tangents(None if isinstance(x, Int8Rows) else x, bias)
    dev = weight.q.device
    if dev.type != "cuda":
        _check_cuda(weight.q, "int8_linear")
    eight = isinstance(x, Int8Rows)
    if not eight and x.dim() != 2:
        raise ValueError("int8_linear expects x shaped [rows, in_features]")
    if x.shape[1] != weight.cols:
        raise ValueError(f"x has {x.shape[1]} features, the weight {weight.cols}")
    if x.device != dev:
        raise RuntimeError(f"input on {x.device} but weight on {dev}")
    if not eight:
        if dtype is not None and dtype != x.dtype:
            raise ValueError("dtype applies to 8-bit input; a tensor's product has its own type")
        dtype = x.dtype
    elif dtype is None:
        if bias is None:
            raise ValueError("int8_linear of 8-bit rows needs the type of y (dtype or bias)")
        dtype = bias.dtype
    mlora_dtype(dtype)
    grad = torch.is_grad_enabled()
    if bias is not None:
        if bias.dtype != dtype or bias.dim() != 1 or bias.shape[0] != weight.q.shape[0] or bias.device != dev:
            raise ValueError("bias must be a vector of y's type on the weight's device, one element per output")
        if grad and bias.requires_grad:
            raise NotImplementedError("the 8-bit linear is frozen: no gradient of its bias")
        if not bias.is_contiguous():
            bias = bias.contiguous()
    if grad and not eight and x.requires_grad:
        _check_dx8(weight)
        return Int8LinearFunction.apply(x, weight.q, weight.scale, bias, weight.cols)
    return _int8_product(x, weight, bias, dtype)


# ---------------------------------------------------------------------------
# C structs for one call
# ---------------------------------------------------------------------------

class _CallArgs:
    """Keeps the numpy arrays behind the ctypes structs alive for one call."""

    def __init__(self, rows, d_in, d_out, dtype, impl, plan: RoutePlan, table: AdapterTable,
                 scaling: np.ndarray, max_ctas: int = 0, out_rows: Optional[torch.Tensor] = None, flags: int = 0,
                 err_word: Optional[torch.Tensor] = None):
        # err_word: a device int32 tensor that receives this call's device-side
        # flags (bounds bit 0, timeout bit 1) instead of the library-wide word
        if err_word is not None and (err_word.dtype != torch.int32 or err_word.device.type != "cuda"):
            raise ValueError("err_word must be a CUDA int32 tensor")
        self.prob = _lib.Problem(rows, d_in, d_out, dtype, _IMPLS[impl], int(max_ctas), int(flags),
                                 err_word.data_ptr() if err_word is not None else None)
        self.err_word = err_word  # kept alive for the call
        self.seg_start = np.ascontiguousarray(plan.seg_start, dtype=np.int32)
        self.seg_adapter = np.ascontiguousarray(plan.seg_adapter, dtype=np.int32)
        self.rank = np.ascontiguousarray(table.rank, dtype=np.int32)
        self.pack_off = np.ascontiguousarray(table.pack_off, dtype=np.int32)
        self.scaling = np.ascontiguousarray(scaling, dtype=np.float32)
        self.route = _lib.Routing(
            len(self.seg_adapter), _lib.i32_ptr(self.seg_start), _lib.i32_ptr(self.seg_adapter),
            table.n, _lib.i32_ptr(self.rank), _lib.i32_ptr(self.pack_off), _lib.f32_ptr(self.scaling),
            table.r_pack, out_rows.data_ptr() if out_rows is not None else None)
        self.out_rows = out_rows  # kept alive for the call

    def sizes(self):
        z = ctypes.c_size_t(0)
        w = ctypes.c_size_t(0)
        _lib.call("mlora_zsave_bytes", ctypes.byref(self.prob), ctypes.byref(self.route), ctypes.byref(z))
        _lib.call("mlora_workspace_bytes", ctypes.byref(self.prob), ctypes.byref(self.route), ctypes.byref(w))
        return int(z.value), int(w.value)


def _call_key(rows, d_in, d_out, dtype, st: "LayerState") -> tuple:
    """All that the routing tables of a call are made from."""
    plan, table = st.plan, st.table
    head = (rows, d_in, d_out, dtype, st.impl, table.r_pack)
    try:
        return (head, table.rank.tobytes(), table.pack_off.tobytes(), st.scaling.tobytes(), plan.seg_start.tobytes(),
                plan.seg_adapter.tobytes())
    except AttributeError:  # lists
        return (head, *[np.asarray(a).tobytes() for a in (table.rank, table.pack_off, st.scaling, plan.seg_start,
                                                          plan.seg_adapter)])


class _Call:
    """One call made with a routing plan: a fresh mlora_problem over a
    mlora_routing and buffer sizes kept for the plan's present content."""

    __slots__ = ("args", "prob", "route", "zbytes", "wbytes", "active", "key", "_scratch")

    def __init__(self, rows, d_in, d_out, dtype, st: "LayerState"):
        plan, table = st.plan, st.table
        perm = plan.perm
        self.key = _call_key(rows, d_in, d_out, dtype, st)
        key = (self.key, None if perm is None else perm.data_ptr())
        kept = plan.calls.get(key)
        if kept is None:
            # copies: what is kept must not change with the caller's arrays
            args = _CallArgs(rows, d_in, d_out, dtype, st.impl,
                             RoutePlan(plan.rows, np.array(plan.seg_start), np.array(plan.seg_adapter)),
                             AdapterTable(table.ids, np.array(table.rank), np.array(table.pack_off), table.r_pack),
                             np.array(st.scaling), out_rows=perm)
            owners = set(args.seg_adapter[np.diff(args.seg_start) > 0].tolist())
            kept = (args, args.sizes(), [i in owners for i in range(table.n)], {})
            if len(plan.calls) >= 8:  # plans or scalings that change from call to call
                plan.calls.clear()
            plan.calls[key] = kept
        # active: the adapters that own rows, whose gradients are written
        self.args, (self.zbytes, self.wbytes), self.active, self._scratch = kept
        word = st.err_word
        if word is not None and (word.dtype != torch.int32 or word.device.type != "cuda"):
            raise ValueError("err_word must be a CUDA int32 tensor")
        self.prob = _lib.Problem(rows, d_in, d_out, dtype, _IMPLS[st.impl], 0, 0,
                                 word.data_ptr() if word is not None else None)
        self.route = self.args.route

    def scratch8(self) -> int:
        """mlora_q8_scratch_bytes of the call."""
        n = self._scratch.get("bytes")
        if n is None:
            sb = ctypes.c_size_t(0)
            _lib.call("mlora_q8_scratch_bytes", ctypes.byref(self.prob), ctypes.byref(self.route), ctypes.byref(sb))
            n = self._scratch["bytes"] = int(sb.value)
        return n


@dataclass
class LayerState:
    """Everything the autograd function needs besides the differentiable inputs."""

    table: AdapterTable
    scaling: np.ndarray
    plan: RoutePlan
    A_pack: torch.Tensor
    B_pack: torch.Tensor
    impl: str = "auto"
    max_ctas: int = 0  # cap on persistent-kernel CTAs (0 = one per SM)
    # device int32 tensor that receives the device-side flags of the calls made
    # with this state (bounds bit 0, timeout bit 1); None = the library-wide word
    err_word: Optional[torch.Tensor] = None
    # the backbone in 8 bits (then W is None), and whether the input is kept
    # in 8 bits for the backward
    base8: Optional["Int8Rows"] = None
    save8: bool = False


def make_resident(st: LayerState, rows: int, d_in: int, d_out: int, dtype: torch.dtype, device) -> torch.Tensor:
    """Upload the routing plan of ``st`` for calls of this shape into a
    workspace kept on the plan (mlora_plan_upload); later forward / backward
    calls with the same plan and shape then issue no host-to-device copy
    (MLORA_PLAN_RESIDENT), which lets a training step be captured into a
    CUDA graph.  Ranks, scalings and segments are part of the uploaded tables:
    layers that differ in them get a workspace each, and a captured graph keeps
    to those it was captured with."""
    code = mlora_dtype(dtype)
    key = _call_key(rows, d_in, d_out, code, st)
    if key in st.plan.resident:
        return st.plan.resident[key]
    args = _CallArgs(rows, d_in, d_out, code, st.impl, st.plan, st.table, st.scaling)
    _, wb = args.sizes()
    ws = torch.empty(max(wb, 1), dtype=torch.uint8, device=device)
    _lib.call("mlora_plan_upload", ctypes.byref(args.prob), ctypes.byref(args.route), _ptr(ws), wb, _stream(device))
    st.plan.resident[key] = ws
    return ws


def _workspace(st: LayerState, args, wb, device):
    """(workspace, flags) of a call: the plan's resident workspace when there
    is one for this shape, else a fresh one the call uploads the plan into."""
    ws = None
    if st.plan.resident:
        p = args.prob
        ws = st.plan.resident.get(args.key if isinstance(args, _Call) else
                                  _call_key(p.rows, p.d_in, p.d_out, p.dtype, st))
    if ws is not None and ws.numel() >= wb and ws.device == device:
        return ws, _lib.PLAN_RESIDENT
    return torch.empty(max(wb, 1), dtype=torch.uint8, device=device), 0


def check_base(x, A, B, W, bias, base8: Optional["Int8Rows"]) -> None:
    """The backbone's operands against the layer's packs: the kernels take all
    sizes from the packs."""
    d_out, d_in = B.shape[0], A.shape[1]
    if W is not None and W.shape != (d_out, d_in):
        raise ValueError(f"backbone {tuple(W.shape)} in a layer of {(d_out, d_in)}")
    if bias is not None:
        if bias.shape != (d_out,):
            raise ValueError(f"bias of shape {tuple(bias.shape)} in a layer of {d_out} outputs")
        if bias.dtype != x.dtype or bias.device != x.device:
            raise RuntimeError(f"input {x.dtype} on {x.device} but bias {bias.dtype} on {bias.device}")
    if base8 is not None:
        if base8.q.device != x.device:
            raise RuntimeError(f"input on {x.device} but the 8-bit backbone on {base8.device}")
        if base8.cols != d_in or base8.q.shape[0] != d_out:
            raise ValueError(f"8-bit backbone {base8.shape} in a layer of {(d_out, d_in)}")


def forward_raw(x, W, bias, st: LayerState, x_sorted=None, rows8: Optional["Int8Rows"] = None):
    """Run mlora_forward; returns (Y in the caller's row order, zsave, x in
    sorted order, call args).  With interleaved ids the rows of X are
    gathered into adapter order and the kernels write each row of Y straight
    to its original position (mlora_routing.out_rows), with no scatter pass.
    With an 8-bit backbone (st.base8) or ``rows8`` the call is
    mlora_forward_q8; ``rows8`` receives the 8-bit rows of the sorted x."""
    rows, d_in = x.shape
    if st.plan.rows != rows:
        raise ValueError(f"the routing plan is of {st.plan.rows} rows, x has {rows}")
    d_out = st.B_pack.shape[0]
    xs = x_sorted if x_sorted is not None else (gather_rows(x, st.plan.perm) if st.plan.perm is not None else x)
    args = _Call(rows, d_in, d_out, mlora_dtype(x.dtype), st)
    zb, wb = args.zbytes, args.wbytes
    dev = x.device
    y = torch.empty(rows, d_out, dtype=x.dtype, device=dev)
    z = torch.empty(max(zb, 1), dtype=torch.uint8, device=dev)
    ws, args.prob.flags = _workspace(st, args, wb, dev)
    if st.base8 is None and rows8 is None:
        _lib.call("mlora_forward", ctypes.byref(args.prob), ctypes.byref(args.route), _ptr(xs), _ptr(W), _ptr(bias),
                  _ptr(st.A_pack), _ptr(st.B_pack), _ptr(y), _ptr(z), _ptr(ws), wb, _stream(dev))
        return y, z, xs, args
    if rows8 is None:
        rows8 = _Scratch8(rows, d_in, dev)
    q8 = _q8_struct(st.base8, rows8)
    _lib.call("mlora_forward_q8", ctypes.byref(args.prob), ctypes.byref(args.route), ctypes.byref(q8), _ptr(xs),
              _ptr(W), _ptr(bias), _ptr(st.A_pack), _ptr(st.B_pack), _ptr(y), _ptr(z), _ptr(ws), wb, _stream(dev))
    return y, z, xs, args


def _no_8_bits(st: LayerState) -> None:
    if st.base8 is not None or st.save8:
        raise NotImplementedError("staged calls have neither a backbone nor saved inputs in 8 bits")


class StagedForward:
    """Forward of one routing plan split into stages and tile ranges (the
    nano-batch pipeline): ``shrink(t0, t1)`` writes the low-rank
    intermediate of tiles [t0, t1) into ``z``; ``main(t0, t1, expand)``
    writes rows [256 t0, 256 t1) of ``y`` (backbone + bias, + LoRA expand when
    ``expand``)."""

    def __init__(self, x, W, bias, st: LayerState, y=None):
        _no_8_bits(st)
        self.x, self.W, self.bias, self.st = x, W, bias, st
        rows, d_in = x.shape
        d_out = st.B_pack.shape[0]
        self.args = _CallArgs(rows, d_in, d_out, mlora_dtype(x.dtype), st.impl, st.plan, st.table, st.scaling,
                              st.max_ctas, err_word=st.err_word)
        zb, wb = self.args.sizes()
        dev = x.device
        self.y = y if y is not None else torch.empty(rows, d_out, dtype=x.dtype, device=dev)
        self.z = torch.empty(max(zb, 1), dtype=torch.uint8, device=dev)
        # the plan's resident workspace when make_resident() uploaded one for
        # this shape: the calls then copy nothing from the host
        self.ws, self.args.prob.flags = _workspace(st, self.args, wb, dev)
        self.wb = wb
        self.n_tiles = int(_lib.lib().mlora_num_tiles(rows))

    def rebind(self, x) -> None:
        """Reuse this object for another call with the same plan and shapes."""
        self.x = x

    def _run(self, stages, t0, t1, bias):
        _lib.call("mlora_forward_staged", ctypes.byref(self.args.prob), ctypes.byref(self.args.route),
                  _ptr(self.x), _ptr(self.W), _ptr(bias), _ptr(self.st.A_pack), _ptr(self.st.B_pack),
                  _ptr(self.y), _ptr(self.z), _ptr(self.ws), self.wb, stages, t0, t1, _stream(self.x.device))

    def shrink(self, t0=0, t1=None):
        self._run(_lib.STAGE_SHRINK, t0, self.n_tiles if t1 is None else t1, None)

    def shrink_main(self, expand=True, add_bias=True):
        """Shrink and mainloop over all tiles in one call: the mainloop is
        launched to overlap the shrink's tail (programmatic dependent launch)."""
        stages = _lib.STAGE_SHRINK | _lib.STAGE_MAIN | (0 if expand else _lib.STAGE_NO_EXPAND)
        self._run(stages, 0, self.n_tiles, self.bias if add_bias else None)

    def main(self, t0=0, t1=None, expand=True, add_bias=True, max_ctas=None):
        """``max_ctas`` (default: the state's) caps the mainloop's CTAs for
        this call, leaving SMs to concurrent communication kernels."""
        stages = _lib.STAGE_MAIN | (0 if expand else _lib.STAGE_NO_EXPAND)
        old = self.args.prob.max_ctas
        if max_ctas is not None:
            self.args.prob.max_ctas = int(max_ctas)
        try:
            self._run(stages, t0, self.n_tiles if t1 is None else t1, self.bias if add_bias else None)
        finally:
            self.args.prob.max_ctas = old

    def push(self, ar, t0=0, t1=None, expand=True, add_bias=True):
        """``main`` whose epilogue writes the partial tiles of [t0, t1) into
        their owner ranks' receive buffers (``ar``: a peer.PeerAllReduce of
        this layer's rows) instead of ``y``; the owners' ``ar.finish`` adds
        them up (mlora_forward_push)."""
        stages = _lib.STAGE_MAIN | (0 if expand else _lib.STAGE_NO_EXPAND)
        _lib.call("mlora_forward_push", ctypes.byref(self.args.prob), ctypes.byref(self.args.route),
                  _ptr(self.x), _ptr(self.W), _ptr(self.bias if add_bias else None), _ptr(self.st.A_pack),
                  _ptr(self.st.B_pack), _ptr(self.z), _ptr(self.ws), self.wb, stages, t0,
                  self.n_tiles if t1 is None else t1, ctypes.byref(ar.ar), _stream(self.x.device))


def backward_raw(dy, xs, W, z, st: LayerState, want_dx: bool, want_dA: bool, want_dB: bool,
                 rows8: Optional["Int8Rows"] = None):
    """Run mlora_backward; returns (dX in the caller's row order or None,
    dA_pack or None, dB_pack or None).  dY is gathered into adapter order;
    dX rows are written straight to their original positions.  With an 8-bit
    backbone or ``rows8`` (the 8-bit rows of the sorted input, in place of
    ``xs``) the call is mlora_backward_q8."""
    rows, d_in, d_out = st.plan.rows, st.A_pack.shape[1], st.B_pack.shape[0]
    dev, dt = st.B_pack.device, st.B_pack.dtype
    # the kernels take their strides and types from the layer: nothing else may differ
    if dy.shape != (rows, d_out):
        raise ValueError(f"dy has shape {tuple(dy.shape)}, the output {(rows, d_out)}")
    if dy.dtype != dt or dy.device != dev:
        raise RuntimeError(f"dy is {dy.dtype} on {dy.device}, the layer {dt} on {dev}")
    if (xs is not None and (xs.shape != (rows, d_in) or xs.dtype != dt or xs.device != dev)) or (
            rows8 is not None and (rows8.shape != (rows, d_in) or rows8.device != dev)):
        raise ValueError(f"the saved input is not that of a call of {rows} rows and {d_in} features")
    call = _Call(rows, d_in, d_out, mlora_dtype(dt), st)
    if z.numel() * z.element_size() < call.zbytes:
        raise ValueError(f"the saved intermediate has {z.numel() * z.element_size()} bytes, the call {call.zbytes}")
    return _backward(call, dy.contiguous(), xs.contiguous() if xs is not None else None, W, z, st, want_dx, want_dA,
                     want_dB, rows8)


def _backward(call: _Call, dy, xs, W, z, st: LayerState, want_dx: bool, want_dA: bool, want_dB: bool, rows8):
    """backward_raw of tensors that belong to the forward ``call``."""
    p = call.prob
    rows, dev, wb = p.rows, dy.device, call.wbytes
    perm = call.args.out_rows
    dys = gather_rows(dy, perm) if perm is not None else dy
    ws, p.flags = _workspace(st, call, wb, dev)
    dx = torch.empty(rows, p.d_in, dtype=dy.dtype, device=dev) if want_dx else None
    # every rank row / column of an adapter that owns rows is written; the
    # rest is never exposed (inactive adapters get None gradients)
    dA = torch.empty_like(st.A_pack) if want_dA else None
    dB = torch.empty_like(st.B_pack) if want_dB else None
    if st.base8 is not None or rows8 is not None:
        grad8 = _Scratch8(rows, p.d_out, dev) if st.base8 is not None and want_dx else None
        q8 = _q8_struct(st.base8, rows8, grad8)
        if rows8 is not None and want_dA:
            q8.scratch_bytes = call.scratch8()
            scratch = torch.empty(max(q8.scratch_bytes, 1), dtype=torch.uint8, device=dev)
            q8.scratch = scratch.data_ptr()
        _lib.call("mlora_backward_q8", ctypes.byref(p), ctypes.byref(call.route), ctypes.byref(q8),
                  _ptr(dys), _ptr(xs), _ptr(W), _ptr(st.A_pack), _ptr(st.B_pack), _ptr(z), _ptr(dx), _ptr(dA),
                  _ptr(dB), _ptr(ws), wb, _stream(dev))
        return dx, dA, dB
    _lib.call("mlora_backward", ctypes.byref(p), ctypes.byref(call.route), _ptr(dys), _ptr(xs), _ptr(W),
              _ptr(st.A_pack), _ptr(st.B_pack), _ptr(z), _ptr(dx), _ptr(dA), _ptr(dB), _ptr(ws), wb,
              _stream(dev))
    return dx, dA, dB


class StagedBackward:
    """Backward of one routing plan split into stages and ranges: ``dz(t0,
    t1)`` writes the dZ intermediate of tiles [t0, t1) into ``dz`` (a zeroed
    caller-visible buffer, so partial results of several ranks can be
    summed); ``dx()``, ``da()`` and ``db(b0, b1)`` (128-row blocks of d_out)
    read it.  ``dB`` starts at zero so that blocks computed elsewhere can be
    summed in."""

    def __init__(self, dy, xs, W, z, st: LayerState):
        _no_8_bits(st)
        self.dy, self.xs, self.W, self.z, self.st = dy, xs, W, z, st
        rows = dy.shape[0]
        d_in = st.A_pack.shape[1]
        d_out = st.B_pack.shape[0]
        dev = dy.device
        self.args = _CallArgs(rows, d_in, d_out, mlora_dtype(dy.dtype), st.impl, st.plan, st.table, st.scaling,
                              st.max_ctas, err_word=st.err_word)
        zb, wb = self.args.sizes()
        self.ws, self.args.prob.flags = _workspace(st, self.args, wb, dev)
        self.wb = wb
        self.dz_bytes = zb
        self.dz = torch.zeros(max(zb, 1), dtype=torch.uint8, device=dev)
        self.dx = torch.empty(rows, d_in, dtype=dy.dtype, device=dev)
        self.dA = torch.zeros_like(st.A_pack)
        self.dB = torch.zeros_like(st.B_pack)
        self.n_tiles = int(_lib.lib().mlora_num_tiles(rows))
        self.n_db = (d_out + 127) // 128

    def rebind(self, dy, xs, z) -> None:
        """Reuse this object (its buffers and call arguments) for another call
        with the same plan and shapes: new dY, X and saved intermediate."""
        self.dy, self.xs, self.z = dy, xs, z

    def zero_partials(self) -> None:
        """Zero dZ and dB before a call that writes only some of their blocks
        (a K-sharded rank's share), so that the ranks' buffers can be summed."""
        self.dz.zero_()
        self.dB.zero_()

    def dz_view(self):
        return self.dz[:self.dz_bytes].view(self.dy.dtype) if self.dz_bytes else None

    def _run(self, stages, t0=0, t1=0, b0=0, b1=0):
        _lib.call("mlora_backward_staged", ctypes.byref(self.args.prob), ctypes.byref(self.args.route),
                  _ptr(self.dy), _ptr(self.xs), _ptr(self.W), _ptr(self.st.A_pack), _ptr(self.st.B_pack),
                  _ptr(self.z), _ptr(self.dz), _ptr(self.dx), _ptr(self.dA), _ptr(self.dB), _ptr(self.ws), self.wb,
                  stages, t0, t1, b0, b1, _stream(self.dy.device))

    def run_dz(self, t0=0, t1=None):
        self._run(_lib.BWD_DZ, t0, self.n_tiles if t1 is None else t1)

    def run_dx(self):
        self._run(_lib.BWD_DX)

    def run_da(self):
        self._run(_lib.BWD_DA)

    def run_db(self, b0=0, b1=None):
        self._run(_lib.BWD_DB, 0, 0, b0, self.n_db if b1 is None else b1)

    def _run_sgd(self, stages, lr, t0=0, t1=0, b0=0, b1=0):
        """A call whose reduction also applies the isolated SGD step (the
        MLORA_BWD_SGD_* stages) with learning rate ``lr``."""
        self.args.prob.lr = float(lr)
        try:
            self._run(stages, t0, t1, b0, b1)
        finally:
            self.args.prob.lr = 0.0

    def run_all(self, sgd_lr: Optional[float] = None):
        """Every stage over all tiles in one call (dZ, then the dX mainloop
        overlapping its tail, then dA and dB in one reduction launch); with
        ``sgd_lr`` the reduction's epilogue also applies the isolated SGD step
        to A_pack and B_pack (every adapter that owns rows)."""
        stages = _lib.BWD_DZ | _lib.BWD_DX | _lib.BWD_DA | _lib.BWD_DB
        if sgd_lr is None:
            self._run(stages, 0, self.n_tiles, 0, self.n_db)
        else:
            self._run_sgd(stages | _lib.BWD_SGD_A | _lib.BWD_SGD_B, sgd_lr, 0, self.n_tiles, 0, self.n_db)

    def run_da_sgd(self, lr: float):
        """dA with the SGD step of A_pack fused into its reduction."""
        self._run_sgd(_lib.BWD_DA | _lib.BWD_SGD_A, lr)

    def run_dadb(self, b0=0, b1=None):
        """dA and dB (d_out blocks [b0, b1)) in one reduction launch."""
        self._run(_lib.BWD_DA | _lib.BWD_DB, 0, 0, b0, self.n_db if b1 is None else b1)


class MultiLoRAFunction(torch.autograd.Function):
    """Y = X W^T + b + per-segment LoRA, with the analytic backward.

    Inputs after ``state``: the per-adapter parameters (A_0, B_0, A_1, ...)
    as views into the packed buffers; gradients are returned for them, so
    autograd accumulates into each adapter's ``.grad`` exactly as for the
    reference module (tlora/multi_lora_linear.py:89-90; grads of adapters
    that own no rows stay None)."""

    @staticmethod
    def forward(ctx, x, W, bias, st: LayerState, *adapter_params):
        ctx.st = st
        if st.base8 is None and not st.save8:
            y, z, xs, ctx.call = forward_raw(x, W, bias, st)
            ctx.save_for_backward(xs, z, W, st.A_pack, st.B_pack)
            return y
        # dA alone reads the input in the backward: kept as it is, or in 8 bits
        keep = any(ctx.needs_input_grad[4::2])
        rows8 = _new_rows8(x.shape[0], x.shape[1], x.device) if keep and st.save8 else None
        y, z, xs, ctx.call = forward_raw(x, W, bias, st, rows8=rows8)
        b8, r8 = st.base8, rows8
        ctx.save_for_backward(xs if keep and not st.save8 else None, z, W, st.A_pack, st.B_pack,
                              *((b8.q, b8.scale) if b8 is not None else (None, None)),
                              *((r8.q, r8.scale) if r8 is not None else (None, None)))
        ctx.d_in = x.shape[1]
        return y

    @staticmethod
    def backward(ctx, dy):
        xs, z, W, _, _, *kept = ctx.saved_tensors
        st: LayerState = ctx.st
        rows8 = _wrap8(kept[2], kept[3], ctx.d_in) if kept and kept[2] is not None else None
        need = ctx.needs_input_grad
        with _on(dy.device):
            # (autograd has checked dy against y; the plan is the forward's, whatever became of it since)
            dx, dA, dB = _backward(ctx.call, dy.contiguous(), xs, W, z, st, need[0], any(need[4::2]), any(need[5::2]),
                                   rows8)
        # one call cuts a pack into all adapters' gradients
        cut, place = st.table.pieces()
        pa = torch.unsafe_split_with_sizes(dA, cut, 0) if dA is not None else None
        pb = torch.unsafe_split_with_sizes(dB, cut, 1) if dB is not None else None
        grads = [None] * (2 * st.table.n)
        for i, act in enumerate(ctx.call.active):
            if not act:
                continue
            if need[4 + 2 * i]:
                grads[2 * i] = pa[place[i]]
            if need[5 + 2 * i]:
                grads[2 * i + 1] = pb[place[i]]
        return (dx, None, None, None, *grads)


class SgdItems:
    """The item array of ``mlora_sgd`` for a fixed list of (param, grad)
    pairs, built once; ``step(lr)`` is one launch with no per-call host
    work beyond the call.  The tensors must stay alive and in place."""

    def __init__(self, params_and_grads):
        self.items, self.dtype, self.device, self.keep = _sgd_items(params_and_grads)

    def step(self, lr: float) -> int:
        if self.items is None:
            return 0
        _lib.call("mlora_sgd", self.items, len(self.items), float(lr), self.dtype, _stream(self.device))
        return len(self.items)


def _sgd_items(params_and_grads):
    items = []
    dtype = None
    device = None
    keep = []
    for p, g in params_and_grads:
        if g is None:
            continue
        if p.dim() != 2 or p.stride(1) != 1 or g.stride(1) != 1:
            raise ValueError("sgd_step_ expects 2-D tensors with unit column stride")
        if g.dtype != p.dtype or g.shape != p.shape:
            raise ValueError("gradient must match the parameter's shape and dtype")
        dt = mlora_dtype(p.dtype)
        if dtype is None:
            dtype, device = dt, p.device
        elif dt != dtype or p.device != device:
            raise ValueError("all tensors of one sgd_step_ call share a dtype and a device")
        keep.append((p, g))
        items.append(_lib.SgdItem(p.data_ptr(), g.data_ptr(), p.shape[0], p.shape[1], p.stride(0), g.stride(0)))
    if not items:
        return None, dtype, device, keep
    return (_lib.SgdItem * len(items))(*items), dtype, device, keep


def sgd_step_(params_and_grads, lr: float) -> int:
    """P <- P - lr * G for the listed (param, grad) pairs in one launch per 64
    tensors (mlora_sgd).  Params are 2-D views with unit column stride."""
    return SgdItems(params_and_grads).step(lr)
