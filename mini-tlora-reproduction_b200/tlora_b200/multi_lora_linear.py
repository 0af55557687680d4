"""Drop-in replacement of the reference's ``tlora/multi_lora_linear.py``.

Same classes, constructor signatures, attributes, ``state_dict`` keys
(``base.weight``, ``base.bias``, ``adapters.<id>.A``, ``adapters.<id>.B``),
``adapter_parameters`` and ``ValueError``s; the same random initialisation
sequence, so a seeded construction yields the same weights as the reference.
Forward and backward run in the native sm_100a library (tcgen05 tensor-core
kernels for bf16, CUDA-core fp32 kernels for fp32) on CUDA tensors; there is
no CPU path and no PyTorch fallback for the computation.

Storage: every adapter's ``A`` [rank, in] and ``B`` [out, rank] is a view into
two packed buffers per module, ``A_pack`` [r_pack, in] and ``B_pack``
[out, r_pack], with each adapter's rank padded to a multiple of 64
(zeros).  The kernels read the packs directly, optimizers update the views in
place, and gradients come back as views of packed gradient buffers.
"""

from __future__ import annotations

import math
import operator
from typing import Dict, Iterable, Optional

import numpy as np
import torch
import torch.nn as nn

from . import ops


class LoRAAdapter(nn.Module):
    """A minimal LoRA branch: delta(x) = scaling * (x @ A^T) @ B^T.

    tlora/multi_lora_linear.py:9-31: A [rank, in] kaiming-uniform(a=sqrt(5)),
    B [out, rank] zeros, alpha defaults to rank, scaling = alpha / rank."""

    def __init__(self, in_features: int, out_features: int, rank: int, alpha: float | None = None):
        super().__init__()
        if rank <= 0:
            raise ValueError("rank must be > 0")
        self.rank = rank
        self.alpha = float(alpha if alpha is not None else rank)
        self.scaling = self.alpha / self.rank
        self.A = nn.Parameter(torch.empty(rank, in_features))
        self.B = nn.Parameter(torch.zeros(out_features, rank))
        nn.init.kaiming_uniform_(self.A, a=math.sqrt(5))
        self.in_features = in_features
        self.out_features = out_features

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """The adapter's delta alone (no backbone), through the native
        delta-only kernel path (the reference kernel's ADD_BASE=False)."""
        lead = x.shape[:-1]
        x2 = x.reshape(-1, x.shape[-1])
        ids = torch.zeros(x2.shape[0], dtype=torch.int64)
        packed = self.__dict__.get("_packed")
        if packed is None or not packed.owns({"0": self}):
            packed = _PackedAdapters({"0": self})
            self.__dict__["_packed"] = packed
        y = packed.apply(x2, ids, None, None, impl="auto")
        return y.reshape(*lead, self.out_features)


class Int8Base(nn.Module):
    """A frozen backbone held in 8 bits: ``weight_q8`` int8 [out, ld] and
    ``weight_scale`` float32 [out] (an ``ops.Int8Rows`` of W's rows, the output
    channels) and the bias as it was.  The scales stay float32 whatever type
    the module is cast to."""

    def __init__(self, rows8: ops.Int8Rows, bias: Optional[torch.Tensor]):
        super().__init__()
        if bias is not None and bias.shape != (rows8.rows,):
            raise ValueError(f"bias of shape {tuple(bias.shape)} for {rows8.rows} output channels")
        self.in_features, self.out_features = rows8.cols, rows8.rows
        self.register_buffer("weight_q8", rows8.q)
        self.register_buffer("weight_scale", rows8.scale)
        self.register_parameter(
            "bias", nn.Parameter(bias.detach().clone(), requires_grad=False) if bias is not None else None)

    @classmethod
    def from_linear(cls, base: nn.Linear) -> "Int8Base":
        return cls(ops.quantize_rows(base.weight.detach()), base.bias)

    @property
    def rows8(self) -> ops.Int8Rows:
        q, scale = self._buffers["weight_q8"], self._buffers["weight_scale"]
        r = self.__dict__.get("_rows8")
        if r is None or r.q is not q or r.scale is not scale:  # moved or replaced buffers
            r = self.__dict__["_rows8"] = ops.Int8Rows(q, scale, self.in_features)
        return r

    def _apply(self, fn, recurse=True):
        scale = self.weight_scale
        super()._apply(fn, recurse)
        if self.weight_scale.dtype != torch.float32:  # .half() and the like: moved, not cast
            self.weight_scale = scale.to(self.weight_scale.device)
        return self

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        lead = x.shape[:-1]
        y = ops.int8_linear(x.reshape(-1, x.shape[-1]), self.rows8, self.bias)
        return y.reshape(*lead, self.out_features)

    def to_linear(self, dtype: torch.dtype) -> nn.Linear:
        base = nn.Linear(self.in_features, self.out_features, bias=self.bias is not None, device=self.weight_q8.device,
                         dtype=dtype)
        with torch.no_grad():
            base.weight.copy_(ops.dequantize_rows(self.rows8, dtype))
            if self.bias is not None:
                base.bias.copy_(self.bias)
        for p in base.parameters():
            p.requires_grad_(False)
        return base


class _Int8BaseMixin:
    """Switching a module's ``base`` between its own type and 8 bits, and how
    its input is kept for the backward."""

    save_input = "full"  # or "int8"

    def quantize_base(self):
        """Hold the frozen backbone in 8 bits (one scale per output channel)
        from now on: forward and dX run the 8-bit product (``ops.int8_linear``)
        with the LoRA terms added as before.  The adapters are untouched.
        ``state_dict`` then has ``base.weight_q8`` and ``base.weight_scale`` in
        place of ``base.weight``.  Returns the module."""
        if not isinstance(self.base, Int8Base):
            self.base = Int8Base.from_linear(self.base)
        return self

    def dequantize_base(self):
        """Back to an ``nn.Linear`` of the adapters' type, with the values the
        8-bit weights stand for.  Returns the module."""
        if isinstance(self.base, Int8Base):
            self.base = self.base.to_linear(next(self._adapter_modules()).A.dtype)
        return self

    def _base_operands(self):
        """(W or None, 8-bit rows or None, bias)."""
        b = self._modules["base"]
        return (None, b.rows8, b._parameters["bias"]) if isinstance(b, Int8Base) else (b.weight, None, b.bias)


_SAVE_INPUT = ("full", "int8")


def _save8(value: str) -> bool:
    if value not in _SAVE_INPUT:
        raise ValueError(f"save_input must be one of {_SAVE_INPUT}, not {value!r}")
    return value == "int8"


class IndependentLoRALinear(_Int8BaseMixin, nn.Module):
    """One LoRA job on its own frozen backbone (tlora/multi_lora_linear.py:34-56)."""

    def __init__(self, in_features: int, out_features: int, rank: int, bias: bool = True,
                 alpha: float | None = None):
        super().__init__()
        self.base = nn.Linear(in_features, out_features, bias=bias)
        for p in self.base.parameters():
            p.requires_grad_(False)
        self.adapter = LoRAAdapter(in_features, out_features, rank, alpha)
        self._packed = None

    def _adapter_modules(self):
        yield self.adapter

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        lead = x.shape[:-1]
        x2 = x.reshape(-1, x.shape[-1])
        ids = torch.zeros(x2.shape[0], dtype=torch.int64)
        if self._packed is None or not self._packed.owns({"0": self.adapter}):
            self._packed = _PackedAdapters({"0": self.adapter})
        W, base8, bias = self._base_operands()
        y = self._packed.apply(x2, ids, W, bias, impl="auto", base8=base8, save8=_save8(self.save_input))
        return y.reshape(*lead, self.base.out_features)


class _PackedAdapters:
    """Packed storage of a set of adapters and the call into the native op.

    The packs are (re)built when the adapters' parameters no longer view them
    (first call, ``.to()``/``.cuda()``, a replaced Parameter); otherwise the
    parameters already live in the packs and nothing is copied."""

    def __init__(self, adapters: Dict[str, LoRAAdapter]):
        self.keys = list(adapters.keys())
        self.adapters = [adapters[k] for k in self.keys]
        self.table = ops.AdapterTable.build([int(k) for k in self.keys], [a.rank for a in self.adapters])
        self.A_pack: Optional[torch.Tensor] = None
        self.B_pack: Optional[torch.Tensor] = None
        self._views = None
        self._scaling = None

    def owns(self, adapters: Dict[str, LoRAAdapter]) -> bool:
        return list(adapters.keys()) == self.keys and all(map(operator.is_, adapters.values(), self.adapters))

    def params(self) -> list:
        """A_0, B_0, A_1, ... as the adapters hold them now."""
        try:  # the parameters' dicts, read directly: attribute lookups cost several times as much
            return [p[k] for p in [ad._parameters for ad in self.adapters] for k in ("A", "B")]
        except KeyError:  # a weight that is no parameter
            return [getattr(ad, k) for ad in self.adapters for k in ("A", "B")]

    def _in_sync(self, params) -> bool:
        # a parameter that no longer views the packs has another address: the
        # packs are alive, so no new storage can share theirs
        return (self._views is not None and params[0].dtype == self.A_pack.dtype and
                [p.data_ptr() for p in params] == self._views)

    def sync(self, params=None):
        if self._in_sync(params if params is not None else self.params()):
            return
        ref = self.adapters[0].A
        dev, dt = ref.device, ref.dtype
        d_in = ref.shape[1]
        d_out = self.adapters[0].B.shape[0]
        R = self.table.r_pack
        A_pack = torch.zeros(R, d_in, device=dev, dtype=dt)
        B_pack = torch.zeros(d_out, R, device=dev, dtype=dt)
        views = []
        with torch.no_grad():
            for i, ad in enumerate(self.adapters):
                if ad.A.device != dev or ad.B.device != dev or ad.A.dtype != dt or ad.B.dtype != dt:
                    raise RuntimeError("all adapters of a module must share one device and dtype")
                o, r = int(self.table.pack_off[i]), int(self.table.rank[i])
                A_pack[o:o + r].copy_(ad.A)
                B_pack[:, o:o + r].copy_(ad.B)
                ad.A.data = A_pack[o:o + r]
                ad.B.data = B_pack[:, o:o + r]
                views += [ad.A.data_ptr(), ad.B.data_ptr()]
        self.A_pack, self.B_pack, self._views = A_pack, B_pack, views

    def scaling(self) -> np.ndarray:
        s = [a.scaling for a in self.adapters]
        if self._scaling is None or self._scaling[0] != s:
            self._scaling = (s, np.array([float(v) for v in s], dtype=np.float32))
        return self._scaling[1]

    def state(self, plan: ops.RoutePlan, impl: str, base8: Optional[ops.Int8Rows] = None,
              save8: bool = False) -> ops.LayerState:
        return ops.LayerState(self.table, self.scaling(), plan, self.A_pack, self.B_pack, impl, base8=base8,
                              save8=save8)

    def operands(self, x, W, bias, base8: Optional[ops.Int8Rows], params: list):
        """(x, W, bias) as the native calls take them, after the checks."""
        if x.device.type != "cuda":
            raise RuntimeError(
                "tlora_b200 computes on CUDA devices only (sm_100a); move the module and inputs to a "
                "B200 with .cuda() -- there is no CPU path")
        self.sync(params)
        A, B = self.A_pack, self.B_pack
        if A.device != x.device:
            raise RuntimeError(f"input on {x.device} but adapters on {A.device}")
        if x.dtype != A.dtype or (W is not None and W.dtype != x.dtype):
            raise RuntimeError(f"dtype mismatch: input {x.dtype}, weights {A.dtype}")
        if x.shape[1] != A.shape[1]:
            raise ValueError(f"x has {x.shape[1]} features, the layer {A.shape[1]}")
        ops.check_base(x, A, B, W, bias, base8)
        if W is not None and W.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("the backbone is frozen: no dW (tlora/multi_lora_linear.py:78-80)")
        return (x.contiguous(), W.contiguous() if W is not None else None,
                bias.contiguous() if bias is not None else None)

    def apply(self, x, ids, W, bias, impl="auto", plan: Optional[ops.RoutePlan] = None,
              base8: Optional[ops.Int8Rows] = None, save8: bool = False):
        params = self.params()
        if ops.forward_ad._current_level >= 0:
            ops._no_tangents(x, W, bias, *params)
        x, Wc, bc = self.operands(x, W, bias, base8, params)
        if plan is None:
            plan = ops.route(ids, self.table, x.device)
        train = torch.is_grad_enabled() and (x.requires_grad or any(p.requires_grad for p in params))
        if base8 is not None and train and x.requires_grad:
            ops._check_dx8(base8)
        # nothing is kept for a backward that cannot follow
        st = self.state(plan, impl, base8, save8 and train)
        with ops._on(x.device):
            if not train:
                return ops.forward_raw(x.detach(), Wc, bc, st)[0]
            return ops.MultiLoRAFunction.apply(x, Wc, bc, st, *params)


class MultiLoRALinear(_Int8BaseMixin, nn.Module):
    """Shared frozen backbone + heterogeneous-rank adapters, one per job.

    tlora/multi_lora_linear.py:59-118.  ``forward(x, adapter_ids)`` takes
    ``x`` [batch, in_features] and per-row adapter ids [batch] in any order;
    rows whose id names no adapter get the backbone output only.  ``impl``
    selects the kernel family: "auto" (tcgen05 for bf16, SIMT otherwise),
    "tc" or "simt".

    ``quantize_base()`` holds the backbone in 8 bits.  ``save_input = "int8"``
    keeps x in 8 bits (one scale per row) between forward and backward instead
    of as it is ("full"): half the saved bytes of a 16-bit layer, and dA is
    computed from the 8-bit rows."""

    def __init__(self, in_features: int, out_features: int, adapter_ranks: Dict[int, int], bias: bool = True):
        super().__init__()
        if not adapter_ranks:
            raise ValueError("adapter_ranks cannot be empty")
        self.base = nn.Linear(in_features, out_features, bias=bias)
        for p in self.base.parameters():
            p.requires_grad_(False)
        self.adapters = nn.ModuleDict(
            {str(adapter_id): LoRAAdapter(in_features, out_features, rank)
             for adapter_id, rank in adapter_ranks.items()})
        self.impl = "auto"
        self._packed: Optional[_PackedAdapters] = None

    def _adapter_modules(self):
        return iter(self.adapters.values())

    def adapter_parameters(self, adapter_id: int) -> Iterable[nn.Parameter]:
        return self.adapters[str(adapter_id)].parameters()

    def _pack(self) -> _PackedAdapters:
        ads = self._modules["adapters"]._modules
        if self._packed is None or not self._packed.owns(ads):
            self._packed = _PackedAdapters(ads)
        return self._packed

    @property
    def adapter_table(self) -> ops.AdapterTable:
        return self._pack().table

    def route(self, adapter_ids: torch.Tensor, device=None) -> ops.RoutePlan:
        """Routing plan of ``adapter_ids``; pass it back as ``plan=`` to reuse
        it across calls with the same ids."""
        dev = torch.device(device) if device is not None else next(self._adapter_modules()).A.device
        return ops.route(adapter_ids, self._pack().table, dev)

    def make_resident(self, plan: ops.RoutePlan) -> None:
        """Upload the routing ``plan`` once into a device workspace kept on the
        plan; calls with ``plan=plan`` then issue no host-to-device copy, so a
        training step with fixed routing can be captured into a CUDA graph
        (tlora_b200.graphs.GraphedTrainStep).  Every layer that uses the plan
        calls this; layers of one shape with the same ranks and scalings share
        a workspace, whose calls must follow one another (one stream, or
        streams that wait for each other).  After a change of the plan or of
        the adapters' ranks or scalings call it again (until then calls upload
        what changed; a captured graph keeps what it was captured with)."""
        pk = self._pack()
        pk.sync()
        st = ops.LayerState(pk.table, pk.scaling(), plan, pk.A_pack, pk.B_pack, self.impl)
        ops.make_resident(st, plan.rows, self.base.in_features, self.base.out_features, pk.A_pack.dtype,
                          pk.A_pack.device)

    def packed(self):
        """(A_pack, B_pack, AdapterTable): the packed adapter storage."""
        p = self._pack()
        p.sync()
        return p.A_pack, p.B_pack, p.table

    def forward(self, x: torch.Tensor, adapter_ids: torch.Tensor, plan: Optional[ops.RoutePlan] = None,
                add_base: bool = True) -> torch.Tensor:
        if x.ndim != 2:
            raise ValueError("Phase 1 expects x shaped [batch, in_features]")
        if adapter_ids.ndim != 1 or adapter_ids.shape[0] != x.shape[0]:
            raise ValueError("adapter_ids must be [batch] and match x.shape[0]")
        W, base8, b = self._base_operands() if add_base else (None, None, None)
        return self._pack().apply(x, adapter_ids, W, b, impl=self.impl, plan=plan, base8=base8,
                                  save8=_save8(self.save_input))

    @torch.no_grad()
    def sgd_step(self, lr: float, adapter_ids: Optional[Iterable[int]] = None) -> int:
        """Isolated SGD over the adapters listed (all by default), one native
        launch: P <- P - lr * P.grad for each listed adapter whose grads are
        set; every other adapter is neither read nor written.  Equivalent to
        one ``torch.optim.SGD(model.adapter_parameters(id), lr)`` step per
        listed adapter (phase3_nano_batch.py:90-107).  Returns the number of
        tensors updated."""
        keys = [str(a) for a in adapter_ids] if adapter_ids is not None else list(self.adapters.keys())
        pairs = []
        for k in keys:
            ad = self.adapters[k]
            for p in (ad.A, ad.B):
                if p.grad is not None:
                    pairs.append((p, p.grad))
        return ops.sgd_step_(pairs, lr)
