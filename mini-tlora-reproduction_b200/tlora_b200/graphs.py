"""CUDA-graph replay of a training step with fixed routing.

A step of the fused layer is a handful of kernel launches plus host work
(routing, plan building, argument packing).  When the job mix of a batch does
not change between steps, the whole step — fused forward, analytic backward
against the upstream gradient, isolated SGD — can be captured once into a
CUDA graph and replayed: the routing plan is uploaded once into a resident
workspace (MultiLoRALinear.make_resident, MLORA_PLAN_RESIDENT), every kernel
and the per-call reset of the work counters become graph nodes, and a replay
costs one launch.

    step = GraphedTrainStep(model, x, adapter_ids, dy, lr=1e-3)
    for batch in batches:          # same rows per adapter each step
        y = step(batch.x, batch.dy)

The step is the module's own call and autograd, so its forward and backward
hooks, the gradient hooks of its parameters and an overridden forward are
captured with it (what they run on the GPU is replayed; the hooks themselves
are called while the step is captured, not at each replay).

Inputs are copied into the graph's static buffers before each replay; the
returned Y, the adapters' .grad and the updated weights live in the graph's
memory and are overwritten by the next replay.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from .multi_lora_linear import MultiLoRALinear


class _Leaves:
    """Stands in for a module's trainable parameters while it is called: leaves
    of their own over the same memory, with the parameters' gradient hooks.
    Autograd's nodes for the parameters themselves may belong to a graph that
    still lives on another stream, which a capture must not meet."""

    def __init__(self, module: nn.Module):
        self.places, self.pairs, made = [], [], {}
        for mod in module.modules():
            for name, p in mod._parameters.items():
                if p is None or not p.requires_grad:
                    continue
                if id(p) not in made:
                    made[id(p)] = leaf = nn.Parameter(p.detach())
                    if p._backward_hooks:
                        leaf._backward_hooks = p._backward_hooks
                    self.pairs.append((p, leaf))
                self.places.append((mod, name, p, made[id(p)]))

    def __enter__(self) -> "_Leaves":
        for mod, name, _, leaf in self.places:
            mod._parameters[name] = leaf
        return self

    def __exit__(self, *exc) -> None:
        for mod, name, p, _ in self.places:
            mod._parameters[name] = p


class GraphedTrainStep:
    def __init__(self, model: MultiLoRALinear, x: torch.Tensor, adapter_ids: torch.Tensor, dy: torch.Tensor,
                 lr: float, warmup: int = 3, need_dx: bool = True):
        if x.device.type != "cuda":
            raise RuntimeError("CUDA graphs need CUDA tensors")
        if dy.device != x.device:
            raise RuntimeError(f"input on {x.device} but dy on {dy.device}")
        self.model = model
        self.lr = float(lr)
        self.plan = model.route(adapter_ids.cpu(), device=x.device)
        model.make_resident(self.plan)
        self.ids = adapter_ids.cpu()
        self.x = x.detach().clone().requires_grad_(need_dx)
        self.dy = dy.detach().to(x.dtype, copy=True)  # the output's type, as autograd casts it
        side = torch.cuda.Stream(x.device)
        side.wait_stream(torch.cuda.current_stream(x.device))
        with torch.cuda.stream(side):  # warm-up off the default stream, as capture requires
            for _ in range(max(1, warmup)):
                self._step()
        torch.cuda.current_stream(x.device).wait_stream(side)
        torch.cuda.synchronize(x.device)
        # what the captured kernels read and update stays, even if the module's
        # weights move, change their type or are replaced (quantize_base)
        pk = model._pack()
        self._kept = [t.detach() for t in (pk.A_pack, pk.B_pack, *model.parameters(), *model.buffers())]
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.y = self._step()

    def _step(self) -> torch.Tensor:
        """One step as a user writes it: the module's call (with its hooks and
        an overridden forward), autograd, the gradients' hooks, the update."""
        m = self.model
        m._pack().sync()
        x = self.x.detach().requires_grad_(self.x.requires_grad)
        with _Leaves(m) as leaves:
            y = m(x, self.ids, plan=self.plan)
        if self.dy.shape != y.shape:
            raise ValueError(f"dy has shape {tuple(self.dy.shape)}, the output {tuple(y.shape)}")
        wanted = ([x] if x.requires_grad else []) + [leaf for _, leaf in leaves.pairs]
        grads = [None] * len(wanted)
        if y.requires_grad:
            grads = list(torch.autograd.grad(y, wanted, self.dy, allow_unused=True))
        self.x.grad = grads.pop(0) if x.requires_grad else None
        adapters = {id(p) for ad in m.adapters.values() for p in ad.parameters()}
        for ad in m.adapters.values():
            ad.A.grad = ad.B.grad = None
        for (p, _), g in zip(leaves.pairs, grads):
            if g is None:
                continue
            if id(p) in adapters or p.grad is None:
                p.grad = g
            else:
                p.grad.add_(g)  # a parameter of the user's own: gradients add up, as ever
            for hook in tuple((p._post_accumulate_grad_hooks or {}).values()):
                hook(p)
        m.sgd_step(self.lr)
        return y.detach()

    def __call__(self, x: Optional[torch.Tensor] = None, dy: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Copy new inputs (same shapes) into the static buffers and replay
        the captured step; returns Y (graph memory)."""
        if x is not None:
            self.x.detach().copy_(x, non_blocking=True)
        if dy is not None:
            self.dy.copy_(dy, non_blocking=True)
        self.graph.replay()
        return self.y

    @property
    def dx(self) -> Optional[torch.Tensor]:
        return self.x.grad
