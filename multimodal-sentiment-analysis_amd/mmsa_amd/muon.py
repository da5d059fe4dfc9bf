"""Orthogonalised updates of weight matrices: the operator, one optimiser step over a list, and the optimiser.

The reference trains every parameter with ``torch.optim.AdamW`` (`CNN implementation/multimodal_train.py:481-485`).  The
Muon rule gives the weight MATRICES (convolutions flattened to [out, in * taps], linear layers) another update: momentum,
then the nearest matrix with all singular values near 1, so that no direction of the gradient dominates the step.
Biases, norms, the embedding and the classifier's last layer stay with AdamW.

The rule and the coefficients of its iteration are K. Jordan and others', "Muon: an optimizer for hidden layers in neural
networks" (2024).
"""
from __future__ import annotations

from typing import List, Sequence, Union

import torch

from . import _lib, ops


def _gpu(ts, what):
    for t in ts:
        if not t.is_cuda:
            raise _lib.MmsaError(f"{what}: tensors must live on the GPU (the HIP kernels have no CPU path)")


def orthogonalize(matrices: Union[torch.Tensor, Sequence[torch.Tensor]], steps: int = 5, eps: float = 1e-7):
    """The Newton-Schulz orthogonalisation of one matrix [rows, cols], or of a list of them in shared launches.

    ``X = u / max(|u|_F, eps)``, then ``steps`` times ``X <- (a I + b S + c S S) X`` with ``S = X X^T`` (on the transpose
    where rows exceed columns) and (a, b, c) = (3.4445, -4.775, 2.0315): singular values that are not tiny end between 0.7
    and 1.2.  float32, bfloat16 or float16 in and out (one type per list), computed about as exactly as with float32
    products.  Returns new contiguous tensors; no gradient flows through.  A list may hold matrices of different
    sizes: tiles and splits are chosen for all that share a launch, so a matrix's last bits can depend on its company.
    """
    single = isinstance(matrices, torch.Tensor)
    ms = [matrices] if single else list(matrices)
    _gpu(ms, "orthogonalize")
    with torch.no_grad():
        dsts = ops.orthogonalize([m if m.is_contiguous() else m.contiguous() for m in ms], None, steps, eps)
    return dsts[0] if single else dsts


def muon_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], momenta: Sequence[torch.Tensor], *,
              lr: float, weight_decay: float = 0.0, momentum: float = 0.95, nesterov: bool = True, steps: int = 5,
              eps: float = 1e-7) -> None:
    """One Muon step over float32 tensors, updating ``params`` and ``momenta`` in place:

    ``m += (1 - momentum)(g - m);  u = g + momentum (m - g) if nesterov else m;``
    ``p = p (1 - lr weight_decay) - lr sqrt(max(1, rows / cols)) orthogonalize(u)``

    A tensor of more than two dimensions is taken as [first, rest].  Parameters and momenta are contiguous and share no
    memory with each other or with a gradient.  The scalars are held by value: a step captured in a HIP graph replays with those of the capture.
    """
    ops.muon_step(params, [g if g.is_contiguous() else g.contiguous() for g in grads], momenta, lr, weight_decay,
                  momentum, nesterov, steps, eps)
    # written through raw pointers: tell autograd (and whoever watches the version counters) that the values changed
    torch.autograd.graph.increment_version([t for t in (*params, *momenta) if not t.is_inference()])


class Muon(torch.optim.Optimizer):
    """Muon over contiguous float32 weight matrices on the GPU, as a ``torch.optim.Optimizer``: the reference's loop
    (`multimodal_train.py:175-195`), its schedulers and ``state_dict`` work on it unchanged.

    Only parameters with at least two dimensions are taken (pass the others to ``torch.optim.AdamW``); a parameter
    without a gradient, or without values, is left alone.  All matrices of a group are updated in shared launches.  A step
    can be captured in a HIP graph once every parameter has had an eager one."""

    def __init__(self, params, lr: float = 0.02, weight_decay: float = 0.0, momentum: float = 0.95,
                 nesterov: bool = True, steps: int = 5, eps: float = 1e-7):
        if lr < 0.0 or weight_decay < 0.0 or not 0.0 <= momentum < 1.0:
            raise ValueError("Muon: lr and weight_decay must not be negative, momentum in [0, 1)")
        ops._ns_args(steps, eps)
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov,
                                      steps=steps, eps=eps))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() < 2 or p.dtype != torch.float32 or not p.is_contiguous():
                self.param_groups.pop()
                raise ValueError("Muon takes contiguous float32 parameters with at least two dimensions, got "
                                 f"{p.dtype} {tuple(p.shape)} with strides {p.stride()}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        todo = []                       # every group is checked before the first one is updated
        for group in self.param_groups:
            ops._ns_args(group["steps"], group["eps"])
            by_device: dict = {}
            for p in group["params"]:
                if p.grad is None or not p.numel():
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("Muon does not take sparse gradients")
                _gpu([p], "Muon")
                if not p.is_contiguous():
                    raise ValueError(f"Muon: parameters must be contiguous, one of {tuple(p.shape)} is not")
                if "momentum_buffer" not in self.state.get(p, ()) and torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("Muon makes its momentum at a parameter's first step, which has to be an eager "
                                       "one: cleared inside a graph, it would be cleared again by every replay")
                by_device.setdefault(p.device, []).append(p)
            todo += [(group, device, ps) for device, ps in by_device.items()]
        for group, device, ps in todo:
            for p in ps:
                state = self.state[p]
                if "momentum_buffer" not in state:
                    state["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            with torch.cuda.device(device):
                muon_step(ps, [p.grad for p in ps], [self.state[p]["momentum_buffer"] for p in ps],
                          lr=float(group["lr"]), weight_decay=group["weight_decay"], momentum=group["momentum"],
                          nesterov=group["nesterov"], steps=group["steps"], eps=group["eps"])
        return loss
