"""Muon: momentum whose update of a weight matrix is orthogonalised, for the matrices of a KAN.

The reference's scripts train with AdamW and LBFGS (run1.py:209, run2.py:174); this is a third optimiser for the same
loops (``PI_DeepONet.fit(optimizer="muon")``, ``bench.py --optimizer muon``): one library call a step, whatever the number
of parameters.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib, functional as K
from ._lib import PdekanMuonParam

__all__ = ["Muon"]


def _matrix_shape(p: torch.Tensor) -> Tuple[int, int]:
    """A weight as the optimiser sees it: one row an output (a KAN's spline weight ``[out, in, coeff]`` is
    ``[out, in * coeff]``); a vector is one row."""
    return (1, p.numel()) if p.dim() < 2 else (p.shape[0], p.numel() // max(1, p.shape[0]))


class Muon(torch.optim.Optimizer):
    """``m <- mu m + (1 - mu) g``; ``u = (1 - mu) g + mu m`` (Nesterov) or ``m``;
    ``p <- (1 - lr decay) p - lr gain NS(u)`` with ``NS`` of :func:`pde_amd.functional.orthogonalize`.

    ``adjust_lr``: the gain of a ``rows x cols`` weight: ``"original"`` sqrt(max(1, rows / cols)), ``"match_rms_adamw"``
    0.2 sqrt(max(rows, cols)) (updates about as large as AdamW's), ``"none"`` 1.  Vectors (biases, norms) are matrices of
    one row: their update is their direction.  ``lr`` may be a float32 tensor on the parameters' device, which a captured
    step reads at every replay.  Parameters are float32 on a ROCm GPU; the step is deterministic, allocates its workspace
    per call and can be captured in a HIP graph once the momentum buffers exist (after one eager step)."""

    def __init__(self, params, lr=0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 ns_steps: int = 5, ns_coefficients: Tuple[float, float, float] = K.NS_COEFFICIENTS, eps: float = 1e-7,
                 adjust_lr: str = "original"):
        defaults = dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, ns_steps=ns_steps,
                        ns_coefficients=tuple(ns_coefficients), eps=eps, adjust_lr=adjust_lr)
        self._check(defaults)
        super().__init__(params, defaults)

    def add_param_group(self, param_group):
        self._check({**self.defaults, **param_group} if hasattr(self, "defaults") else param_group)
        super().add_param_group(param_group)

    @staticmethod
    def _check(group) -> None:
        lr = group["lr"]
        if not isinstance(lr, torch.Tensor) and not 0.0 <= lr < float("inf"):
            raise ValueError(f"pde_amd: lr must be finite and not negative, got {lr}")
        if not 0.0 <= group["momentum"] < 1.0:
            raise ValueError(f"pde_amd: momentum must lie in [0, 1), got {group['momentum']}")
        if not 0.0 <= group["weight_decay"] < float("inf"):
            raise ValueError(f"pde_amd: weight_decay must be finite and not negative, got {group['weight_decay']}")
        if group["adjust_lr"] not in ("original", "match_rms_adamw", "none"):
            raise ValueError(f"pde_amd: adjust_lr must be 'original', 'match_rms_adamw' or 'none', got {group['adjust_lr']!r}")
        K.ns_settings(group["ns_steps"], group["eps"], group["ns_coefficients"])

    @staticmethod
    def _gain(rows: int, cols: int, kind: str) -> float:
        if kind == "original":
            return max(1.0, rows / cols) ** 0.5
        return 0.2 * max(rows, cols) ** 0.5 if kind == "match_rms_adamw" else 1.0

    @torch.no_grad()
    def step(self, closure=None) -> Optional[torch.Tensor]:
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_device = {}
            for p in group["params"]:
                if p.grad is not None and p.numel():
                    by_device.setdefault(p.device, []).append(p)
            for device, params in by_device.items():
                self._step_on(device, params, group)
        return loss

    def _step_on(self, device, params, group) -> None:
        desc = (PdekanMuonParam * len(params))()
        keep = []                                        # contiguous copies of gradients, until the launch
        for d, p in zip(desc, params):
            g = p.grad
            if not p.is_cuda:
                raise RuntimeError(f"pde_amd: a parameter is on {p.device}; Muon runs only on a ROCm GPU "
                                   "(there is no CPU implementation in this package)")
            if p.dtype != torch.float32 or g.dtype != torch.float32:
                raise TypeError(f"pde_amd: Muon takes float32 parameters and gradients, got {p.dtype} and {g.dtype}")
            if g.layout != torch.strided:
                raise RuntimeError("pde_amd: Muon takes dense gradients")
            if not p.is_contiguous():
                raise RuntimeError("pde_amd: Muon takes contiguous parameters")
            if g.device != device:
                raise RuntimeError(f"pde_amd: a parameter on {device} has its gradient on {g.device}")
            state = self.state[p]
            m = state.get("momentum_buffer")
            if m is None:
                with K._on(device):
                    capturing = torch.cuda.is_current_stream_capturing()
                if capturing:
                    raise RuntimeError("pde_amd: run one eager Muon step before capturing one (its momentum buffers "
                                       "would be cleared at every replay)")
                m = state["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
            if not (m.is_contiguous() and m.dtype == torch.float32 and m.device == device and m.numel() == p.numel()):
                raise RuntimeError("pde_amd: a momentum buffer is not a contiguous float32 tensor of its parameter's size")
            if not g.is_contiguous():
                g = g.contiguous()
                keep.append(g)
            rows, cols = _matrix_shape(p)
            d.param, d.grad, d.momentum, d.rows, d.cols = p.data_ptr(), g.data_ptr(), m.data_ptr(), rows, cols
            d.gain = self._gain(rows, cols, group["adjust_lr"])
        if len({d.param for d in desc}) < len(params):
            raise RuntimeError("pde_amd: two parameters of one group share their memory")
        lr, lr_ptr = group["lr"], None
        if isinstance(lr, torch.Tensor):
            if lr.is_cuda:
                if lr.device != device or lr.dtype != torch.float32 or lr.numel() != 1:
                    raise RuntimeError("pde_amd: a tensor lr must be one float32 number on the parameters' device")
                lr_ptr, lr = lr.data_ptr(), 0.0
            else:
                lr = float(lr)
        steps, eps, c = K.ns_settings(group["ns_steps"], group["eps"], group["ns_coefficients"])
        lib = _lib.load()
        need = lib.pdekan_muon_workspace_bytes(desc, len(params))
        if need == 0:
            _lib.check(-1)
        ws = K._workspace(need, device)
        with K._on(device):
            rc = lib.pdekan_muon_step(desc, len(params), lr, lr_ptr, group["momentum"], int(group["nesterov"]),
                                      group["weight_decay"], steps, c, eps, ws.data_ptr(), need, K._raw_stream(device))
        _lib.check(rc)
        # written through their addresses: an autograd graph that saved them has to know
        torch.autograd.graph.increment_version([*params, *[self.state[p]["momentum_buffer"] for p in params]])
