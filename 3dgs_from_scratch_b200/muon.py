"""Orthogonalised updates for matrix parameters on this library's kernels.

The trainer's optimizer (dp.FlatParams, gs_adam_step) scales every element of
the Gaussians' parameters by its own history. A dense matrix trained next to
them (the projections of a recurrence, a decoder of features) can instead take
an update whose singular values are all near 1: momentum, a few Newton-Schulz
products that orthogonalise it, and the weight update, in one call
(`muon_step`), or the orthogonalisation alone (`orthogonalize`). No counterpart
in the reference, whose optimizer is Adam.

Calls run on the current stream of the tensors' device with no host
synchronisation and can be captured in a CUDA graph.
"""
from __future__ import annotations

import math

import torch

from . import _native as nat
from .recurrence import _TYPES, on_device

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _check_matrices(name, t):
    if t.dim() not in (2, 3) or 0 in t.shape[-2:]:
        raise ValueError(f"{name} expects (rows, cols) matrices or a (batch, rows, cols) stack of them")
    if t.dtype not in _TYPES:
        raise ValueError(f"{name} runs on float32, bfloat16 or float16")
    if not t.is_cuda:
        raise ValueError(f"{name} runs on CUDA tensors")


def _check_steps(name, steps, coefficients, eps):
    if int(steps) != steps or not 1 <= steps <= 100:
        raise ValueError(f"{name} takes 1 to 100 steps")
    if len(coefficients) != 3 or not all(math.isfinite(v) for v in coefficients):
        raise ValueError("coefficients are the three of a x + b x^3 + c x^5")
    if not eps > 0:
        raise ValueError("eps must be positive")


def _scratch(batch, rows, cols, kind, dev):
    nbytes = nat.size_query("gs_orthogonalize_scratch_bytes", batch, rows, cols, kind)
    return torch.empty(nbytes, dtype=torch.uint8, device=dev), nbytes


def orthogonalize(update: torch.Tensor, steps: int = 5, coefficients=COEFFICIENTS,
                  eps: float = 1e-7) -> torch.Tensor:
    """The update with its singular values brought near 1 by `steps` of
    X = a X + (b A + c A A) X, A = X X^T, from X = update / max(norm, eps).

    (rows, cols) or (batch, rows, cols), each matrix by itself; any strides;
    float32, bfloat16 or float16. Returns a new contiguous tensor of the same
    shape and type. Coefficients under which the singular values or b A + c A A
    could pass 8, or A itself 15, are refused. Not differentiable: the
    result is detached."""
    _check_matrices("orthogonalize", update)
    _check_steps("orthogonalize", steps, coefficients, eps)
    dev, (rows, cols) = update.device, update.shape[-2:]
    batch = update.shape[0] if update.dim() == 3 else 1
    out = torch.empty(update.shape, dtype=update.dtype, device=dev)
    if batch == 0:
        return out
    kind = _TYPES[update.dtype]
    st = update.stride()
    scratch, nbytes = _scratch(batch, rows, cols, kind, dev)
    with on_device(dev):
        nat.call("gs_orthogonalize", batch, rows, cols, kind, update.data_ptr(),
                 st[0] if update.dim() == 3 else 0, st[-2], st[-1], out.data_ptr(), int(steps),
                 *coefficients, eps, scratch.data_ptr(), nbytes, nat.stream_ptr(dev))
    return out


def muon_step(param: torch.Tensor, grad: torch.Tensor, momentum: torch.Tensor, lr: float,
              beta: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
              scale: float | None = None, steps: int = 5, coefficients=COEFFICIENTS,
              eps: float = 1e-7) -> None:
    """One optimizer step of a matrix parameter, in place:

    momentum = beta momentum + (1 - beta) grad; the update is beta momentum +
    (1 - beta) grad with nesterov, else the momentum; param = (1 - lr
    weight_decay) param - lr scale orthogonalize(update). scale defaults to
    sqrt(max(1, rows / cols)).

    param and momentum are float32 and contiguous, (rows, cols) or a
    (batch, rows, cols) stack; grad has their shape, of any supported type. The
    three share no memory.
    Like the Adam step it is skipped, as a whole, while the device status word
    holds an error of an earlier kernel (gs_check_status)."""
    _check_matrices("muon_step", param)
    _check_matrices("muon_step", grad)
    _check_steps("muon_step", steps, coefficients, eps)
    if param.dtype != torch.float32 or momentum.dtype != torch.float32:
        raise ValueError("muon_step updates float32 parameters and momentum")
    if grad.shape != param.shape or momentum.shape != param.shape:
        raise ValueError("param, grad and momentum must have the same shape")
    if grad.device != param.device or momentum.device != param.device:
        raise ValueError("muon_step runs on CUDA tensors of one device")
    if not param.is_contiguous() or not momentum.is_contiguous():
        raise ValueError("muon_step updates contiguous tensors")
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
                   for t in (param, momentum, grad) if t.is_contiguous())
    if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
        raise ValueError("param, grad and momentum must not share memory")
    if not 0.0 <= beta < 1.0:
        raise ValueError("beta must be in [0, 1)")
    dev, (rows, cols) = param.device, param.shape[-2:]
    batch = param.shape[0] if param.dim() == 3 else 1
    if batch == 0:
        return
    if scale is None:
        scale = math.sqrt(max(1.0, rows / cols))
    grad = grad.contiguous()
    scratch, nbytes = _scratch(batch, rows, cols, _TYPES[torch.float32], dev)
    with on_device(dev):
        nat.call("gs_muon_step", batch, rows, cols, _TYPES[grad.dtype], param.data_ptr(),
                 grad.data_ptr(), momentum.data_ptr(), lr, beta, int(nesterov), weight_decay, scale,
                 int(steps), *coefficients, eps, scratch.data_ptr(), nbytes, nat.stream_ptr(dev))
    # written behind autograd's back: a graph that still holds the old values says so
    torch.autograd.graph.increment_version((param, momentum))
