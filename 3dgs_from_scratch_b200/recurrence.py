"""A gated linear recurrence with its gradients on this library's kernels.

h_t = g_t h_{t-1} + x_t over packed or batched sequences, the gates shared by
groups of channels. The blend kernels run one such chain (three colours, gates
1 - alpha, over the tiles' lists); this is the same chain for any number of
channels and any sequences: features composited over per-ray lists (back to
front: gate 1 - alpha, x = alpha * feature, `initial` the background, the
final state the pixel), or a state carried over the frames of a scene. No
counterpart in the reference.

Both directions run on the current stream of x's device, with no host
synchronisation, and can be captured in a CUDA graph.
"""
from __future__ import annotations

import contextlib

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _native as nat

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


_HERE = contextlib.nullcontext()


def on_device(dev):
    """The device's context where it is not the current one."""
    return _HERE if dev.index == torch._C._cuda_getDevice() else torch.cuda.device(dev)


def _rows_of(t, channels):
    """t as rows of adjacent channels with one stride between all of them, at
    16-byte boundaries, and that stride; a copy where it does not lie so."""
    st = t.stride()
    step = st[-2]
    plain = channels == 1 or st[-1] == 1
    if t.dim() == 3 and t.shape[0] > 1:
        if t.shape[1] == 1:
            step = st[0]
        else:
            plain = plain and st[0] == t.shape[1] * step
    if plain and t.data_ptr() % 16 == 0 and (step == channels or step * t.element_size() % 16 == 0):
        return t, step
    return t.clone(memory_format=torch.contiguous_format), channels


def _check(x, gate, initial, offsets):
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (x, gate, initial)):
        raise NotImplementedError("gated_scan has no forward-mode derivative")
    if x.dim() != 2 and (x.dim() != 3 or offsets is not None):
        raise ValueError("gated_scan expects x of shape (rows, channels), with offsets or as one "
                         "sequence, or (batch, rows, channels)")
    if gate.dim() != x.dim() or gate.shape[:-1] != x.shape[:-1]:
        raise ValueError("gated_scan expects a gate of x's shape but for the last dimension")
    channels, gates = x.shape[-1], gate.shape[-1]
    if channels < 1 or gates < 1 or channels % gates:
        raise ValueError("the gates of a row must divide its channels")
    if x.dtype not in _TYPES or gate.dtype not in (x.dtype, torch.float32):
        raise ValueError("gated_scan runs on float32, bfloat16 or float16, with gates of the same "
                         "type or float32")
    if not x.is_cuda or gate.device != x.device:
        raise ValueError("gated_scan runs on CUDA tensors of one device")
    if offsets is not None:
        if offsets.dim() != 1 or offsets.shape[0] < 2 or offsets.dtype not in (torch.int32, torch.int64):
            raise ValueError("offsets must hold one int32 or int64 row number more than there are "
                             "sequences")
        if offsets.device != x.device:
            raise ValueError("gated_scan runs on CUDA tensors of one device")
        sequences = offsets.shape[0] - 1
    else:
        sequences = x.shape[0] if x.dim() == 3 else 1
    if initial is not None:
        if tuple(initial.shape) != (sequences, channels) or not initial.is_floating_point():
            raise ValueError("initial must be floating point of shape (sequences, channels)")
        if initial.device != x.device:
            raise ValueError("gated_scan runs on CUDA tensors of one device")
    return sequences


def _work(name, sizes, like, *more):
    """Memory of a size query (None, 0 where there is none), on `like`'s device."""
    nbytes = nat.size_query(name, *sizes, *more)
    return (like.new_empty(-(-nbytes // like.element_size())) if nbytes else None), nbytes


def _states_like(initial, shape, like):
    """An empty tensor of one fp32 state a sequence."""
    if initial is not None and initial.dtype == torch.float32:
        return torch.empty_like(initial, memory_format=torch.contiguous_format)
    return like.new_empty(shape, dtype=torch.float32)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _states(t):
    """States as the kernels read them."""
    if t is None or t.dtype == torch.float32 and t.is_contiguous():
        return t
    return t.to(torch.float32).contiguous()


def _forward(x, gate, initial, offsets, reverse, sequences, keep):
    dev, channels, gates = x.device, x.shape[-1], gate.shape[-1]
    h = torch.empty_like(x, memory_format=torch.contiguous_format)
    final = _states_like(initial, (sequences, channels), x)
    rows = x.numel() // channels
    if sequences == 0 or rows == 0 and offsets is None:
        final.zero_() if initial is None else final.copy_(initial)
        return h, final, None, None
    # (without rows the offsets are still looked at)
    (xr, x_step), (gr, g_step) = _rows_of(x, channels), _rows_of(gate, gates)
    init, offs = _states(initial), offsets
    if offs is not None:
        if offs.dtype == torch.int64:  # beyond 32 bits stays out of range
            offs = offs.clamp(-1, 2 ** 31 - 1).to(torch.int32)
        offs = offs.contiguous()
    sizes = (rows, sequences, int(offs is None), channels, gates, _TYPES[x.dtype], _TYPES[gate.dtype])
    saved = _work("gs_gated_scan_saved_bytes", sizes, h)[0] if keep else None
    scratch, nbytes = _work("gs_gated_scan_scratch_bytes", sizes, h, 0)
    with on_device(dev):
        nat.call("gs_gated_scan_forward", rows, sequences, channels, gates, sizes[5], sizes[6],
                 xr.data_ptr(), x_step, gr.data_ptr(), g_step, _ptr(init), _ptr(offs), int(reverse),
                 h.data_ptr(), final.data_ptr(), _ptr(saved), _ptr(scratch), nbytes,
                 nat.stream_ptr(dev))
    return h, final, saved, offs


def _backward(ctx, grad_h, grad_final):
    x, gate, initial, offs, saved = ctx.saved_tensors
    dev, channels, gates, sequences = x.device, x.shape[-1], gate.shape[-1], ctx.sequences
    want = initial is not None and ctx.needs_input_grad[2]
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    dgate = torch.empty_like(gate, memory_format=torch.contiguous_format)
    dfinal = _states(grad_final)
    rows = x.numel() // channels
    if sequences == 0 or rows == 0:
        dinit = None
        if want:
            dinit = torch.zeros_like(initial) if dfinal is None else dfinal.to(initial.dtype)
        return dx, dgate, dinit, None, None, None
    (xr, x_step), (gr, g_step) = _rows_of(x, channels), _rows_of(gate, gates)
    dh, dh_step = (None, channels) if grad_h is None else _rows_of(grad_h, channels)
    init = _states(initial)
    dinit = _states_like(initial, (sequences, channels), dx) if want else None
    sizes = (rows, sequences, int(offs is None), channels, gates, _TYPES[x.dtype], _TYPES[gate.dtype])
    scratch, nbytes = _work("gs_gated_scan_scratch_bytes", sizes, dx, 1)
    with on_device(dev):
        nat.call("gs_gated_scan_backward", rows, sequences, channels, gates, sizes[5], sizes[6],
                 xr.data_ptr(), x_step, gr.data_ptr(), g_step, _ptr(init), _ptr(offs),
                 int(ctx.reverse), saved.data_ptr(), _ptr(dh), dh_step, _ptr(dfinal), dx.data_ptr(),
                 dgate.data_ptr(), _ptr(dinit), _ptr(scratch), nbytes, nat.stream_ptr(dev))
    if want and initial.dtype != torch.float32:
        dinit = dinit.to(initial.dtype)
    return dx, dgate, dinit, None, None, None


_backward_once = once_differentiable(_backward)


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, initial, offsets, reverse, sequences):
        h, final, saved, offs = _forward(x, gate, initial, offsets, reverse, sequences, True)
        ctx.save_for_backward(x, gate, initial, offs, saved)
        ctx.reverse, ctx.sequences = reverse, sequences
        ctx.set_materialize_grads(False)
        return h, final

    @staticmethod
    def backward(ctx, grad_h, grad_final):
        # a graph of the backward (create_graph) is refused when it is used
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, grad_h, grad_final)


def gated_scan(x: torch.Tensor, gate: torch.Tensor, initial: torch.Tensor | None = None,
               offsets: torch.Tensor | None = None, reverse: bool = False):
    """h_t = gate_t h_{t-1} + x_t over every sequence; returns (h, final).

    x is (batch, rows, channels), or (rows, channels) with `offsets`: sequence
    s is the rows offsets[s]..offsets[s + 1] - 1 (ascending row numbers on the
    device; sequences may be empty, rows behind the last one or before the
    first give zeros; offsets that do not ascend within the rows are reported
    by gs_check_status). (rows, channels) without offsets is one sequence. gate
    has x's shape but for its last dimension, which divides the channels:
    channel c takes gate c // (channels // gates). initial (sequences, channels)
    is the state before the first row (zeros without it); final (sequences,
    channels), fp32, the state after the last one (initial where a sequence is
    empty), so that a sequence can be continued, a row at a time if need be.
    reverse runs every sequence from its last row to its first.

    float32, bfloat16 or float16; gates of x's type or float32. The recurrence
    runs in fp32 and h is rounded once. Differentiable w.r.t. x, gate and
    initial (once, in reverse mode), through h and final."""
    sequences = _check(x, gate, initial, offsets)
    if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad or
                                    initial is not None and initial.requires_grad):
        return _GatedScan.apply(x, gate, initial, offsets, bool(reverse), sequences)
    return _forward(x, gate, initial, offsets, reverse, sequences, False)[:2]
