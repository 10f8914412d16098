"""The norm of a model's gradients and their clipping on MI355X (no counterpart in
the reference): ``gradient_norm(grads)`` and ``clip_gradients(grads, max_norm)``
over any number of tensors.

All arithmetic runs in the HIP kernels of libozaki_amd.so (C ABI:
include/ozaki_amd.h), on the tensors' device and its current stream; nothing
waits for the host.  Wrong shapes raise AssertionError, types without a kernel
NotImplementedError, tensors off the GPU RuntimeError.
"""
from __future__ import annotations

from array import array

import torch
from torch.autograd import forward_ad

from . import _lib
from .linear import _FLOAT, _bound, _bytes, _call, _no_tangent, _on_one_gpu, _require_dtype, _workspace
from .ozaki import _TORCH_TO_OZK

_CODES = {d: _TORCH_TO_OZK[d] for d in _FLOAT}


def _is_dense(t: torch.Tensor) -> bool:
    """Whether t's elements, in some order, are one range of memory."""
    if t.is_neg():      # they are the negatives of what is there
        return False
    if t.is_contiguous():
        return True
    at = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != at:
            return False
        at *= size
    return True


def _checked(name, tensors):
    """The tensors as a list, and the types' codes."""
    tensors = list(tensors)
    assert tensors, f"{name} needs at least one tensor"
    dev = tensors[0].get_device()
    codes = [_CODES.get(t.dtype) for t in tensors]
    if dev < 0 or any([t.get_device() != dev for t in tensors]):
        _on_one_gpu(*tensors)
    if None in codes:
        _require_dtype(name, tensors[codes.index(None)].dtype, _FLOAT)
    if torch.is_grad_enabled() and any([t.requires_grad for t in tensors]):
        raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad() or on "
                           "detached tensors")
    _no_tangent(name, *tensors)
    return tensors, codes


class _Table:
    """Host arrays of addresses, element counts and types, as the C calls take them."""

    def __init__(self, ins, outs, codes):
        self.held = (array("Q", [t.data_ptr() for t in ins]), array("q", [t.numel() for t in ins]),
                     array("i", codes), None if outs is None else array("Q", [t.data_ptr() for t in outs]))
        self.ins, self.counts, self.codes = (a.buffer_info()[0] for a in self.held[:3])
        self.outs = None if outs is None else self.held[3].buffer_info()[0]


def gradient_norm(grads) -> torch.Tensor:
    """The Euclidean norm of all tensors' elements taken as one vector: float32, on
    their device, summed in 64 bits in the same order every time.

    grads: tensors of any shapes, float32 / float16 / bfloat16 in any mix, on one GPU
    """
    grads = list(grads)
    if grads and grads[0].is_cuda and forward_ad._current_level < 0:
        norm = _bound("gradient_norm", grads[0].device, grads)
        if norm is not None:
            return norm
    grads, codes = _checked("gradient_norm", grads)
    grads = [t if t.is_contiguous() or _is_dense(t) else t.contiguous() for t in grads]   # (of any sign)
    dev, n = grads[0].device, len(grads)
    table = _Table(grads, None, codes)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    size = _bytes("ozk_gradient_norm_workspace_bytes", n)
    ws, wsp = _workspace(size, dev)
    _call("ozk_gradient_norm", dev, table.ins, table.counts, table.codes, n, norm.data_ptr(), wsp, size)
    del ws
    return norm


def clip_gradients(grads, max_norm: float, *, out=None) -> torch.Tensor:
    """Scales all tensors by min(1, max_norm / norm), their norm as gradient_norm's,
    and returns that norm (before the scaling; the host does not wait for it).

    Args:
        grads: as for gradient_norm; no tensor twice, and none on another's elements, with
             gaps or without (views that interleave are taken; the host decides it from
             their strides, in 2^16 steps for two tensors, and past that refuses)
        max_norm: >= 0
        out: tensors of the same shapes and dtypes that take the results; default:
             the gradients themselves, in place
    The scaling goes by the norm in 64 bits, also where float32 holds it as infinity.
    An infinite element makes everything finite 0 (with an infinite max_norm nothing
    changes), a NaN everything NaN.
    """
    grads = list(grads)
    out = None if out is None else list(out)
    if grads and grads[0].is_cuda and forward_ad._current_level < 0:
        norm = _bound("clip_gradients", grads[0].device, grads, grads if out is None else out,
                      float(max_norm))
        if norm is not None:
            return norm
    # what the call does not take as it is: layouts other than contiguous, and mistakes
    grads, codes = _checked("clip_gradients", grads)
    assert max_norm >= 0, f"max_norm must be >= 0, got {max_norm}"
    ins, to, back = grads, grads, ()
    if out is None:
        whole = all([t.is_contiguous() and not t.is_neg() for t in grads])
    else:
        to, kinds = _checked("clip_gradients", out)
        assert len(to) == len(grads), f"out must have {len(grads)} tensors, got {len(to)}"
        if kinds != codes or [t.shape for t in to] != [t.shape for t in grads]:
            for g, o in zip(grads, to):
                assert o.shape == g.shape and o.dtype == g.dtype, \
                    f"out must match: {tuple(g.shape)} {g.dtype}, got {tuple(o.shape)} {o.dtype}"
        if grads[0].get_device() != to[0].get_device():
            _on_one_gpu(grads[0], to[0])
        whole = all([t.is_contiguous() and not t.is_neg() for t in grads + to])
    outs = to
    if not whole:
        ins, to, back = _through_copies(grads, to)
    dev, n = grads[0].device, len(grads)
    table = _Table(ins, to, codes)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    size = _bytes("ozk_gradient_norm_workspace_bytes", n)
    ws, wsp = _workspace(size, dev)
    try:
        _call("ozk_clip_gradients", dev, table.ins, table.outs, table.counts, table.codes, n,
              float(max_norm), norm.data_ptr(), wsp, size)
    except _lib.OzakiLibError as e:
        if e.status == _lib.OZK_ERR_SHAPE:
            raise AssertionError("tensors to clip share memory") from None
        raise
    del ws
    for o, t in back:
        o.copy_(t)
    # written behind autograd's back
    torch.autograd.graph.increment_version(outs)
    return norm


def _through_copies(grads, outs):
    """Tensors with gaps, or laid out other than their result, by copies: the inputs,
    the outputs, and (result, copy) to copy back."""
    # (the copies are apart, whatever their tensors are)
    assert not _lib.torch_binding().share_memory(grads, outs), "tensors to clip share memory"
    ins, to, back = list(grads), list(outs), []
    for i, (g, o) in enumerate(zip(grads, outs)):
        if (g is o or g.stride() == o.stride() or g.is_contiguous() and o.is_contiguous()) \
                and _is_dense(g) and _is_dense(o):
            continue
        ins[i] = g.resolve_neg().contiguous()
        to[i] = torch.empty_like(ins[i])
        back.append((o, to[i]))
    return ins, to, back
