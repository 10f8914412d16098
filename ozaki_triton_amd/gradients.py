"""The norm of a model's gradients and their clipping on MI355X (no counterpart in
the reference): ``gradient_norm(grads)`` and ``clip_gradients(grads, max_norm)``
over any number of tensors.

All arithmetic runs in the HIP kernels of libozaki_amd.so (C ABI:
include/ozaki_amd.h), on the tensors' device and its current stream; nothing
waits for the host.  Wrong shapes raise AssertionError, types without a kernel
NotImplementedError, tensors off the GPU RuntimeError.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .linear import _FLOAT, _bytes, _call, _no_grad, _on_one_gpu, _require_dtype, _workspace
from .ozaki import _TORCH_TO_OZK


def _is_dense(t: torch.Tensor) -> bool:
    """Whether t's elements, in some order, are one range of memory."""
    if t.is_contiguous():
        return True
    at = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != at:
            return False
        at *= size
    return True


def _tensors(name, grads):
    grads = list(grads)
    assert grads, f"{name} needs at least one tensor"
    _on_one_gpu(*grads)
    for t in grads:
        if t.dtype not in _FLOAT:
            _require_dtype(name, t.dtype, _FLOAT)
    return grads


def _pointers(tensors):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])


def _described(tensors):
    n = len(tensors)
    return ((ctypes.c_int64 * n)(*[t.numel() for t in tensors]),
            (ctypes.c_int * n)(*[_TORCH_TO_OZK[t.dtype] for t in tensors]))


def gradient_norm(grads) -> torch.Tensor:
    """The Euclidean norm of all tensors' elements taken as one vector: float32, on
    their device, summed in 64 bits in the same order every time.

    grads: tensors of any shapes, float32 / float16 / bfloat16 in any mix, on one GPU
    """
    grads = _tensors("gradient_norm", grads)
    _no_grad("gradient_norm", *grads)
    grads = [t if _is_dense(t) else t.contiguous() for t in grads]
    dev, n = grads[0].device, len(grads)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    size = _bytes("ozk_gradient_norm_workspace_bytes", n)
    ws, wsp = _workspace(size, dev)
    _call("ozk_gradient_norm", dev, _pointers(grads), *_described(grads), n, norm.data_ptr(), wsp, size)
    del ws
    return norm


def clip_gradients(grads, max_norm: float, *, out=None) -> torch.Tensor:
    """Scales all tensors by min(1, max_norm / norm), their norm as gradient_norm's,
    and returns that norm (before the scaling; the host does not wait for it).

    Args:
        grads: as for gradient_norm; no tensor twice, and none on another's elements
        max_norm: >= 0
        out: tensors of the same shapes and dtypes that take the results; default:
             the gradients themselves, in place
    A norm of infinity makes everything finite 0, one of NaN everything NaN.
    """
    grads = _tensors("clip_gradients", grads)
    outs = grads if out is None else list(out)
    assert max_norm >= 0, f"max_norm must be >= 0, got {max_norm}"
    if outs is not grads:
        assert len(outs) == len(grads), f"out must have {len(grads)} tensors, got {len(outs)}"
        for g, o in zip(grads, outs):
            assert o.shape == g.shape and o.dtype == g.dtype, \
                f"out must match: {tuple(g.shape)} {g.dtype}, got {tuple(o.shape)} {o.dtype}"
        _on_one_gpu(grads[0], *outs)
    _no_grad("clip_gradients", *grads)
    if outs is not grads:
        _no_grad("clip_gradients", *outs)
    # tensors with gaps, or laid out other than their result, go through copies
    ins, to = grads, outs
    back = []
    for i, (g, o) in enumerate(zip(grads, outs)):
        if g is o and _is_dense(g) or (g.is_contiguous() and o.is_contiguous()):
            continue
        if g.stride() == o.stride() and _is_dense(g):
            continue
        assert all(s or n <= 1 for s, n in zip(o.stride(), o.shape)), \
            "out must not be expanded: its elements share memory"
        if ins is grads:
            ins, to = list(grads), list(outs)
        ins[i] = g.contiguous()
        to[i] = torch.empty_like(ins[i])
        back.append((o, to[i]))
    dev, n = grads[0].device, len(grads)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    size = _bytes("ozk_gradient_norm_workspace_bytes", n)
    ws, wsp = _workspace(size, dev)
    try:
        _call("ozk_clip_gradients", dev, _pointers(ins), _pointers(to), *_described(ins), n,
              float(max_norm), norm.data_ptr(), wsp, size)
    except _lib.OzakiLibError as e:
        if e.status == _lib.OZK_ERR_SHAPE:
            raise AssertionError("tensors to clip share memory") from None
        raise
    del ws
    for o, t in back:
        o.copy_(t)
    # written behind autograd's back
    torch.autograd.graph.increment_version([t for t in outs if not t.is_inference()])
    return norm
