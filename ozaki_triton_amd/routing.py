"""The router of a layer of experts on MI355X (no counterpart in the reference):
``route_tokens(logits, k)`` chooses each token's experts and makes what
``grouped_matmul`` needs, with the counts of the experts and the loss that
balances them.

All arithmetic runs in the HIP kernels of libozaki_amd.so (C ABI:
include/ozaki_amd.h), on the tensors' device and its current stream; nothing
waits for the host.  Wrong shapes raise AssertionError, types without a kernel
NotImplementedError, tensors off the GPU RuntimeError.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib
from .linear import _FLOAT, _bytes, _call, _no_tangent, _on_one_gpu, _require_dtype, _workspace
from .ozaki import _TORCH_TO_OZK


class Routing(NamedTuple):
    """What route_tokens gives (T tokens, E experts, k of them to a token).

    A layer of experts with it:

        r = route_tokens(logits, k)
        y = grouped_matmul(x[r.order // k], W, r.offsets)    # rows sorted by expert
        out = (y[r.place] * r.weights[..., None]).sum(1)     # back to their tokens
    """
    experts: torch.Tensor        # (T, k) int32, E for masked tokens
    weights: torch.Tensor        # (T, k) float32, 0 for masked tokens
    order: torch.Tensor          # (T k,) int32: slots t k + j sorted by expert, masked ones last
    place: torch.Tensor          # (T, k) int32: the slots' places in it
    offsets: torch.Tensor        # (E + 1,) int32: where each expert's slots begin and the last end
    counts: torch.Tensor         # (E,) int32
    balance_loss: torch.Tensor   # () float32


def _route_forward(logits, mask, k, normalize):
    T, E = logits.shape
    dev, n = logits.device, T * k
    ints = torch.empty(3 * n + 2 * E + 1, dtype=torch.int32, device=dev)
    experts, order, place, offsets, counts = ints.split_with_sizes((n, n, n, E + 1, E))
    weights = torch.empty((T, k), dtype=torch.float32, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    at = ints.data_ptr()
    size = _bytes("ozk_route_workspace_bytes", T, E, k)
    ws, wsp = _workspace(size, dev)
    _call("ozk_route", dev, logits.data_ptr(), _TORCH_TO_OZK[logits.dtype], logits.stride(0),
          None if mask is None else mask.data_ptr(), T, E, k, 1 if normalize else 0, at,
          weights.data_ptr(), at + 4 * n, at + 8 * n, at + 12 * n, at + 12 * n + 4 * (E + 1),
          loss.data_ptr(), wsp, size)
    del ws
    return experts.view(T, k), weights, order, place.view(T, k), offsets, counts, loss


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, mask, k, normalize, rest):
        """The differentiable two; the others go into the list `rest`."""
        experts, weights, order, place, offsets, counts, loss = _route_forward(logits, mask, k, normalize)
        rest += (experts, order, place, offsets, counts)
        ctx.save_for_backward(logits, mask, weights, experts, counts)
        ctx.normalize = normalize
        ctx.set_materialize_grads(False)
        return weights, loss

    @staticmethod
    def backward(ctx, dweights, dloss):
        # (the wrapper that refuses a second derivative costs 4 us: only where one is asked for)
        if torch.is_grad_enabled():
            return _Route.backward_once(ctx, dweights, dloss)
        return _Route.gradients(ctx, dweights, dloss)

    @staticmethod
    def gradients(ctx, dweights, dloss):
        if dweights is None and dloss is None:
            return None, None, None, None, None
        logits, mask, weights, experts, counts = ctx.saved_tensors
        T, k = experts.shape
        if dweights is not None:
            dweights = dweights.contiguous()
        dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        _call("ozk_route_backward", logits.device, logits.data_ptr(), _TORCH_TO_OZK[logits.dtype],
              logits.stride(0), None if mask is None else mask.data_ptr(), T, counts.shape[0], k,
              1 if ctx.normalize else 0, experts.data_ptr(), weights.data_ptr(), counts.data_ptr(),
              None if dweights is None else dweights.data_ptr(),
              None if dloss is None else dloss.data_ptr(), dlogits.data_ptr())
        return dlogits, None, None, None, None

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward_once(ctx, dweights, dloss):
        return _Route.gradients(ctx, dweights, dloss)


def route_tokens(logits: torch.Tensor, k: int, *, mask: torch.Tensor | None = None,
                 normalize: bool = True) -> Routing:
    """Each token's k experts, their weights, and the slots' order for grouped_matmul.

    Args:
        logits: (T, E) float32 / float16 / bfloat16, up to 1024 experts
        k: experts of a token: those of the greatest logits, the greatest first, of
           equal ones the lowest index, NaN above all
        mask: (T,) bool, False for tokens that are left out (padding): they go to
              expert E, which has no group, with weight 0
        normalize: weights are softmax(logits) over the sum of the k; else as they are
    Returns:
        Routing.  ``balance_loss`` is E sum_e f_e P_e with f_e the share of the slots
        that expert e has and P_e the mean of softmax(logits)[:, e], over the tokens
        that are not left out (0 if there is none).  weights and balance_loss are
        differentiable in logits (reverse mode, once; f as a constant).
    """
    assert logits.dim() == 2, f"logits must be [tokens, experts], got {tuple(logits.shape)}"
    T, E = logits.shape
    assert 1 <= E <= _lib.OZK_MAX_EXPERTS, f"experts must be 1 .. {_lib.OZK_MAX_EXPERTS}, got {E}"
    assert 1 <= k <= E, f"k must be 1 .. {E}, got {k}"
    assert mask is None or (mask.shape == (T,) and mask.dtype == torch.bool), \
        f"mask must be {(T,)} bool, got {tuple(mask.shape)} {mask.dtype}"
    _on_one_gpu(logits, mask)
    _require_dtype("route_tokens", logits.dtype, _FLOAT)
    _no_tangent("route_tokens", logits)
    if logits.stride(1) != 1 and E != 1:
        logits = logits.contiguous()
    if mask is not None and mask.stride(0) != 1:
        mask = mask.contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        rest: list = []
        weights, loss = _Route.apply(logits, mask, k, normalize, rest)
        experts, order, place, offsets, counts = rest
        return Routing(experts, weights, order, place, offsets, counts, loss)
    return Routing(*_route_forward(logits, mask, k, normalize))
