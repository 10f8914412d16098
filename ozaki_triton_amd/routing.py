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
from .linear import _FLOAT, _bound, _no_tangent, _on_one_gpu, _require_dtype


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
    _no_tangent("route_tokens", logits)
    if logits.is_cuda:
        out = _bound("route", logits.device, logits, mask, k, normalize)
        if out is not None:
            return Routing(*out)
    # one of these says what is wrong
    assert logits.dim() == 2, f"logits must be [tokens, experts], got {tuple(logits.shape)}"
    T, E = logits.shape
    assert 1 <= E <= _lib.OZK_MAX_EXPERTS, f"experts must be 1 .. {_lib.OZK_MAX_EXPERTS}, got {E}"
    assert 1 <= k <= E, f"k must be 1 .. {E}, got {k}"
    assert mask is None or (mask.shape == (T,) and mask.dtype == torch.bool), \
        f"mask must be {(T,)} bool, got {tuple(mask.shape)} {mask.dtype}"
    _on_one_gpu(logits, mask)
    _require_dtype("route_tokens", logits.dtype, _FLOAT)
    raise AssertionError("route_tokens: arguments not taken")
