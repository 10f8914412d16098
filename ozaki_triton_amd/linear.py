"""Products for a model's linear layers on MI355X (no counterpart in the
reference):

* ``grouped_matmul(A, B, offsets)``: rows sorted by expert, each group times its
  expert's matrix; differentiable, ``grouped_matmul_backward`` on its own;
* ``quantize_w4`` / ``dequantize_w4`` / ``matmul_w4``: weights of 4 bits in groups
  with scales, and their product with a few rows of activations;
* ``orthogonalize(G)``: the Newton-Schulz orthogonalisation of an update.

All arithmetic runs in the HIP kernels of libozaki_amd.so (C ABI:
include/ozaki_amd.h), on the tensors' device and its current stream; nothing
waits for the host.  Wrong shapes raise AssertionError, types without a kernel
NotImplementedError, tensors off the GPU RuntimeError.
"""
from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd import forward_ad

from . import _lib
from .ozaki import _RAW_STREAM, _TORCH_TO_OZK, _require_gpu, _stream

_HALF = (torch.float16, torch.bfloat16)
_OFFSETS = (torch.int32, torch.int64)
_FLOAT = (torch.float32, torch.float16, torch.bfloat16)
_MAX_STRIDE = 1 << 22      # the kernels' limit on the distance of two rows
_MAX_BATCH = 65535         # matrices that one orthogonalisation takes


def _require_dtype(name: str, dtype: torch.dtype, allowed) -> None:
    if dtype not in allowed:
        raise NotImplementedError(
            f"{name}: {dtype} is not implemented by the MI355X kernels (implemented: "
            f"{', '.join(str(d).replace('torch.', '') for d in allowed)})")


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _on_one_gpu(a: torch.Tensor, *others) -> None:
    """_require_gpu's check without its sets: host time counts in calls of a few us."""
    if a.is_cuda:
        dev = a.device
        for t in others:
            if t is not None and t.device != dev:
                break
        else:
            return
    _require_gpu(a, *(t for t in others if t is not None))


def _no_tangent(name: str, *tensors) -> None:
    """Forward-mode derivatives would be lost without a word: there are none here."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{name} has no forward-mode derivative: call it on primal tensors")


_FUNCTIONS: dict = {}


def _call(name: str, dev: torch.device, *args) -> None:
    """Library call `name` on dev's current stream, its last argument."""
    fn = _FUNCTIONS.get(name)
    if fn is None:
        fn = _FUNCTIONS[name] = getattr(_lib.load(), name)
    idx = dev.index
    if _RAW_STREAM is not None and idx == _current_device():
        st = fn(*args, _RAW_STREAM(idx))
    else:
        with torch.cuda.device(dev):
            st = fn(*args, _stream(dev))
    if st:
        _lib.check(name, st)


@functools.lru_cache(maxsize=1024)
def _i64(*vals):
    return _lib.i64arr(vals)


@functools.lru_cache(maxsize=1024)
def _bytes(name: str, *args) -> int:
    """Workspace query `name`: it depends on nothing but its arguments (of a pointer
    its alignment, which is passed in its place; strides come as a tuple)."""
    n = ctypes.c_size_t(0)
    args = [_i64(*a) if isinstance(a, tuple) else a for a in args]
    _lib.check(name, getattr(_lib.load(), name)(*args, ctypes.byref(n)))
    return n.value


def _workspace(nbytes: int, dev: torch.device):
    """Scratch on dev's current stream, the one the kernels run on (so it needs no
    record_stream), and its address."""
    if not nbytes:
        return None, None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    return ws, ws.data_ptr()


def _rows(t: torch.Tensor):
    """t [rows, columns] with its columns contiguous, and its rows' distance, which
    the kernels take up to a limit.  (Strides of dims of size 1 mean nothing, to
    contiguous() either: one row of a longer tensor keeps the distance of its rows.)"""
    if t.shape[0] <= 1 and (t.stride(1) == 1 or t.shape[1] <= 1):
        return t, 0
    if (t.stride(1) == 1 or t.shape[1] == 1) and t.stride(0) < _MAX_STRIDE:
        return t, t.stride(0)
    return t.contiguous(), t.shape[1]


def _matrices(t: torch.Tensor):
    """t [groups, K, N] with K or N contiguous, and its strides, one of K and N 1 and
    the other within the kernels' limit.  Strides of dims of size 1 as in _rows."""
    (G, K, N), (s_g, s_k, s_n) = t.shape, t.stride()
    if G <= 1:
        s_g = 0
    if (s_n == 1 or N == 1) and (s_k < _MAX_STRIDE or K <= 1):
        return t, (s_g, s_k if K > 1 else 0, 1)
    if (s_k == 1 or K == 1) and (s_n < _MAX_STRIDE or N <= 1):
        return t, (s_g, 1, s_n if N > 1 else 0)
    return t.contiguous(), (K * N, N, 1)


# ============================================================
# grouped products
# ============================================================

def _grouped_checks(A, B, offsets):
    a, b, dev = A.shape, B.shape, A.device
    if (len(a) == 2 and len(b) == 3 and a[1] == b[1] and A.dtype in _HALF and B.dtype == A.dtype
            and offsets.shape == (b[0] + 1,) and offsets.dtype in _OFFSETS and dev.type == "cuda"
            and B.device == dev and offsets.device == dev):
        return
    # one of these says what is wrong
    assert A.dim() == 2, f"A must be [rows, K], got {tuple(A.shape)}"
    assert B.dim() == 3, f"B must be [groups, K, N], got {tuple(B.shape)}"
    assert A.shape[1] == B.shape[1], f"contraction dim mismatch: A K={A.shape[1]}, B K={B.shape[1]}"
    assert A.dtype == B.dtype, f"A/B dtype mismatch: {A.dtype} vs {B.dtype}"
    assert offsets.dim() == 1 and offsets.shape[0] == B.shape[0] + 1, \
        f"offsets must be [groups + 1] = [{B.shape[0] + 1}], got {tuple(offsets.shape)}"
    if offsets.dtype not in _OFFSETS:
        raise NotImplementedError(f"offsets must be int32 or int64, got {offsets.dtype}")
    _on_one_gpu(A, B, offsets)
    _require_dtype("grouped_matmul", A.dtype, _HALF)


def _grouped_forward(A, B, offsets):
    T, K = A.shape
    G, _, N = B.shape
    dtype, dev = A.dtype, A.device
    sa, sb = A.stride(), B.stride()
    pitch = sa[0]
    if sa[1] != 1 or pitch >= _MAX_STRIDE:
        A, pitch = _rows(A)
    if not ((sb[2] == 1 and sb[1] < _MAX_STRIDE) or (sb[1] == 1 and sb[2] < _MAX_STRIDE)):
        B, sb = _matrices(B)
    if offsets.stride(0) != 1:
        offsets = offsets.contiguous()
    C = A.new_empty((T, N))
    ap, bp = A.data_ptr(), B.data_ptr()
    ws = wsp = None
    n = 0
    # whole 16-byte pieces need no workspace: most calls spare the query
    if (ap | bp | (pitch | sb[0] | sb[1] * sb[2] | K | N) * 2) & 15:
        n = _bytes("ozk_grouped_matmul_workspace_bytes", ap & 15, pitch, bp & 15, sb, T, K, N, G)
        ws, wsp = _workspace(n, dev)
    _call("ozk_grouped_matmul", dev, ap, pitch, bp, _i64(*sb), offsets.data_ptr(),
          offsets.element_size(), T, K, N, G, _TORCH_TO_OZK[dtype], C.data_ptr(), N, wsp, n)
    del ws
    return C


def _grouped_wgrad(A, D, offsets, G):
    T, K = A.shape
    N = D.shape[1]
    (A, sa), (D, sd) = _rows(A), _rows(D)
    if offsets.stride(0) != 1:
        offsets = offsets.contiguous()
    dtype, dev = A.dtype, A.device
    dB = A.new_empty((G, K, N))
    ap, dp = A.data_ptr(), D.data_ptr()
    n = _bytes("ozk_grouped_matmul_wgrad_workspace_bytes", ap & 15, sa, dp & 15, sd, T, K, N, G)
    ws, wsp = _workspace(n, dev)
    _call("ozk_grouped_matmul_wgrad", dev, ap, sa, dp, sd, offsets.data_ptr(),
          offsets.element_size(), T, K, N, G, _TORCH_TO_OZK[dtype], dB.data_ptr(),
          _i64(K * N, N), wsp, n)
    del ws
    return dB


class _GroupedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, A, B, offsets):
        ctx.save_for_backward(A, B, offsets)
        return _grouped_forward(A, B, offsets)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dC):
        A, B, offsets = ctx.saved_tensors
        dA = _grouped_forward(dC, B.mT, offsets) if ctx.needs_input_grad[0] else None
        dB = _grouped_wgrad(A, dC, offsets, B.shape[0]) if ctx.needs_input_grad[1] else None
        return dA, dB, None


def grouped_matmul(A: torch.Tensor, B: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """C[t] = A[t] @ B[g] for the rows offsets[g] <= t < offsets[g + 1].

    Args:
        A: (rows, K) float16 / bfloat16, sorted by group
        B: (groups, K, N), dtype of A; a transposed view (K contiguous) is read in place
        offsets: (groups + 1,) int32 / int64 on the device, not decreasing; never
                 read by the host.  Rows before offsets[0] and from
                 offsets[groups] on belong to no group.
    Returns:
        C: (rows, N), dtype of A, summed in float32 and rounded once; zeros in the
        rows of no group.  Differentiable in A and B (reverse mode, once).
    """
    _grouped_checks(A, B, offsets)
    _no_tangent("grouped_matmul", A, B)
    if torch.is_grad_enabled() and (A.requires_grad or B.requires_grad):
        return _GroupedMatmul.apply(A, B, offsets)
    return _grouped_forward(A, B, offsets)


def grouped_matmul_backward(dC: torch.Tensor, A: torch.Tensor, B: torch.Tensor,
                            offsets: torch.Tensor):
    """The gradients (dA, dB) of grouped_matmul(A, B, offsets) for dC (rows, N):
    dA[t] = dC[t] @ B[g]^T, zeros in the rows of no group; dB[g] = A[rows of g]^T
    @ dC[rows of g], zeros for a group without rows.  Both have A's dtype; they are
    not differentiable themselves."""
    _grouped_checks(A, B, offsets)
    assert dC.shape == (A.shape[0], B.shape[2]), \
        f"dC must be {(A.shape[0], B.shape[2])}, got {tuple(dC.shape)}"
    assert dC.dtype == A.dtype, f"dC/A dtype mismatch: {dC.dtype} vs {A.dtype}"
    _on_one_gpu(dC, A)
    _no_tangent("grouped_matmul_backward", dC, A, B)
    return _grouped_forward(dC, B.mT, offsets), _grouped_wgrad(A, dC, offsets, B.shape[0])


# ============================================================
# 4-bit weights
# ============================================================

_GROUPS = (32, 64, 128)


def _no_grad(name: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad() or on "
                                   "detached tensors")
    _no_tangent(name, *tensors)


def _w4_checks(packed, scales, zeros, group_size, K):
    assert group_size in _GROUPS, f"group_size must be 32, 64 or 128, got {group_size}"
    assert packed.dim() == 2 and packed.dtype == torch.uint8, \
        f"packed must be a 2-d uint8 tensor, got {packed.dtype} {tuple(packed.shape)}"
    assert packed.shape[1] >= (K + 31) // 32 * 16, \
        f"packed has {packed.shape[1]} bytes a row, K={K} needs {(K + 31) // 32 * 16}"
    want = (packed.shape[0], (K + group_size - 1) // group_size)
    assert scales.shape == want, f"scales must be {want}, got {tuple(scales.shape)}"
    assert zeros is None or (zeros.shape == want and zeros.dtype == torch.uint8), \
        f"zeros must be {want} uint8, got {zeros.dtype} {tuple(zeros.shape)}"


def _w4_operands(packed, scales, zeros, K):
    """The three as the kernels read them: rows contiguous, packed ones 16-byte aligned
    and no closer than they are long."""
    if (packed.stride(1) != 1 or packed.stride(0) % 16 or packed.data_ptr() % 16
            or packed.stride(0) < (K + 31) // 32 * 16):
        if packed.shape[1] % 16:
            packed = torch.nn.functional.pad(packed, (0, -packed.shape[1] % 16))
        packed = packed.clone(memory_format=torch.contiguous_format)
    if scales.stride(1) != 1:
        scales = scales.contiguous()
    if zeros is not None and zeros.stride(1) != 1:
        zeros = zeros.contiguous()
    return packed, scales, zeros


def quantize_w4(W: torch.Tensor, group_size: int = 128, *, zeros: bool = False):
    """W (N, K) to 4 bits in groups of ``group_size`` (32, 64 or 128) along K.

    Returns (packed, scales, zeros) with W[n, k] ~ (q - z) * s:
        packed: (N, ceil(K / 32) * 16) uint8, q of 0 .. 15, k even in the low half
                of byte k // 2
        scales: (N, ceil(K / group_size)), dtype of W (float32 / float16 / bfloat16):
                max |w| / 7, or with ``zeros`` the range of the group and 0, over 15
        zeros:  the same of uint8, or None: every z is 8
    q = round(w / s) + z, ties to even, within 0 .. 15; NaN counts as 0.
    """
    assert W.dim() == 2, f"W must be [N, K], got {tuple(W.shape)}"
    assert group_size in _GROUPS, f"group_size must be 32, 64 or 128, got {group_size}"
    _on_one_gpu(W)
    _require_dtype("quantize_w4", W.dtype, _FLOAT)
    _no_grad("quantize_w4", W)
    N, K = W.shape
    groups = -(-K // group_size)
    W = W if W.stride(1) == 1 or K == 1 else W.contiguous()
    dev = W.device
    packed = torch.empty((N, (K + 31) // 32 * 16), dtype=torch.uint8, device=dev)
    scales = W.new_empty((N, groups))
    z = torch.empty((N, groups), dtype=torch.uint8, device=dev) if zeros else None
    _call("ozk_quantize_w4", dev, W.data_ptr(), _TORCH_TO_OZK[W.dtype], N, K, W.stride(0),
          group_size, packed.data_ptr(), packed.shape[1], scales.data_ptr(), groups,
          z.data_ptr() if zeros else None, groups)
    return packed, scales, z


def dequantize_w4(packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None,
                  *, group_size: int = 128, K: int | None = None,
                  dtype: torch.dtype | None = None) -> torch.Tensor:
    """The weights (N, K) that quantize_w4's tensors stand for, in ``dtype``
    (default: the scales' dtype; float32 scales go with any).  K defaults to what
    the packed rows hold."""
    K = packed.shape[-1] * 2 if K is None else K
    _w4_checks(packed, scales, zeros, group_size, K)
    dtype = scales.dtype if dtype is None else dtype
    _on_one_gpu(packed, scales, zeros)
    _require_dtype("dequantize_w4", dtype, _FLOAT)
    _no_grad("dequantize_w4", scales)
    assert scales.dtype in (dtype, torch.float32), \
        f"scales must be {dtype} or float32, got {scales.dtype}"
    packed, scales, zeros = _w4_operands(packed, scales, zeros, K)
    N, dev = packed.shape[0], packed.device
    W = torch.empty((N, K), dtype=dtype, device=dev)
    _call("ozk_dequantize_w4", dev, packed.data_ptr(), packed.stride(0), scales.data_ptr(),
          _TORCH_TO_OZK[scales.dtype], scales.stride(0),
          None if zeros is None else zeros.data_ptr(), 0 if zeros is None else zeros.stride(0),
          group_size, N, K, W.data_ptr(), _TORCH_TO_OZK[dtype], K)
    return W


def matmul_w4(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor,
              zeros: torch.Tensor | None = None, *, group_size: int = 128) -> torch.Tensor:
    """y = x @ W^T for W (N, K) of 4 bits (quantize_w4).

    Args:
        x: (..., K) float32 / float16 / bfloat16; meant for few rows (one token of
           each sequence), taken in any number
        packed, scales, zeros: quantize_w4's; scales in x's dtype or float32
    Returns:
        y: (..., N), dtype of x, summed in float32 and rounded once.  A row of x
        with an infinity or NaN gives a row of NaN; finite ones do not.
    """
    assert x.dim() >= 1 and x.shape[-1] >= 1, f"x must be [..., K], got {tuple(x.shape)}"
    K, dtype, dev = x.shape[-1], x.dtype, x.device
    _w4_checks(packed, scales, zeros, group_size, K)
    assert scales.dtype == dtype or scales.dtype == torch.float32, \
        f"scales must be {dtype} or float32, got {scales.dtype}"
    _on_one_gpu(x, packed, scales, zeros)
    _require_dtype("matmul_w4", dtype, _FLOAT)
    _no_grad("matmul_w4", x, scales)
    packed, scales, zeros = _w4_operands(packed, scales, zeros, K)
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    if x2.stride(1) != 1 and K != 1:
        x2 = x2.contiguous()
    M, N = x2.shape[0], packed.shape[0]
    y = x2.new_empty((M, N))
    code = _TORCH_TO_OZK[dtype]
    n = _bytes("ozk_matmul_w4_workspace_bytes", code, M, N, K, group_size)
    ws, wsp = _workspace(n, dev)
    _call("ozk_matmul_w4", dev, x2.data_ptr(), code, x2.stride(0), packed.data_ptr(),
          packed.stride(0), scales.data_ptr(), _TORCH_TO_OZK[scales.dtype], scales.stride(0),
          None if zeros is None else zeros.data_ptr(), 0 if zeros is None else zeros.stride(0),
          group_size, M, N, K, y.data_ptr(), N, wsp, n)
    del ws
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)


# ============================================================
# orthogonalisation
# ============================================================

def orthogonalize(G: torch.Tensor, steps: int = 5, coefficients=(3.4445, -4.7750, 2.0315),
                  eps: float = 1e-7) -> torch.Tensor:
    """G's nearest matrix with singular values about 1, by Newton-Schulz products:
    X = G / (|G|_F + eps), then ``steps`` times with S = X X^T (X^T X where G is tall)
    X <- a X + (b S + c S S) X.

    Args:
        G: (..., M, N) float32 / float16 / bfloat16, each matrix on its own
        coefficients: (a, b, c) of every step, or a sequence of ``steps`` such triples
    Returns:
        X: the shape and dtype of G.  Products are fp32-grade (two fp16 slices, sums
        in fp32), whatever G's dtype and the coefficients.  A zero matrix stays
        zero; one with an infinity or NaN becomes NaN.
    """
    assert G.dim() >= 2, f"G must be [..., M, N], got {tuple(G.shape)}"
    assert 1 <= steps <= 64, f"steps must be 1 .. 64, got {steps}"
    co = tuple(coefficients)
    triples = [co] * steps if len(co) == 3 and not hasattr(co[0], "__len__") else co
    assert len(triples) == steps and all(len(t) == 3 for t in triples), \
        f"coefficients must be one triple or {steps}, got {coefficients!r}"
    _on_one_gpu(G)
    _require_dtype("orthogonalize", G.dtype, _FLOAT)
    _no_grad("orthogonalize", G)
    if G.numel() == 0:
        return torch.empty_like(G, memory_format=torch.contiguous_format)
    M, N = G.shape[-2:]
    G3 = G if G.dim() == 3 else G.reshape(-1, M, N)
    if G3.stride(2) != 1 and N != 1:
        G3 = G3.contiguous()
    B, dev = G3.shape[0], G.device
    if B > _MAX_BATCH:
        return torch.cat([orthogonalize(g, steps, triples, eps) for g in G3.split(_MAX_BATCH)]).view(G.shape)
    out = torch.empty((B, M, N), dtype=G.dtype, device=dev)
    n = _bytes("ozk_orthogonalize_workspace_bytes", B, M, N, steps)
    ws, wsp = _workspace(n, dev)
    flat = (ctypes.c_double * (3 * steps))(*[float(v) for t in triples for v in t])
    _call("ozk_orthogonalize", dev, G3.data_ptr(), _TORCH_TO_OZK[G.dtype], B, M, N,
          _i64(*G3.stride()[:2]), flat, steps, float(eps), out.data_ptr(), _i64(M * N, N), wsp, n)
    del ws
    return out.view(G.shape)
