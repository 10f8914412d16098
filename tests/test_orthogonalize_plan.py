"""The plan of an orthogonalisation -- which products it runs, on what scales --
carried out on the CPU: matrices as two fp16 slices, products as the slice pairs
hh, hl, lh.  The result, before its last rounding, is held to four times the error
that the same steps have in plain fp32, whatever the result's dtype."""
import ctypes

import pytest
import torch

from ozaki_triton_amd import _lib

STANDARD, QUINTIC = (3.4445, -4.7750, 2.0315), (1.875, -1.25, 0.375)
DTYPES = {"fp32": _lib.OZK_F32, "fp16": _lib.OZK_F16, "bf16": _lib.OZK_BF16}


def _plan(m, n, triples, dtype):
    """The products, as ((kind, L, R, Y, D), (f, f_y, f_i)), and X's first scale."""
    co = (ctypes.c_double * (3 * len(triples)))(*[v for t in triples for v in t])
    buffers, factors = (ctypes.c_int * (5 * 256))(), (ctypes.c_float * (3 * 256))()
    scale, ops = ctypes.c_float(0), ctypes.c_int(0)
    _lib.check("ozk_debug_orth_plan", _lib.load().ozk_debug_orth_plan(
        m, n, co, len(triples), dtype, buffers, factors, ctypes.byref(scale), ctypes.byref(ops)))
    return [(buffers[5 * i:5 * i + 5], factors[3 * i:3 * i + 3]) for i in range(ops.value)], scale.value


def _slices(v):
    v = v.float()
    h = v.half()
    return h.double(), (v - h.float()).half().double()


def _run(G, triples, dtype, eps=1e-7):
    """X of the plan, as fp32 values before they are rounded to the result's dtype."""
    plan, scale = _plan(*G.shape, triples, dtype)
    held = {-1: _slices(G.double() / (G.double().norm() + eps) * scale)}
    eye = torch.eye(G.shape[0], dtype=torch.float64)
    for (kind, L, R, Y, D), (f, f_y, f_i) in plan:
        (lh, ll), (rh, rl) = held[L], held[R]
        if kind == 0:
            rh, rl = rh.T, rl.T
        v = (lh @ rh + lh @ rl + ll @ rh).float().double() * f
        if Y != -9:
            v = v + sum(held[Y]) * f_y
        if f_i:
            v = v + f_i * eye
        if kind == 3:
            return v.float()
        held[D] = _slices(v)


def _steps(G, triples, dtype, eps=1e-7):
    X = (G.double() / (G.double().norm() + eps)).to(dtype)
    for a, b, c in triples:
        A = X @ X.T
        X = a * X + (b * A + c * (A @ A)) @ X
    return X


def _matrix(kind, m, n):
    g = torch.Generator().manual_seed(m + n)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    if kind == "low rank":
        return r(m, 3) @ r(3, n)
    if kind == "four decades":
        u, v = torch.linalg.qr(r(m, m))[0], torch.linalg.qr(r(n, m))[0]
        return u @ torch.diag(torch.logspace(0, -4, m, dtype=torch.float64)) @ v.T
    return r(m, n)


def _check(kind, m, n, triples, dtype):
    G = _matrix(kind, m, n)
    if dtype != _lib.OZK_F32:
        G = G.to(torch.bfloat16).double()
    want, plain = _steps(G, triples, torch.float64), _steps(G, triples, torch.float32)
    off = lambda y: float((y.double() - want).norm() / want.norm())  # noqa: E731
    got = off(_run(G, triples, dtype))
    assert got <= 4 * max(off(plain), 2.0 ** -24), (got, off(plain))


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
@pytest.mark.parametrize("kind", ["gauss", "four decades", "low rank"])
@pytest.mark.parametrize("triples", [
    [STANDARD] * 5, [QUINTIC] * 8, [(1.5, -0.5, 0.0)] * 4,
    # a scale, or nothing, at the end: the last slope is 0 and says nothing of the others
    [STANDARD] * 7 + [(0.2, 0.0, 0.0)], [STANDARD] * 9 + [(0.2, 0.0, 0.0)],
    [STANDARD] * 6 + [(1.0, 0.0, 0.0)]])
def test_last_steps_are_as_near_as_steps_by_themselves(triples, kind, dtype):
    for m, n in ((64, 200), (48, 96), (40, 44)):
        _check(kind, m, n, triples, dtype)


def test_last_steps_run_together_where_they_may():
    """Two of five with the standard coefficients, from twice as long as high on."""
    kinds = lambda *a: [b[0] for b, _ in _plan(*a)[0]]  # noqa: E731
    own = [0, 1, 2] * 4 + [0, 1, 3]
    assert kinds(64, 127, [STANDARD] * 5, _lib.OZK_BF16) == own
    assert kinds(64, 200, [STANDARD] * 5, _lib.OZK_F32) == own
    assert kinds(64, 200, [STANDARD] * 5, _lib.OZK_BF16) == [0, 1, 2] * 3 + [0, 1, 1, 1, 1, 1, 3]
