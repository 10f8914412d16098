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
    norm_x, norm_b = 1.0, 1.0      # measured ones
    if all(kind != 4 for (kind, *_), _ in plan):
        norm_x = norm_b = None
    held = {-1: _slices(G.double() / (G.double().norm() + eps) * scale)}
    eye = torch.eye(G.shape[0], dtype=torch.float64)
    for (kind, L, R, Y, D), (f, f_y, f_i) in plan:
        (lh, ll), (rh, rl) = held[L], held[R]
        if kind == 0:
            rh, rl = rh.T, rl.T
        if norm_x is not None and kind != 0:
            f, f_y = (f * norm_x ** 4, f_y * norm_x ** 2) if kind == 4 else (f * norm_b * norm_x, f_y * norm_x)
        v = (lh @ rh + lh @ rl + ll @ rh).float().double() * f
        if Y != -9:
            v = v + sum(held[Y]) * f_y
        if f_i:
            v = v + f_i * eye
        if kind == 3:
            return v.float()
        if kind >= 4:
            norm = float(v.norm())
            v = v * (scale / norm if norm else 0.0)
            norm_x, norm_b = (norm_x, norm) if kind == 4 else (norm, norm_b)
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


# Coefficients that overshoot at 1: step by step a bound over whole intervals grows to
# 1.99, 1.99, 2.2, 6.6, 4.6e3, 8e17 and 1e89, where no value of [0, 1] gets past 2.
OVERSHOOTING = [(8.28721201814563, -23.595886519098837, 17.300387312530933),
                (4.107059111542203, -2.9478499167379106, 0.5448431082926601),
                (3.9486908534822946, -2.908902115962949, 0.5518191394370137),
                (3.3184196573706015, -2.488488024314874, 0.51004894012372),
                (2.300652019954817, -1.6689039845747493, 0.4188073119525673),
                (1.891301407787398, -1.2679958271945868, 0.37680408948524835), (1.875, -1.25, 0.375)]


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES.keys())
@pytest.mark.parametrize("triples", [OVERSHOOTING, OVERSHOOTING[:3], [(40.0, -30.0, 10.0)] * 2,
                                     [STANDARD, (1e-3, 0.0, 0.0), (900.0, -4e8, 0.0)]])
def test_bounds_that_no_matrix_reaches(triples, dtype):
    for m, n in ((64, 200), (96, 160), (256, 512)):
        _check("gauss", m, n, triples, dtype)
    _check("four decades", 64, 200, triples, dtype)


def test_scales_are_measured_where_the_bounds_are_wide():
    kinds = lambda t: [b[0] for b, _ in _plan(64, 200, t, _lib.OZK_BF16)[0]]  # noqa: E731
    assert kinds(OVERSHOOTING) == [0, 4, 5] * 6 + [0, 4, 3]
    assert kinds([(1e4, 0.0, -1e6)]) == [0, 4, 3]
    for t in ([STANDARD] * 9, [QUINTIC] * 64, [(1.5, -0.5, 0.0)] * 20):
        assert 4 not in kinds(t)


def test_last_steps_run_together_where_they_may():
    """Two of five with the standard coefficients, from twice as long as high on."""
    kinds = lambda *a: [b[0] for b, _ in _plan(*a)[0]]  # noqa: E731
    own = [0, 1, 2] * 4 + [0, 1, 3]
    assert kinds(64, 127, [STANDARD] * 5, _lib.OZK_BF16) == own
    assert kinds(64, 200, [STANDARD] * 5, _lib.OZK_F32) == own
    assert kinds(64, 200, [STANDARD] * 5, _lib.OZK_BF16) == [0, 1, 2] * 3 + [0, 1, 1, 1, 1, 1, 3]
