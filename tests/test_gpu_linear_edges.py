"""Operators for linear layers on the GPU at the edges of their ranges, against plain
computations in 64 bits; tolerances as in test_gpu_linear.py, unless a test derives
its own."""
import math

import pytest
import torch
from test_gpu_linear import BF, COEFFICIENTS, F16, F32, _gen, _steps

import ozaki_triton_amd as ozk

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# orthogonalisation
# ---------------------------------------------------------------------------

def _four_decades(seed, m, n, dtype):
    r = lambda *s: torch.randn(*s, generator=_gen(seed), device="cuda", dtype=torch.float64)  # noqa: E731
    u, v = torch.linalg.qr(r(m, m))[0], torch.linalg.qr(r(n, m))[0]
    return (u @ torch.diag(torch.logspace(0, -4, m, device="cuda", dtype=torch.float64)) @ v.T).to(dtype)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("triples", [[COEFFICIENTS] * 5, [COEFFICIENTS] * 7 + [(0.2, 0.0, 0.0)],
                                     [COEFFICIENTS] * 6 + [(1.0, 0.0, 0.0)]])
def test_orthogonalize_long_rounds_like_fp32(triples, dtype):
    """16-bit results of long matrices: an error of a given size moves a share of the
    entries over to the next 16-bit number in proportion, and four times the error of
    plain fp32 is allowed, so four times the entries (and 5 deviations of their count)."""
    for m, n in ((256, 1024), (1024, 256)):
        G = _four_decades(3, min(m, n), max(m, n), dtype)
        G = G if m < n else G.T
        want = _steps(G.cpu().double(), triples, 1e-7, torch.float64).to(dtype)
        plain = _steps(G.cpu().float(), triples, 1e-7, F32).to(dtype)
        moved = lambda y: int((y.cpu() != want).sum())  # noqa: E731
        got, allowed = moved(ozk.orthogonalize(G, len(triples), triples)), 4 * moved(plain)
        assert got <= allowed + 5 * math.sqrt(allowed) + 5, (got, allowed)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
def test_orthogonalize_zero_matrix_without_eps(dtype):
    """A zero matrix stays zero, also where nothing is added to its norm of 0."""
    G = torch.randn(3, 40, 50, generator=_gen(1), device="cuda").to(dtype)
    G[1] = 0
    for g in (G, G.mT):
        X = ozk.orthogonalize(g, eps=0.0)
        assert not X[1].any()
        assert all(torch.equal(X[i], ozk.orthogonalize(g[i], eps=0.0)) for i in (0, 2))
        assert torch.isfinite(X).all()
