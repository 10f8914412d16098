"""Operators for linear layers on the GPU at the edges of their ranges, against plain
computations in 64 bits; tolerances as in test_gpu_linear.py, unless a test derives
its own."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fw
from test_gpu_linear import (BF, COEFFICIENTS, F16, F32, ROUND, _check_grouped, _check_orth, _check_w4, _gen,
                             _offsets, _random_w4, _randn, _steps, _unpack)
from test_orthogonalize_plan import OVERSHOOTING, STANDARD

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
@pytest.mark.parametrize("triples", [OVERSHOOTING, [(40.0, -30.0, 10.0)] * 2, [(9.0, 2e3, -3e3)],
                                     [STANDARD, (1e-3, 0.0, 0.0), (900.0, -4e8, 0.0)]])
def test_orthogonalize_bounds_that_no_matrix_reaches(triples, dtype):
    """Schedules whose bound on the singular values grows far past the matrices' own."""
    for shape in ((64, 200), (96, 160), (160, 96), (256, 512), (3, 65, 40), (2, 3, 40, 24), (700, 1100)):
        G = _randn(1, *shape, dtype=dtype)
        want = _steps(G.cpu().double(), triples, 1e-7, torch.float64)
        if bool((want.abs() < torch.finfo(dtype).max).all()):
            _check_orth(G, len(triples), triples)
            continue
        # entries past the type's range become infinities, the others are held to the same
        got = ozk.orthogonalize(G, len(triples), triples).cpu()
        inside = want.abs() < torch.finfo(dtype).max * 0.999
        assert bool((got == want.to(dtype))[want.abs() > torch.finfo(dtype).max * 1.001].all())
        off = lambda y: float((y.double() - want)[inside].norm() / want[inside].norm())  # noqa: E731
        plain = _steps(G.cpu().float(), triples, 1e-7, F32)
        assert off(got) <= 4 * max(off(plain), 2.0 ** -24) + ROUND[dtype]


def test_orthogonalize_measured_scales_are_each_matrix_own():
    """Matrices of a batch beside a zero one, one with a NaN and one of rank 1 (all of
    its norm in one value) are what they are alone; a schedule that diverges gives no
    finite value."""
    G = _randn(1, 5, 64, 80, dtype=F32)
    G[1], G[2, 3, 4], G[4] = 0, math.nan, _randn(2, 64, 1, dtype=F32) * _randn(3, 80, dtype=F32)
    X = ozk.orthogonalize(G, 7, OVERSHOOTING)
    assert not X[1].any() and X[2].isnan().all()
    for i in (0, 3, 4):
        assert torch.equal(X[i], _check_orth(G[i], 7, OVERSHOOTING)) and torch.isfinite(X[i]).all()
    assert not torch.isfinite(ozk.orthogonalize(G[0], 6, (40.0, -30.0, 10.0))).any()


def test_orthogonalize_measured_scales_in_a_graph():
    G = _randn(1, 2, 100, 160)
    graph = torch.cuda.CUDAGraph()
    ozk.orthogonalize(G, 7, OVERSHOOTING)
    with torch.cuda.graph(graph):
        got = ozk.orthogonalize(G, 7, OVERSHOOTING)
    for n in range(3):
        G.copy_(_randn(2 + n, 2, 100, 160))
        want = ozk.orthogonalize(G, 7, OVERSHOOTING)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


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


@pytest.mark.parametrize("shape", [(0, 48), (48, 0), (0, 0), (2, 3, 0, 5), (2, 0, 4, 5), (0, 4, 5), (3, 4, 0)])
def test_orthogonalize_empty(shape):
    G = torch.zeros(shape, dtype=BF, device="cuda")
    X = ozk.orthogonalize(G)
    assert X.shape == shape and X.dtype == BF and X.data_ptr() == 0


def test_orthogonalize_more_matrices_than_a_launch_counts():
    G = _randn(1, 2, 33000, 3, 5, dtype=F32)
    X = ozk.orthogonalize(G)
    assert X.shape == G.shape
    for b, n in ((0, 0), (1, 32534), (1, 32535), (1, 32999)):     # 65535 = 33000 + 32535
        assert torch.equal(X[b, n], ozk.orthogonalize(G[b, n]))


# ---------------------------------------------------------------------------
# grouped products
# ---------------------------------------------------------------------------

def test_grouped_single_rows_of_longer_tensors():
    """The last token of one sequence, a matrix with one row or one column: their strides
    are those of what they were cut from, past the kernels' limit."""
    h, d = _randn(1, 1, 2048, 4096), _randn(2, 1, 40000, 136)
    last, grad, B = h[:, -1], d[:, -1], _randn(3, 1, 4096, 136)
    assert last.stride(0) >= 1 << 22 and grad.stride(0) >= 1 << 22 and last.is_contiguous()
    offsets = _offsets([1])
    _check_grouped(last, B, grad, offsets)
    far = torch.zeros(1, 8, (1 << 22) + 24, dtype=BF, device="cuda")
    far[:, :, :64] = _randn(4, 1, 8, 64)
    A, D, offsets = _randn(5, 50, 8), _randn(6, 50, 64), _offsets([40])
    _check_grouped(A[:, 3:4], far[:, 3:4, :64], D, offsets)                   # K = 1
    _check_grouped(D, far[:, 3:4, :64].mT, A[:, 3:4], offsets)                # N = 1
    _check_grouped(A, far[:, :, 5:6], D[:, 5:6], offsets)
    _check_grouped(A[:, 3:4], far[:, 3:4, 5:6], D[:, 5:6], offsets)           # both
    one = far[0, 3, 5].expand(1, 1, 1).as_strided((1, 1, 1), (7, 7, 7))
    _check_grouped(A[:, 3:4], one, D[:, 5:6], offsets)


@pytest.mark.parametrize("rows, N", [(2, 64), (64, 3)])
def test_grouped_rows_longer_than_their_distance_may_be(rows, N):
    """One row (column) for all, of more elements than rows may be apart, and no whole 16-byte
    pieces: 64 copies of it on rows of their own end past the tiles' 31-bit offsets."""
    K, offsets = (1 << 24) + 500001, _offsets([rows])
    whole = lambda seed, *s: torch.randint(-2, 3, s, generator=_gen(seed), device="cuda",  # noqa: E731
                                           dtype=torch.int8).to(BF)
    a, b = whole(1, 1, K), whole(2, 1, 1, K).mT
    want = (a.double() @ b[0].double()).to(BF)          # every sum is a whole number, and exact
    assert bool(want.any()) and 63 * 2 * K > 1 << 31
    C = ozk.grouped_matmul(a.expand(rows, K), b.expand(1, K, N), offsets)
    assert torch.equal(C, want.expand(rows, N))


def test_forward_mode_is_refused():
    """A tangent is not dropped: none of the operators has a forward-mode derivative."""
    A, B, D, offsets = _randn(1, 6, 32), _randn(2, 1, 32, 40), _randn(3, 6, 40), _offsets([6])
    weights, G = ozk.quantize_w4(_randn(4, 40, 32), 32), _randn(5, 8, 16)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: ozk.grouped_matmul(dual(A), B, offsets),
                     lambda: ozk.grouped_matmul(A, dual(B), offsets),
                     lambda: ozk.grouped_matmul_backward(dual(D), A, B, offsets),
                     lambda: ozk.matmul_w4(dual(A), *weights, group_size=32),
                     lambda: ozk.quantize_w4(dual(B[0].T), 32),
                     lambda: ozk.orthogonalize(dual(G))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert torch.equal(ozk.grouped_matmul(A, B, offsets), ozk.grouped_matmul(A, B, offsets))
    assert ozk.orthogonalize(G).shape == G.shape


# ---------------------------------------------------------------------------
# 4-bit weights
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("N, K, group", [(5, 33, 32), (3, 64, 64), (4, 1000, 128), (2, 513, 32)])
def test_quantize_leaves_what_lies_between_its_rows(N, K, group):
    """Packed rows, scales and zero points inside wider buffers (the C call): the bytes
    between the rows, and those behind the last one, stay."""
    lib, W = ozk.ozaki._lib, _randn(1, N, K, dtype=F32)
    groups, width, stride, apart = -(-K // group), -(-K // 32) * 16, -(-K // 32) * 16 + 48, -(-K // group) + 3
    packed = torch.full((N * stride + 512,), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((N * apart + 64,), -7.0, device="cuda")
    zeros = torch.full((N * apart + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    lib.check("ozk_quantize_w4", lib.load().ozk_quantize_w4(
        W.data_ptr(), lib.OZK_F32, N, K, K, group, packed.data_ptr(), stride, scales.data_ptr(), apart,
        zeros.data_ptr(), apart, torch.cuda.current_stream().cuda_stream))
    want = ozk.quantize_w4(W, group, zeros=True)
    for got, columns, distance, w, other in ((packed, width, stride, want[0], 0xA5),
                                             (scales, groups, apart, want[1], -7.0),
                                             (zeros, groups, apart, want[2], 0xA5)):
        rows = got[:N * distance].view(N, distance)
        assert torch.equal(rows[:, :columns], w)
        assert bool((rows[:, columns:] == other).all()) and bool((got[N * distance:] == other).all())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M, N, K", [(1, 200, 512), (3, 9000, 256), (20, 300, 1024), (40, 300, 640), (2, 64, 16384)])
def test_w4_activations_up_to_the_largest(dtype, group, M, N, K):
    """Finite x gives finite y where y itself is: the two sums that are subtracted are up to
    31 times sum |x|, past fp32's range here.  Powers of two change nothing else."""
    packed, scales, z = _random_w4(2, N, K, group, dtype, True)
    scales = (scales.float() / 64).to(dtype)
    x = _randn(1, M, K, dtype=dtype)
    y = ozk.matmul_w4(x, packed, scales, z, group_size=group)
    for power in (123, 60, -60):
        big = ozk.matmul_w4((x.double() * 2.0 ** power).to(dtype), packed, scales, z, group_size=group)
        assert torch.equal(big.double(), y.double() * 2.0 ** power)
    x[:, ::7] = 3.3e38
    x[:, 1::7] = -3.3e38
    _check_w4(x, packed, (scales.double() / 2 ** 7).to(dtype), z, group)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M, N, K", [
    (1, 4096, 1024), (5, 1000, 2047), (16, 512, 4096),         # one block of 16 columns a workgroup
    (2, 8208, 1024), (4, 9001, 515),                           # few rows, many columns
    (6, 4112, 1000), (17, 300, 2048), (32, 9000, 640),         # many of both
    (33, 260, 1024), (65, 130, 2048), (150, 300, 700),
    (1, 64, 16384), (3, 100, 8191), (20, 70, 16384)])          # K in ranges
def test_w4_full_precision_activations_in_every_shape(M, N, K, group, zeros):
    """fp32 x at fp32's accuracy: within four times the error of a plain fp32 product (x cut to
    16 bits is 30 times as far off, to 8 bits 8000 times)."""
    x, (p, s, z) = _randn(1, M, K, dtype=F32), _random_w4(2, N, K, group, F32, zeros)
    W = ozk.dequantize_w4(p, s, z, group_size=group, K=K)
    want = x.cpu().double() @ W.cpu().double().T
    off = lambda y: float((y.cpu().double() - want).norm() / want.norm())  # noqa: E731
    plain = off(x.cpu() @ W.cpu().T)
    assert off(ozk.matmul_w4(x, p, s, z, group_size=group)) <= 4 * max(plain, 2.0 ** -24)


def _format(W, group, zeros):
    """q, s and z of the format by its definition, in fp32 as stated."""
    N, K = W.shape
    w = torch.nn.functional.pad(W.cpu().float(), (0, -K % group)).view(N, -1, group)
    lo, hi = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
    s = (((hi - lo) * (1 / 15)) if zeros else torch.maximum(hi, -lo) * (1 / 7)).to(W.dtype).float()
    over = lambda a, b: torch.where(b > 0, torch.round(a / b), torch.zeros_like(a))  # noqa: E731
    z = over(-lo, s).clamp(0, 15) if zeros else torch.full_like(s, 8)
    q = (over(w, s[..., None].expand_as(w)) + z[..., None]).clamp(0, 15)
    return q.view(N, -1)[:, :K].long(), s, z


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize_is_the_format_to_the_last_value(dtype, zeros, group):
    """q and z equal the definition's, at ties of a power-of-two scale (k + 1/2 steps, to the
    even one), at quotients beside them, and on random weights of any size."""
    g = _gen(9)
    ties = torch.randint(-14, 15, (64, 4 * group), generator=g, device="cuda").float() / 2
    if zeros:
        ties = ties.clamp(-7, 7)
        ties[:, ::group], ties[:, 1::group] = -7.5, 7.5         # s = 1, z = 7.5 to even
        ties[32:, ::group], ties[32:, 1::group] = -4.5, 10.5
    else:
        ties[:, ::group] = 7.0                                  # s = 1
    ties = ties * 2.0 ** torch.randint(-8, 8, (64, 1), generator=g, device="cuda")
    beside = ties * (1 + torch.finfo(dtype).eps * torch.randint(-1, 2, ties.shape, generator=g, device="cuda"))
    sizes = 10.0 ** torch.linspace(-4, 4 if dtype == F16 else 30, 64, device="cuda")[:, None]
    for W in (ties, beside, _randn(1, 64, 4 * group, dtype=F32) * sizes, _randn(2, 7, 3 * group + 5, dtype=F32),
              _randn(3, 64, group, dtype=F32).abs(), -_randn(4, 64, group, dtype=F32).abs()):
        W = W.to(dtype)
        q, s, z = _format(W, group, zeros)
        packed, scales, got_z = ozk.quantize_w4(W, group, zeros=zeros)
        assert torch.equal(scales.cpu().float(), s)
        assert not zeros or torch.equal(got_z.cpu().float(), z)
        assert torch.equal(_unpack(packed, W.shape[1]), q)
    # (the first weights do hold ties)
    steps = ties.to(dtype).cpu().float().view(64, 4, group) / _format(ties.to(dtype), group, zeros)[1][..., None]
    assert int((steps % 1 == 0.5).sum()) > 1000


@pytest.mark.parametrize("dtype", [BF, F32])
def test_quantize_ranges_past_the_largest_float(dtype):
    """Weights of both signs near the type's largest: their range is past it, their scale
    is not.  Each comes back within half a step (and a whole one at the ends)."""
    W = (_randn(1, 6, 96, dtype=F32) / 5).clamp(-1, 1)
    W[:, ::32], W[:, 1::32] = 1, -0.8
    W = (W * 3e38).to(dtype)
    packed, scales, z = ozk.quantize_w4(W, 32, zeros=True)
    step = scales.cpu().double().repeat_interleave(32, 1)
    assert bool(((step > 3.5e37) & (step < 3.7e37)).all()) and bool((z == 7).all())      # 1.8 / 15, 0.8 / 0.12
    off = (ozk.dequantize_w4(packed, scales, z, group_size=32).cpu().double() - W.cpu().double()).abs()
    assert bool((off <= step * 1.01).all()) and float((off <= step * 0.51).double().mean()) > 0.9


def test_w4_packed_rows_past_4_gib():
    """Rows whose first byte lies past 2^32."""
    N, K = (1 << 16) + 5, 1 << 17
    packed = torch.zeros(N, K // 2, dtype=torch.uint8, device="cuda")
    rows = torch.tensor([0, 1, 4, 1 << 16, N - 4, N - 1], device="cuda")   # 1, 4: where 32 bits would read
    p, s, z = _random_w4(2, 6, K, 128, BF, True)
    packed[rows] = p
    scales = torch.ones(N, K // 128, dtype=BF, device="cuda")
    zeros = torch.zeros(N, K // 128, dtype=torch.uint8, device="cuda")
    scales[rows], zeros[rows] = s, z
    for M in (2, 20):
        _check_w4(_randn(1, M, K), packed, scales, zeros, 128, rows.cpu())
    W = ozk.dequantize_w4(packed[-6:], scales[-6:], zeros[-6:])
    assert torch.equal(W[2], ozk.dequantize_w4(p[4:5], s[4:5], z[4:5])[0])
    assert torch.equal(W[5], ozk.dequantize_w4(p[5:], s[5:], z[5:])[0])
    # the whole of it back to weights and to 4 bits again
    back = ozk.dequantize_w4(packed, scales, zeros)
    assert torch.equal(back[rows], ozk.dequantize_w4(p, s, z))
    again, s2, z2 = ozk.quantize_w4(back, zeros=True)
    for got, want in zip((again[rows], s2[rows], z2[rows]), ozk.quantize_w4(back[rows], zeros=True)):
        assert torch.equal(got, want)


def test_dequantize_has_no_gradient():
    """Scales that want a gradient are refused, as by matmul_w4."""
    p, s, z = _random_w4(2, 30, 64, 32, BF, True)
    want = ozk.dequantize_w4(p, s, z, group_size=32)
    s.requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        ozk.dequantize_w4(p, s, z, group_size=32)
    with torch.no_grad():
        assert torch.equal(ozk.dequantize_w4(p, s, z, group_size=32), want)


def test_w4_rows_that_overlap():
    """One packed row, scale and zero point for all rows of W, and rows that overlap."""
    x, (p, s, z) = _randn(1, 3, 96), _random_w4(2, 1, 96, 32, BF, True)
    one = ozk.matmul_w4(x, p, s, z, group_size=32)
    wide = [t.expand(20, -1) for t in (p, s, z)]
    assert torch.equal(ozk.matmul_w4(x, *wide, group_size=32), one.expand(3, 20))
    assert torch.equal(ozk.dequantize_w4(*wide, group_size=32), ozk.dequantize_w4(p, s, z, group_size=32).expand(20, 96))
    p, s, z = _random_w4(3, 4, 32, 32, BF, True)
    windows = p.flatten().as_strided((2, 48), (16, 1))
    for n in range(2):
        got = ozk.matmul_w4(x, windows, s[:2].expand(2, 3), z[:2].expand(2, 3), group_size=32)[:, n]
        assert torch.equal(got, ozk.matmul_w4(x, windows[n:n + 1].clone(), s[n:n + 1].expand(1, 3),
                                              z[n:n + 1].expand(1, 3), group_size=32)[:, 0])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_w4_more_rows_than_a_launch_counts(dtype):
    """65535 blocks of 64 rows (fp32: of 32) and some more."""
    M, (p, s, z) = 65535 * (32 if dtype == F32 else 64) + 70, _random_w4(2, 5, 32, 32, dtype, True)
    x = _randn(1, M, 33, dtype=dtype)[:, 1:]
    y = ozk.matmul_w4(x, p, s, z, group_size=32)
    for rows in (slice(0, 100), slice(M // 2, M // 2 + 100), slice(M - 200, M)):
        assert torch.equal(y[rows], ozk.matmul_w4(x[rows], p, s, z, group_size=32))
