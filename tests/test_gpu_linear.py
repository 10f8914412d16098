"""Operators for linear layers on the GPU, against plain computations in 64 bits.

Tolerances.  Products of 16-bit values are exact in fp32, so a result differs
from the exact one by its sums in fp32 -- (terms) 2^-23 of the sum of the terms'
magnitudes covers rounding and truncating adders in any order -- and by its one
rounding to 16 bits: 2^-8 of the value for bfloat16 (8 significant bits), 2^-11 for
float16 (11; and half the smallest subnormal, 2^-25).  Orthogonalised matrices are held to four
times the error that the same steps have in plain fp32: slices of 22 bits against
24."""
import math

import pytest
import torch

import ozaki_triton_amd as ozk

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
ROUND = {BF: 2.0 ** -8, F16: 2.0 ** -11, F32: 2.0 ** -24}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(seed, *size, dtype=BF):
    return torch.randn(*size, generator=_gen(seed), device="cuda").to(dtype)


def _offsets(counts, dtype=torch.int32, start=0):
    return torch.tensor([start] + counts, device="cuda").cumsum(0).to(dtype)


def _close(got, want, magnitude, terms, dtype):
    """got against want (64 bits) with `magnitude` the sum of the terms' magnitudes."""
    bound = ROUND[dtype] * 1.01 * want.abs() + terms * 2.0 ** -23 * magnitude + 2.0 ** -25
    assert got.dtype == dtype and got.shape == want.shape
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())


def _grouped(A, B, ends):
    """C and the magnitudes of its terms, group by group."""
    C = torch.zeros(A.shape[0], B.shape[2], dtype=torch.float64, device=A.device)
    mag = C.clone()
    for g, (lo, hi) in enumerate(zip(ends, ends[1:])):
        b = B[g].double()
        C[lo:hi] = A[lo:hi].double() @ b
        mag[lo:hi] = A[lo:hi].double().abs() @ b.abs()
    return C, mag


def _wgrad(A, D, ends):
    dB = torch.zeros(len(ends) - 1, A.shape[1], D.shape[1], dtype=torch.float64, device=A.device)
    mag = dB.clone()
    for g, (lo, hi) in enumerate(zip(ends, ends[1:])):
        a = A[lo:hi].double().T.contiguous()
        dB[g] = a @ D[lo:hi].double()
        mag[g] = a.abs() @ D[lo:hi].double().abs()
    return dB, mag


def _check_grouped(A, B, D, offsets):
    ends = offsets.tolist()
    rows = max((hi - lo for lo, hi in zip(ends, ends[1:])), default=0)
    K, N = B.shape[1:]
    _close(ozk.grouped_matmul(A, B, offsets), *_grouped(A, B, ends), K, A.dtype)
    dA, dB = ozk.grouped_matmul_backward(D, A, B, offsets)
    _close(dA, *_grouped(D, B.mT, ends), N, A.dtype)
    _close(dB, *_wgrad(A, D, ends), rows + 16, A.dtype)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("bt", [False, True])
@pytest.mark.parametrize("counts, K, N, spare", [
    ([1], 64, 64, 0), ([1], 1, 1, 0), ([0], 64, 64, 0), ([0, 0, 3], 8, 8, 5),
    ([5, 0, 130, 1, 64], 128, 256, 0), ([5, 0, 130, 1, 64], 72, 136, 7),
    ([33, 31, 0, 2], 73, 137, 1), ([31, 33, 65], 65, 130, 0), ([257, 300], 100, 500, 3),
    ([700, 1, 512], 264, 520, 0), ([1000, 0], 250, 257, 0), ([3] * 70, 40, 48, 2),
    ([0] * 61 + [2, 0, 9], 40, 48, 2), ([2, 1, 0, 0, 4, 1, 3, 2], 1024, 200, 0),
    ([1, 2, 1], 1023, 65, 0), ([2600], 520, 264, 9), ([4000], 24, 33, 0),
])
def test_grouped(dtype, bt, counts, K, N, spare):
    rows = sum(counts) + spare
    A, D = _randn(1, rows, K, dtype=dtype), _randn(3, rows, N, dtype=dtype)
    B = _randn(2, len(counts), N, K, dtype=dtype)
    _check_grouped(A, B.mT if bt else B.mT.contiguous(), D, _offsets(counts))


@pytest.mark.parametrize("counts, K, N", [
    ([1500, 900], 1001, 1003), ([300, 200, 100], 513, 515), ([900], 4097, 257),
    ([64], 2049, 2047), ([5000, 3000], 220, 103), ([2500], 1344, 1001)])
def test_grouped_copied_operands(counts, K, N):
    """Sizes whose rows are copied to whole 16-byte pieces first, at aligned and
    misaligned addresses, by both layouts of B; without the copies' workspace the
    same products go through registers."""
    offsets = _offsets(counts)
    A, D, B = _randn(1, sum(counts), K), _randn(3, sum(counts), N), _randn(2, len(counts), K, N)
    _check_grouped(A, B, D, offsets)
    _check_grouped(A, B.mT.contiguous().mT, D, offsets)
    buffer = torch.empty(A.numel() + 3, dtype=BF, device="cuda")
    A2 = buffer[3:].view(A.shape).copy_(A)
    assert A2.data_ptr() % 16 == 6
    assert torch.equal(ozk.grouped_matmul(A2, B, offsets), ozk.grouped_matmul(A, B, offsets))
    lib, C = ozk.ozaki._lib, torch.empty(sum(counts), N, dtype=BF, device="cuda")
    lib.check("ozk_grouped_matmul", lib.load().ozk_grouped_matmul(
        A.data_ptr(), K, B.data_ptr(), lib.i64arr((K * N, N, 1)), offsets.data_ptr(), 4, A.shape[0],
        K, N, len(counts), lib.OZK_BF16, C.data_ptr(), N, None, 0,
        torch.cuda.current_stream().cuda_stream))
    _close(C, *_grouped(A, B, offsets.tolist()), K, BF)


@pytest.mark.parametrize("counts, K, N", [
    ([600] * 4, 256, 8192), ([900, 1300, 1000], 192, 16384),   # the largest tiles
    ([1000, 500, 500], 1024, 4096), ([300, 700], 2048, 2048), ([1000, 3000], 264, 2056),
    ([40] * 8, 2048, 2048),       # 128 x 128, four stages
    ([700, 500], 4096, 256),      # two groups of waves on a tile's stages
    ([3, 0, 2], 4096, 1024), ([70, 90], 520, 520)])
def test_grouped_tiles(counts, K, N):
    offsets, rows = _offsets(counts), sum(counts)
    for bt in (False, True):
        B = _randn(2, len(counts), N, K)
        _check_grouped(_randn(1, rows, K), B.mT if bt else B.mT.contiguous(), _randn(3, rows, N), offsets)


@pytest.mark.parametrize("counts, K, N", [
    ([1] * 30 + [90, 500, 60, 200], 520, 264),     # every class of length
    ([0] * 63 + [300], 136, 72), ([300] + [0] * 62 + [7], 512, 320), ([3] * 64 + [400], 136, 200),
    ([10, 900, 10, 10], 2048, 2048), ([200] * 4, 2048, 2056), ([20, 900] * 4, 2048, 2048),
    ([40] * 8, 2048, 2048), ([300, 100, 80], 1288, 2056), ([90, 110, 100], 1304, 1112),
    ([0, 5000, 0, 30], 64, 64)])
def test_grouped_gradient_of_uneven_groups(counts, K, N):
    """Every tile of dB is written once, whatever the order of the groups: by length
    where they differ, their own where not or where they are many."""
    A, D, offsets = _randn(1, sum(counts), K), _randn(3, sum(counts), N), _offsets(counts)
    B = torch.zeros(len(counts), K, N, dtype=BF, device="cuda")
    stale = torch.full((len(counts), K, N), math.nan, dtype=BF, device="cuda")
    del stale    # the memory that dB is likely to get
    _, dB = ozk.grouped_matmul_backward(D, A, B, offsets)
    _close(dB, *_wgrad(A, D, offsets.tolist()), max(counts) + 16, BF)


def test_grouped_offsets_inside_the_rows():
    """int64 offsets that start after row 0: the rows before and after get zeros."""
    A, B, D = _randn(1, 90, 64), _randn(2, 3, 64, 72), _randn(3, 90, 72)
    offsets = _offsets([20, 0, 41], torch.int64, start=13)
    _check_grouped(A, B, D, offsets)
    C = ozk.grouped_matmul(A, B, offsets)
    assert not C[:13].any() and not C[74:].any()


def test_grouped_offsets_past_the_rows_are_cut():
    A, B = _randn(1, 90, 64), _randn(2, 3, 64, 72)
    cut = ozk.grouped_matmul(A, B, torch.tensor([0, 30, 90, 90], device="cuda"))
    for off in ([-5, 30, 1000, 1 << 40], [0, 30, 91, 91]):
        assert torch.equal(ozk.grouped_matmul(A, B, torch.tensor(off, device="cuda")), cut)


def test_grouped_without_rows_groups_or_columns():
    z = lambda *s: torch.zeros(*s, dtype=BF, device="cuda")  # noqa: E731
    off = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    assert ozk.grouped_matmul(z(0, 8), z(2, 8, 4), off(3)).shape == (0, 4)
    assert ozk.grouped_matmul(z(3, 8), z(2, 8, 0), off(3)).shape == (3, 0)
    A = _randn(1, 5, 8)
    assert not ozk.grouped_matmul(A, z(0, 8, 4), off(1)).any()
    assert not ozk.grouped_matmul(z(5, 0), z(1, 0, 4), _offsets([5])).any()
    dA, dB = ozk.grouped_matmul_backward(z(0, 4), z(0, 8), _randn(2, 2, 8, 4), off(3))
    assert dA.shape == (0, 8) and dB.shape == (2, 8, 4) and not dB.any()


def test_grouped_strides_and_alignments():
    """Rows of a wider buffer, from an odd column, every other row, a transposed
    A, one matrix for every group."""
    counts, K, N = [40, 0, 77], 64, 96
    offsets = _offsets(counts)
    wide, D = _randn(1, 117, 200), _randn(3, 234, N)
    B = _randn(2, 3, K + 3, N + 5)
    for A in (wide[:, :K], wide[:, 1:1 + K], wide[:, 8:8 + K], _randn(4, K, 117).T):
        for b in (B[:, :K, :N], B[:, 1:1 + K, 3:3 + N], B[1:2, :K, :N].expand(3, K, N),
                  _randn(5, K, 3, N).transpose(0, 1), _randn(6, K, N, 3).permute(2, 0, 1)):
            _check_grouped(A, b, D[::2], offsets)


def test_grouped_rows_do_not_leak():
    """NaN and infinities in other groups', spare rows and matrices stay there."""
    counts = [37, 20, 0, 50]
    A, B, D = _randn(1, 120, 72), _randn(2, 4, 72, 64), _randn(3, 120, 64)
    offsets = _offsets(counts)
    C, (dA, dB) = ozk.grouped_matmul(A, B, offsets), ozk.grouped_matmul_backward(D, A, B, offsets)
    for bad in (math.nan, math.inf):
        A2, B2, D2 = A.clone(), B.clone(), D.clone()
        A2[37:57], D2[37:57], B2[1], B2[2] = bad, bad, bad, bad
        A2[107:], D2[107:] = bad, bad
        C2, (dA2, dB2) = ozk.grouped_matmul(A2, B2, offsets), ozk.grouped_matmul_backward(D2, A2, B2, offsets)
        keep = [t for t in range(120) if not 37 <= t < 57]
        assert torch.equal(C2[keep], C[keep]) and torch.equal(dA2[keep], dA[keep])
        assert torch.equal(dB2[[0, 2, 3]], dB[[0, 2, 3]])
        assert not torch.isfinite(C2[37:57]).any() and not torch.isfinite(dB2[1]).any()
    one = A.clone()
    one[3, 5] = math.inf                 # one infinity: its row, with the matrix' signs
    want = torch.where(B[0, 5] > 0, math.inf, -math.inf).to(BF)
    assert torch.equal(ozk.grouped_matmul(one, B, offsets)[3], want)


def test_grouped_repeats_bit_for_bit():
    """Partial sums are joined in one order."""
    A, D = _randn(1, 20000, 64), _randn(3, 20000, 80)
    B, offsets = _randn(2, 2, 64, 80), _offsets([15000, 5000])
    first = ozk.grouped_matmul_backward(D, A, B, offsets)
    for _ in range(5):
        again = ozk.grouped_matmul_backward(D, A, B, offsets)
        assert all(torch.equal(x, y) for x, y in zip(first, again))


def test_grouped_gradient():
    """Autograd against the explicit backward, and against differences: small whole
    numbers make every product and sum exact, so the differences are too."""
    g = torch.Generator().manual_seed(0)
    whole = lambda *s: torch.randint(-2, 3, s, generator=g).to("cuda", BF)  # noqa: E731
    A, B, R = whole(50, 24), whole(1, 24, 16), whole(50, 16)
    offsets = _offsets([20, 0, 25])
    Ag, Bg = A.clone().requires_grad_(), B.clone().requires_grad_()
    (ozk.grouped_matmul(Ag, Bg.expand(3, 24, 16), offsets).float() * R).sum().backward()
    dA, dB = ozk.grouped_matmul_backward(R, A, B.expand(3, 24, 16), offsets)
    assert torch.equal(Ag.grad, dA) and torch.equal(Bg.grad, dB.float().sum(0, True).to(BF))
    f = lambda a, b: float((ozk.grouped_matmul(a, b.expand(3, 24, 16), offsets).double() * R.double()).sum())  # noqa: E731
    for seed in range(3):
        V, W = torch.roll(A, seed, 0), torch.roll(B, seed, 1)
        assert (f(A + V, B) - f(A - V, B)) / 2 == float((dA.double() * V.double()).sum())
        assert (f(A, B + W) - f(A, B - W)) / 2 == float((dB.double().sum(0, True) * W.double()).sum())
    only = B.clone().requires_grad_()
    ozk.grouped_matmul(A, only.expand(3, 24, 16), offsets).sum().backward()
    assert only.grad is not None
    with torch.no_grad():
        assert not ozk.grouped_matmul(Ag, Bg.expand(3, 24, 16), offsets).requires_grad


def test_grouped_on_its_stream_and_in_a_graph():
    A, B, D, offsets = _randn(1, 600, 128), _randn(2, 2, 128, 96), _randn(3, 600, 96), _offsets([250, 350])
    want = (ozk.grouped_matmul(A, B, offsets), *ozk.grouped_matmul_backward(D, A, B, offsets))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = (ozk.grouped_matmul(A, B, offsets), *ozk.grouped_matmul_backward(D, A, B, offsets))
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = (ozk.grouped_matmul(A, B, offsets), *ozk.grouped_matmul_backward(D, A, B, offsets))
    for n in range(3):
        offsets.copy_(_offsets([100 * n, 500 - 50 * n]))
        want = (ozk.grouped_matmul(A, B, offsets), *ozk.grouped_matmul_backward(D, A, B, offsets))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_grouped_rows_past_4_gib():
    rows, K, N = (1 << 20) + 77, 2112, 64
    A = torch.zeros(rows, K, dtype=BF, device="cuda")
    at = [0, 1 << 19, (1 << 20) - 1, rows - 1]
    A[at] = _randn(1, 4, K)
    B, offsets = _randn(2, 2, K, N), _offsets([1 << 19, rows - (1 << 19)])
    C = ozk.grouped_matmul(A, B, offsets)
    for t in at:
        b = B[int(t >= 1 << 19)].double()
        _close(C[t], A[t].double() @ b, A[t].double().abs() @ b.abs(), K, BF)
    D = torch.ones(rows, N, dtype=BF, device="cuda")
    _, dB = ozk.grouped_matmul_backward(D, A, B, offsets)
    want = torch.stack((A[0].double(), A[at[1:]].double().sum(0)))[:, :, None].expand(2, K, N)
    _close(dB, want, want.abs() + 12, 8, BF)


# ---------------------------------------------------------------------------
# 4-bit weights
# ---------------------------------------------------------------------------

def _reference_quantize(W, group, zeros):
    """The format by its definition, in fp32 as stated: q, s, z."""
    W = W.float().cpu().nan_to_num(nan=0.0, posinf=math.inf, neginf=-math.inf)
    N, K = W.shape
    q, s, z = torch.zeros(N, K), [], []
    for lo in range(0, K, group):
        w = W[:, lo:lo + group]
        hi_, lo_ = w.amax(1).clamp(min=0), w.amin(1).clamp(max=0)
        s.append((hi_ - lo_) * (1 / 15) if zeros else torch.maximum(hi_, -lo_) * (1 / 7))
    return W, torch.stack(s, 1)


def _unpack(packed, K):
    p = packed.cpu().long()
    return torch.stack((p & 15, p >> 4), -1).flatten(1)[:, :K]


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("N, K, group", [(1, 1, 32), (3, 31, 32), (5, 33, 64), (64, 256, 128),
                                         (7, 1000, 128), (65, 513, 32), (2, 2047, 64)])
def test_quantize(dtype, zeros, N, K, group):
    W = _randn(1, N, K, dtype=dtype)
    W[0, :min(K, group)] = 0                                  # a group of zeros
    if N > 1:
        W[1] = W[1].abs()                                     # one side of zero
    packed, scales, z = ozk.quantize_w4(W, group, zeros=zeros)
    assert packed.shape == (N, (K + 31) // 32 * 16) and scales.dtype == dtype
    assert (z is None) == (not zeros)
    Wf, s = _reference_quantize(W, group, zeros)
    s = s.to(dtype).float()
    assert torch.equal(scales.cpu().float(), s)
    wide = lambda t: t.repeat_interleave(group, 1)[:, :K]  # noqa: E731
    q = _unpack(packed, K)
    zf = wide(z.cpu().float()) if zeros else torch.full((N, K), 8.0)
    # within half a step of the weight (and its rounding), or at an end of the range
    value, step = (q - zf) * wide(s), wide(s)
    off = (value - Wf).abs()
    ends = (q == 0) | (q == 15)
    assert bool(((off <= step * 0.5001) | ends).all())
    # the ends are at most a whole step away: the scale's and zero point's rounding
    assert bool((off <= step * 1.01 + 2.0 ** -24).all())
    assert bool((q[wide(s) == 0] == zf[wide(s) == 0]).all())
    back = ozk.dequantize_w4(packed, scales, z, group_size=group, K=K)
    assert torch.equal(back.cpu(), value.to(dtype))


def test_quantize_special_values():
    W = _randn(1, 4, 64, dtype=F32)
    W[1, 3], W[2, :32] = math.nan, math.nan
    packed, scales, _ = ozk.quantize_w4(W, 32)
    q = _unpack(packed, 64)
    assert q[1, 3] == 8 and bool((q[2, :32] == 8).all()) and scales[2, 0] == 0
    clean = W.nan_to_num(nan=0.0)
    assert all(torch.equal(x, y) for x, y in zip(ozk.quantize_w4(clean, 32)[:2], (packed, scales)))
    tiny = torch.full((1, 32), 1e-45, device="cuda")           # the scale is a subnormal, or zero
    p, s, z = ozk.quantize_w4(tiny, 32, zeros=True)
    assert torch.isfinite(ozk.dequantize_w4(p, s, z, group_size=32)).all()
    big = torch.full((1, 32), 3e38, device="cuda")
    assert torch.isfinite(ozk.dequantize_w4(*ozk.quantize_w4(big, 32), group_size=32)).all()
    assert ozk.quantize_w4(W[:0], 32)[0].shape == (0, 32)


def test_quantize_reads_strided_weights():
    W = _randn(1, 96, 200)
    for w in (W[:, 1:101], W[::2, :64], W.T):
        for a, b in zip(ozk.quantize_w4(w, 32, zeros=True), ozk.quantize_w4(w.contiguous(), 32, zeros=True)):
            assert torch.equal(a, b)


def _random_w4(seed, N, K, group, dtype, zeros):
    g, groups = _gen(seed), -(-K // group)
    packed = torch.randint(0, 256, (N, (K + 31) // 32 * 16), generator=g, device="cuda").to(torch.uint8)
    scales = (torch.rand(N, groups, generator=g, device="cuda") + 0.1).to(dtype) / 16
    z = torch.randint(0, 16, (N, groups), generator=g, device="cuda").to(torch.uint8) if zeros else None
    return packed, scales, z


def _check_w4(x, packed, scales, z, group, rows=None):
    y = ozk.matmul_w4(x, packed, scales, z, group_size=group)
    K = x.shape[-1]
    assert y.dtype == x.dtype and y.shape == (*x.shape[:-1], packed.shape[0])
    keep = slice(None) if rows is None else rows
    wide = lambda t: t[keep].double().cpu().repeat_interleave(group, 1)[:, :K]  # noqa: E731
    q, zf = _unpack(packed[keep], K).double(), 8.0 if z is None else wide(z)
    x2 = x.reshape(-1, K).double().cpu()
    # the two sums that are formed: (16 + q) x and (16 + z) x
    _close(y.reshape(-1, packed.shape[0])[:, keep].cpu(), x2 @ ((q - zf) * wide(scales)).T,
           x2.abs() @ ((32 + q + zf) * wide(scales)).T, K + 32, x.dtype)
    return y


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M, N, K, zeros", [
    (1, 1, 1, True), (1, 16, 32, False), (1, 17, 129, True), (2, 300, 1000, False),
    (4, 64, 2047, True), (5, 100, 96, True), (16, 129, 4100, False), (17, 65, 513, True),
    (32, 200, 1024, False), (33, 64, 640, True), (64, 130, 2048, False), (65, 70, 300, True),
    (150, 48, 257, False), (3, 2, 16384, True), (40, 40, 8191, False),
])
def test_w4(dtype, group, M, N, K, zeros):
    _check_w4(_randn(1, M, K, dtype=dtype), *_random_w4(2, N, K, group, dtype, zeros), group)


def test_w4_full_precision_activations():
    """fp32 x loses nothing to its slices: as near as plain fp32 products."""
    x, (p, s, z) = _randn(1, 6, 4096, dtype=F32), _random_w4(2, 512, 4096, 128, F32, True)
    W = ozk.dequantize_w4(p, s, z, group_size=128)
    want = x.double() @ W.double().T
    off = lambda y: float((y.double() - want).norm() / want.norm())  # noqa: E731
    assert off(ozk.matmul_w4(x, p, s, z, group_size=128)) <= 4 * max(off(x @ W.T), 2.0 ** -24)


def test_w4_scales_of_32_bits_and_layouts():
    x, (p, s, z) = _randn(1, 3, 200), _random_w4(2, 50, 200, 32, F32, True)
    want = _check_w4(x, p, s, z, 32)
    wide = torch.zeros(50, 200, dtype=torch.uint8, device="cuda")
    wide[:, 16:16 + p.shape[1]] = p
    for packed in (wide[:, 16:16 + p.shape[1]], wide[:, 16:], p.T.contiguous().T):
        assert torch.equal(ozk.matmul_w4(x, packed, s, z, group_size=32), want)
    assert torch.equal(ozk.matmul_w4(x, p, s.T.contiguous().T, z.T.contiguous().T, group_size=32), want)
    xs = torch.zeros(3, 401, dtype=BF, device="cuda")
    xs[:, 1:401:2] = x
    assert torch.equal(ozk.matmul_w4(xs[:, 1:401:2], p, s, z, group_size=32), want)
    xs[:, 3:203] = x
    assert torch.equal(ozk.matmul_w4(xs[:, 3:203], p, s, z, group_size=32), want)
    assert torch.equal(ozk.matmul_w4(x.view(3, 1, 200), p, s, z, group_size=32), want.view(3, 1, 50))
    assert torch.equal(ozk.matmul_w4(x[0], p, s, z, group_size=32), want[0])
    assert ozk.matmul_w4(x[:0], p, s, z, group_size=32).shape == (0, 50)
    assert ozk.matmul_w4(x, p[:0], s[:0], z[:0], group_size=32).shape == (3, 0)


def test_w4_rows_do_not_leak():
    x, (p, s, z) = _randn(1, 20, 512), _random_w4(2, 100, 512, 64, BF, True)
    want = ozk.matmul_w4(x, p, s, z, group_size=64)
    x[3, 100], x[17, 5] = math.nan, math.inf
    s[40, 2] = math.nan
    got = ozk.matmul_w4(x, p, s, z, group_size=64)
    assert got[3].isnan().all() and got[17].isnan().all() and got[:, 40].isnan().all()
    keep = [m for m in range(20) if m not in (3, 17)]
    cols = [n for n in range(100) if n != 40]
    assert torch.equal(got[keep][:, cols], want[keep][:, cols])
    # what lies past K in the last bytes of a row is not read into the result
    x, (p, s, z) = _randn(1, 2, 40), _random_w4(2, 30, 40, 32, BF, True)
    want = ozk.matmul_w4(x, p, s, z, group_size=32)
    p[:, 20:] = 255
    assert torch.equal(ozk.matmul_w4(x, p, s, z, group_size=32), want)


def test_w4_packed_past_4_gib():
    N, K = 1 << 16, 1 << 17
    packed = torch.zeros(N, K // 2, dtype=torch.uint8, device="cuda")
    rows = torch.tensor([0, N // 2, N - 1], device="cuda")
    p, s, z = _random_w4(2, 3, K, 128, BF, True)
    packed[rows] = p
    scales = torch.ones(N, K // 128, dtype=BF, device="cuda")
    zeros = torch.zeros(N, K // 128, dtype=torch.uint8, device="cuda")
    scales[rows], zeros[rows] = s, z
    _check_w4(_randn(1, 2, K), packed, scales, zeros, 128, rows.cpu())


def test_w4_has_no_gradient():
    p, s, z = _random_w4(2, 30, 64, 32, BF, True)
    x = _randn(1, 2, 64).requires_grad_()
    with pytest.raises(RuntimeError):
        ozk.matmul_w4(x, p, s, z, group_size=32)
    with torch.no_grad():
        assert not ozk.matmul_w4(x, p, s, z, group_size=32).requires_grad


def test_w4_on_its_stream_and_in_a_graph():
    x, w = _randn(1, 2, 16384), _random_w4(2, 64, 16384, 128, BF, True)   # K is cut
    want = ozk.matmul_w4(x, *w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ozk.matmul_w4(x, *w)
    for n in range(3):
        x.copy_(_randn(5 + n, 2, 16384))
        want = ozk.matmul_w4(x, *w)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ozk.matmul_w4(x, *w)
    side.synchronize()
    assert torch.equal(got, want)


# ---------------------------------------------------------------------------
# orthogonalisation
# ---------------------------------------------------------------------------

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _steps(G, triples, eps, dtype):
    X = G.to(dtype)
    flip = X.shape[-2] > X.shape[-1]
    if flip:
        X = X.mT.contiguous()
    norm = X.double().square().sum((-2, -1), keepdim=True).sqrt() + eps
    X = (X.double() / norm).to(dtype)
    for a, b, c in triples:
        A = X @ X.mT.contiguous()
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.mT if flip else X


def _check_orth(G, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    triples = [coefficients] * steps if isinstance(coefficients[0], float) else coefficients
    got = ozk.orthogonalize(G, steps, coefficients, eps)
    assert got.dtype == G.dtype and got.shape == G.shape
    g = G.cpu()
    want = _steps(g.double(), triples, eps, torch.float64)
    plain = _steps(g.float(), triples, eps, F32)
    off = lambda y: float((y.double() - want).norm() / want.norm())  # noqa: E731
    rounding = 0.0 if G.dtype == F32 else ROUND[G.dtype]
    # half a unit of fp32 is the least that a plain computation is off
    assert off(got.cpu()) <= 4 * max(off(plain), 2.0 ** -24) + rounding, (off(got.cpu()), off(plain))
    return got


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (7, 1), (31, 33), (64, 64), (65, 40), (100, 200),
                                   (200, 100), (128, 1000), (257, 130), (3, 64, 96), (2, 3, 40, 24),
                                   (300, 520), (520, 300)])
def test_orthogonalize(dtype, shape):
    _check_orth(_randn(1, *shape, dtype=dtype))


@pytest.mark.parametrize("steps, coefficients", [
    (1, COEFFICIENTS), (2, COEFFICIENTS), (10, (1.875, -1.25, 0.375)), (3, (1.5, -0.5, 0.0)),
    (3, [(3.4445, -4.7750, 2.0315), (2.5, -3.0, 1.5), (1.875, -1.25, 0.375)]),
    (2, (40.0, -30.0, 10.0)),                     # leaves the unit interval: the scales follow
])
def test_orthogonalize_steps(steps, coefficients):
    _check_orth(_randn(2, 96, 160, dtype=F32), steps, coefficients)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
@pytest.mark.parametrize("shape, steps, coefficients", [
    ((64, 200), 5, COEFFICIENTS), ((300, 64), 6, COEFFICIENTS), ((3, 40, 130), 2, COEFFICIENTS),
    ((100, 1000), 8, (1.875, -1.25, 0.375)), ((65, 400), 4, (1.5, -0.5, 0.0)),
    ((33, 100), 3, [(3.4445, -4.7750, 2.0315), (2.5, -3.0, 1.5), (1.875, -1.25, 0.375)])])
def test_orthogonalize_long(dtype, shape, steps, coefficients):
    """Matrices three times longer than high and more: the last steps run on the
    square matrices alone, as many as the dtype's precision bears."""
    _check_orth(_randn(7, *shape, dtype=dtype), steps, coefficients)


def test_orthogonalize_long_of_any_condition():
    """Singular values over four decades, and a matrix of rank 3."""
    g = _gen(8)
    u, v = (torch.linalg.qr(torch.randn(n, 48, generator=g, device="cuda"))[0] for n in (48, 200))
    G = u @ torch.diag(torch.logspace(0, -4, 48, device="cuda")) @ v.T
    low = _randn(5, 40, 3, dtype=F32) @ _randn(6, 3, 160, dtype=F32)
    for dtype in (BF, F16):
        # the values that bfloat16 has of G are other ones: compare on those
        for m in (G, low):
            x = m.to(dtype)
            got, want = ozk.orthogonalize(x).double(), _steps(x.cpu().double(), [COEFFICIENTS] * 5, 1e-7, torch.float64)
            off = float((got.cpu() - want).norm() / want.norm())
            # half a unit for the rounding, half a unit for the steps
            assert off <= 2 * ROUND[dtype], (dtype, off)


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e25])
def test_orthogonalize_scale(scale):
    """Gradients of any size: the squares are summed in 64 bits."""
    _check_orth(_randn(3, 64, 80, dtype=F32) * scale, eps=0.0)


def test_orthogonalize_singular_values():
    """Converged steps give orthonormal rows; a matrix of low rank keeps its rank."""
    G = _randn(4, 48, 200, dtype=F32)
    X = ozk.orthogonalize(G, 30, (1.875, -1.25, 0.375)).double()
    assert float((X @ X.T - torch.eye(48, device="cuda")).abs().max()) < 1e-5
    low = _randn(5, 64, 3, dtype=F32) @ _randn(6, 3, 90, dtype=F32)
    s = torch.linalg.svdvals(_check_orth(low).double().cpu())
    assert 0.6 < float(s[2]) and float(s[0]) < 1.3 and float(s[3]) < 1e-3


def test_orthogonalize_special_values():
    G = _randn(1, 4, 64, 48, dtype=F32)
    G[1] = 0
    G[2, 5, 6], G[3, 0, 0] = math.nan, math.inf
    X = ozk.orthogonalize(G)
    assert torch.equal(X[0], ozk.orthogonalize(G[0])) and not X[1].any()
    assert X[2].isnan().all() and not torch.isfinite(X[3]).any()
    assert ozk.orthogonalize(G[:, :0]).shape == (4, 0, 48)
    assert ozk.orthogonalize(G[:0]).shape == (0, 64, 48)


def test_orthogonalize_strides():
    wide = _randn(1, 2, 90, 300, dtype=F32)
    for G in (wide[:, ::2, 1:78], wide.mT[:, 3:60], wide[:1].expand(2, 90, 300)):
        assert torch.equal(ozk.orthogonalize(G), ozk.orthogonalize(G.contiguous()))


def test_orthogonalize_large_tiles():
    """Sizes that take the largest tiles, with ragged edges, and a long batch."""
    _check_orth(_randn(1, 1100, 2500, dtype=BF), 2)
    _check_orth(_randn(1, 40, 200, 232, dtype=F32), 2)


@pytest.mark.parametrize("shape, steps", [((2000, 2100), 2), ((4100, 4100), 1), ((16, 333, 700), 3),
                                          ((700, 1500), 4)])
def test_orthogonalize_every_square_tile(shape, steps):
    """Symmetric products in tiles of 96 and 256, with ragged edges, and a chain of
    products on a matrix twice as long as high."""
    G = _randn(1, *shape, dtype=BF)
    got = ozk.orthogonalize(G, steps)
    for g, y in zip(G.view(-1, *shape[-2:]), got.view(-1, *shape[-2:])):
        want = _steps(g.double(), [COEFFICIENTS] * steps, 1e-7, torch.float64)
        plain = _steps(g.float(), [COEFFICIENTS] * steps, 1e-7, F32)
        off = lambda t: float((t.double() - want).norm() / want.norm())  # noqa: E731
        assert off(y) <= 4 * max(off(plain), 2.0 ** -24) + ROUND[BF]


def test_orthogonalize_in_a_graph():
    G = _randn(1, 2, 100, 160)
    graph = torch.cuda.CUDAGraph()
    ozk.orthogonalize(G)
    with torch.cuda.graph(graph):
        got = ozk.orthogonalize(G)
    for n in range(3):
        G.copy_(_randn(2 + n, 2, 100, 160))
        want = ozk.orthogonalize(G)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ozk.orthogonalize(G)
    side.synchronize()
    assert torch.equal(got, want)
