"""gradient_norm and clip_gradients against sums in 64 bits.  Each rounding is off by
at most half a step, relative: 2^-24 (fp32), finfo.eps / 2."""
import math

import pytest
import torch

import ozaki_triton_amd as ozk

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def _norm(tensors):
    return math.sqrt(sum(float(t.double().square().sum()) for t in tensors))


def _tensors(sizes, dtypes, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [((0.1 + i % 3) * torch.randn(s, generator=g, device="cuda")).to(dtypes[i % len(dtypes)])
            for i, s in enumerate(sizes)]


def _check(before, after, limit, norm):
    want = _norm(before)
    assert norm.shape == () and norm.dtype == F32
    # the sums in 64 bits: n 2^-53 of them at most
    assert abs(float(norm) - want) <= 2 * U * want
    by = min(1.0, limit / want) if want else 1.0
    for b, a in zip(before, after):
        assert a.dtype == b.dtype and a.shape == b.shape
        exact = b.double() * by
        info = torch.finfo(b.dtype)
        # fp32: one rounding, by in 64 bits; 16 bits: by, the product and the result
        tol = exact.abs() * (info.eps / 2 + (2.1 * U if b.dtype != F32 else 2.0 ** -45)) + info.tiny * info.eps / 2
        assert bool(((a.double() - exact).abs() <= tol).all())


SIZES = [[1], [0], [7, 0, 3], [64], [2047, 2048, 2049], [100000], [1 << 20, 1024, 5, 1 << 16],
         [s * 37 % 5000 for s in range(130)], [3] * 300, [(3, 5, 7), (16, 16), ()], [3000000, 11]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("dtypes", [[F32], [BF], [F16], [BF, F32, F16]], ids=["f32", "bf16", "f16", "mixed"])
def test_norm_and_clip(gpu, sizes, dtypes):
    grads = _tensors(sizes, dtypes)
    want = _norm(grads)
    norm = ozk.gradient_norm(grads)
    assert abs(float(norm) - want) <= 2 * U * want
    for part in (0.3, 1.5):
        limit = part * want
        work = [t.clone() for t in grads]
        _check(grads, work, limit, ozk.clip_gradients(work, limit)) if part > 1 else None
        if part < 1:
            got = ozk.clip_gradients(work, limit)
            _check(grads, work, limit, got)
        else:
            assert all(torch.equal(a, b) for a, b in zip(work, grads))
        out = [torch.full_like(t, 9.0) for t in grads]
        keep = [t.clone() for t in grads]
        _check(grads, out, limit, ozk.clip_gradients(grads, limit, out=out))
        assert all(torch.equal(a, b) for a, b in zip(keep, grads))
        assert all(torch.equal(a, b) for a, b in zip(out, work))


def test_range(gpu):
    """Squares past fp32's range at both ends."""
    for value in (1e-30, 2.0 ** -149, 1e20, 3e38):
        t = [torch.full((1000,), value, device="cuda"), torch.full((24,), value, device="cuda")]
        want = _norm(t)
        norm = float(ozk.gradient_norm(t))
        if want > 3.4028235e38:
            assert norm == math.inf
        else:
            # a subnormal norm is rounded to whole steps of 2^-149
            assert abs(norm - want) <= 2 * U * want + 2.0 ** -150
        work = [a.clone() for a in t]
        ozk.clip_gradients(work, want / 1024)
        for a, b in zip(work, t):
            exact = b.double() / 1024
            assert bool(((a.double() - exact).abs() <= 2 * U * exact + 2.0 ** -150).all())
    big = [torch.full((64,), 1e4, device="cuda", dtype=F16), torch.full((9,), 1e38, device="cuda", dtype=BF)]
    assert abs(float(ozk.gradient_norm(big)) / _norm(big) - 1) <= 2 * U


def test_factors_below_32_bits(gpu):
    """max_norm over the norm below fp32's least: results that are ordinary values."""
    for dtype, value, limit in ((BF, 3e38, 1e-5), (BF, 1e30, 1e-20), (F32, 3e38, 1e-30)):
        t = [torch.full((n,), value, device="cuda").to(dtype) for n in (3000, 13)]
        want = [a.double() * (limit / _norm(t)) for a in t]
        ozk.clip_gradients(t, limit)
        for a, w in zip(t, want):
            # one rounding to the type, those of the factor and of 32 bits far below it
            u = torch.finfo(dtype).eps / 2
            assert bool(((a.double() - w).abs() <= (u + 4 * U) * w).all())


def test_infinite_nan_and_zero(gpu):
    inf, nan = float("inf"), float("nan")
    for bad in (inf, -inf):
        t = [torch.ones(5000, device="cuda"), torch.tensor([1.0, bad], device="cuda", dtype=BF)]
        norm = ozk.clip_gradients(t, 1.0)
        assert float(norm) == inf
        assert not t[0].any() and t[1][0] == 0 and torch.isnan(t[1][1])
    t = [torch.ones(5000, device="cuda"), torch.tensor([1.0, nan], device="cuda", dtype=F16)]
    assert math.isnan(float(ozk.clip_gradients(t, 1.0)))
    assert all(bool(torch.isnan(x).all()) for x in t)
    t = [torch.zeros(5000, device="cuda"), torch.zeros(3, device="cuda", dtype=BF)]
    assert float(ozk.clip_gradients(t, 0.0)) == 0.0 and not any(x.any() for x in t)
    t = [torch.ones(50, device="cuda")]
    ozk.clip_gradients(t, inf)
    assert bool((t[0] == 1).all())
    ozk.clip_gradients(t, 0.0)
    assert not t[0].any()


def test_layouts(gpu):
    """Tensors with gaps, permuted and misaligned ones; elements beside them stay."""
    base = torch.randn(64, 48, device="cuda")
    keep = base.clone()
    views = [base[:30, :20], base[:30, 20:47], base[40:].mT, base[31:39, ::2]]
    half = torch.randn(1001, device="cuda").to(BF)
    odd = half[1:]
    before = [v.clone() for v in views] + [odd.clone()]
    norm = ozk.gradient_norm(views + [odd])
    assert abs(float(norm) - _norm(before)) <= 2 * U * _norm(before)
    first = half[0].clone()
    got = ozk.clip_gradients(views + [odd], 1.0)
    _check(before, views + [odd], 1.0, got)
    assert half[0] == first
    touched = torch.zeros_like(base, dtype=torch.bool)
    for v in (touched[:30, :20], touched[:30, 20:47], touched[40:], touched[31:39, ::2]):
        v.fill_(True)
    assert torch.equal(base[~touched], keep[~touched])
    # results laid out otherwise
    g = [torch.randn(50, 70, device="cuda"), torch.randn(8, 9, device="cuda").mT]
    out = [torch.zeros(70, 50, device="cuda").mT, torch.zeros(9, 8, device="cuda")]
    _check(g, out, 2.0, ozk.clip_gradients(g, 2.0, out=out))


def test_refusals_on_the_gpu(gpu):
    t = torch.ones(100, device="cuda")
    for bad in ([t, t], [t, t[50:]], [t[:60], t[50:]]):
        with pytest.raises(AssertionError):
            ozk.clip_gradients(bad, 1.0)
    assert bool((t == 1).all())
    assert abs(float(ozk.gradient_norm([t, t])) - math.sqrt(200)) < 1e-5
    with pytest.raises(AssertionError):
        ozk.clip_gradients([t[:1].expand(5)], 1.0)
    gaps = torch.ones(10, 10, device="cuda")
    with pytest.raises(AssertionError):
        ozk.clip_gradients([gaps[:, ::2], gaps[:, ::2]], 1.0)
    assert bool((gaps == 1).all())
    with pytest.raises(AssertionError):
        ozk.clip_gradients([t], 1.0, out=[t, t])
    with pytest.raises(AssertionError):
        ozk.clip_gradients([t], 1.0, out=[t[:50]])
    with pytest.raises(AssertionError):
        ozk.clip_gradients([t], -1.0)
    with pytest.raises(NotImplementedError):
        ozk.clip_gradients([t.double()], 1.0)
    with pytest.raises(RuntimeError):
        ozk.clip_gradients([t, torch.ones(3)], 1.0)
    with pytest.raises(RuntimeError):
        ozk.gradient_norm([t.clone().requires_grad_()])
    # autograd is told that a saved tensor has changed
    a, w = t.clone(), t.clone().requires_grad_()
    y = (a * w).sum()
    ozk.clip_gradients([a], 1.0)
    with pytest.raises(RuntimeError):
        y.backward()


def test_same_bits_every_time_and_on_any_stream(gpu):
    grads = _tensors([1 << 18, 333, 1 << 16, 5], [BF, F32])
    first, out0 = ozk.gradient_norm(grads), [torch.empty_like(t) for t in grads]
    ozk.clip_gradients(grads, 3.0, out=out0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            out = [torch.empty_like(t) for t in grads]
            got.append((ozk.clip_gradients(grads, 3.0, out=out), out))
    torch.cuda.synchronize()
    for norm, out in got:
        assert torch.equal(norm, first) and all(torch.equal(a, b) for a, b in zip(out, out0))


def test_captured(gpu):
    grads = _tensors([5000, 77, 1 << 16], [BF, F32, F16])
    ozk.clip_gradients([t.clone() for t in grads], 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ozk.clip_gradients(grads, 2.0)
    for seed in range(4):
        new = _tensors([5000, 77, 1 << 16], [BF, F32, F16], seed=seed)
        for t, n in zip(grads, new):
            t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        want = ozk.clip_gradients(new, 2.0)
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(grads, new))


def test_past_32_bits(gpu):
    """More than 2^32 bytes and 2^31 elements in one tensor."""
    n = (1 << 31) + 12345
    t = torch.zeros(n, device="cuda", dtype=BF)
    t[-1], t[0], t[n // 2] = 3.0, 4.0, 12.0
    assert float(ozk.gradient_norm([t])) == 13.0
    ozk.clip_gradients([t], 6.5)
    assert [float(t[i]) for i in (n - 1, 0, n // 2)] == [1.5, 2.0, 6.0]


def test_parameters_gradients_in_place(gpu):
    """As a training loop calls it: the .grad of parameters, the parameters' own flags unchanged."""
    ps = [torch.randn(40, 30, device="cuda").to(BF).requires_grad_(), torch.randn(30, device="cuda", requires_grad=True)]
    sum(p.float().square().sum() for p in ps).backward()
    before = [p.grad.clone() for p in ps]
    norm = ozk.clip_gradients((p.grad for p in ps), 1.0)      # any iterable
    _check(before, [p.grad for p in ps], 1.0, norm)
    assert all(p.requires_grad and not p.grad.requires_grad for p in ps)
    with torch.inference_mode():
        t = [torch.ones(10, device="cuda")]
        ozk.clip_gradients(t, 1.0)
    assert abs(float(t[0].norm()) - 1) < 1e-6


def test_overlaps_of_tensors_with_gaps(gpu):
    """Refused like those of contiguous ones, before anything is written."""
    base = torch.ones(64, 48, device="cuda")
    for bad in ([base, base[:, ::2]], [base[:, :4], base[:, 2:6]], [base[:8], base[::2]],
                [base.as_strided((5, 5), (3, 2))]):
        with pytest.raises(AssertionError, match="share memory"):
            ozk.clip_gradients(bad, 1.0)
    g = [torch.ones(64, 4, device="cuda") for _ in range(2)]
    for out in ([base[:, :4], base[:, 2:6]], [base[:, 44:], base[:1, 44:].expand(64, 4)]):
        with pytest.raises(AssertionError, match="share memory"):
            ozk.clip_gradients(g, 1.0, out=out)
    assert bool((base == 1).all()) and all(bool((t == 1).all()) for t in g)
    # columns of one tensor, apart
    views = [base[:, i::3] for i in range(3)]
    before = [v.clone() for v in views]
    _check(before, views, 3.0, ozk.clip_gradients(views, 3.0))


def _split_cases(dtype, n):
    """Values and limits where a factor rounded to 32 bits first and one in 64 bits lead to
    neighbouring values of the dtype."""
    g = torch.Generator().manual_seed(3)
    v = (1 + torch.rand(1 << 20, generator=g)).to(dtype)
    limit = torch.rand(1 << 20, generator=g, dtype=torch.float64) * math.sqrt(n)
    by = limit / (math.sqrt(n) * v.double())
    mantissa, exponent = torch.frexp(by)
    first = torch.ldexp(v.float() * mantissa.float(), exponent).to(dtype)
    at = torch.nonzero(first != (v.double() * by).float().to(dtype))[:8, 0]
    assert len(at) >= 4
    return [(float(v[i]), float(limit[i])) for i in at]


@pytest.mark.parametrize("dtype", [BF, F16])
def test_equal_values_stay_equal(gpu, dtype):
    """Wherever they lie: a tensor's last elements are no 16 bytes."""
    n = 4099
    for value, limit in _split_cases(dtype, n):
        t = torch.full((n,), value, device="cuda").to(dtype)
        ozk.clip_gradients([t], limit)
        assert bool((t == t[0]).all()), (value, limit)


def test_norms_past_float32(gpu):
    """A norm that float32 holds as infinity scales by its value; an infinite limit changes nothing."""
    for dtype in (F32, BF):
        t = [torch.full((n,), 3e38, device="cuda").to(dtype) for n in (3000, 13)]
        before = [a.clone() for a in t]
        assert float(ozk.clip_gradients(t, 1.0)) == math.inf
        u = torch.finfo(dtype).eps / 2 + 4 * U
        for a, b in zip(t, before):
            want = b.double() / _norm(before)
            assert bool(((a.double() - want).abs() <= u * want).all())
        t = [torch.tensor([1.0, math.inf, -2.0], device="cuda").to(dtype)]
        before = [a.clone() for a in t]
        assert float(ozk.clip_gradients(t, math.inf)) == math.inf
        assert torch.equal(t[0], before[0])
