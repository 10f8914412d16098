"""fused_linear and its gradients against the formula in 64 bits.

u = 2^-24 is half a step of fp32, h half a step of the dtype, both relative.  A sum
of n products in fp32, in any order, is off by at most n u times the sum of their
sizes; activations by their slope (at most 1.13) times that and 2^-18 |z| of their
own (exp2's argument, the fitted tail); each rounding to the dtype by h."""
import ctypes
import math

import pytest
import torch

import ozaki_triton_amd as ozk
from ozaki_triton_amd import _lib

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16
U = 2.0 ** -24
ACTS = (None, "relu", "gelu", "gelu_tanh", "silu")


def _act(z, act):
    """act(z) and its derivative in 64 bits."""
    if act is None:
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        below = 0.5 * torch.erfc(z * -math.sqrt(0.5))   # (1 + erf loses the lower tail)
        return z * below, below + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    slope = math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * slope


def _half(dtype):
    return torch.finfo(dtype).eps / 2, torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def _inputs(M, N, K, dtype, seed=0, wt=False, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, W, b, res = scale * r(M, K), r(N, K) / math.sqrt(max(K, 1)), r(N), r(M, N)
    x, W, b, res, dy = (t.to(dtype) for t in (x, W, b, res, r(M, N)))
    return x, W.mT.contiguous().mT if wt else W, b, res, dy


def _check(y, x, W, b, res, act):
    K, (h, least) = x.shape[-1], _half(x.dtype)
    xd, Wd = x.double(), W.double().mT.contiguous()
    z, size = xd @ Wd, xd.abs() @ Wd.abs()
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    want, _ = _act(z, act)
    tol = 1.13 * (K + 4) * U * size + 2 ** -18 * z.abs()
    if res is not None:
        want = want + res.double()
    tol = tol + (h + 2 * U) * (want.abs() + tol) + least
    if res is not None:
        tol = tol + U * res.double().abs()
    off = (y.double() - want).abs()
    assert y.shape == want.shape and y.dtype == x.dtype
    assert bool((off <= tol).all()), float((off / tol).max())


SHAPES = [
    (1, 4096, 4096), (1, 1, 1), (1, 17, 100), (3, 1000, 2047), (16, 64, 512), (17, 250, 129), (31, 96, 8),
    (33, 512, 1000), (64, 40, 4100), (65, 128, 256), (100, 1, 72), (128, 256, 4096), (200, 72, 2056),
    (257, 300, 64), (500, 1030, 200), (1999, 520, 1000), (1024, 2048, 1024), (4096, 4100, 136),
    (700, 333, 1001), (90, 90, 4097), (2, 60, 4097), (20, 48, 1025), (9, 50, 2049), (32, 33, 4159), (2300, 8, 3000), (70, 2000, 7)]


@pytest.mark.parametrize("M, N, K", SHAPES)
@pytest.mark.parametrize("wt", [False, True])
def test_products(gpu, M, N, K, wt):
    for dtype in (BF, F16):
        x, W, b, res, _ = _inputs(M, N, K, dtype, seed=M + N, wt=wt)
        _check(ozk.fused_linear(x, W), x, W, None, None, None)
        act = ACTS[(M + N + K) % 5]
        y = ozk.fused_linear(x, W, b, activation=act, residual=res)
        _check(y, x, W, b, res, act)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M, N, K", [(2, 300, 64), (150, 200, 96), (130, 64, 8192), (8192, 2050, 64)])
def test_epilogues(gpu, M, N, K, act):
    for dtype in (BF, F16):
        x, W, b, res, _ = _inputs(M, N, K, dtype, seed=1, scale=3.0)
        for bias in (None, b):
            for residual in (None, res):
                y = ozk.fused_linear(x, W, bias, activation=act, residual=residual)
                _check(y, x, W, bias, residual, act)


@pytest.mark.parametrize("act", ACTS)
def test_activations_over_their_range(gpu, act):
    """x W^T = x where W is one column of 1: the activation alone, at every value."""
    for dtype in (BF, F16):
        bits = torch.arange(-32768, 32768, dtype=torch.int32, device="cuda").to(torch.int16)
        x = bits.view(dtype)
        x = x[torch.isfinite(x)][:, None].contiguous()
        one = torch.ones(1, 1, dtype=dtype, device="cuda")
        h, least = _half(dtype)
        for rows in (x, x[:50], x[-50:]):
            y = ozk.fused_linear(rows, one, activation=act).double()
            z = rows.double()
            want = z.clamp(min=0) if act == "relu" else _act(z, act)[0]
            if act == "gelu_tanh":     # tanh + 1 loses what is far below 0, in 64 bits from -8 on
                u = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
                want = z * torch.sigmoid(u)
            # relative, down to the values whose exponential the hardware flushes to 0
            tol = (h + 2 ** -16) * want.abs() + least + 2 ** -126 * z.abs().clamp(min=1)
            assert bool(((y - want).abs() <= tol).all()), (act, dtype, float(((y - want).abs() / tol).max()))


def test_infinities_and_nan(gpu):
    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[1.0], [inf], [-inf], [nan]], device="cuda", dtype=BF)
    for M in (4, 200):
        rows = x if M == 4 else x.repeat(50, 1)
        one = torch.ones(1, 1, dtype=BF, device="cuda")
        for act in ACTS:
            y = ozk.fused_linear(rows, one, activation=act)[:4, 0].float()
            assert y[1] == inf and y[3] != y[3]
            assert y[2] == (-inf if act is None else 0.0) or (act in ("gelu", "gelu_tanh", "silu") and y[2] != y[2])
        # a row's infinity stays in its row
        a, W, b, _, _ = _inputs(M, 100, 72, BF)
        clean = ozk.fused_linear(a, W, b, activation="gelu")
        a[1, 3] = nan
        y = ozk.fused_linear(a, W, b, activation="gelu")
        assert bool(torch.isnan(y[1]).all())
        keep = torch.arange(M, device="cuda") != 1
        assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("M, N, K", [(5, 70, 300), (64, 33, 65), (300, 200, 136), (260, 515, 520), (100, 64, 2048)])
def test_whole_numbers_are_exact(gpu, M, N, K):
    """Small whole numbers: every sum is exact, so is every gradient, in any order."""
    g = torch.Generator(device="cuda").manual_seed(3)
    draw = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device="cuda").to(F16)  # noqa: E731
    keep = (torch.rand(M, K, generator=g, device="cuda") < 0.2).to(F16)
    x, W, b = draw(-2, 3, M, K) * keep, draw(-1, 2, N, K), draw(-3, 4, N)
    res, dy = draw(-5, 6, M, N), draw(-1, 2, M, N)
    for wt in (False, True):
        leaves = [t.clone().requires_grad_() for t in (x, W.mT.contiguous().mT if wt else W, b, res)]
        y = ozk.fused_linear(leaves[0], leaves[1], leaves[2], activation="relu", residual=leaves[3])
        grads = torch.autograd.grad(y, leaves, dy)
        z = x.double() @ W.double().mT.contiguous() + b.double()
        dz = dy.double() * (z > 0)
        assert torch.equal(y.double(), z.clamp(min=0) + res.double())
        for got, want in zip(grads, (dz @ W.double(), dz.mT.contiguous() @ x.double(), dz.sum(0), dy.double())):
            assert torch.equal(got.double(), want)


@pytest.mark.parametrize("M, N, K", [(1, 100, 64), (16, 333, 200), (40, 512, 1000), (300, 72, 2056), (1999, 520, 1000),
                                     (1024, 1024, 512), (129, 1001, 130), (3000, 136, 72), (90, 2, 3)])
@pytest.mark.parametrize("act", ACTS)
def test_gradients(gpu, M, N, K, act):
    for dtype in (BF, F16):
        x, W, b, res, dy = _inputs(M, N, K, dtype, seed=K, wt=(M + N) % 2 == 1)
        leaves = [t.requires_grad_() for t in (x, W, b, res)]
        y = ozk.fused_linear(x, W, b, activation=act, residual=res)
        dx, dW, db, dres = torch.autograd.grad(y, leaves, dy)
        x, W, b, res = (t.detach() for t in leaves)
        _check(y.detach(), x, W, b, res, act)
        assert torch.equal(dres, dy)
        h, least = _half(dtype)
        z = x.double() @ W.double().mT.contiguous() + b.double()
        dz = dy.double() * _act(z, act)[1]
        if act == "relu":
            # next to 0 either side is right: leave those rows and columns out
            near = z.abs() < (K + 4) * U * (x.double().abs() @ W.double().mT.contiguous().abs() + b.double().abs())
        else:
            near = torch.zeros_like(z, dtype=torch.bool)
        # z to h |z| moves the derivative by at most 0.8 of that; dz to h
        zero = 0.0 if act in (None, "relu") else 1.0
        e = dy.double().abs() * zero * (0.8 * (h * z.abs() + least + (K + 4) * U * 4) + 2 ** -17)
        e = e + (h * dz.abs() + least if act is not None else 0.0)
        Wa, xa = W.double().abs(), x.double().abs()
        size = dz.abs() + e
        for got, want, tol, skip in (
                (dx, dz @ W.double(), e @ Wa + (N + 2) * U * (size @ Wa), near.any(1)[:, None]),
                (dW, dz.mT.contiguous() @ x.double(), e.mT.contiguous() @ xa + (M + 2) * U * (size.mT.contiguous() @ xa),
                 near.any(0)[:, None]),
                (db, dz.sum(0), e.sum(0) + (M + 2) * U * size.sum(0), near.any(0))):
            tol = tol + (h + U) * (want.abs() + tol) + least
            off = (got.double() - want).abs()
            assert got.shape == want.shape and got.dtype == dtype
            assert bool(((off <= tol) | skip).all()), float((off / tol).max())
            # the roundings are as good as independent: far below their worst case together
            if act != "relu" and want.numel() > 1000:
                assert float((got.double() - want).norm()) <= 2 * h * float(want.norm())


def test_gradients_against_differences(gpu):
    """d/dt of <y(x + t dx), dy>, with y in 64 bits from the formula, not from its derivative."""
    M, N, K = 70, 90, 64
    for act in ACTS[2:]:
        x, W, b, _, dy = _inputs(M, N, K, F16, seed=5)
        leaves = [t.requires_grad_() for t in (x, W, b)]
        grads = torch.autograd.grad(ozk.fused_linear(x, W, b, activation=act), leaves, dy)
        vals = [t.detach().double() for t in leaves]
        g = torch.Generator(device="cuda").manual_seed(7)
        for i in range(3):
            d = torch.randn(vals[i].shape, generator=g, device="cuda", dtype=torch.float64)

            def at(t):
                v = [w + t * d if j == i else w for j, w in enumerate(vals)]
                return float((_act(v[0] @ v[1].mT.contiguous() + v[2], act)[0] * dy.double()).sum())
            slope = (at(1e-4) - at(-1e-4)) / 2e-4
            got = float((grads[i].double() * d).sum())
            # each of n gradients is off by about h times itself, with signs as they fall
            tol = 16 * 2.0 ** -11 * float((grads[i].double() * d).norm()) + 1e-6 * abs(slope)
            assert abs(got - slope) <= tol, (act, i, got, slope)


def test_only_what_is_wanted(gpu):
    x, W, b, res, dy = _inputs(150, 96, 72, BF)
    whole = None
    for need in ((1, 1, 1, 1), (1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (0, 1, 1, 0)):
        for act in (None, "silu"):
            ts = [t.clone().requires_grad_(bool(n)) for t, n in zip((x, W, b, res), need)]
            y = ozk.fused_linear(ts[0], ts[1], ts[2], activation=act, residual=ts[3])
            y.backward(dy)
            if all(need):
                whole = {**(whole or {}), act: [t.grad for t in ts]}
            for t, n, want in zip(ts, need, whole[act]):
                assert (t.grad is None) == (not n) and (not n or torch.equal(t.grad, want))
    with torch.no_grad():
        assert not ozk.fused_linear(x.clone().requires_grad_(), W).requires_grad


def test_layouts(gpu):
    """Rows with gaps, views, expanded and misaligned operands give the bits of copies."""
    base = torch.randn(400, 600, device="cuda").to(BF)
    flat = torch.randn(200 * 136 + 1, device="cuda").to(BF)
    b = torch.randn(400, device="cuda").to(BF)[::2]
    for M in (10, 200):
        xs = [base[:M, 8:144], base[:M, 3:139], base[:M, ::2][:, :136], base[:136, :M].mT,
              flat[1:1 + M * 136].view(M, 136), base[:1, :136].expand(M, 136)]
        Ws = [base[200:400, 16:152], base[200:400, 1:137], base[:136, 100:300].mT, base[:136, 101:301].mT,
              base[:272:2, ::3][:, :200].mT, base[:1, :136].expand(200, 136)]
        r = base[:M, 7:207]
        for x in xs:
            for W in Ws:
                y = ozk.fused_linear(x, W, b, activation="gelu", residual=r)
                _check(y, x, W, b, r, "gelu")
    # any number of dims
    x = base[:60, :136].reshape(3, 4, 5, 136)
    r = base[:60, :200].reshape(3, 4, 5, 200)
    y = ozk.fused_linear(x, Ws[0], b, residual=r)
    assert torch.equal(y.view(60, 200), ozk.fused_linear(x.reshape(60, 136), Ws[0], b, residual=r.reshape(60, 200)))
    assert ozk.fused_linear(x[0, 0, 0], Ws[0]).shape == (200,)
    # a gradient that comes expanded or with gaps
    for act in (None, "silu"):
        t = base[:100, :136].clone().requires_grad_()
        W = Ws[0].clone().requires_grad_()
        ozk.fused_linear(t, W, activation=act).sum().backward()
        ones = torch.ones(100, 200, device="cuda", dtype=BF)
        got = torch.autograd.grad(ozk.fused_linear(t, W, activation=act), (t, W), ones)
        assert torch.equal(t.grad, got[0]) and torch.equal(W.grad, got[1])
        dy = base[:100, 11:211]
        for a, c in zip(torch.autograd.grad(ozk.fused_linear(t, W, activation=act), (t, W), dy),
                        torch.autograd.grad(ozk.fused_linear(t, W, activation=act), (t, W), dy.contiguous())):
            assert float((a.double() - c.double()).norm()) <= 2.0 ** -8 * float(c.double().norm())


def test_empty(gpu):
    for M, N, K in ((0, 5, 7), (4, 0, 7), (4, 5, 0), (100, 5, 0), (0, 0, 0)):
        x, W, b, res, dy = _inputs(M, N, K, BF)
        leaves = [t.requires_grad_() for t in (x, W, b, res)]
        y = ozk.fused_linear(x, W, b, activation="gelu", residual=res)
        grads = torch.autograd.grad(y, leaves, dy)
        z = b.detach().double().expand(M, N)
        assert y.shape == (M, N)
        if M and N:
            want = _act(z, "gelu")[0] + res.detach().double()
            assert float((y.detach().double() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max()) + 1e-5
        assert [g.shape for g in grads] == [t.shape for t in leaves]
        if K == 0 and M and N:
            want = (dy.double() * _act(z, "gelu")[1]).sum(0)
            assert float((grads[2].double() - want).abs().max()) <= 2.0 ** -6 * float(want.abs().max())
        elif M == 0:
            assert not grads[1].any() and not grads[2].any()
        elif N == 0:
            assert not grads[0].any()
    x = torch.zeros(2, 0, 8, device="cuda", dtype=BF)
    assert ozk.fused_linear(x, torch.zeros(3, 8, device="cuda", dtype=BF)).shape == (2, 0, 3)


def test_relu_keeps_its_side(gpu):
    """Sums too small for the dtype have a derivative of 1 above 0 and of 0 below."""
    tiny = torch.full((80, 64), 2.0 ** -20, device="cuda", dtype=F16)
    for sign in (1.0, -1.0):
        W = torch.full((40, 64), sign * 2.0 ** -20, device="cuda", dtype=F16)
        x = tiny.clone().requires_grad_()
        b = torch.zeros(40, device="cuda", dtype=F16).requires_grad_()
        ozk.fused_linear(x, W, b, activation="relu").backward(torch.ones(80, 40, device="cuda", dtype=F16))
        assert bool((b.grad == (80 if sign > 0 else 0)).all())


def test_large_rows(gpu):
    """Rows that lie 2^22 elements and more apart are copied, those closer are read in place;
    byte offsets past 2^32."""
    flat = torch.randn((1 << 31) // 2 + 4096, device="cuda", dtype=BF)
    for M, pitch in ((300, 1 << 21), (250, (1 << 22) + 8), (40, (1 << 22) + 8)):
        x = flat.as_strided((M, 64), (pitch, 1))
        W = torch.randn(80, 64, device="cuda").to(BF)
        _check(ozk.fused_linear(x, W), x.contiguous(), W, None, None, None)
        _check(ozk.fused_linear(W, x), W, x.contiguous(), None, None, None)


def test_same_bits_every_time_and_on_any_stream(gpu):
    x, W, b, res, dy = _inputs(520, 300, 2048, BF)
    leaves = [t.requires_grad_() for t in (x, W, b)]

    def step():
        y = ozk.fused_linear(x, W, b, activation="gelu", residual=res)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    first = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            results.append(step())
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, c) for a, c in zip(r, first))


def test_captured(gpu):
    """A captured step of forward and backward, replayed on new values between eager calls."""
    x, W, b, res, dy = _inputs(200, 130, 264, BF)
    leaves = [t.requires_grad_() for t in (x, W, b)]

    def step():
        y = ozk.fused_linear(x, W, b, activation="silu", residual=res)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        with torch.no_grad():
            for t, n in zip((x, W, b, res, dy), _inputs(200, 130, 264, BF, seed=seed)):
                t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, c in zip(got, step()):
            assert torch.equal(a, c)


def test_refusals_on_the_gpu(gpu):
    x, W = torch.zeros(2, 8, device="cuda"), torch.zeros(3, 8, device="cuda")
    with pytest.raises(NotImplementedError):
        ozk.fused_linear(x, W)
    with pytest.raises(RuntimeError):
        ozk.fused_linear(x.to(BF), W.to(BF), torch.zeros(3, dtype=BF))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.to(BF), x.to(BF))
        with pytest.raises(RuntimeError):
            ozk.fused_linear(dual, W.to(BF))
    t = x.to(BF).requires_grad_()
    g, = torch.autograd.grad(ozk.fused_linear(t, W.to(BF)).sum(), t, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_gradients_without_a_bias(gpu):
    x, W, b, res, dy = _inputs(120, 96, 72, BF)
    for need in ((1, 1, 1), (0, 0, 1), (1, 0, 0), (0, 1, 1)):
        for act in (None, "gelu_tanh"):
            ts = [t.clone().requires_grad_(bool(n)) for t, n in zip((x, W, res), need)]
            ozk.fused_linear(ts[0], ts[1], activation=act, residual=ts[2]).backward(dy)
            zero = torch.zeros_like(b).requires_grad_()
            us = [t.clone().requires_grad_() for t in (x, W, res)]
            want = torch.autograd.grad(ozk.fused_linear(us[0], us[1], zero, activation=act, residual=us[2]), us, dy)
            for t, n, w in zip(ts, need, want):
                assert (t.grad is None) == (not n) and (not n or torch.equal(t.grad, w))


def test_backward_twice_and_recorded(gpu):
    """A kept graph gives the same gradients again; a recorded backward pass has their values and
    refuses a second derivative, in a sum with something that has one too."""
    x, W, b, _, dy = _inputs(120, 96, 72, BF)
    leaves = [t.requires_grad_() for t in (x, W, b)]
    y = ozk.fused_linear(x, W, b, activation="silu")
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    recorded = torch.autograd.grad(y, leaves, dy, create_graph=True)
    for a, c, d in zip(first, again, recorded):
        assert torch.equal(a, c) and torch.equal(a, d.detach())
    with pytest.raises(RuntimeError, match="twice"):
        (recorded[0].float().square().sum() + x.float().sum()).backward()
    # a saved operand that has changed meanwhile is noticed
    y = ozk.fused_linear(x, W, b, activation="silu")
    with torch.no_grad():
        W.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward(dy)


def test_inference_mode(gpu):
    x, W, b, res, _ = _inputs(70, 96, 72, BF)
    want = ozk.fused_linear(x, W, b, activation="gelu", residual=res)
    with torch.inference_mode():
        y = ozk.fused_linear(x, W.requires_grad_(), b, activation="gelu", residual=res)
    assert torch.equal(y, want) and not y.requires_grad


def test_saved_tensor_hooks(gpu):
    """Saved tensors that travel to the host and back; ones that come back as something else."""
    x, W, b, _, dy = _inputs(70, 96, 72, BF)
    leaves = [t.requires_grad_() for t in (x, W, b)]

    def grads():
        return torch.autograd.grad(ozk.fused_linear(x, W, b, activation="gelu"), leaves, dy)
    want = grads()
    with torch.autograd.graph.save_on_cpu():
        assert all(torch.equal(a, c) for a, c in zip(grads(), want))
    # same values, other strides
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.mT.contiguous().mT):
        for a, c in zip(grads(), want):
            assert bool(((a.double() - c.double()).abs() <= 2.0 ** -7 * c.double().abs() + 1e-2).all())
    for back in (lambda t: t.cpu(), lambda t: t[:1], lambda t: t.half(), lambda t: t[..., None]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
            with pytest.raises(RuntimeError, match="saved"):
                grads()


@pytest.mark.parametrize("M, N, K", [(1, 64, 64), (3, 70, 100), (4, 33, 4097), (20, 50, 1025), (33, 65, 72), (130, 200, 136),
                                     (300, 72, 2056), (64, 40, 99)])
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_nothing_beside_the_operands_counts(gpu, M, N, K, offset):
    """Operands inside tensors of NaN: neither results nor gradients have one."""
    def inside(rows, columns):
        big = torch.full((rows + 3, columns + 24), math.nan, device="cuda", dtype=BF)
        big[1:1 + rows, offset:offset + columns] = torch.randn(rows, columns, device="cuda").to(BF)
        return big[1:1 + rows, offset:offset + columns]
    for W in (inside(N, K), inside(K, N).mT):
        x, b, res = inside(M, K), inside(1, N)[0], inside(M, N)
        leaves = [t.detach().requires_grad_() for t in (x, W, b, res)]
        y = ozk.fused_linear(leaves[0], leaves[1], leaves[2], activation="gelu", residual=leaves[3])
        _check(y.detach(), x, W, b, res, "gelu")
        for g in torch.autograd.grad(y, leaves, inside(M, N)):
            assert bool(torch.isfinite(g).all())


def test_past_32_bits(gpu):
    """More than 2^31 results: the first, middle and last rows and columns, and their gradients."""
    M, N, K = 70000, 31000, 16
    x, W, b = (torch.randn(*s, device="cuda").to(BF) for s in ((M, K), (N, K), (N,)))
    dy = torch.randn(N, device="cuda").to(BF).expand(M, N)
    leaves = [t.requires_grad_() for t in (x, W, b)]
    y = ozk.fused_linear(x, W, b, activation="relu")
    for rows in (slice(0, 100), slice(34600, 34800), slice(M - 100, M)):
        _check(y[rows].detach(), x[rows].detach(), W.detach(), b.detach(), None, "relu")
    dx, dW, db = torch.autograd.grad(y, leaves, dy)
    last = slice(M - 50, M)
    dz = torch.where(y[last].detach() > 0, dy[last].double(), 0.0)   # relu's side as computed
    size = dz.abs() @ W.detach().double().abs()
    want = dz @ W.detach().double()
    assert bool(((dx[last].double() - want).abs() <= (1.13 * N * U + 2.0 ** -8) * size).all())
    columns = slice(N - 40, N)
    dz = torch.where(y[:, columns].detach() > 0, dy[:, columns].double(), 0.0).mT.contiguous()
    size = dz.abs() @ x.detach().double().abs()
    assert bool(((dW[columns].double() - dz @ x.detach().double()).abs() <= (1.13 * M * U + 2.0 ** -8) * size).all())
    assert bool(((db[columns].double() - dz.sum(1)).abs() <= (M * U + 2.0 ** -8) * dz.abs().sum(1)).all())


@pytest.mark.parametrize("M, N, K", [(33, 70, 1001), (40, 2500, 2861), (45, 7000, 2861), (64, 129, 515), (100, 60, 4097),
                                     (113, 33, 1810), (128, 1000, 999), (129, 1000, 999), (47, 90, 8191), (97, 1, 77)])
def test_rows_off_16_bytes(gpu, M, N, K):
    """Whole range of rows that are no 16-byte pieces: with few of them, copied, and read as they are."""
    for dtype, act in ((BF, "gelu"), (F16, None)):
        x, W, b, res, _ = _inputs(M, N, K, dtype)
        _check(ozk.fused_linear(x, W, b, activation=act, residual=res), x, W, b, res, act)
        # rows that are whole pieces apart but begin off them
        x, W = (torch.nn.functional.pad(t, (1, 16 - (K + 1) % 8))[:, 1:1 + K] for t in (x, W))
        _check(ozk.fused_linear(x, W, b, activation=act), x, W, b, None, act)


@pytest.mark.parametrize("act", ACTS[2:])
def test_smallest_results(gpu, act):
    """Far below 0 results and derivatives keep their relative accuracy as long as they are normal
    numbers: bf16 has fp32's range, and the exponentials in them leave it first.

    exp2's argument, up to 2^7 in size there, has at most 8 roundings of 2^-24 (gelu_tanh): 2^-14
    relative in the result; then one rounding to bf16, of the derivative one more factor of that size."""
    bits = torch.arange(-32768, 0, dtype=torch.int32, device="cuda").to(torch.int16)
    x = bits.view(BF)
    x = x[(x.float() <= -8) & (x.float() > -300)]
    z, h = x.double(), _half(BF)[0]
    if act == "gelu_tanh":
        slope = 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
        s = torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        want, steep = z * s, s * (1 + z * slope * (1 - s))
    else:
        want, steep = _act(z, act)
        if act == "gelu":        # Phi + z phi, of which the second is larger
            steep = 0.5 * torch.erfc(z * -math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    for rows in (x, x[:3], x[-40:]):
        n = rows.shape[0]
        first = 0 if rows.data_ptr() == x.data_ptr() else x.shape[0] - n
        a = rows[:, None].contiguous().requires_grad_()
        y = ozk.fused_linear(a, torch.ones(1, 1, dtype=BF, device="cuda"), activation=act)
        d, = torch.autograd.grad(y, a, torch.ones_like(y))
        for got, exact in ((y, want), (d, steep)):
            exact = exact[first:first + n]
            off = (got.detach().double()[:, 0] - exact).abs()
            # (below 2^-126 they may come out as 0)
            tol = torch.where(exact.abs() >= 2.0 ** -126, (h + 2.0 ** -13) * exact.abs(), 2.0 ** -126)
            assert bool((off <= tol).all()), [(float(z[first + i]), float(got[i]), float(exact[i]))
                                              for i in torch.nonzero(off > tol)[:5, 0].tolist()]


@pytest.mark.parametrize("act", [None, "silu"])
def test_wide_results(gpu, act):
    """Rows of 2^22 results and more: a gradient that the backward pass does not take is refused
    before the forward pass, that of one row has the formula's values."""
    N, K = (1 << 22) + 3, 8
    x, W, b, _, dy = _inputs(2, N, K, F16)
    _check(ozk.fused_linear(x, W, b, activation=act), x, W, b, None, act)
    for leaf in (x, W, b):
        leaf.requires_grad_()
        with pytest.raises(RuntimeError, match="columns"):
            ozk.fused_linear(x, W, b, activation=act)
        with torch.no_grad():
            assert ozk.fused_linear(x, W, b, activation=act).shape == (2, N)
        leaf.requires_grad_(False)
    res = dy.clone().requires_grad_()       # its gradient is dy
    g, = torch.autograd.grad(ozk.fused_linear(x, W, b, activation=act, residual=res), res, dy)
    assert torch.equal(g, dy)
    x, dy = x[:1], dy[:1]
    leaves = [t.requires_grad_() for t in (x, W, b)]
    dx, dW, db = torch.autograd.grad(ozk.fused_linear(*leaves, activation=act), leaves, dy)
    x, W, b = (t.detach() for t in leaves)
    h, least = _half(F16)
    z = x.double() @ W.double().mT.contiguous() + b.double()
    dz = dy.double() * _act(z, act)[1]
    # as in test_gradients: z in 16 bits, dz rounded, the sums of N or one product
    e = (h * dz.abs() + least + dy.double().abs() * (0.8 * (h * z.abs() + least + (K + 4) * U * 4) + 2 ** -17)
         if act else torch.zeros_like(dz))
    for got, want, tol in ((dx, dz @ W.double(), e @ W.double().abs() + (N + 2) * U * ((dz.abs() + e) @ W.double().abs())),
                           (dW, dz.mT.contiguous() @ x.double(), e.mT.contiguous() @ x.double().abs()),
                           (db, dz[0], e[0])):
        tol = tol + (h + U) * (want.abs() + tol) + 2 * least
        assert bool(((got.double() - want).abs() <= tol).all())
    # (N terms whose roundings are as good as independent)
    want = dz @ W.double()
    assert float((dx.double() - want).norm()) <= 2 * h * float(want.norm()) + 4 * h * float((dz.mT.contiguous() * W.double()).norm())


def test_one_long_row(gpu):
    """One row of 2^22 elements has no distance to a next one, also where it comes with gaps."""
    K = 1 << 22
    x = torch.randn(K, 2, device="cuda").to(F16)[:, :1].mT
    V = (torch.randn(K, 3, device="cuda") / math.sqrt(K)).to(F16)
    _check(ozk.fused_linear(x, V.mT), x, V.mT, None, None, None)
    w = torch.randn(K, 2, device="cuda").to(F16)[:, 1:].mT / 64
    _check(ozk.fused_linear(x, w.contiguous()), x, w, None, None, None)
    w = (torch.randn(K, 2, device="cuda") / 64).to(F16)[:, 1:].mT
    _check(ozk.fused_linear(x, w), x, w, None, None, None)


@pytest.mark.parametrize("M, N, K", [(130, 64, 8191), (200, 72, 4099), (129, 520, 16383), (33, 3000, 8191), (500, 64, 16385)])
@pytest.mark.parametrize("wt", [False, True])
def test_partial_sums_without_copies(gpu, M, N, K, wt):
    """The C call with room for the partial sums of K ranges but not for copies of rows off 16 bytes."""
    L, n = _lib.load(), ctypes.c_size_t(0)
    for dtype, act in ((BF, "gelu"), (F16, None)):
        x, W, b, res, _ = _inputs(M, N, K, dtype, wt=wt)
        s = _lib.i64arr(W.stride())
        size = lambda k, *strides: (L.ozk_linear_workspace_bytes(  # noqa: E731
            x.data_ptr(), strides[0], W.data_ptr(), _lib.i64arr(strides[1:]), M, N // 8 * 8, k, ctypes.byref(n)), n.value)
        # rows that are whole 16 bytes need the partial sums alone
        status, sums = size(K // 8 * 8, K // 8 * 8, *((1, N // 8 * 8) if wt else (K // 8 * 8, 1)))
        assert status == _lib.OZK_OK and sums >= 2 * M * (N // 8 * 8) * 4
        assert L.ozk_linear_workspace_bytes(x.data_ptr(), K, W.data_ptr(), s, M, N, K, ctypes.byref(n)) == _lib.OZK_OK
        assert n.value > sums
        for room in (n.value, n.value - 1):
            ws = torch.full((room + 64,), 0xAB, dtype=torch.uint8, device="cuda")
            y = torch.full((M, N), math.nan, device="cuda", dtype=dtype)
            z = torch.full((M, N), math.nan, device="cuda", dtype=dtype)
            assert L.ozk_linear(x.data_ptr(), K, W.data_ptr(), s, b.data_ptr(), res.data_ptr(), N, ACTS.index(act), M, N, K,
                                _lib.OZK_BF16 if dtype == BF else _lib.OZK_F16, y.data_ptr(), N, z.data_ptr(),
                                ws.data_ptr(), room, torch.cuda.current_stream().cuda_stream) == _lib.OZK_OK
            _check(y, x, W, b, res, act)
            _check(z, x, W, b, None, None)
            assert bool((ws[room:] == 0xAB).all())
        assert L.ozk_linear(x.data_ptr(), K, W.data_ptr(), s, None, None, 0, 0, M, N, K, _lib.OZK_F16, y.data_ptr(), N, None,
                            ws.data_ptr(), sums // 2, None) == _lib.OZK_ERR_WORKSPACE
