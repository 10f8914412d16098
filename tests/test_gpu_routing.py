"""route_tokens against plain torch: whole numbers exactly, the rest in 64 bits.

u = 2^-24.  A softmax value is off by the rounding of l - max (u |l - max|), those
of the exponential, the sum of E terms and a division: under (40 + |l - max|) u
relative for up to 1024 experts (a lane adds at most 16, six exchanges follow)."""
import pytest
import torch

import ozaki_triton_amd as ozk

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


def _plain(logits, k, mask, normalize):
    T, E = logits.shape
    l = logits.double()
    valid = torch.ones(T, dtype=torch.bool, device="cuda") if mask is None else mask
    chosen = torch.sort(-l, dim=1, stable=True).indices[:, :k]
    p = torch.softmax(l, 1)
    w = p.gather(1, chosen)
    if normalize:
        w = torch.softmax(l.gather(1, chosen), 1)
    w = torch.where(valid[:, None], w, 0.0)
    experts = torch.where(valid[:, None], chosen, E)
    flat = experts.flatten()
    order = torch.sort(flat, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(T * k, device="cuda")
    counts = torch.bincount(flat, minlength=E + 1)[:E]
    offsets = torch.nn.functional.pad(counts.cumsum(0), (1, 0))
    n = int(valid.sum())
    P = p[valid].sum(0)
    loss = E * (counts.double() * P).sum() / (n * k * n) if n else torch.zeros((), device="cuda", dtype=torch.float64)
    return dict(experts=experts, weights=w, order=order, place=place.view(T, k), offsets=offsets,
                counts=counts, balance_loss=loss), p, valid, n


def _check(logits, k, mask=None, normalize=True):
    r = ozk.route_tokens(logits, k, mask=mask, normalize=normalize)
    want, p, valid, n = _plain(logits.detach(), k, mask, normalize)
    for name in ("experts", "order", "place", "offsets", "counts"):
        got = getattr(r, name)
        assert got.dtype == torch.int32 and got.shape == want[name].shape
        assert torch.equal(got.long(), want[name]), name
    spread = 40 + (logits.detach().double().amax(1) - logits.detach().double().gather(
        1, want["experts"].clamp(max=logits.shape[1] - 1)).amin(1)).clamp(max=150)[:, None]
    assert r.weights.dtype == F32
    assert bool(((r.weights.double() - want["weights"]).abs() <=
                 2 * spread * U * want["weights"] + 2.0 ** -126)[valid].all())   # (below: subnormal, or 0)
    assert not r.weights[~valid].any()
    # every p is within that for differences up to 40 (smaller ones do not count), and
    # a lane adds up to 64 tokens before the sums go on in 64 bits
    assert abs(float(r.balance_loss.detach()) - float(want["balance_loss"])) <= 160 * U * float(want["balance_loss"])
    return r, want, p, valid, n


def _logits(T, E, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (2 * torch.randn(T, E, generator=g, device="cuda")).to(dtype)


CASES = [(1, 1, 1), (1, 2, 2), (1, 64, 8), (3, 5, 5), (16, 16, 2), (63, 7, 3), (64, 8, 1), (65, 9, 2), (100, 33, 4),
         (1000, 64, 8), (1025, 40, 3), (4099, 40, 3), (2000, 128, 8), (777, 129, 5), (500, 256, 8), (300, 300, 7),
         (200, 512, 2), (130, 1000, 10), (90, 1024, 4), (50, 1024, 1024), (5000, 4, 4), (70000, 8, 2),
         (10, 300, 280), (40, 300, 280), (1, 600, 2), (5, 1024, 3)]   # the last: about 64 KiB of LDS


@pytest.mark.parametrize("T, E, k", CASES)
@pytest.mark.parametrize("dtype", [F32, BF, F16])
def test_routing(gpu, T, E, k, dtype):
    logits = _logits(T, E, dtype, seed=T + E)
    _check(logits, k)
    _check(logits, k, normalize=False)
    mask = torch.rand(T, device="cuda") < 0.6
    _check(logits, k, mask)
    _check(logits, k, mask, normalize=False)


def test_ties_zeros_and_signs(gpu):
    """Of equal logits the lowest index, 0 and -0 equal."""
    for E, k in ((6, 3), (16, 4), (64, 64), (300, 9)):
        for dtype in (F32, BF, F16):
            g = torch.Generator(device="cuda").manual_seed(E)
            logits = torch.randint(-1, 2, (500, E), generator=g, device="cuda").to(dtype)
            logits = torch.where(torch.rand(500, E, generator=g, device="cuda") < 0.5, -logits, logits)
            assert bool((logits.float().view(torch.int32) == -2147483648).any())
            _check(logits, k)
            _check(torch.zeros(70, E, device="cuda", dtype=dtype), k)


def test_one_expert_takes_all(gpu):
    logits = torch.zeros(5000, 32, device="cuda")
    logits[:, 5] = 30.0
    r, *_ = _check(logits, 1)
    assert int(r.counts[5]) == 5000 and abs(float(r.balance_loss) - 32) < 1e-3


def test_infinities_and_nan(gpu):
    inf, nan = float("inf"), float("nan")
    # experts that are switched off: probability and weight 0
    logits = _logits(600, 20, F32)
    logits[:, 3:18] = -inf
    logits[::2, :3] = -inf
    r, *_ = _check(logits, 4)
    assert torch.isfinite(r.weights).all() and bool((r.weights[::2, 2:] == 0).all())
    # rows that have no softmax: NaN in their weights and the loss, everything else in order
    for bad in (nan, inf, -inf):
        logits = _logits(600, 20, F32)
        if bad == -inf:
            logits[7] = -inf
        else:
            logits[7, 11] = bad
        r = ozk.route_tokens(logits, 4)
        assert bool(torch.isnan(r.weights[7]).any()) and torch.isnan(r.balance_loss)
        keep = torch.arange(600, device="cuda") != 7
        assert torch.isfinite(r.weights[keep]).all()
        experts = r.experts.long()
        assert int(experts.min()) >= 0 and int(experts.max()) < 20
        assert all(len(set(row)) == 4 for row in experts[5:9].tolist())
        if bad != -inf:
            assert experts[7, 0] == 11
        assert torch.equal(torch.sort(r.order.long()).values, torch.arange(2400, device="cuda"))
        # masked out, the row is not looked at
        mask = keep
        r = ozk.route_tokens(logits, 4, mask=mask)
        assert torch.isfinite(r.weights).all() and torch.isfinite(r.balance_loss)
        logits.requires_grad_()
        r = ozk.route_tokens(logits, 4, mask=mask)
        d, = torch.autograd.grad(r.balance_loss + r.weights.square().sum(), logits)
        assert torch.isfinite(d).all() and not d[7].any()


def test_lowest_values(gpu):
    """Experts switched off by the type's lowest value, some or all of them."""
    for dtype in (F32, BF, F16):
        low = torch.finfo(dtype).min
        logits = _logits(500, 24, dtype)
        logits[:, 5:20] = low
        logits[3] = low
        logits[4] = torch.finfo(dtype).max
        logits[5, ::2] = torch.finfo(dtype).max
        logits[5, 1::2] = low
        logits.requires_grad_()
        r, want, p, *_ = _check(logits, 6)
        assert torch.isfinite(r.weights).all() and torch.isfinite(r.balance_loss)
        d, = torch.autograd.grad(r.balance_loss * 500 + r.weights.square().sum(), logits)
        assert torch.isfinite(d).all()
        assert not d[6:, 5:20].any()


def test_nothing_left(gpu):
    for T in (0, 1, 70, 5000):
        logits = _logits(T, 12, F32).requires_grad_()
        mask = torch.zeros(T, dtype=torch.bool, device="cuda")
        r = ozk.route_tokens(logits, 3, mask=mask)
        assert float(r.balance_loss.detach()) == 0 and not r.weights.any() and not r.counts.any() and not r.offsets.any()
        assert bool((r.experts == 12).all())
        assert torch.equal(r.order, torch.arange(3 * T, device="cuda", dtype=torch.int32))
        assert torch.equal(r.place.flatten(), r.order)
        d, = torch.autograd.grad(r.balance_loss + r.weights.sum(), logits)
        assert d.shape == (T, 12) and not d.any()


@pytest.mark.parametrize("T, E, k", [(1, 1, 1), (5, 3, 2), (16, 16, 2), (333, 40, 3), (3000, 64, 8), (200, 100, 100),
                                     (70, 300, 7), (64, 1024, 5), (4099, 8, 1)])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF, F16])
def test_gradients(gpu, T, E, k, normalize, dtype):
    for masked in (False, True):
        mask = torch.rand(T, device="cuda") < 0.7 if masked else None
        logits = _logits(T, E, dtype, seed=T).requires_grad_()
        dw = torch.randn(T, k, device="cuda")
        dloss = torch.tensor(1.7 * T, device="cuda")
        r, want, p, valid, n = _check(logits, k, mask, normalize)
        dl, = torch.autograd.grad([r.weights, r.balance_loss], [logits], [dw, dloss])
        only_w, = torch.autograd.grad(ozk.route_tokens(logits, k, mask=mask, normalize=normalize).weights, logits, dw)
        only_l, = torch.autograd.grad(ozk.route_tokens(logits, k, mask=mask, normalize=normalize).balance_loss,
                                      logits, dloss)
        # the formula in 64 bits
        w, dwd = want["weights"], torch.where(valid[:, None], dw.double(), 0.0)
        at = want["experts"].clamp(max=E - 1)
        p = torch.where(valid[:, None], p, 0.0)
        zero = torch.zeros_like(p)
        g_loss = (1.7 * T * E * want["counts"].double() / max(n * k * n, 1)).expand(T, E)
        if normalize:
            direct = zero.scatter_add(1, at, w * (dwd - (w * dwd).sum(1, keepdim=True)))
            direct_size = zero.scatter_add(1, at, w * (dwd.abs() + (w * dwd.abs()).sum(1, keepdim=True)))
            g_w = zero
        else:
            direct = direct_size = zero
            g_w = zero.scatter_add(1, at, dwd)
        for got, g, d, d_size in ((dl, g_loss + g_w, direct, direct_size), (only_w, g_w, direct, direct_size),
                                  (only_l, g_loss, zero, zero)):
            exact = d + p * (g - (p * g).sum(1, keepdim=True))
            size = d_size + p * (g.abs() + (p * g.abs()).sum(1, keepdim=True))
            # weights and softmax to 100 u for differences up to 30 in the logits, sums of E + k terms
            half = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
            least = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
            tol = (200 + k) * U * size + half * exact.abs() * 1.01 + least
            assert got.dtype == dtype and got.shape == (T, E)
            assert bool(((got.double() - exact).abs() <= tol).all()), \
                float(((got.double() - exact).abs() / tol).max())


def test_gradients_against_differences(gpu):
    """Along random directions, where the choice does not change; f is a constant."""
    T, E, k = 40, 24, 3
    logits = _logits(T, E, F32, seed=9).requires_grad_()
    dw = torch.randn(T, k, device="cuda")
    for normalize in (True, False):
        r = ozk.route_tokens(logits, k, normalize=normalize)
        dl, = torch.autograd.grad((r.weights * dw).sum() + 3.0 * r.balance_loss, logits)
        f = r.counts.double() / (T * k)
        at = r.experts.long()
        base = logits.detach().double()

        def value(l):
            p = torch.softmax(l, 1)
            w = p.gather(1, at)
            if normalize:
                w = w / w.sum(1, keepdim=True)
            return float((w * dw.double()).sum() + 3.0 * E * (f * p.mean(0)).sum())
        for seed in range(3):
            g = torch.Generator(device="cuda").manual_seed(seed)
            d = torch.randn(T, E, generator=g, device="cuda", dtype=torch.float64)
            slope = (value(base + 1e-5 * d) - value(base - 1e-5 * d)) / 2e-5
            got = float((dl.double() * d).sum())
            assert abs(got - slope) <= 1e-5 * float((dl.double().abs() * d.abs()).sum())


def test_layouts(gpu):
    base = _logits(300, 200, F32)
    for logits in (base[:, 3:43], base[:, ::2][:, :40], base[:40, :].mT, base[:1, :40].expand(300, 40), base[:, :1]):
        k = min(3, logits.shape[1])
        mask = (torch.arange(2 * logits.shape[0], device="cuda") % 5 != 0)[::2]
        a = ozk.route_tokens(logits, k, mask=mask)
        b = ozk.route_tokens(logits.contiguous(), k, mask=mask.contiguous())
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        _check(logits, k, mask)


def test_same_bits_every_time_and_on_any_stream(gpu):
    logits = _logits(9000, 64, BF).requires_grad_()
    dw = torch.randn(9000, 8, device="cuda")

    def step():
        r = ozk.route_tokens(logits, 8)
        return [t.detach() for t in r] + list(torch.autograd.grad((r.weights * dw).sum() + r.balance_loss, logits))
    first = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(step())
    torch.cuda.synchronize()
    for r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, first))


def test_captured(gpu):
    for T in (40, 3000):
        logits = _logits(T, 64, F32).requires_grad_()
        mask = torch.ones(T, dtype=torch.bool, device="cuda")
        dw = torch.randn(T, 4, device="cuda")

        def step():
            r = ozk.route_tokens(logits, 4, mask=mask)
            return [t.detach() for t in r] + list(torch.autograd.grad((r.weights * dw).sum() + r.balance_loss, logits))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for seed in range(4):
            with torch.no_grad():
                logits.copy_(_logits(T, 64, F32, seed=seed))
                mask.copy_(torch.rand(T, device="cuda") < 0.2 + 0.2 * seed)
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in out]
            assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_refusals_on_the_gpu(gpu):
    logits = _logits(10, 8, F32)
    with pytest.raises(NotImplementedError):
        ozk.route_tokens(logits.double(), 2)
    with pytest.raises(RuntimeError):
        ozk.route_tokens(logits, 2, mask=torch.ones(10, dtype=torch.bool))
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError):
            ozk.route_tokens(torch.autograd.forward_ad.make_dual(logits, logits), 2)
    t = logits.requires_grad_()
    g, = torch.autograd.grad(ozk.route_tokens(t, 2).weights.sum(), t, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_layer_of_experts(gpu):
    """The router with the grouped products, against every expert on every token: with
    grouped_matmul's roundings (bf16 products of 64 terms)."""
    T, E, k, width = 300, 6, 2, 64
    x = torch.randn(T, width, device="cuda").to(BF)
    W = (torch.randn(E, width, width, device="cuda") / 8).to(BF)
    logits = (x.float() @ torch.randn(width, E, device="cuda") / 8).requires_grad_()
    mask = torch.rand(T, device="cuda") < 0.8
    r = ozk.route_tokens(logits, k, mask=mask)
    y = ozk.grouped_matmul(x[r.order // k], W, r.offsets)
    out = (y[r.place].float() * r.weights[..., None]).sum(1)
    out.sum().backward()
    full = torch.stack([x.float() @ W[e].float() for e in range(E)], 1).double()
    l = logits.detach().double().requires_grad_()
    top = torch.topk(l, k, dim=1)
    w = torch.softmax(top.values, 1) * mask[:, None]
    want = (full.gather(1, top.indices[..., None].expand(T, k, width)) * w[..., None]).sum(1)
    want.sum().backward()
    # each product is rounded to 2^-8 of itself
    size = (full.abs().gather(1, top.indices[..., None].expand(T, k, width)) * w.detach()[..., None]).sum(1)
    assert bool(((out.double() - want).abs() <= 2.0 ** -8 * size + 1e-5).all())
    assert not out[~mask].any()
    tol = 2.0 ** -7 * full.abs().sum(2).amax(1)[:, None] + 1e-5
    assert bool(((logits.grad.double() - l.grad).abs() <= tol).all())


def test_recorded_and_changed(gpu):
    """A recorded backward pass has the same values; what it needs and was changed is noticed."""
    logits = _logits(200, 16, F32).requires_grad_()
    r = ozk.route_tokens(logits, 3)
    dw = torch.randn(200, 3, device="cuda")
    a, = torch.autograd.grad(r.weights, logits, dw, retain_graph=True)
    b, = torch.autograd.grad(r.weights, logits, dw, create_graph=True)
    assert torch.equal(a, b.detach())
    with pytest.raises(RuntimeError, match="twice"):
        b.sum().backward()
    for name in ("experts", "counts"):
        r = ozk.route_tokens(logits, 3)
        getattr(r, name).add_(1000)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            (r.weights * dw).sum().backward()
    with torch.inference_mode():
        q = ozk.route_tokens(logits, 3)
    assert torch.equal(q.order, r.order) and not q.weights.requires_grad


def test_results_are_each_others_own(gpu):
    """What the backward pass does not need may be changed in place before it."""
    logits = _logits(200, 16, F32).requires_grad_()
    dw = torch.randn(200, 3, device="cuda")
    want, = torch.autograd.grad(ozk.route_tokens(logits, 3).weights, logits, dw)
    r = ozk.route_tokens(logits, 3)
    r.order.div_(3, rounding_mode="floor")
    r.place.add_(7)
    r.offsets.zero_()
    got, = torch.autograd.grad(r.weights, logits, dw)
    assert torch.equal(got, want)


def test_saved_tensor_hooks(gpu):
    """Saved tensors that travel to the host and back; ones that come back as something else."""
    logits = _logits(300, 20, BF).requires_grad_()
    mask = torch.rand(300, device="cuda") < 0.9
    dw = torch.randn(300, 4, device="cuda")

    def grad():
        r = ozk.route_tokens(logits, 4, mask=mask)
        return torch.autograd.grad([r.weights, r.balance_loss], logits, [dw, dw[0, 0]])[0]
    want = grad()
    with torch.autograd.graph.save_on_cpu():
        assert torch.equal(grad(), want)
    for back in (lambda t: t.cpu(), lambda t: t[:1], lambda t: t.double(), lambda t: t[..., None]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, back):
            with pytest.raises(RuntimeError, match="saved"):
                grad()


def test_past_32_bits(gpu):
    """More than 2^31 logits: the first and the last tokens, the whole order, their gradients."""
    T, E, k = 4300000, 512, 2
    logits = torch.randn(T, E, device="cuda").to(BF).requires_grad_()
    r = ozk.route_tokens(logits, k)
    ends = [slice(0, 500), slice(T - 500, T)]
    for s in ends:
        want, *_ = _plain(logits[s].detach(), k, None, True)
        assert torch.equal(r.experts[s].long(), want["experts"])
        # (2 spread U as above, spread below 64)
        assert bool(((r.weights[s].double() - want["weights"]).abs() <= 128 * U).all())
    slots = torch.arange(T * k, device="cuda")
    sorted_experts = r.experts.flatten()[r.order.long()]
    assert torch.equal(r.order[r.place.flatten().long()].long(), slots)
    assert bool((sorted_experts.diff() >= 0).all())
    assert bool(((r.order.diff() > 0) | (sorted_experts.diff() > 0)).all())   # their own order within one
    assert torch.equal(r.counts.long(), torch.bincount(r.experts.flatten(), minlength=E))
    assert torch.equal(r.offsets.diff(), r.counts)
    dw = torch.randn(T, k, device="cuda")
    d, = torch.autograd.grad(r.weights, logits, dw)
    for s in ends:
        w, g = r.weights[s].detach().double(), dw[s].double()
        want = torch.zeros(500, E, device="cuda", dtype=torch.float64).scatter_(
            1, r.experts[s].long(), w * (g - (w * g).sum(1, keepdim=True)))
        # a weight's error by the difference of two terms that have it, too
        tol = 2.0 ** -8 * want.abs() + 3 * 128 * U * g.abs().sum(1, keepdim=True)
        assert bool(((d[s].double() - want).abs() <= tol).all())
