"""The operators of a training step together: router, grouped products, dense products
with their epilogues, clipping, orthogonalised update; eager and captured."""
import math
import threading

import pytest
import torch

import ozaki_triton_amd as ozk

pytestmark = pytest.mark.gpu

F16 = torch.float16
T, WIDTH, HIDDEN, OUT, E, K = 200, 64, 96, 40, 5, 2


def _setup(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    p = dict(router=r(WIDTH, E) / 8, up=(r(E, WIDTH, HIDDEN) / 8).to(F16), down=(r(E, HIDDEN, WIDTH) / 10).to(F16),
             shared=(r(HIDDEN, WIDTH) / 8).to(F16), back=(r(WIDTH, HIDDEN) / 10).to(F16),
             head=(r(OUT, WIDTH) / 8).to(F16), bias=r(OUT).to(F16))
    return r(T, WIDTH).to(F16), torch.rand(T, generator=g, device="cuda") < 0.85, r(T, OUT).to(F16), p


def _step(x, mask, dy, p):
    """One layer's outputs, balance loss and gradients, these clipped to half their norm's bound."""
    r = ozk.route_tokens(x.float() @ p["router"], K, mask=mask)
    h = ozk.grouped_matmul(x[r.order // K], p["up"], r.offsets).relu()
    y = ozk.grouped_matmul(h, p["down"], r.offsets)
    y = (y[r.place].float() * r.weights[..., None]).sum(1).to(F16)
    s = ozk.fused_linear(ozk.fused_linear(x, p["shared"], activation="gelu"), p["back"], residual=x)
    out = ozk.fused_linear(s + y, p["head"], p["bias"], activation="silu")
    grads = list(torch.autograd.grad([out, r.balance_loss], list(p.values()),
                                     [dy, torch.full((), 30.0, device="cuda")]))
    norm = ozk.clip_gradients(grads, 20.0)
    with torch.no_grad():
        update = ozk.orthogonalize(grads[5])
    return [out.detach(), r.balance_loss.detach(), norm, update, *grads]


def _exact(x, mask, dy, p):
    """The same in 64 bits, every expert on every token."""
    p = {n: v.detach().double().requires_grad_() for n, v in p.items()}
    x, dy = x.double(), dy.double()
    logits = x @ p["router"]
    chosen = torch.sort(-logits.detach(), dim=1, stable=True).indices[:, :K]
    w = torch.softmax(logits.gather(1, chosen), 1) * mask[:, None]
    every = torch.stack([(x @ p["up"][e]).relu() @ p["down"][e] for e in range(E)], 1)
    y = (every.gather(1, chosen[..., None].expand(T, K, WIDTH)) * w[..., None]).sum(1)
    u = x @ p["shared"].T
    s = (u * 0.5 * torch.erfc(-u / math.sqrt(2))) @ p["back"].T + x
    z = (s + y) @ p["head"].T + p["bias"]
    out = z * torch.sigmoid(z)
    n = mask.sum()
    counts = torch.bincount(chosen[mask].flatten(), minlength=E).double()
    loss = E * (counts / (n * K) * torch.softmax(logits, 1)[mask].mean(0)).sum()
    grads = torch.autograd.grad([out, loss], list(p.values()), [dy, torch.full_like(loss, 30.0)])
    norm = math.sqrt(sum(float(v.square().sum()) for v in grads))
    return out, loss, norm, [v * min(1.0, 20.0 / norm) for v in grads]


def test_step_against_64_bits(gpu):
    x, mask, dy, p = _setup()
    for v in p.values():
        v.requires_grad_()
    out, loss, norm, update, *grads = _step(x, mask, dy, p)
    want, want_loss, want_norm, want_grads = _exact(x, mask, dy, p)
    # a path has about ten roundings to fp16, each half a step (2^-11) of its tensor's norm at
    # most, through maps that do not enlarge norms much: three times their sum
    tol = 30 * 2.0 ** -11
    off = lambda a, b: float((a.detach().double() - b.detach()).norm() / b.detach().norm())  # noqa: E731
    assert off(out, want) <= tol
    # logits in fp32 (64 terms)
    assert abs(float(loss) - float(want_loss.detach())) <= 1e-5 * float(want_loss.detach())
    assert want_norm > 20.0                                # the gradients are scaled
    assert abs(float(norm) - want_norm) <= tol * want_norm
    for name, got, exact in zip(p, grads, want_grads):
        assert off(got, exact) <= tol, name
    # singular values near 1, along the gradient
    s = torch.linalg.svdvals(update.float())
    assert float(s.max()) < 1.3 and float((update.float() * grads[5].float()).sum()) > 0


def test_step_captured(gpu):
    """One graph of the whole step, replayed on new inputs between eager steps."""
    x, mask, dy, p = _setup()
    for v in p.values():
        v.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _step(x, mask, dy, p)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = _step(x, mask, dy, p)
    for seed in range(1, 5):
        nx, nmask, ndy, np_ = _setup(seed)
        with torch.no_grad():
            for old, new in zip((x, mask, dy, *p.values()), (nx, nmask, ndy, *np_.values())):
                old.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in results]
        eager = _step(x, mask, dy, p)
        for a, b in zip(got, eager):
            # (torch's own reductions and scatters run in both)
            assert float((a.double() - b.double()).norm()) <= 1e-3 * float(b.double().norm()) + 1e-12
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])


def test_threads(gpu):
    """Steps of several threads at once, each on a stream of its own, have the same bits."""
    x, W = (torch.randn(*s, device="cuda").to(torch.bfloat16) for s in ((333, 520), (700, 520)))
    logits = torch.randn(3000, 64, device="cuda")

    def step():
        a, w, t = (v.detach().requires_grad_() for v in (x, W, logits))
        y = ozk.fused_linear(a, w, activation="gelu")
        r = ozk.route_tokens(t, 4)
        (y.float().square().sum() + r.balance_loss + r.weights.square().sum()).backward()
        norm = ozk.clip_gradients([a.grad, w.grad, t.grad], 1.0)
        return [y.detach(), a.grad, w.grad, t.grad, norm, *(v.detach() for v in r)]
    want = step()
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(10):
                got = step()
                stream.synchronize()
                if not all(torch.equal(u, v) for u, v in zip(got, want)):
                    wrong.append(i)
        wrong.append(None)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == [None] * 4


def test_capture_beside_an_eager_graph(gpu):
    """A captured backward pass of leaves that an eager graph holds is refused, and works once that is gone."""
    x = torch.randn(64, 64, device="cuda").to(F16)
    W = torch.randn(64, 64, device="cuda").to(F16).requires_grad_()
    logits = torch.randn(40, 8, device="cuda").requires_grad_()
    dy, dw = torch.randn(64, 64, device="cuda").to(F16), torch.randn(40, 2, device="cuda")
    calls = [(lambda: ozk.fused_linear(x, W), W, dy), (lambda: ozk.route_tokens(logits, 2).weights, logits, dw)]
    for forward, leaf, seed in calls:
        want, = torch.autograd.grad(forward(), leaf, seed)
        keep = forward()
        # on another stream, but not captured: as ever
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got, = torch.autograd.grad(forward(), leaf, seed)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="default stream"):
            with torch.cuda.graph(graph):
                torch.autograd.grad(forward(), leaf, seed)
        torch.cuda.synchronize()
        del keep
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, = torch.autograd.grad(forward(), leaf, seed)
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


def test_nodes_called_by_hand(gpu):
    """A backward node called outside autograd's engine runs where it is called: in a capture on
    another stream than its forward pass's it is captured, and behind work on its own stream."""
    x, W = (torch.randn(*s, device="cuda").to(F16).requires_grad_() for s in ((64, 72), (80, 72)))
    logits = torch.randn(40, 8, device="cuda").requires_grad_()
    y, r = ozk.fused_linear(x, W, activation="silu"), ozk.route_tokens(logits, 2)
    dy, dw = torch.randn(64, 80, device="cuda").to(F16), torch.randn(40, 2, device="cuda")
    nothing = [None] * 7

    def route(dw):
        grads = list(nothing)
        grads[1] = dw
        return r.weights.grad_fn(*grads)      # one result: not a tuple

    def calls():
        dx, dW = y.grad_fn(dy)[:2]
        return [dx, dW, route(dw)]

    def want():
        return [*torch.autograd.grad(y, (x, W), dy, retain_graph=True),
                *torch.autograd.grad(r.weights, logits, dw, retain_graph=True)]
    assert all(torch.equal(a, b) for a, b in zip(calls(), want()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls()
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        dy.copy_(torch.randn(64, 80, device="cuda", generator=g))
        dw.copy_(torch.randn(40, 2, device="cuda", generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want()))
    # 40 products of 4096 before dy is there
    side, a = torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(40):
            a = a @ a * 1e-2
        dy.copy_(torch.where(a[:64, :80] == a[:64, :80], 2.0, 3.0))
        dw.fill_(0.5)
        got = calls()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want()))


def test_nodes_called_by_hand_with_other_gradients(gpu):
    """Gradients of another shape, type or device than the results raise before a launch."""
    x, b = torch.randn(16, 24, device="cuda").to(F16), torch.zeros(40, device="cuda", dtype=F16).requires_grad_()
    W = torch.randn(40, 24, device="cuda").to(F16)
    logits = torch.randn(16, 8, device="cuda").requires_grad_()
    r = ozk.route_tokens(logits, 2)
    ok = torch.ones(16, 40, device="cuda", dtype=F16)
    for y in (ozk.fused_linear(x, W, b), ozk.fused_linear(x, W, b, activation="silu"),
              ozk.fused_linear(x.clone().requires_grad_(), W)):
        y.grad_fn(ok)
        for bad in (ok[:15], ok[:, :39], ok[0], ok.float(), ok.cpu(), ok[None]):
            with pytest.raises(RuntimeError, match="another shape, type or device"):
                y.grad_fn(bad)
    dw, dl = torch.ones(16, 2, device="cuda"), torch.ones((), device="cuda")
    call = lambda w, l: r.weights.grad_fn(None, w, None, None, None, None, l)  # noqa: E731
    want, = torch.autograd.grad([r.weights, r.balance_loss], logits, [dw, dl], retain_graph=True)
    assert torch.equal(call(dw, dl), want)
    for w, l in ((dw[:15], dl), (dw[:, :1], None), (dw.half(), dl), (dw.cpu(), None), (dw, dl.cpu()),
                 (None, dl.double()), (None, dl[None])):
        with pytest.raises(RuntimeError, match="another shape, type or device"):
            call(w, l)


def test_capture_beside_an_eager_graph_further_on(gpu):
    """The same where the leaf lies behind other nodes: behind the reshape of an x of three dims, or
    the caller's own operations; a leaf whose gradient is not wanted does not matter."""
    x = torch.randn(4, 16, 64, device="cuda").to(F16).requires_grad_()
    W = torch.randn(64, 64, device="cuda").to(F16).requires_grad_()
    logits = torch.randn(40, 8, device="cuda").requires_grad_()
    dy, dw = torch.randn(4, 16, 64, device="cuda").to(F16), torch.randn(40, 2, device="cuda")
    calls = [(lambda: ozk.fused_linear(x, W.detach(), activation="gelu"), x, dy),
             (lambda: ozk.fused_linear(x.detach(), (2 * W).mT.contiguous()), W, dy),
             (lambda: ozk.route_tokens(3 * logits.view(8, 40).view(40, 8), 2).weights, logits, dw)]
    for forward, leaf, seed in calls:
        want, = torch.autograd.grad(forward(), leaf, seed)
        keep = forward()
        with pytest.raises(RuntimeError, match="default stream"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.autograd.grad(forward(), leaf, seed)
        torch.cuda.synchronize()
        del keep
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, = torch.autograd.grad(forward(), leaf, seed)
        for _ in range(3):
            got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
    # not wanted: the eager graph holds W alone, the gradient is x's
    want, = torch.autograd.grad(ozk.fused_linear(x, W), x, dy)
    keep = ozk.fused_linear(x.detach(), W)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(ozk.fused_linear(x, W), x, dy)
    for _ in range(3):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
    assert keep.requires_grad


def test_transforms_are_refused(gpu):
    """Tensors of torch.func's transforms have no memory of their own: an error, never a wrong result."""
    x, W = torch.randn(4, 16, 24, device="cuda").to(F16), torch.randn(40, 24, device="cuda").to(F16)
    b, logits = torch.zeros(4, 40, device="cuda", dtype=F16), torch.randn(4, 16, 8, device="cuda")
    masks = torch.ones(4, 16, dtype=torch.bool, device="cuda")
    grads = torch.ones(4, 100, device="cuda")
    calls = [
        lambda: torch.func.vmap(lambda t: ozk.fused_linear(t, W))(x),
        lambda: torch.func.vmap(lambda t: ozk.fused_linear(x[0], W, t))(b),
        lambda: torch.func.vmap(lambda t: ozk.fused_linear(x[0], W, residual=t))(x.new_zeros(4, 16, 40)),
        lambda: torch.func.vmap(lambda t: ozk.route_tokens(t, 2).weights)(logits),
        lambda: torch.func.vmap(lambda t: ozk.route_tokens(logits[0], 2, mask=t).weights)(masks),
        lambda: torch.func.vmap(lambda t: ozk.gradient_norm([t]))(grads),
        lambda: torch.func.vmap(lambda t: ozk.clip_gradients([t], 1.0))(grads),
        lambda: torch.func.grad(lambda t: ozk.fused_linear(t, W).float().sum())(x[0]),
        lambda: torch.func.grad(lambda t: ozk.fused_linear(x[0], t).float().sum())(W),
        lambda: torch.func.grad(lambda t: ozk.route_tokens(t, 2).balance_loss)(logits[0]),
        lambda: torch.func.jvp(lambda t: ozk.fused_linear(t, W), (x[0],), (x[1],)),
    ]
    t, r = x[0].clone().requires_grad_(), logits[0].clone().requires_grad_()
    y, w = ozk.fused_linear(t, W, activation="silu"), ozk.route_tokens(r, 2).weights
    calls += [
        lambda: torch.autograd.grad(y, t, torch.ones(3, 16, 40, device="cuda", dtype=F16), is_grads_batched=True),
        lambda: torch.autograd.grad(w, r, torch.ones(3, 16, 2, device="cuda"), is_grads_batched=True),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(RuntimeError):
            call()
            print("taken:", i)
    assert bool((grads == 1).all())
