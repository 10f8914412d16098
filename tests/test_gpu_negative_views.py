"""Imaginary parts of conjugates: tensors that stand for the negatives of their memory.  Each
call gives what it gives for a written-out copy."""
import pytest
import torch

import ozaki_triton_amd as ozk

pytestmark = pytest.mark.gpu

F16, F32 = torch.float16, torch.float32


def _negative(*shape, dtype=F32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    v = torch.view_as_complex(torch.randn(*shape, 2, device="cuda", generator=g).to(dtype)).conj().imag
    assert v.is_neg()
    return v


@pytest.mark.parametrize("M, N, K", [(5, 40, 1), (1, 1, 24), (70, 33, 24), (1, 40, 1)])
def test_fused_linear(gpu, M, N, K):
    ts = [_negative(*s, dtype=F16, seed=i) for i, s in enumerate(((M, K), (N, K), (N,), (M, N)))]
    dy = _negative(M, N, dtype=F16, seed=9)
    for act in (None, "gelu"):
        leaves = [t.detach().requires_grad_() for t in ts]
        plain = [t.detach().clone().requires_grad_() for t in ts]
        assert all(t.is_neg() for t in leaves) and not any(t.is_neg() for t in plain)
        call = lambda x, W, b, r: ozk.fused_linear(x, W, b, activation=act, residual=r)  # noqa: E731
        y, want = call(*leaves), call(*plain)
        assert torch.equal(y, want)
        for a, b in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(want, plain, dy.clone())):
            assert torch.equal(a, b)
        with torch.no_grad():
            assert torch.equal(call(*leaves), want)


@pytest.mark.parametrize("T, E, k", [(1, 8, 1), (40, 8, 2), (5, 1, 1)])
def test_route_tokens(gpu, T, E, k):
    logits, dw, dl = _negative(T, E), _negative(T, k, seed=1), _negative(seed=2)
    for normalize in (True, False):
        a, b = logits.detach().requires_grad_(), logits.clone().requires_grad_()
        r, want = (ozk.route_tokens(t, k, normalize=normalize) for t in (a, b))
        assert all(torch.equal(u, v) for u, v in zip(r, want))
        got, = torch.autograd.grad([r.weights, r.balance_loss], a, [dw, dl])
        exact, = torch.autograd.grad([want.weights, want.balance_loss], b, [dw.clone(), dl.clone()])
        assert torch.equal(got, exact)


@pytest.mark.parametrize("shape", [(), (1,), (1, 1), (50, 3)])
def test_clip_gradients(gpu, shape):
    beside = torch.randn(100, device="cuda")
    v = _negative(*shape)
    plain, norm = v.clone(), ozk.gradient_norm([v, beside])
    assert torch.equal(norm, ozk.gradient_norm([plain, beside]))
    want = [torch.empty_like(plain), torch.empty_like(beside)]
    ozk.clip_gradients([plain, beside], 1.0, out=want)
    for of, to in ((v, torch.empty_like(plain)), (plain, _negative(*shape, seed=4))):
        out = [to, torch.empty_like(beside)]
        ozk.clip_gradients([of, beside], 1.0, out=out)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    ozk.clip_gradients([v, beside], 1.0)
    assert torch.equal(v, want[0]) and torch.equal(beside, want[1])
