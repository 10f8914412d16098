"""The dense product with its epilogue, the router and gradient clipping: what
needs no GPU -- argument checks of the Python functions and of the C calls,
workspace sizes."""
import ctypes

import pytest
import torch

import ozaki_triton_amd as ozk
from ozaki_triton_amd import _lib
from ozaki_triton_amd.gradients import _is_dense

BF, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def _p(x=1 << 20):
    """A non-null pointer that no checked call reads."""
    return ctypes.c_void_p(x)


def _b(*v):
    return _lib.i64arr(v)


def _z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("args, kw, error", [
    ((_z(2, 8), _z(3, 8)), {}, RuntimeError),                                   # on the CPU
    ((_z(2, 8), _z(3, 8), _z(3)), dict(activation="gelu", residual=_z(2, 3)), RuntimeError),
    ((_z(2, 8), _z(3, 9)), {}, AssertionError),
    ((_z(2, 8), _z(1, 3, 8)), {}, AssertionError),
    ((torch.zeros((), dtype=BF), _z(3, 8)), {}, AssertionError),
    ((_z(2, 8), _z(3, 8, dtype=F16)), {}, AssertionError),
    ((_z(2, 8), _z(3, 8), _z(2)), {}, AssertionError),
    ((_z(2, 8), _z(3, 8), _z(3, dtype=F32)), {}, AssertionError),
    ((_z(2, 8), _z(3, 8)), dict(activation="tanh"), AssertionError),
    ((_z(2, 8), _z(3, 8)), dict(residual=_z(3)), AssertionError),               # not broadcast
    ((_z(2, 8), _z(3, 8)), dict(residual=_z(2, 3, dtype=F16)), AssertionError),
    ((_z(4, 2, 8), _z(3, 8)), dict(residual=_z(8, 3)), AssertionError),
])
def test_fused_linear_refuses(args, kw, error):
    with pytest.raises(error):
        ozk.fused_linear(*args, **kw)


@pytest.mark.parametrize("logits, k, mask, error", [
    (torch.zeros(4, 8), 2, None, RuntimeError),
    (torch.zeros(4, 8), 0, None, AssertionError),
    (torch.zeros(4, 8), 9, None, AssertionError),
    (torch.zeros(4, 0), 1, None, AssertionError),
    (torch.zeros(4, 1025), 1, None, AssertionError),
    (torch.zeros(2, 4, 8), 1, None, AssertionError),
    (torch.zeros(4, 8), 2, torch.ones(3, dtype=torch.bool), AssertionError),
    (torch.zeros(4, 8), 2, torch.ones(4), AssertionError),
])
def test_route_tokens_refuses(logits, k, mask, error):
    with pytest.raises(error):
        ozk.route_tokens(logits, k, mask=mask)


def test_gradients_refuse():
    g = [torch.zeros(4), torch.zeros(2, 3, dtype=BF)]
    for call in (ozk.gradient_norm, lambda t: ozk.clip_gradients(t, 1.0)):
        with pytest.raises(RuntimeError):
            call(g)
        with pytest.raises(AssertionError):
            call([])
    for bad in (-1.0, float("nan")):
        with pytest.raises((AssertionError, RuntimeError)):
            ozk.clip_gradients(g, bad)


def test_dense_layouts():
    t = torch.zeros(4, 6, 5)
    for dense in (t, t.mT, t.permute(2, 0, 1), t[1:3], t[:, :, :0], torch.zeros(()), t[:1].mT):
        assert _is_dense(dense), (dense.shape, dense.stride())
    for gaps in (t[:, :5], t[..., ::2], torch.zeros(1, 3).expand(4, 3), t.mT[:, 1:]):
        assert not _is_dense(gaps), (gaps.shape, gaps.stride())


def test_linear_c_calls_check_before_they_launch():
    L = _lib.load()
    f = lambda **k: L.ozk_linear(*{**dict(  # noqa: E731
        x=_p(), xs=8, W=_p(), ws=_b(8, 1), b=None, r=None, rs=0, act=0, M=4, N=3, K=8,
        d=_lib.OZK_BF16, y=_p(), ys=3, z=None, w=None, n=0, st=None), **k}.values())
    assert f(d=_lib.OZK_F32) == f(d=_lib.OZK_F64) == _lib.OZK_ERR_DTYPE
    assert f(ws=None) == f(x=None) == f(W=None) == f(y=None) == _lib.OZK_ERR_NULL
    assert f(M=-1) == f(ws=_b(8, 2)) == f(xs=-1) == f(ys=-1) == f(rs=-1) == f(act=5) == f(act=-1) \
        == f(M=1 << 40, K=1 << 30) == _lib.OZK_ERR_SHAPE
    assert f(xs=1 << 22) == f(ws=_b(1 << 22, 1)) == f(ws=_b(1, 1 << 22)) == _lib.OZK_ERR_TOO_LARGE
    assert f(M=0) == f(N=0) == _lib.OZK_OK
    assert f(M=128, K=1 << 14) == _lib.OZK_ERR_WORKSPACE      # few tiles, long K: partial sums
    assert f(w=_p(8), n=64) == _lib.OZK_ERR_WORKSPACE
    g = lambda **k: L.ozk_linear_backward(*{**dict(  # noqa: E731
        dy=_p(), ds=3, z=_p(), x=_p(), xs=8, W=_p(), ws=_b(8, 1), act=2, M=4, N=3, K=8,
        d=_lib.OZK_F16, dx=_p(), dxs=8, dW=_p(), dws=8, db=_p(), w=None, n=0, st=None), **k}.values())
    assert g(d=_lib.OZK_F32) == _lib.OZK_ERR_DTYPE
    assert g(dy=None) == g(z=None) == g(x=None) == g(W=None) == g(ws=None) == _lib.OZK_ERR_NULL
    assert g(ds=-1) == g(dxs=-1) == g(dws=-1) == g(act=9) == g(K=-1) == _lib.OZK_ERR_SHAPE
    assert g() == g(w=_p(16), n=1 << 20) == g(w=_p(), n=16) == _lib.OZK_ERR_WORKSPACE
    assert g(ds=1 << 22) == _lib.OZK_ERR_TOO_LARGE
    n = ctypes.c_size_t(0)
    q = lambda act, want: (L.ozk_linear_backward_workspace_bytes(  # noqa: E731
        None, 4096, None, 2048, None, _b(2048, 1), act, 8192, 4096, 2048, want, ctypes.byref(n)), n.value)
    assert q(0, 3) == (_lib.OZK_OK, 0)                        # dy is dz
    assert q(2, 3) == (_lib.OZK_OK, 8192 * 4096 * 2)
    assert q(2, 4)[1] < 8192 * 4096                             # db alone: no dz
    assert q(2, 8)[0] == q(7, 1)[0] == _lib.OZK_ERR_SHAPE


def test_route_c_calls_check_before_they_launch():
    L = _lib.load()
    f = lambda **k: L.ozk_route(*{**dict(  # noqa: E731
        l=_p(), d=_lib.OZK_F32, ls=8, m=None, T=4, E=8, k=2, norm=1, e=_p(), w=_p(), o=_p(), p=_p(),
        off=_p(), c=_p(), loss=_p(), ws=None, n=0, st=None), **k}.values())
    assert f(d=_lib.OZK_F64) == f(d=_lib.OZK_I8) == _lib.OZK_ERR_DTYPE
    assert f(E=0) == f(k=0) == f(k=9) == f(T=-1) == f(ls=-1) == _lib.OZK_ERR_SHAPE
    assert f(E=1025) == f(T=1 << 31) == f(T=1 << 29, k=8) == _lib.OZK_ERR_TOO_LARGE
    for name in ("l", "e", "w", "o", "p", "off", "c", "loss"):
        assert f(**{name: None}) == _lib.OZK_ERR_NULL, name
    assert f(T=1 << 15) == f(T=1 << 15, ws=_p(8), n=1 << 20) == _lib.OZK_ERR_WORKSPACE
    b = lambda **k: L.ozk_route_backward(*{**dict(  # noqa: E731
        l=_p(), d=_lib.OZK_F32, ls=8, m=None, T=4, E=8, k=2, norm=1, e=_p(), w=_p(), c=_p(), dw=_p(),
        dl=_p(), out=_p(), st=None), **k}.values())
    assert b(d=_lib.OZK_F64) == _lib.OZK_ERR_DTYPE
    assert b(k=9) == _lib.OZK_ERR_SHAPE
    for name in ("l", "e", "w", "c", "out"):
        assert b(**{name: None}) == _lib.OZK_ERR_NULL, name
    assert b(T=0) == _lib.OZK_OK
    # tokens of a workgroup fit its LDS whatever E and k are; the places stay below 2^31
    n = ctypes.c_size_t(0)
    for E in (1, 7, 8, 64, 500, 1024):
        for k in (1, min(E, 8), E):
            for T in (0, 1, 64, 4097, 1 << 20):
                assert L.ozk_route_workspace_bytes(T, E, k, ctypes.byref(n)) == _lib.OZK_OK
                assert n.value % (8 * E) == 0 and n.value < 1 << 33


def test_gradient_c_calls_check_before_they_launch():
    L = _lib.load()
    vp = lambda *v: (ctypes.c_void_p * len(v))(*v)  # noqa: E731
    ints = lambda *v: (ctypes.c_int * len(v))(*v)  # noqa: E731
    a, n = 1 << 20, ctypes.c_size_t(0)
    assert L.ozk_gradient_norm_workspace_bytes(2, ctypes.byref(n)) == _lib.OZK_OK
    room = n.value
    two = dict(g=vp(a, a + 4096), c=_b(16, 16), d=ints(_lib.OZK_F32, _lib.OZK_BF16), t=2, norm=_p(),
               ws=_p(1 << 24), n=room, st=None)
    f = lambda **k: L.ozk_gradient_norm(*{**two, **k}.values())  # noqa: E731
    assert f(t=-1) == f(c=_b(16, -1)) == _lib.OZK_ERR_SHAPE
    assert f(g=None) == f(c=None) == f(d=None) == f(norm=None) == f(g=vp(a, None)) == _lib.OZK_ERR_NULL
    assert f(d=ints(_lib.OZK_F32, _lib.OZK_F64)) == _lib.OZK_ERR_DTYPE
    assert f(ws=None) == f(n=room - 1) == f(ws=_p(8)) == _lib.OZK_ERR_WORKSPACE
    c = lambda g, o, counts=(16, 16), limit=1.0, **k: L.ozk_clip_gradients(  # noqa: E731
        vp(*g), o if o is None else vp(*o), _b(*counts), ints(_lib.OZK_F32, _lib.OZK_F32), 2, limit,
        *{**dict(norm=_p(), ws=_p(1 << 24), n=8, st=None), **k}.values())
    for limit in (-1.0, float("nan")):
        assert c((a, a + 64), (a, a + 64), limit=limit, n=room) == _lib.OZK_ERR_SHAPE
    assert c((a, a + 64), None, n=room) == c((a, a + 64), (a, None), n=room) == _lib.OZK_ERR_NULL
    assert c((a, a + 64), (a, a + 64)) == _lib.OZK_ERR_WORKSPACE
    for g, o in (((a, a), (a, a)),                     # the same tensor twice
                 ((a, a + 60), (a, a + 60)),           # one on the other's end
                 ((a, a + 64), (a + 64, a)),           # results exchanged
                 ((a, a + 64), (a + 4, a + 4096)),     # a result beside its own tensor
                 ((a, a + 64), (a + 4096, a + 4100)),  # results on each other
                 ((a, a + 64), (a + 4096, a + 32))):   # a result on another tensor
        assert c(g, o, n=room) == _lib.OZK_ERR_SHAPE, (g, o)


def test_module_on_pytorchs_side():
    """It is built for this interpreter and torch, and takes nothing that is off the GPU."""
    m = _lib.torch_binding()
    x, W = _z(2, 8), _z(3, 8)
    assert m.linear(x, W, None, None, 0, 0) is None
    assert m.route(torch.zeros(4, 8), None, 2, True, 0) is None
    assert m.gradient_norm([torch.zeros(4)], 0) is None and m.gradient_norm([], 0) is None
    assert m.clip_gradients([torch.zeros(4)], [torch.zeros(4)], 1.0, 0) is None


def test_a_missing_module_is_named(monkeypatch):
    import builtins
    real = builtins.__import__

    def absent(name, globals=None, locals=None, fromlist=(), level=0):
        if fromlist and "_ozk_torch" in fromlist:
            raise ImportError("absent")
        return real(name, globals, locals, fromlist, level)
    monkeypatch.setattr(_lib, "_binding", None)
    monkeypatch.setattr(builtins, "__import__", absent)
    with pytest.raises(ImportError, match="_ozk_torch.so is not built"):
        _lib.torch_binding()


def test_wide_results_have_the_gradients_of_one_row():
    """Rows of 2^22 elements: one row of them needs no distance between rows, with an activation as without."""
    L, n = _lib.load(), ctypes.c_size_t(0)
    q = lambda M, N, act, dy: L.ozk_linear_backward_workspace_bytes(  # noqa: E731
        None, dy, None, 8, None, _b(8, 1), act, M, N, 8, 7, ctypes.byref(n))
    for act in (0, 2):
        for N in (1 << 22, (1 << 22) - 3, (1 << 23) + 5):
            assert q(1, N, act, 0) == _lib.OZK_OK
    assert q(2, 1 << 22, 0, 1 << 22) == q(2, 1 << 22, 2, 1 << 22) == _lib.OZK_ERR_TOO_LARGE
    assert q(2, (1 << 22) - 8, 2, (1 << 22) - 8) == q(2, (1 << 22) - 1, 0, (1 << 22) - 1) == _lib.OZK_OK
