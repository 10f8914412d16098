"""Operators for linear layers: what needs no GPU -- argument checks of the
Python functions and of the C calls, workspace sizes."""
import ctypes

import pytest
import torch

import ozaki_triton_amd as ozk
from ozaki_triton_amd import _lib

BF, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
OFF = torch.tensor([0, 2, 4], dtype=torch.int32)


def _p(x=1 << 20):
    """A non-null pointer that no checked call reads."""
    return ctypes.c_void_p(x)


def _b(*v):
    return _lib.i64arr(v)


@pytest.mark.parametrize("A, B, offsets, error", [
    (torch.zeros(4, 8, dtype=BF), torch.zeros(2, 8, 3, dtype=BF), OFF, RuntimeError),      # on the CPU
    (torch.zeros(4, 8, 1, dtype=BF), torch.zeros(2, 8, 3, dtype=BF), OFF, AssertionError),
    (torch.zeros(4, 8, dtype=BF), torch.zeros(8, 3, dtype=BF), OFF, AssertionError),
    (torch.zeros(4, 7, dtype=BF), torch.zeros(2, 8, 3, dtype=BF), OFF, AssertionError),
    (torch.zeros(4, 8, dtype=BF), torch.zeros(2, 8, 3, dtype=F16), OFF, AssertionError),
    (torch.zeros(4, 8, dtype=BF), torch.zeros(3, 8, 3, dtype=BF), OFF, AssertionError),    # G + 1 offsets
    (torch.zeros(4, 8, dtype=BF), torch.zeros(2, 8, 3, dtype=BF), OFF.float(), NotImplementedError),
])
def test_grouped_matmul_refuses(A, B, offsets, error):
    with pytest.raises(error):
        ozk.grouped_matmul(A, B, offsets)
    with pytest.raises(error):
        ozk.grouped_matmul_backward(torch.zeros(4, 3, dtype=BF), A, B, offsets)


def test_grouped_matmul_backward_refuses_other_gradients():
    A, B = torch.zeros(4, 8, dtype=BF), torch.zeros(2, 8, 3, dtype=BF)
    for dC in (torch.zeros(4, 4, dtype=BF), torch.zeros(4, 3, dtype=F16)):
        with pytest.raises((AssertionError, RuntimeError)):
            ozk.grouped_matmul_backward(dC, A, B, OFF)


def _w4(N=4, K=40, group=32, dtype=BF, zeros=True):
    groups = -(-K // group)
    return (torch.zeros(N, (K + 31) // 32 * 16, dtype=torch.uint8), torch.ones(N, groups, dtype=dtype),
            torch.zeros(N, groups, dtype=torch.uint8) if zeros else None)


def test_w4_refuses():
    x = torch.zeros(2, 40, dtype=BF)
    p, s, z = _w4()
    with pytest.raises(RuntimeError):
        ozk.matmul_w4(x, p, s, z, group_size=32)            # on the CPU
    for args, kw in (((x, p, s, z), dict(group_size=48)), ((x, p.int(), s, z), dict(group_size=32)),
                     ((x, p[:, :16], s, z), dict(group_size=32)),
                     ((x, p, s[:, :1], z), dict(group_size=32)),
                     ((x, p, s, z.int()), dict(group_size=32)),
                     ((x, p, s.half(), z), dict(group_size=32)),
                     ((x[:, :0], p, s, z), dict(group_size=32))):
        with pytest.raises(AssertionError):
            ozk.matmul_w4(*args, **kw)
    with pytest.raises(AssertionError):
        ozk.quantize_w4(torch.zeros(3, 4, 5))
    with pytest.raises(AssertionError):
        ozk.quantize_w4(torch.zeros(4, 64), 16)
    with pytest.raises(RuntimeError):
        ozk.quantize_w4(torch.zeros(4, 64), 32)
    with pytest.raises(AssertionError):
        ozk.dequantize_w4(p, s, z, group_size=32, K=200)
    with pytest.raises(RuntimeError):
        ozk.dequantize_w4(p, s, z, group_size=32, K=40)


def test_orthogonalize_refuses():
    G = torch.zeros(4, 8)
    with pytest.raises(RuntimeError):
        ozk.orthogonalize(G)
    for kw in (dict(steps=0), dict(steps=65), dict(coefficients=(1.0, 2.0)),
               dict(steps=3, coefficients=[(1.0, 2.0, 3.0)] * 2)):
        with pytest.raises(AssertionError):
            ozk.orthogonalize(G, **kw)
    with pytest.raises(AssertionError):
        ozk.orthogonalize(G[0])


def test_c_calls_check_before_they_launch():
    L = _lib.load()
    g = lambda **k: L.ozk_grouped_matmul(*{**dict(  # noqa: E731
        A=_p(), a=8, B=_p(), bs=_b(24, 3, 1), off=_p(), ob=4, T=4, K=8, N=3, G=2,
        d=_lib.OZK_BF16, C=_p(), c=3, ws=None, n=0, st=None), **k}.values())
    assert g(d=_lib.OZK_F32) == _lib.OZK_ERR_DTYPE
    assert g(ob=2) == _lib.OZK_ERR_DTYPE
    assert g(bs=None) == g(C=None) == g(off=None) == g(A=None) == g(B=None) == _lib.OZK_ERR_NULL
    assert g(T=-1) == g(bs=_b(24, 3, 2)) == g(c=-1) == g(a=-1) == _lib.OZK_ERR_SHAPE
    assert g(T=1 << 40, K=1 << 30) == _lib.OZK_ERR_SHAPE
    assert g(a=1 << 22) == g(bs=_b(24, 1 << 22, 1)) == _lib.OZK_ERR_TOO_LARGE
    assert g(T=0) == g(N=0) == _lib.OZK_OK
    w = lambda **k: L.ozk_grouped_matmul_wgrad(*{**dict(  # noqa: E731
        A=_p(), a=8, D=_p(), ds=3, off=_p(), ob=4, T=4, K=8, N=3, G=2, d=_lib.OZK_BF16,
        dB=_p(), db=_b(24, 3), ws=None, n=0, st=None), **k}.values())
    assert w(d=_lib.OZK_I8) == _lib.OZK_ERR_DTYPE
    assert w(db=None) == w(dB=None) == w(A=None) == w(D=None) == w(off=None) == _lib.OZK_ERR_NULL
    assert w(K=-1) == w(db=_b(24, -3)) == _lib.OZK_ERR_SHAPE
    assert w(ds=1 << 22) == _lib.OZK_ERR_TOO_LARGE
    assert w(T=1 << 16, G=1) == _lib.OZK_ERR_WORKSPACE       # few tiles, many rows: partial sums
    assert w(G=0) == _lib.OZK_OK
    m = lambda **k: L.ozk_matmul_w4(*{**dict(  # noqa: E731
        x=_p(), d=_lib.OZK_BF16, xs=64, p=_p(), ps=32, s=_p(), sd=_lib.OZK_BF16, ss=2, z=None,
        zs=0, group=32, M=2, N=4, K=64, y=_p(), ys=4, ws=None, n=0, st=None), **k}.values())
    assert m(d=_lib.OZK_F64) == m(sd=_lib.OZK_F16) == _lib.OZK_ERR_DTYPE
    assert m(group=16) == m(K=0) == m(M=-1) == m(ps=24) == m(ps=16) == m(p=_p(8)) == _lib.OZK_ERR_SHAPE
    assert m(x=None) == m(p=None) == m(s=None) == m(y=None) == _lib.OZK_ERR_NULL
    assert m(K=1 << 14, ps=1 << 13) == _lib.OZK_ERR_WORKSPACE
    assert m(M=0) == m(N=0) == _lib.OZK_OK
    o = lambda **k: L.ozk_orthogonalize(*{**dict(  # noqa: E731
        G=_p(), d=_lib.OZK_F32, b=1, M=4, N=8, gs=_b(32, 8), co=(ctypes.c_double * 3)(1, 2, 3),
        steps=1, eps=1e-7, out=_p(), os=_b(32, 8), ws=None, n=0, st=None), **k}.values())
    assert o(d=_lib.OZK_F64) == _lib.OZK_ERR_DTYPE
    assert o(steps=0) == o(steps=65) == o(M=-1) == o(gs=_b(-1, 8)) == _lib.OZK_ERR_SHAPE
    assert o(co=None) == o(gs=None) == o(os=None) == o(G=None) == o(out=None) == _lib.OZK_ERR_NULL
    assert o() == o(ws=_p(8), n=1 << 30) == _lib.OZK_ERR_WORKSPACE
    assert o(b=1 << 16) == _lib.OZK_ERR_TOO_LARGE
    assert o(b=0) == o(M=0) == _lib.OZK_OK


def _bytes(fn, *args):
    n = ctypes.c_size_t(0)
    assert getattr(_lib.load(), fn)(*args, ctypes.byref(n)) == _lib.OZK_OK
    return n.value


def test_workspace_sizes():
    # many tiles, or few rows: no partial sums; one tile under many rows: some
    assert _bytes("ozk_grouped_matmul_wgrad_workspace_bytes", 0, 2048, 0, 1024, 16384, 2048, 1024, 32) == 0
    assert _bytes("ozk_grouped_matmul_wgrad_workspace_bytes", 0, 64, 0, 64, 64, 64, 64, 1) == 0
    assert _bytes("ozk_grouped_matmul_wgrad_workspace_bytes", 0, 64, 0, 64, 1 << 15, 64, 64, 1) % (64 * 64 * 4) == 0
    assert _bytes("ozk_grouped_matmul_wgrad_workspace_bytes", 0, 64, 0, 64, 1 << 15, 64, 64, 1) > 0
    # rows that are no whole 16-byte pieces, by size, distance or address: copies
    # where there is enough to multiply
    w = lambda a, sa, T, K, N: _bytes("ozk_grouped_matmul_workspace_bytes", a, sa, 0,  # noqa: E731
                                      _b(K * N, N, 1), T, K, N, 4)
    assert w(0, 1024, 8192, 1024, 1024) == w(0, 1001, 64, 1001, 1024) == 0
    assert w(0, 1001, 8192, 1001, 1024) == w(2, 1008, 8192, 1001, 1024) == 8192 * 1008 * 2
    assert w(2, 1024, 8192, 1024, 1024) == w(0, 1025, 8192, 1024, 1024) == 8192 * 1024 * 2
    assert w(0, 1001, 8192, 1001, 1003) == 8192 * 1008 * 2 + 4 * 1001 * 1008 * 2
    assert _bytes("ozk_matmul_w4_workspace_bytes", _lib.OZK_BF16, 1, 0, 64, 32) == 0
    assert _bytes("ozk_matmul_w4_workspace_bytes", _lib.OZK_BF16, 1, 64, 1 << 14, 128) % (64 * 4) == 0
    # X twice and two square matrices, 4 bytes an element, columns up to whole 32
    one = _bytes("ozk_orthogonalize_workspace_bytes", 1, 64, 100, 1)
    two = _bytes("ozk_orthogonalize_workspace_bytes", 1, 64, 100, 2)
    assert two - one == 64 * 128 * 4 and one >= 64 * 128 * 4 + 2 * 64 * 64 * 4
    assert _bytes("ozk_orthogonalize_workspace_bytes", 1, 100, 64, 2) == two


@pytest.mark.parametrize("m, n, squares", [(64, 127, 2), (64, 128, 5), (64, 150, 5), (64, 192, 5),
                                           (700, 1399, 2), (700, 1400, 5), (700, 1500, 5), (1, 1, 2)])
def test_orthogonalize_workspace_holds_the_chain(m, n, squares):
    """From twice as long as high on the last steps run on the square matrix alone,
    which takes three more of them."""
    up = lambda v: -(-v // 32) * 32  # noqa: E731
    for batch in (1, 3):
        want = batch * (2 * m * up(n) + squares * m * up(m)) * 4
        for shape in ((m, n), (n, m)):   # and the partial sums of the norm
            got = _bytes("ozk_orthogonalize_workspace_bytes", batch, *shape, 5)
            assert want < got <= want + 64 * 1024


def test_strides_of_single_rows_mean_nothing():
    """A dim of size 1 keeps the stride of the tensor it was cut from, contiguous() leaves
    it, and the kernels have a limit."""
    from ozaki_triton_amd.linear import _MAX_STRIDE, _matrices, _rows
    far = _MAX_STRIDE + 8
    strided = lambda size, stride: torch.empty(1, dtype=BF).as_strided(  # noqa: E731
        size, stride) if 0 in size or all(n == 1 for n in size) else \
        torch.empty(sum((n - 1) * s for n, s in zip(size, stride)) + 1, dtype=BF).as_strided(size, stride)
    for t in (strided((1, 64), (far, 1)), strided((1, 1), (far, far)), strided((0, 64), (far, 1)),
              strided((3, 1), (2, far)), strided((1, 8), (far, 3)), strided((3, 8), (far, 1))):
        r, pitch = _rows(t)
        assert r.shape == t.shape and pitch < _MAX_STRIDE
        assert r.shape[1] <= 1 or r.stride(1) == 1
        assert r.shape[0] <= 1 or pitch == r.stride(0)
    for size, stride in (((1, 1, 64), (far, far, 1)), ((1, 1, 1), (far, far, far)), ((1, 1, 1), (7, 7, 7)),
                         ((1, 8, 1), (far, 1, far)), ((1, 8, 1), (far, 2, far)), ((1, 8, 1), (far, far, 1)),
                         ((1, 1, 8), (far, far, 3)), ((2, 1, 8), (far, far, 1)), ((1, 4, 3), (far, 3, 1)),
                         ((1, 4, 3), (far, 1, 4)), ((2, 4, 3), (2, 6, 2)), ((0, 4, 3), (far, far, far))):
        t = strided(size, stride)
        b, (s_g, s_k, s_n) = _matrices(t)
        assert b.shape == t.shape and 1 in (s_k, s_n) and max(s_k, s_n) < _MAX_STRIDE
        for dim, s in enumerate((s_g, s_k, s_n)):
            assert b.shape[dim] <= 1 or b.numel() == 0 or s == b.stride(dim), (size, stride)
