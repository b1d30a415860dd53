"""Checks of the arguments of the experts' operators and of the 4-bit matrices: no GPU needed, every call is refused (or has
nothing to do) before anything is launched.  And the plain implementations against differences."""
import ctypes

import numpy as np
import pytest

import experts_oracle as ref

P = 1 << 20  # an address that nothing looks at


def _refused(miw, code, call, *args, **kw):
    with pytest.raises(miw.MIWError) as e:
        call(*args, **kw)
    assert e.value.code == code, e.value


def test_route_refusals(miw):
    E, L = miw.EXPERTS, miw._lib
    ok = dict(tokens=8, experts=16, top=2)
    arrays = [P] * 6
    _refused(miw, L.ERR_INVALID_SHAPE, E.route, *arrays, **{**ok, "top": 0})
    _refused(miw, L.ERR_INVALID_SHAPE, E.route, *arrays, **{**ok, "top": 17})
    _refused(miw, L.ERR_INVALID_SHAPE, E.route, *arrays, tokens=8, experts=4, top=5)
    _refused(miw, L.ERR_INVALID_SHAPE, E.route, *arrays, **{**ok, "experts": 1025})
    _refused(miw, L.ERR_INVALID_SHAPE, E.route, *arrays, **{**ok, "tokens": -1})
    _refused(miw, L.ERR_INVALID_SHAPE, E.route, *arrays, tokens=1 << 28, experts=16, top=8)
    _refused(miw, L.ERR_INVALID_VALUE, E.route, *arrays, **ok, ld=15)
    for i in range(6):
        _refused(miw, L.ERR_NULL_POINTER, E.route, *[None if i == j else P for j in range(6)], **ok)
        _refused(miw, L.ERR_MISALIGNED, E.route, *[P + 1 if i == j else P for j in range(6)], **ok)
    assert E.route_workspace(8, 16, 2) == 0
    need = E.route_workspace(5000, 16, 2)
    assert need > 0 and need % 4 == 0
    _refused(miw, L.ERR_NULL_POINTER, E.route, *arrays, tokens=5000, experts=16, top=2)
    lib = L.load()
    assert lib.miw_route(1, 5000, 16, 2, 0, 0, P, P, P, P, P, P, P, need - 1, None) == L.ERR_INVALID_VALUE
    assert lib.miw_route(3, 8, 16, 2, 0, 0, P, P, P, P, P, P, None, 0, None) == L.ERR_INVALID_TYPE
    assert lib.miw_route_workspace(8, 16, 2, None) == L.ERR_NULL_POINTER
    grad = [P] * 5
    _refused(miw, L.ERR_INVALID_VALUE, E.route_grad, *grad, **ok, ldd=3)
    for i in range(5):
        _refused(miw, L.ERR_NULL_POINTER, E.route_grad, *[None if i == j else P for j in range(5)], **ok)
    E.route_grad(None, None, None, None, None, tokens=0, experts=16, top=2)  # nothing to do


def test_grouped_refusals(miw):
    E, L = miw.EXPERTS, miw._lib
    ok = dict(rows=10, groups=3, n=8, k=16)
    four = [P] * 4
    for i in range(4):
        _refused(miw, L.ERR_NULL_POINTER, E.grouped_gemm, *[None if i == j else P for j in range(4)], **ok)
        _refused(miw, L.ERR_MISALIGNED, E.grouped_gemm, *[P + 1 if i == j else P for j in range(4)], **ok)
    for bad in (dict(n=0), dict(k=0), dict(groups=0), dict(rows=-1), dict(rows=1 << 31), dict(n=1 << 27), dict(a_rows=9), dict(a_rows=-1)):
        _refused(miw, L.ERR_INVALID_SHAPE, E.grouped_gemm, *four, **{**ok, **bad})
    for bad in (dict(lda=15), dict(ldw=15), dict(ldd=7), dict(stride_w=-8), dict(lda=1 << 40)):
        _refused(miw, L.ERR_INVALID_VALUE, E.grouped_gemm, *four, **{**ok, **bad})
    _refused(miw, L.ERR_INVALID_VALUE, E.grouped_gemm, *four, **ok, w_layout=miw.WMMA.RowMajor, ldw=7)
    _refused(miw, L.ERR_INVALID_SHAPE, E.grouped_gemm, *four, **ok, gather=P)  # a_rows is not known
    _refused(miw, L.ERR_INVALID_TYPE, E.grouped_gemm, *four, **ok, dtype=np.float32)
    _refused(miw, L.ERR_INVALID_TYPE, E.grouped_gemm, *four, **ok, d_type=miw.BFloat16)
    _refused(miw, L.ERR_INVALID_SHAPE, E.grouped_gemm, *four, **{**ok, "n": 7}, epilogue=E.GATED_SILU)
    with pytest.raises(ValueError):
        E.grouped_gemm(*four, **ok, epilogue="relu")
    with pytest.raises(TypeError):
        E.grouped_gemm(*four, **ok, dtype=np.int8)
    E.grouped_gemm(None, None, None, None, **{**ok, "rows": 0})
    lib = L.load()
    assert lib.miw_grouped_gemm(0, 0, 2, 0, 10, 3, 8, 16, 0, 0, 0, 0, 0, P, P, P, P, None, None) == L.ERR_INVALID_LAYOUT
    assert lib.miw_grouped_gemm(0, 0, 1, 2, 10, 3, 8, 16, 0, 0, 0, 0, 0, P, P, P, P, None, None) == L.ERR_INVALID_VALUE
    ok = dict(rows=10, groups=3, m=8, n=16)
    for i in range(4):
        _refused(miw, L.ERR_NULL_POINTER, E.grouped_wgrad, *[None if i == j else P for j in range(4)], **ok)
    for bad in (dict(m=0), dict(n=0), dict(groups=65537), dict(b_rows=9)):
        _refused(miw, L.ERR_INVALID_SHAPE, E.grouped_wgrad, *four, **{**ok, **bad})
    for bad in (dict(lda=7), dict(ldb=15), dict(ldd=15), dict(stride_d=127)):
        _refused(miw, L.ERR_INVALID_VALUE, E.grouped_wgrad, *four, **ok, **bad)
    _refused(miw, L.ERR_INVALID_TYPE, E.grouped_wgrad, *four, **ok, d_type=miw.BFloat16)


def test_combine_refusals(miw):
    E, L = miw.EXPERTS, miw._lib
    ok = dict(tokens=4, top=2, n=8, rows=8)
    for i in range(3):
        _refused(miw, L.ERR_NULL_POINTER, E.combine, *[None if i == j else P for j in range(3)], **ok)
        _refused(miw, L.ERR_MISALIGNED, E.combine, *[P + 1 if i == j else P for j in range(3)], **ok)
    for bad in (dict(tokens=-1), dict(top=0), dict(n=0), dict(rows=-1), dict(tokens=1 << 24)):
        _refused(miw, L.ERR_INVALID_SHAPE, E.combine, P, P, P, **{**ok, **bad})
    for bad in (dict(ldh=7), dict(ldy=7)):
        _refused(miw, L.ERR_INVALID_VALUE, E.combine, P, P, P, **ok, **bad)
    _refused(miw, L.ERR_INVALID_TYPE, E.combine, P, P, P, **ok, dtype=np.float32)
    E.combine(None, None, None, **{**ok, "tokens": 0})
    for i in range(4):  # (the fifth, dgates, may be left out)
        _refused(miw, L.ERR_NULL_POINTER, E.combine_grad, *[None if i == j else P for j in range(5)], **ok)
    _refused(miw, L.ERR_MISALIGNED, E.combine_grad, P, P, P, P, P + 2, **ok)
    _refused(miw, L.ERR_INVALID_VALUE, E.combine_grad, P, P, P, P, P, **ok, lddh=7)


def test_mxfp4_refusals(miw):
    Q, L = miw.MXFP4, miw._lib
    ok = dict(rows=6, k=100)
    for call in (Q.quantize, Q.dequantize):
        for i in range(3):
            _refused(miw, L.ERR_NULL_POINTER, call, *[None if i == j else P for j in range(3)], **ok)
        for bad in (dict(rows=-1), dict(k=0), dict(k=1 << 27)):
            _refused(miw, L.ERR_INVALID_SHAPE, call, P, P, P, **{**ok, **bad})
        for bad in (dict(ld=99), dict(ldq=48), dict(ldq=72), dict(lds=5), dict(lds=7)):
            _refused(miw, L.ERR_INVALID_VALUE, call, P, P, P, **ok, **bad)
        call(None, None, None, rows=0, k=5)
    _refused(miw, L.ERR_MISALIGNED, Q.quantize, P, P + 8, P, **ok)
    _refused(miw, L.ERR_MISALIGNED, Q.dequantize, P, P + 8, P, **ok)
    assert Q.codes_bytes(6, 100) == 6 * 64 and Q.scales_bytes(5, 257) == 2 * 6 * 8
    ok = dict(m=5, n=6, k=64)
    for i in range(5):
        _refused(miw, L.ERR_NULL_POINTER, Q.gemm, *[None if i == j else P for j in range(5)], **ok)
    for i in range(4):
        _refused(miw, L.ERR_MISALIGNED, Q.gemm, *[P + 8 if i == j else P for j in range(5)], **ok)
    for bad in (dict(lda=16), dict(ldb=40), dict(lds_a=4), dict(lds_b=9), dict(ldd=5)):
        _refused(miw, L.ERR_INVALID_VALUE, Q.gemm, *[P] * 5, **ok, **bad)
    ok = dict(rows=5, groups=2, n=6, k=64)
    for i in range(6):
        _refused(miw, L.ERR_NULL_POINTER, Q.grouped_gemm, *[None if i == j else P for j in range(6)], **ok)
    _refused(miw, L.ERR_MISALIGNED, Q.grouped_gemm, *[P] * 6, **ok, stride_w=8)
    _refused(miw, L.ERR_MISALIGNED, Q.grouped_gemm, *[P] * 6, **ok, stride_ws=24)
    _refused(miw, L.ERR_INVALID_SHAPE, Q.grouped_gemm, *[P] * 6, **ok, gather=P)
    Q.gemm(None, None, None, None, None, m=0, n=6, k=64)


def test_valid_calls_need_init(miw):
    """A call that is right in itself is refused without a device (in a process that never chose one)."""
    lib = ctypes.CDLL(miw._lib.LIB_PATH)
    if lib.miw_init(0) == 0:
        pytest.skip("there is a device")
    E, L = miw.EXPERTS, miw._lib
    _refused(miw, L.ERR_NOT_INITIALIZED, E.combine, P, P, P, tokens=4, top=2, n=8, rows=8)
    _refused(miw, L.ERR_NOT_INITIALIZED, E.grouped_gemm, P, P, P, P, rows=10, groups=3, n=8, k=16)
    _refused(miw, L.ERR_NOT_INITIALIZED, miw.MXFP4.quantize, P, P, P, rows=6, k=100)


@pytest.mark.parametrize("over_all", [False, True])
def test_route_gradient_formula_against_differences(over_all):
    rng = np.random.default_rng(5)
    z = rng.normal(size=(7, 12))
    z[2, 3] = -np.inf
    top, h = 4, 1e-6
    chosen = ref.route(z, top, over_all)[0]
    dg = rng.normal(size=(7, top))
    got = ref.route_grad(z, chosen, dg, over_all)
    for t in range(7):
        for e in range(12):
            if np.isneginf(z[t, e]):
                continue
            up, down = z.copy(), z.copy()
            up[t, e] += h
            down[t, e] -= h
            slope = (ref.route(up, top, over_all)[1] - ref.route(down, top, over_all)[1]) * dg / (2 * h)
            # central differences of a smooth function: h^2 times its third derivative, and rounding 2^-52 / h
            assert abs(slope.sum() - got[t, e]) < 1e-8


def test_grouped_gradients_against_differences():
    """dX = dY W^T and dW = X^T dY of Y = X[gather] W_g, where the oracle's product is linear in each."""
    rng = np.random.default_rng(6)
    offsets, gather = np.array([0, 3, 3, 5]), np.array([1, 0, 1, 2, 0])
    x, w, dy = rng.normal(size=(3, 4)), rng.normal(size=(3, 4, 6)), rng.normal(size=(5, 6))
    loss = lambda x, w: (ref.grouped(x, w, offsets, gather, np.zeros((5, 6)))[0] * dy).sum()  # noqa: E731
    dx_rows = ref.grouped(dy, w.transpose(0, 2, 1), offsets, None, np.zeros((5, 4)))[0]
    dx = np.zeros((3, 4))
    np.add.at(dx, gather, dx_rows)
    for i in range(3):
        for c in range(4):
            step = np.zeros((3, 4))
            step[i, c] = 1.0
            assert abs(loss(x + step, w) - loss(x - step, w) - 2 * dx[i, c]) < 1e-11
    for g in range(3):
        rows = slice(offsets[g], offsets[g + 1])
        dw = x[gather[rows]].T @ dy[rows]
        for i in range(4):
            step = np.zeros((3, 4, 6))
            step[g, i, 2] = 1.0
            assert abs(loss(x, w + step) - loss(x, w - step) - 2 * dw[i, 2]) < 1e-11
