"""Operands whose rows and groups lie more than 4 GiB, or 2^31 elements, from the first: every offset is one of 64 bits.  Whole
numbers, so that sums are exact."""
import numpy as np
import pytest

import experts_oracle as ref

pytestmark = pytest.mark.gpu


class Rows:
    """Rows (of the last axis) at a pitch in bytes, groups at a stride, in memory that is otherwise not written."""

    def __init__(self, gpu, shape, dtype, pitch, stride=0):
        self.lib, self.shape, self.dtype = gpu._lib.load(), shape, np.dtype(dtype)
        self.at = [g * stride + r * pitch for g in range(shape[0]) for r in range(shape[1])]
        self.array = gpu.DeviceArray.undef(np.uint8, self.at[-1] + shape[2] * self.dtype.itemsize)
        assert self.at[-1] > 1 << 32

    def put(self, values):
        values = np.ascontiguousarray(values, self.dtype).reshape(len(self.at), -1)
        for at, row in zip(self.at, values):
            assert self.lib.miw_memcpy_h2d(self.array.ptr + at, row.ctypes.data, row.nbytes) == 0
        return self

    def get(self):
        out = np.empty((len(self.at), self.shape[2]), self.dtype)
        for at, row in zip(self.at, out):
            assert self.lib.miw_memcpy_d2h(row.ctypes.data, self.array.ptr + at, row.nbytes) == 0
        return out.reshape(self.shape)


def _numbers(rng, *shape):
    return rng.integers(-2, 3, shape).astype(np.float16)


def _sizes(gpu, offsets):
    return ref.upload(gpu, np.array(offsets, np.int32))


# ldw of 64: weights dense within a group (tiles); of 2^23: a row of weights every 16 MiB (the kernel for any pitch).
@pytest.mark.parametrize("layout", ["col", "row"])
@pytest.mark.parametrize("ldw", [64, 1 << 23])
def test_grouped_gemm(gpu, ldw, layout):
    rng = np.random.default_rng(1)
    rows, groups, n, k, pitch, stride = 140, 3, 64, 64, 1 << 25, 3 << 30
    a, w, offsets, gather = _numbers(rng, rows, k), _numbers(rng, groups, n, k), [3, 20, 101, 138], rng.permutation(rows).astype(np.int32)
    A, D = Rows(gpu, (1, rows, k), np.float16, 2 * pitch).put(a), Rows(gpu, (1, rows, n), np.float32, 4 * pitch)
    W = Rows(gpu, (groups, n, k), np.float16, 2 * ldw, 2 * stride).put(w if layout == "col" else w.transpose(0, 2, 1))
    gpu.EXPERTS.grouped_gemm(A.array, W.array, D.array, _sizes(gpu, offsets), rows=rows, groups=groups, n=n, k=k, d_type=np.float32, gather=ref.upload(gpu, gather), a_rows=rows,
                             lda=pitch, ldw=ldw, stride_w=stride, ldd=pitch, w_layout=gpu.WMMA.ColMajor if layout == "col" else gpu.WMMA.RowMajor)
    got = D.get()[0]
    for g in range(groups):
        for r in range(offsets[g], offsets[g + 1]):
            assert np.array_equal(got[r], w[g].astype(np.float64) @ a[gather[r]]), (g, r)


def test_grouped_gemm_few_rows(gpu):
    """Few rows a group, weights far from each other."""
    rng = np.random.default_rng(2)
    groups, n, k, stride = 4, 48, 264, 3 << 29
    a, w, offsets = _numbers(rng, 9, k), _numbers(rng, groups, n, k), [0, 2, 2, 5, 9]
    W, D = Rows(gpu, (groups, n, k), np.float16, 2 * k, 2 * stride).put(w), ref.upload(gpu, np.zeros((9, n), np.float32))
    gpu.EXPERTS.grouped_gemm(ref.upload(gpu, a), W.array, D, _sizes(gpu, offsets), rows=9, groups=groups, n=n, k=k, d_type=np.float32, stride_w=stride)
    got = D.to_host().reshape(9, n)
    for g in range(groups):
        for r in range(offsets[g], offsets[g + 1]):
            assert np.array_equal(got[r], w[g].astype(np.float64) @ a[r])


# ldb of 2^21 elements: tiles; of 2^25: the kernel for any pitch.
@pytest.mark.parametrize("b_rows,ldb", [(1200, 1 << 21), (90, 1 << 25)])
def test_grouped_wgrad(gpu, b_rows, ldb):
    rng = np.random.default_rng(3)
    rows, groups, m, n = 90, 2, 72, 136
    a, b, offsets = _numbers(rng, rows, m), _numbers(rng, b_rows, n), [1, 50, 89]
    gather = rng.integers(0, b_rows, rows).astype(np.int32)
    gather[60] = b_rows - 1
    A, B, D = Rows(gpu, (1, rows, m), np.float16, 1 << 26).put(a), Rows(gpu, (1, b_rows, n), np.float16, 2 * ldb).put(b), Rows(gpu, (groups, m, n), np.float32, 1 << 27, 3 << 32)
    gpu.EXPERTS.grouped_wgrad(A.array, B.array, D.array, _sizes(gpu, offsets), rows=rows, groups=groups, m=m, n=n, gather=ref.upload(gpu, gather), b_rows=b_rows, lda=1 << 25,
                              ldb=ldb, ldd=1 << 25, stride_d=3 << 30)
    got = D.get()
    for g in range(groups):
        r = slice(offsets[g], offsets[g + 1])
        assert np.array_equal(got[g], a[r].astype(np.float64).T @ b[gather[r]].astype(np.float64))


@pytest.mark.parametrize("n", [64, 37])
def test_join_and_activation(gpu, n):
    E, rng, pitch = gpu.EXPERTS, np.random.default_rng(n), 1 << 27
    rows, tokens = 24, 12
    h, dy = _numbers(rng, rows, n), _numbers(rng, tokens, n)
    place = rng.permutation(rows).astype(np.int32).reshape(tokens, 2)
    H, dY = Rows(gpu, (1, rows, n), np.float16, 2 * pitch).put(h), Rows(gpu, (1, tokens + 8, n), np.float16, 2 * pitch).put(np.concatenate([dy, np.zeros((8, n))]))
    Y, dH, dg = Rows(gpu, (1, tokens + 8, n), np.float16, 2 * pitch).put(np.zeros((tokens + 8, n))), Rows(gpu, (1, rows, n), np.float16, 2 * pitch), ref.upload(gpu, np.zeros(rows, np.float32))
    at = ref.upload(gpu, place)
    E.combine(H.array, at, Y.array, tokens=tokens, top=2, n=n, rows=rows, ldh=pitch, ldy=pitch)
    E.combine_grad(dY.array, H.array, at, dH.array, dg, tokens=tokens, top=2, n=n, rows=rows, ldh=pitch, ldy=pitch, lddh=pitch)
    assert np.array_equal(Y.get()[0, :tokens], h[place].sum(1))
    assert np.array_equal(dH.get()[0][place], np.repeat(dy[:, None], 2, 1))
    assert np.array_equal(dg.to_host().reshape(tokens, 2), (dy[:, None].astype(np.float64) * h[place]).sum(2))
    if n % 2:
        return
    A, dZ = Rows(gpu, (1, rows, n // 2), np.float16, 2 * pitch), Rows(gpu, (1, rows, n), np.float16, 2 * pitch)
    E.gated_silu(H.array, A.array, rows=rows, n=n, ldz=pitch, lda=pitch)
    E.gated_silu_grad(H.array, A.array, dZ.array, rows=rows, n=n, ldz=pitch, ldda=pitch, lddz=pitch)
    near, back = ref.upload(gpu, h), ref.upload(gpu, np.zeros((rows, n), np.float16))
    a = ref.upload(gpu, np.zeros((rows, n // 2), np.float16))
    E.gated_silu(near, a, rows=rows, n=n)
    E.gated_silu_grad(near, a, back, rows=rows, n=n)
    assert np.array_equal(A.get()[0].ravel(), a.to_host()) and np.array_equal(dZ.get()[0].ravel(), back.to_host())


# Codes 2^22 bytes apart: tiles; 2^28: the kernel for any pitch.
@pytest.mark.parametrize("rows,ldq", [(1100, 1 << 22), (40, 1 << 28)])
def test_mxfp4(gpu, rows, ldq):
    Q, rng = gpu.MXFP4, np.random.default_rng(rows)
    k, n = 288, 64
    x, w = _numbers(rng, rows, k), _numbers(rng, n, k)
    X = ref.upload(gpu, x)
    codes, near = Rows(gpu, (1, rows, Q.codes_bytes(1, k)), np.uint8, ldq), ref.upload(gpu, np.zeros(Q.codes_bytes(rows, k), np.uint8))
    scales, back = ref.upload(gpu, np.zeros(Q.scales_bytes(rows, k), np.uint8)), ref.upload(gpu, np.zeros((rows, k), np.float16))
    Q.quantize(X, codes.array, scales, rows=rows, k=k, ldq=ldq)
    Q.quantize(X, near, scales, rows=rows, k=k)
    assert np.array_equal(codes.get()[0].ravel(), near.to_host())
    Q.dequantize(codes.array, scales, back, rows=rows, k=k, dtype=np.float16, ldq=ldq)
    assert np.array_equal(back.to_host().reshape(rows, k), x)  # (whole numbers up to 2 are values of the format)
    wc, ws = ref.upload(gpu, np.zeros(Q.codes_bytes(n, k), np.uint8)), ref.upload(gpu, np.zeros(Q.scales_bytes(n, k), np.uint8))
    Q.quantize(ref.upload(gpu, w), wc, ws, rows=n, k=k)
    want = x.astype(np.float64) @ w.T.astype(np.float64)
    D = ref.upload(gpu, np.zeros((rows, n), np.float32))
    Q.gemm(codes.array, scales, wc, ws, D, m=rows, n=n, k=k, d_type=np.float32, lda=ldq)
    assert np.array_equal(D.to_host().reshape(rows, n), want)
    D = ref.upload(gpu, np.zeros((n, rows), np.float32))
    Q.gemm(wc, ws, codes.array, scales, D, m=n, n=rows, k=k, d_type=np.float32, ldb=ldq)
    assert np.array_equal(D.to_host().reshape(n, rows), want.T)
