"""Matrices beyond what the caches hold, which the kernels that touch every element once stream past them: bit for bit what the
same rows give in parts that are not streamed (those are compared with 64-bit implementations elsewhere)."""
import numpy as np
import pytest

from experts_oracle import KINDS, upload

pytestmark = pytest.mark.gpu

PARTS = 4


def _matrix(kind, rows, n, seed):
    """A random matrix without the time that normal numbers take: random bits with exponents around 1."""
    bits = np.random.default_rng(seed).integers(0, 1 << 16, size=(rows, n), dtype=np.uint16)
    if kind.name == "f16":
        return ((bits & 0x8FFF) | 0x3000).view(np.float16)
    return (bits & 0x81FF) | 0x3F00


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_combine_and_its_gradient(gpu, kind):
    kind, E, rng = KINDS[kind], gpu.EXPERTS, np.random.default_rng(1)
    tokens, top, n = 3203, 3, 8192
    rows = tokens * top
    assert 2 * rows * n > 100 << 20
    H, dY = upload(gpu, _matrix(kind, rows, n, 2)), upload(gpu, _matrix(kind, tokens, n, 3))
    gates, place = rng.random((tokens, top)).astype(np.float32), rng.permutation(rows).astype(np.int32).reshape(tokens, top)
    place[rng.random((tokens, top)) < 0.05] = -1
    out = []
    for parts in (1, PARTS):
        Y, dH, dg = (upload(gpu, np.zeros(s, T)) for s, T in ((tokens * n, kind.dtype), (rows * n, kind.dtype), (rows, np.float32)))
        G, P = upload(gpu, gates), upload(gpu, place)
        step = -(-tokens // parts)
        for t in range(0, tokens, step):
            sizes = dict(tokens=min(step, tokens - t), top=top, n=n, rows=rows, dtype=kind.marker(gpu), gates=G.ptr + 4 * t * top)
            E.combine(H, P.ptr + 4 * t * top, Y.ptr + 2 * t * n, **sizes)
            E.combine_grad(dY.ptr + 2 * t * n, H, P.ptr + 4 * t * top, dH, dg.ptr + 4 * t * top, **sizes)
        out.append([v.to_host().view(np.uint32 if v is dg else np.uint16) for v in (Y, dH, dg)])
    for whole, parts in zip(*out):
        assert whole.any() and np.array_equal(whole, parts)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_gated_silu_and_its_gradient(gpu, kind):
    kind, E = KINDS[kind], gpu.EXPERTS
    rows, n = 8203, 8192
    Z, dA = upload(gpu, _matrix(kind, rows, n, 4)), upload(gpu, _matrix(kind, rows, n // 2, 5))
    out = []
    for parts in (1, PARTS):
        A, dZ = upload(gpu, np.zeros(rows * n // 2, kind.dtype)), upload(gpu, np.zeros(rows * n, kind.dtype))
        step = -(-rows // parts)
        for r in range(0, rows, step):
            sizes = dict(rows=min(step, rows - r), n=n, dtype=kind.marker(gpu))
            E.gated_silu(Z.ptr + 2 * r * n, A.ptr + r * n, **sizes)
            E.gated_silu_grad(Z.ptr + 2 * r * n, dA.ptr + r * n, dZ.ptr + 2 * r * n, **sizes)
        out.append([v.to_host().view(np.uint16) for v in (A, dZ)])
    for whole, parts in zip(*out):
        assert whole.any() and np.array_equal(whole, parts)


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
def test_mxfp4_quantize_and_back(gpu, kind):
    kind, Q = KINDS[kind], gpu.MXFP4
    size = np.dtype(kind.dtype).itemsize
    rows, k = (8200, 8190) if size == 2 else (4104, 8188)
    ld = -(-k // 8) * 8
    x = _matrix(KINDS["f16"], rows, ld, 6).astype(np.float32) if size == 4 else _matrix(kind, rows, ld, 6)
    X, codes_pitch = upload(gpu, x), -(-k // 32) * 16
    out = []
    for parts in (1, PARTS):
        codes, scales, back = upload(gpu, np.zeros(Q.codes_bytes(rows, k), np.uint8)), upload(gpu, np.zeros(Q.scales_bytes(rows, k), np.uint8)), upload(gpu, np.zeros(rows * ld, kind.dtype))
        step = rows // parts
        for r in range(0, rows, step):
            sizes = dict(rows=step, k=k, dtype=kind.marker(gpu), ld=ld, lds=rows)
            # (two rows of scales are 16 bytes)
            assert step * parts == rows and r % 2 == 0
            Q.quantize(X.ptr + size * r * ld, codes.ptr + r * codes_pitch, scales.ptr + 8 * r, **sizes)
            Q.dequantize(codes.ptr + r * codes_pitch, scales.ptr + 8 * r, back.ptr + size * r * ld, **sizes)
        out.append([v.to_host().view(np.uint8) for v in (codes, scales, back)])
    for whole, parts in zip(*out):
        assert whole.any() and np.array_equal(whole, parts)
