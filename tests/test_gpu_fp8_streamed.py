"""8-bit conversions and the activation that keeps 8 bits on matrices beyond what the caches hold, which their kernels stream past them: bit for bit what the same rows give
in parts that are not streamed (those are compared with 64-bit implementations elsewhere)."""
import numpy as np
import pytest

from experts_oracle import KINDS, upload
from test_gpu_experts_streamed import _matrix

pytestmark = pytest.mark.gpu

STREAMED = 96 << 20  # bytes of a matrix


def _parts(rows, parts):
    """(first, count): firsts are multiples of four, on which panels of scales may be shared."""
    step = -(-rows // parts // 4) * 4
    return [(r, min(step, rows - r)) for r in range(0, rows, step)]


@pytest.mark.parametrize("form", ["e4m3", "e5m2"])
@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
def test_quantize_and_back(gpu, kind, form):
    kind, Q = KINDS[kind], gpu.FP8
    size, form = np.dtype(kind.dtype).itemsize, {"e4m3": Q.E4M3, "e5m2": Q.E5M2}[form]
    rows, k, ld = (6203, 8200, 8208) if size == 2 else (3103, 8200, 8204)
    assert size * rows * k > STREAMED > size * rows * k / 2 and k % 128
    X = upload(gpu, _matrix(KINDS["f16"], rows, ld, 6).astype(np.float32) if size == 4 else _matrix(kind, rows, ld, 6))
    ldq, lds, out = Q.codes_bytes(1, k), -(-rows // 4) * 4, []
    for parts in (1, 3):
        codes, scales, back = upload(gpu, np.zeros(rows * ldq, np.uint8)), upload(gpu, np.zeros(Q.scales_bytes(rows, k), np.uint8)), upload(gpu, np.zeros(rows * ld, kind.dtype))
        for r, n in _parts(rows, parts):
            sizes = dict(rows=n, k=k, dtype=kind.marker(gpu), format=form, ld=ld, lds=lds)
            assert parts == 1 or size * n * k < STREAMED
            Q.quantize(X.ptr + size * r * ld, codes.ptr + r * ldq, scales.ptr + 4 * r, **sizes)
            Q.dequantize(codes.ptr + r * ldq, scales.ptr + 4 * r, back.ptr + size * r * ld, **sizes)
        out.append([v.to_host().view(np.uint8) for v in (codes, scales, back)])
    for whole, parts in zip(*out):
        assert whole.any() and np.array_equal(whole, parts)
    assert not out[0][2].reshape(rows, ld * size)[:, k * size:].any()


@pytest.mark.parametrize("again", ["without", "beside", "in place"])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_kept_activation(gpu, kind, again):
    kind, Q, rows, n = KINDS[kind], gpu.FP8, 6203, 8200
    assert 2 * rows * n > STREAMED > rows * n
    Z, given = upload(gpu, _matrix(kind, rows, n, 4)), _matrix(kind, rows, n // 2, 5)
    ldq, lds, out = Q.codes_bytes(1, n), -(-rows // 4) * 4, []
    for parts in (1, 3):
        codes, scales = upload(gpu, np.zeros(rows * ldq, np.uint8)), upload(gpu, np.zeros(Q.scales_bytes(rows, n), np.uint8))
        A, dZ, other = (upload(gpu, np.zeros(m, kind.dtype)) for m in (rows * n // 2, rows * n, rows * n // 2))
        dA = upload(gpu, given)
        made = {"without": None, "beside": other, "in place": dA}[again]
        for r, m in _parts(rows, parts):
            sizes = dict(rows=m, n=n, dtype=kind.marker(gpu), lds=lds)
            assert parts == 1 or 2 * m * n < STREAMED
            Q.gated_silu(Z.ptr + 2 * r * n, A.ptr + r * n, codes.ptr + r * ldq, scales.ptr + 4 * r, **sizes)
            Q.gated_silu_grad(codes.ptr + r * ldq, scales.ptr + 4 * r, dA.ptr + r * n, dZ.ptr + 2 * r * n, A=None if made is None else made.ptr + r * n, **sizes)
        out.append([v.to_host().view(np.uint8) for v in (A, codes, scales, dZ, dA, other)])
    for i, (whole, parts) in enumerate(zip(*out)):
        assert whole.any() == (i < 5 or again == "beside") and np.array_equal(whole, parts), i
    assert again == "in place" or np.array_equal(out[0][4].view(kind.dtype).reshape(given.shape).view(np.uint16), given.view(np.uint16))
