"""Every kernel that a product grouped by expert can run on, named in the test, which asks the library's rule for it: short and long sums,
widths and sums that no tile or chunk divides, groups of very different size with empty ones among them.  Whole numbers, so that sums are exact in
whatever order."""
import numpy as np
import pytest

import experts_oracle as ref
from experts_oracle import KINDS, upload
from grouped_choice import grouped_kernel
from test_gpu_experts import _sizes_of

pytestmark = pytest.mark.gpu

NARROW = [("narrow 1 1 8", 11, 1, 200, 72), ("narrow 1 1 8", 13, 2, 200, 2088), ("narrow 1 2 2", 60, 20, 392, 72), ("narrow 1 2 2", 60, 20, 392, 584), ("narrow 1 2 4", 60, 20, 392, 1096),
          ("narrow 1 2 4", 66, 40, 264, 2120), ("narrow 2 1 8", 29, 1, 200, 72), ("narrow 2 1 8", 60, 2, 200, 2088), ("narrow 4 1 8", 62, 1, 200, 72), ("narrow 4 1 8", 180, 3, 392, 2088)]
TILES = [("tile 128x64", 90, 1, 200, 72), ("tile 128x64", 500, 7, 520, 584), ("tile 128x128", 3500, 70, 264, 584), ("tile 128x128", 3800, 70, 264, 1096), ("tile 256x128", 1400, 70, 392, 72),
         ("tile 256x128", 1400, 70, 392, 584), ("tile 256x256", 16000, 40, 264, 72), ("tile 256x256", 16000, 40, 264, 584)]
ROW_TILES = TILES[:4] + [("tile 256x128", 210, 70, 392, 72), ("tile 256x128", 210, 70, 392, 584)] + TILES[6:]
PRODUCTS = [("col",) + s for s in NARROW + TILES] + [("row",) + s for s in ROW_TILES]
MXFP4 = [("narrow 1 1 8", 11, 1, 200, 100), ("narrow 1 1 8", 13, 2, 200, 4500), ("narrow 1 2 2", 60, 20, 392, 100), ("narrow 1 2 2", 60, 20, 392, 1300), ("narrow 1 2 4", 60, 20, 392, 4500),
         ("narrow 2 1 8", 29, 1, 200, 100), ("narrow 2 1 8", 60, 2, 200, 4500), ("narrow 4 1 8", 62, 1, 200, 100), ("narrow 4 1 8", 180, 3, 392, 4500), ("tile 128x64", 90, 1, 200, 100),
         ("tile 128x64", 500, 7, 520, 1300), ("tile 128x128", 3500, 70, 264, 100), ("tile 128x128", 3500, 70, 264, 1300), ("tile 256x128", 1400, 70, 392, 100), ("tile 256x128", 1400, 70, 392, 1300),
         ("tile 256x256", 10500, 70, 520, 100), ("tile 256x256", 10500, 70, 520, 1300)]
SUMS = [("tile 128x64", 3, 1, 584, 200), ("tile 128x64", 700, 2, 200, 136), ("tile 128x128", 15, 5, 1096, 264), ("tile 128x128", 2100, 70, 72, 200), ("tile 256x128", 60, 20, 1096, 264),
        ("tile 256x128", 1500, 20, 1096, 264), ("tile 256x256", 22000, 20, 1096, 264)]


def _offsets(rng, groups, rows):
    offsets = _sizes_of(groups, rows, rng, 0.2)
    return np.clip(offsets, 3, rows - 2) if groups > 1 else offsets


def _parts(offsets):
    return [(g, slice(a, b)) for g, (a, b) in enumerate(zip(offsets, offsets[1:])) if a < b]


def _check_outside(got, offsets):
    assert np.all(got[:offsets[0]] == 99) and np.all(got[offsets[-1]:] == 99)


# The gated form of exact sums: exp's argument is rounded after it is scaled (|g| 2^-24 of the result, and a quarter of that from log2 e itself), exp, the
# sum, the quotient and the product add at most some eight units; below -88 exp overflows and the result is a zero.
def _check_gated(got, z, okind):
    with np.errstate(over="ignore"):
        want = ref.gated(z.astype(np.float64))
    gate = np.abs(z[..., 0::2])
    far = np.abs(okind.load(got) - want)
    assert np.all(far <= ((2 * gate + 16) * 2.0 ** -24 + okind.roundoff * 1.01) * np.abs(want) + (2.0 ** -25 if okind.name == "f16" else 1e-30)), far.max()


@pytest.mark.parametrize("kind,out", [("f16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("epilogue", [None, "gated_silu"])
@pytest.mark.parametrize("layout,kernel,rows,groups,n,k", PRODUCTS)
def test_grouped_gemm(gpu, layout, kernel, rows, groups, n, k, epilogue, kind, out):
    assert grouped_kernel(gpu, rows=rows, groups=groups, n=n, k=k, layout=layout)[0] == kernel
    rng, kind, okind = np.random.default_rng(rows + n + k), KINDS[kind], KINDS[out]
    offsets, a_rows = _offsets(rng, groups, rows), rows // 2 + 7
    gather = rng.integers(0, a_rows, rows).astype(np.int32)
    a, w = rng.integers(-1, 2, (a_rows, k)).astype(np.float32), rng.integers(-1, 2, (groups, k, n)).astype(np.float32)
    width = n if epilogue is None else n // 2
    D = upload(gpu, np.full((rows, width), okind.store(np.float64(99)), okind.dtype))
    gpu.EXPERTS.grouped_gemm(upload(gpu, kind.store(a)), upload(gpu, kind.store(w.transpose(0, 2, 1) if layout == "col" else w)), D, upload(gpu, offsets), rows=rows, groups=groups, n=n,
                             k=k, dtype=kind.marker(gpu), d_type=okind.marker(gpu), gather=upload(gpu, gather), a_rows=a_rows, epilogue=epilogue,
                             w_layout=gpu.WMMA.ColMajor if layout == "col" else gpu.WMMA.RowMajor)
    got = D.to_host().reshape(rows, width)
    for g, r in _parts(offsets):
        z = a[gather[r]] @ w[g]
        if epilogue is None:
            assert np.array_equal(got[r], okind.store(z)), g
        else:
            _check_gated(got[r], z, okind)
    _check_outside(okind.load(got), offsets)


@pytest.mark.parametrize("epilogue,out", [(None, "f32"), ("gated_silu", "f32"), ("gated_silu", "f16"), (None, "bf16")])
@pytest.mark.parametrize("kernel,rows,groups,n,k", MXFP4)
def test_mxfp4_grouped_gemm(gpu, kernel, rows, groups, n, k, epilogue, out):
    """Magnitudes 0 and 1, scales of 1 and 2; in the gated form of 1 / 4 and 1 / 8, so that gates are of order one."""
    assert grouped_kernel(gpu, rows=rows, groups=groups, n=n, k=k, mxfp4=True)[0] == kernel
    Q, rng, okind = gpu.MXFP4, np.random.default_rng(rows + n + k), KINDS[out]
    offsets, a_rows = _offsets(rng, groups, rows), rows // 2 + 7
    gather = rng.integers(0, a_rows, rows).astype(np.int32)
    least = 127 if epilogue is None else 124

    def matrix(rows):
        blocks = -(-k // 32)
        value = rng.choice(np.array([0, 2, 8 + 2], np.uint8), (rows, 32 * blocks))
        value[:, k:] = 0
        scales = rng.integers(least, least + 2, (rows, blocks)).astype(np.uint8)
        x = np.where(value & 8, -1, 1) * ref.E2M1[value & 7] * np.exp2(np.repeat(scales.astype(np.float32), 32, 1) - 127)
        return (value[:, 0::2] | value[:, 1::2] << 4).astype(np.uint8), ref.panels(scales, fill=255), x[:, :k].astype(np.float32)

    a, w = matrix(a_rows), [matrix(n) for _ in range(groups)]
    width = n if epilogue is None else n // 2
    D = upload(gpu, np.full((rows, width), okind.store(np.float64(99)), okind.dtype))
    Q.grouped_gemm(upload(gpu, a[0]), upload(gpu, a[1]), upload(gpu, np.stack([x[0] for x in w])), upload(gpu, np.stack([x[1] for x in w])), D, upload(gpu, offsets), rows=rows,
                   groups=groups, n=n, k=k, d_type=okind.marker(gpu), gather=upload(gpu, gather), a_rows=a_rows, epilogue=epilogue)
    got = D.to_host().reshape(rows, width)
    for g, r in _parts(offsets):
        z = a[2][gather[r]] @ w[g][2].T
        if epilogue is None:
            assert np.array_equal(got[r], okind.store(z)), g
        else:
            _check_gated(got[r], z, okind)
    _check_outside(okind.load(got), offsets)


@pytest.mark.parametrize("kind,out", [("f16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("kernel,rows,groups,m,n", SUMS)
def test_grouped_wgrad(gpu, kernel, rows, groups, m, n, kind, out):
    assert grouped_kernel(gpu, rows=rows, groups=groups, n=n, m=m)[0] == kernel
    rng, kind, okind = np.random.default_rng(rows + n), KINDS[kind], KINDS[out]
    offsets, b_rows = _offsets(rng, groups, rows) if rows > 20 else np.linspace(0, rows, groups + 1).astype(np.int32), rows // 2 + 7
    gather = rng.integers(0, b_rows, rows).astype(np.int32)
    a, b = rng.integers(-1, 2, (rows, m)).astype(np.float32), rng.integers(-1, 2, (b_rows, n)).astype(np.float32)
    before = rng.integers(-9, 10, (groups, m, n)).astype(np.float32)
    args = [upload(gpu, v) for v in (kind.store(a), kind.store(b), okind.store(before), offsets)]
    sizes = dict(rows=rows, groups=groups, m=m, n=n, dtype=kind.marker(gpu), d_type=okind.marker(gpu), gather=upload(gpu, gather), b_rows=b_rows)
    want = np.zeros((groups, m, n), np.float32)
    for g, r in _parts(offsets):
        want[g] = a[r].T @ b[gather[r]]
    gpu.EXPERTS.grouped_wgrad(*args, accumulate=True, **sizes)
    assert np.array_equal(args[2].to_host().reshape(want.shape), okind.store(before + want))
    gpu.EXPERTS.grouped_wgrad(*args, **sizes)
    assert np.array_equal(args[2].to_host().reshape(want.shape), okind.store(want))
