"""The experts' operators and the 4-bit matrices on the GPU, through the Python entry points, against 64-bit
implementations.

Tolerances.  A Float32 sum of K products, in whatever order, is within K * 2^-24 of the sum of the products' magnitudes
(products of 16-bit and 4-bit values are exact in Float32); two more roundings for what joins partial sums.  Rounding to
the result's type adds half a unit in its last place, 2^-11 or 2^-8 of the result, and 2^-25 below Float16's smallest normal.
Results that are whole numbers below 2^11 (2^8 for bfloat16) are exact."""
import numpy as np
import pytest

import experts_oracle as ref
from experts_oracle import KINDS, upload

pytestmark = pytest.mark.gpu


def _bound(size, exact, terms, kind):
    return (terms + 2) * 2.0 ** -24 * size + kind.roundoff * np.abs(exact) * 1.01 + 2.0 ** -25


def _check(got, exact, size, terms, kind):
    assert got.shape == exact.shape
    far = np.abs(got - exact) - _bound(size, exact, terms, kind)
    assert np.all(far <= 0), (float(far.max()), np.unravel_index(int(far.argmax()), far.shape))


def _padded(kind, a, pitch, fill=np.nan):
    """Rows of `a` at a pitch, with what lies between rows filled by NaN."""
    out = np.full(a.shape[:-1] + (pitch,), fill)
    out[..., :a.shape[-1]] = a
    with np.errstate(invalid="ignore"):
        return np.full(out.shape, 0x7FC0, np.uint16) if kind.name == "bf16" and np.isnan(out).all() else _store(kind, out)


def _store(kind, a):
    nan = np.isnan(a)
    stored = kind.store(np.where(nan, 0.0, a))
    stored[nan] = 0x7FC0 if kind.name == "bf16" else np.nan
    return stored


# ------------------------------------------------------------------------------------- routing

def _route(gpu, z, kind, top, over_all, ld=0, dgates=None, ldd=0):
    tokens, experts = z.shape
    E = gpu.EXPERTS
    stored = _store(kind, np.where(np.isneginf(z) | np.isposinf(z), 0.0, z))
    inf = np.isinf(z)
    if inf.any():
        stored[inf] = np.where(z[inf] > 0, 0x7F80, 0xFF80) if kind.name == "bf16" else z[inf]
    if ld:
        pad = np.zeros((tokens, ld), stored.dtype)
        pad[:, :experts] = stored
        stored = pad
    dz = upload(gpu, stored)
    i32 = lambda *shape: upload(gpu, np.full(shape, 12345, np.int32))  # noqa: E731
    chosen, gates, offsets, rows, place = i32(tokens, top), upload(gpu, np.full((tokens, top), 7.0, np.float32)), i32(experts + 1), i32(tokens * top), i32(tokens, top)
    need = E.route_workspace(tokens, experts, top)
    workspace = upload(gpu, np.full(max(16, need), 77, np.uint8))
    sizes = dict(tokens=tokens, experts=experts, top=top, dtype=kind.marker(gpu), over_all=over_all, ld=ld)
    E.route(dz, chosen, gates, offsets, rows, place, workspace=workspace, **sizes)
    out = [chosen.to_host().reshape(tokens, top), gates.to_host().reshape(tokens, top), offsets.to_host(), rows.to_host(), place.to_host().reshape(tokens, top)]
    if dgates is not None:
        width = ldd or experts
        back = upload(gpu, np.full((tokens, width), 9, kind.dtype))
        E.route_grad(dz, chosen, gates, upload(gpu, dgates.astype(np.float32)), back, ldd=ldd, **sizes)
        out.append(back.to_host().reshape(tokens, width))
    return out


@pytest.mark.parametrize("over_all", [False, True])
@pytest.mark.parametrize("tokens,experts,top,kind,ld", [
    (1, 1, 1, "f32", 0), (1, 8, 2, "bf16", 0), (3, 5, 5, "f16", 9), (16, 64, 4, "f32", 0), (64, 64, 16, "f32", 0), (65, 63, 1, "bf16", 0), (129, 65, 8, "f32", 70),
    (300, 256, 8, "f16", 0), (777, 257, 3, "bf16", 0), (2050, 130, 6, "f32", 0), (4099, 1024, 2, "f16", 0), (1000, 7, 7, "bf16", 0)])
def test_route(gpu, tokens, experts, top, kind, ld, over_all):
    kind, rng = KINDS[kind], np.random.default_rng(tokens * 31 + experts)
    # values of one decimal have ties in plenty; every fourth expert is off, some tokens have one or none
    z = kind.load(kind.store(np.round(rng.normal(size=(tokens, experts)) * 2, 1)))
    z[rng.random((tokens, experts)) < 0.25] = -np.inf
    if tokens > 2:
        z[1] = -np.inf
        z[2] = np.where(np.arange(experts) == experts - 1, 1.0, -np.inf)
    dgates = rng.normal(size=(tokens, top)).astype(np.float32)
    got = _route(gpu, z, kind, top, over_all, ld, dgates, ldd=experts + 3 if ld else 0)
    want = ref.route(z, top, over_all)
    for g, w in zip((got[0], got[2], got[3], got[4]), (want[0], want[2], want[3], want[4])):
        assert np.array_equal(g, w)
    # exp of a Float32 argument x: |x| * 2^-23 from the product with log2 e, and a few units in the last place; |x| <= 20
    assert np.allclose(got[1], want[1], rtol=64 * 2.0 ** -23, atol=1e-30)
    exact = ref.route_grad(z, want[0], dgates.astype(np.float64), over_all)
    back = got[5]
    if ld:
        assert np.all(back[:, experts:] == 9)
        back = back[:, :experts]
    # a gate times a difference of at most 2 sum |g dg|, of gates that are off by 64 * 2^-23
    size = np.abs(dgates).max(1, keepdims=True) * 2
    assert np.all(np.abs(kind.load(back) - exact) <= kind.roundoff * np.abs(exact) * 1.01 + 200 * 2.0 ** -23 * size + 2.0 ** -25)


def test_route_extremes(gpu):
    """The types' lowest and highest values, infinities, NaN, zeros of both signs, equal logits."""
    f32 = np.finfo(np.float32)
    for kind, low in (("f32", f32.min), ("f16", -65504.0), ("bf16", -3.3895313892515355e38)):
        kind = KINDS[kind]
        z = np.array([[low, low, low, low], [low, -np.inf, low, 0.0], [np.inf, 1.0, np.inf, -low], [0.0, -0.0, 0.0, -1.0], [-np.inf] * 4, [-np.inf, low, -np.inf, -np.inf]])
        z = np.where(np.isinf(z), z, kind.load(kind.store(np.where(np.isinf(z), 0, z))))
        for over_all in (False, True):
            got, want = _route(gpu, z, kind, 2, over_all), ref.route(z, 2, over_all)
            for g, w in zip((got[0], got[2], got[3], got[4]), (want[0], want[2], want[3], want[4])):
                assert np.array_equal(g, w), (kind.name, over_all, g, w)
            assert np.allclose(got[1], want[1], rtol=1e-5, atol=1e-30) and np.isfinite(got[1]).all()
    z = np.array([[np.nan, 1.0, np.nan, 2.0], [np.nan] * 4], np.float32)
    E = gpu.EXPERTS
    out = [upload(gpu, np.zeros(n, t)) for n, t in ((6, np.int32), (6, np.float32), (5, np.int32), (6, np.int32), (6, np.int32))]
    back = upload(gpu, np.ones((2, 4), np.float32))
    E.route(upload(gpu, z), *out, tokens=2, experts=4, top=3)
    assert out[0].to_host().tolist() == [3, 1, -1, -1, -1, -1] and out[4].to_host().tolist() == [1, 0, -1, -1, -1, -1]
    E.route_grad(upload(gpu, z), out[0], out[1], upload(gpu, np.array([1, 1] + [np.nan] * 4, np.float32)), back, tokens=2, experts=4, top=3)
    assert np.isfinite(back.to_host()).all() and not back.to_host()[4:].any()


def test_route_of_no_tokens_writes_the_offsets(gpu):
    offsets = upload(gpu, np.full(6, 5, np.int32))
    gpu.EXPERTS.route(None, None, None, offsets, None, None, tokens=0, experts=5, top=2)
    assert not offsets.to_host().any()


# ------------------------------------------------------------------------------------- products grouped by expert

def _sizes_of(groups, rows, rng, empty):
    """Rows of each group: `empty` says which share has none."""
    weight = rng.random(groups) * (rng.random(groups) >= empty)
    if not weight.sum():
        weight[-1] = 1
    cut = np.floor(np.cumsum(weight) / weight.sum() * rows + 1e-9).astype(int)
    return np.concatenate([[0], cut]).astype(np.int32)


SHAPES = [  # rows, groups, n, k: one row; no group of more than a few rows; nothing even; more groups than a wavefront has lanes; whole tiles; long sums
    (1, 1, 1, 1), (1, 3, 16, 8), (5, 2, 37, 45), (33, 4, 40, 24), (70, 7, 72, 64), (130, 130, 24, 40), (200, 3, 136, 72), (257, 5, 264, 200), (40, 64, 64, 512),
    (300, 2, 256, 1032), (600, 200, 48, 96), (129, 1, 520, 328), (1030, 6, 272, 136)]


@pytest.mark.parametrize("layout", ["col", "row"])
@pytest.mark.parametrize("kind,out", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("rows,groups,n,k", SHAPES)
def test_grouped_gemm(gpu, rows, groups, n, k, kind, out, layout):
    rng = np.random.default_rng(rows * 7 + n)
    kind, okind = KINDS[kind], KINDS[out]
    offsets = _sizes_of(groups, rows, rng, 0.3)
    if groups > 1 and rows > 20:  # positions before the first group and behind the last
        offsets = np.clip(offsets, 3, rows - 2)
    a_rows = max(1, rows // 2)
    gather = rng.integers(0, a_rows, rows).astype(np.int32) if rows % 2 else None
    a = kind.load(kind.store(rng.normal(size=(a_rows if gather is not None else rows, k))))
    w = kind.load(kind.store(rng.normal(size=(groups, k, n)) * 0.1))
    stored_w = w.transpose(0, 2, 1) if layout == "col" else w
    D = upload(gpu, np.full((rows, n), 99, okind.dtype))
    gpu.EXPERTS.grouped_gemm(upload(gpu, kind.store(a)), upload(gpu, kind.store(stored_w)), D, upload(gpu, offsets), rows=rows, groups=groups, n=n, k=k,
                             dtype=kind.marker(gpu), d_type=okind.marker(gpu), w_layout=gpu.WMMA.ColMajor if layout == "col" else gpu.WMMA.RowMajor,
                             gather=None if gather is None else upload(gpu, gather), a_rows=len(a))
    got = D.to_host().reshape(rows, n)
    exact, size = ref.grouped(a, w, offsets, gather, np.zeros((rows, n)))
    inside = (np.arange(rows) >= offsets[0]) & (np.arange(rows) < offsets[-1])
    assert np.all(got[~inside] == 99)
    _check(okind.load(got)[inside], exact[inside], size[inside], k, okind)


@pytest.mark.parametrize("layout", ["col", "row"])
@pytest.mark.parametrize("pitch", [8, 3])
@pytest.mark.parametrize("rows,groups,n,k", [(50, 3, 72, 40), (300, 2, 264, 136), (20, 30, 128, 256)])
def test_grouped_gemm_pitches_with_nan_between_rows(gpu, rows, groups, n, k, pitch, layout):
    """Pitches and strides beyond the extents, NaN in everything that is no operand, whole numbers: the results are exact, and
    D's own padding stays."""
    rng = np.random.default_rng(n + pitch)
    kind = KINDS["f16"]
    offsets = _sizes_of(groups, rows, rng, 0.2)
    a, w = rng.integers(-2, 3, (rows + 4, k)).astype(float), rng.integers(-1, 2, (groups, k, n)).astype(float)
    gather = rng.permutation(rows + 4)[:rows].astype(np.int32)
    unused = np.setdiff1d(np.arange(rows + 4), gather)
    a_stored = _padded(kind, a, k + pitch)
    a_stored[unused] = np.nan
    w_stored = _padded(kind, w.transpose(0, 2, 1) if layout == "col" else w, (k if layout == "col" else n) + pitch)
    lines = w_stored.shape[1]
    w_stored = np.concatenate([w_stored, np.full((groups, 2, w_stored.shape[2]), np.nan, np.float16)], 1)  # two more lines from group to group
    D = upload(gpu, np.full((rows, n + pitch), 99, np.float32))
    gpu.EXPERTS.grouped_gemm(upload(gpu, a_stored), upload(gpu, w_stored), D, upload(gpu, offsets), rows=rows, groups=groups, n=n, k=k, d_type=np.float32,
                             w_layout=gpu.WMMA.ColMajor if layout == "col" else gpu.WMMA.RowMajor, gather=upload(gpu, gather), a_rows=rows + 4, lda=k + pitch,
                             ldw=w_stored.shape[2], stride_w=(lines + 2) * w_stored.shape[2], ldd=n + pitch)
    got = D.to_host().reshape(rows, n + pitch)
    exact, _ = ref.grouped(a, w, offsets, gather, np.full((rows, n), 99.0))
    assert np.array_equal(got[:, :n], exact) and np.all(got[:, n:] == 99)


@pytest.mark.parametrize("rows,groups,n,k,address", [(9, 2, 16, 8, 0), (100, 3, 38, 64, 0), (100, 3, 130, 64, 2), (260, 2, 512, 72, 0), (31, 40, 64, 128, 0)])
@pytest.mark.parametrize("out", ["f16", "f32"])
def test_grouped_gemm_gated(gpu, rows, groups, n, k, address, out):
    rng = np.random.default_rng(n)
    kind, okind = KINDS["f16"], KINDS[out]
    offsets = _sizes_of(groups, rows, rng, 0.3)
    a, w = kind.load(kind.store(rng.normal(size=(rows, k)))), kind.load(kind.store(rng.normal(size=(groups, k, n)) * 0.2))
    D = upload(gpu, np.full(rows * (n // 2) + 8, 99, okind.dtype))
    gpu.EXPERTS.grouped_gemm(upload(gpu, kind.store(a)), upload(gpu, kind.store(w.transpose(0, 2, 1))), D.ptr + address * okind.dtype().itemsize, upload(gpu, offsets),
                             rows=rows, groups=groups, n=n, k=k, d_type=okind.marker(gpu), epilogue=gpu.EXPERTS.GATED_SILU)
    got = D.to_host()
    assert np.all(got[:address] == 99) and np.all(got[address + rows * (n // 2):] == 99)
    got = okind.load(got[address:address + rows * (n // 2)].reshape(rows, n // 2))
    exact, size = ref.grouped(a, w, offsets, None, np.zeros((rows, n)))
    # silu(g) v: its slopes are at most 1.1 |v| and |silu(g)| <= |g|; the quotient and exp add some units of 2^-23
    error = (k + 2) * 2.0 ** -24 * (1.1 * size[:, 0::2] * np.abs(exact[:, 1::2]) + np.abs(exact[:, 0::2]) * size[:, 1::2])
    want = ref.gated(exact)
    far = np.abs(got - want) - (error + (okind.roundoff * 1.01 + 64 * 2.0 ** -23) * np.abs(want) + 2.0 ** -25)
    assert far.max() <= 0, far.max()


@pytest.mark.parametrize("kind,out", [("f16", "f32"), ("bf16", "f32"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("rows,groups,m,n", [
    (1, 1, 1, 1), (5, 2, 37, 45), (64, 1, 64, 64), (70, 5, 24, 72), (130, 130, 24, 16), (200, 3, 136, 72), (257, 4, 264, 200), (1000, 3, 136, 264), (67, 2, 128, 256), (300, 80, 16, 24)])
def test_grouped_wgrad(gpu, rows, groups, m, n, kind, out, accumulate):
    rng = np.random.default_rng(rows + n)
    kind, okind = KINDS[kind], KINDS[out]
    offsets = _sizes_of(groups, rows, rng, 0.3)
    if groups > 1 and rows > 20:
        offsets = np.clip(offsets, 3, rows - 2)
    b_rows = max(1, rows // 2)
    gather = rng.integers(0, b_rows, rows).astype(np.int32) if rows % 2 else None
    a = kind.load(kind.store(rng.normal(size=(rows, m))))
    b = kind.load(kind.store(rng.normal(size=(b_rows if gather is not None else rows, n))))
    before = okind.load(okind.store(rng.normal(size=(groups, m, n))))
    D = upload(gpu, okind.store(before))
    gpu.EXPERTS.grouped_wgrad(upload(gpu, kind.store(a)), upload(gpu, kind.store(b)), D, upload(gpu, offsets), rows=rows, groups=groups, m=m, n=n,
                              dtype=kind.marker(gpu), d_type=okind.marker(gpu), gather=None if gather is None else upload(gpu, gather), b_rows=len(b), accumulate=accumulate)
    got = okind.load(D.to_host().reshape(groups, m, n))
    taken = b if gather is None else b[gather]
    for g in range(groups):
        r = slice(offsets[g], offsets[g + 1])
        exact, size = a[r].T @ taken[r], np.abs(a[r]).T @ np.abs(taken[r])
        if accumulate:
            exact, size = exact + before[g], size + np.abs(before[g])
        if offsets[g] == offsets[g + 1]:
            assert np.array_equal(got[g], exact)
        _check(got[g], exact, size, rows + 1, okind)


@pytest.mark.parametrize("rows,groups,m,n", [(100, 4, 136, 72), (333, 3, 264, 264), (77, 6, 40, 39)])
def test_grouped_wgrad_infinities_stay_in_their_group(gpu, rows, groups, m, n):
    """An infinity in a group's last row, NaN in rows of no group: neighbours and padding never meet them."""
    rng = np.random.default_rng(rows)
    offsets = np.clip(_sizes_of(groups, rows, rng, 0.0), 2, rows - 3)
    a, b = rng.integers(-2, 3, (rows, m)).astype(np.float16), rng.integers(-2, 3, (rows, n)).astype(np.float16)
    a[:2] = np.nan
    b[rows - 3:] = np.nan
    last = offsets[1] - 1
    a[last], b[last] = 0, 1
    a[last, 5] = 1
    b[last, 7] = np.inf
    D = upload(gpu, np.zeros((groups, m, n), np.float32))
    gpu.EXPERTS.grouped_wgrad(upload(gpu, a), upload(gpu, b), D, upload(gpu, offsets), rows=rows, groups=groups, m=m, n=n)
    got = D.to_host().reshape(groups, m, n)
    for g in range(groups):
        r = slice(offsets[g], offsets[g + 1])
        with np.errstate(invalid="ignore"):
            exact = a[r].astype(np.float64).T @ b[r].astype(np.float64)
        if g == 0:
            assert got[0, 5, 7] == np.inf
            finite = np.delete(got[0], 7, 1)
            assert np.array_equal(finite, np.delete(exact, 7, 1))
        else:
            assert np.array_equal(got[g], exact)


# Products large enough for every tile, with edges on all sides and groups of very different size; whole numbers, so that the results
# are exact whatever the order of the sums.
def _large_groups(groups, rows):
    if groups == 1:
        return np.array([0, rows], np.int32)
    cut = (np.arange(groups + 1) / groups) ** 1.7 * (rows - 5)
    offsets = np.concatenate([[0], np.floor(cut[1:]) + 3]).astype(np.int32)
    offsets[1] = offsets[0] = 2  # (the first group has no rows, and the last ones have no group)
    return offsets


@pytest.mark.parametrize("layout", ["col", "row"])
@pytest.mark.parametrize("rows,groups,n,k,kind,out", [
    (4000, 1, 4088, 72, "f16", "f16"), (8150, 3, 8184, 136, "bf16", "f32"), (2900, 3, 4096, 1000, "f16", "f32"), (1000, 4, 2056, 328, "bf16", "bf16"), (500, 12, 1032, 200, "f16", "f16")])
def test_grouped_gemm_large(gpu, rows, groups, n, k, kind, out, layout):
    rng = np.random.default_rng(rows)
    kind, okind = KINDS[kind], KINDS[out]
    offsets = _large_groups(groups, rows)
    a_rows = rows // 2 + 7
    gather = rng.integers(0, a_rows, rows).astype(np.int32)
    a, w = rng.integers(-1, 2, (a_rows, k)).astype(np.float32), rng.integers(-1, 2, (groups, k, n)).astype(np.float32)
    D = upload(gpu, np.full((rows, n), 99, okind.dtype))
    gpu.EXPERTS.grouped_gemm(upload(gpu, kind.store(a)), upload(gpu, kind.store(w.transpose(0, 2, 1) if layout == "col" else w)), D, upload(gpu, offsets), rows=rows,
                             groups=groups, n=n, k=k, dtype=kind.marker(gpu), d_type=okind.marker(gpu), gather=upload(gpu, gather), a_rows=a_rows,
                             w_layout=gpu.WMMA.ColMajor if layout == "col" else gpu.WMMA.RowMajor)
    got = D.to_host().reshape(rows, n)
    for g in range(groups):
        r = slice(offsets[g], offsets[g + 1])
        assert np.array_equal(got[r], okind.store(a[gather[r]] @ w[g])), g
    assert np.all(got[:offsets[0]] == 99) and np.all(got[offsets[-1]:] == 99)


@pytest.mark.parametrize("rows,groups,m,n,kind,out", [(150, 1, 3496, 3592, "bf16", "f32"), (700, 3, 1992, 2056, "f16", "f32"), (900, 5, 1000, 1032, "bf16", "bf16"), (3000, 1, 520, 264, "f16", "f32")])
def test_grouped_wgrad_large(gpu, rows, groups, m, n, kind, out):
    rng = np.random.default_rng(rows)
    kind, okind = KINDS[kind], KINDS[out]
    offsets = _large_groups(groups, rows)
    b_rows = rows // 2 + 7
    gather = rng.integers(0, b_rows, rows).astype(np.int32)
    a, b = rng.integers(-1, 2, (rows, m)).astype(np.float32), rng.integers(-1, 2, (b_rows, n)).astype(np.float32)
    D = upload(gpu, np.full((groups, m, n), 99, okind.dtype))
    args = upload(gpu, kind.store(a)), upload(gpu, kind.store(b)), D, upload(gpu, offsets)
    sizes = dict(rows=rows, groups=groups, m=m, n=n, dtype=kind.marker(gpu), d_type=okind.marker(gpu), gather=upload(gpu, gather), b_rows=b_rows)
    gpu.EXPERTS.grouped_wgrad(*args, **sizes)
    want = np.stack([a[offsets[g]:offsets[g + 1]].T @ b[gather[offsets[g]:offsets[g + 1]]] for g in range(groups)])
    assert np.array_equal(D.to_host().reshape(groups, m, n), okind.store(want))
    if out == "f32":
        gpu.EXPERTS.grouped_wgrad(*args, accumulate=True, **sizes)
        assert np.array_equal(D.to_host().reshape(groups, m, n), 2 * want)


@pytest.mark.parametrize("rows,groups,m,n,kind,out", [(1601, 1, 3496, 3592, "bf16", "f32"), (4703, 3, 2056, 1992, "f16", "f16"), (1537, 1, 3592, 3496, "f16", "f32")])
def test_grouped_wgrad_large_and_long(gpu, rows, groups, m, n, kind, out):
    """Sums so long that the largest tile takes them (with an empty group among three)."""
    test_grouped_wgrad_large(gpu, rows, groups, m, n, kind, out)


def test_grouped_gemm_offsets_and_gather_outside(gpu):
    """Offsets and rows that lie outside are taken as the nearest inside: nothing else is read or written."""
    rng = np.random.default_rng(1)
    a, w = rng.integers(-2, 3, (6, 16)).astype(np.float16), rng.integers(-2, 3, (3, 24, 16)).astype(np.float16)
    offsets, gather = np.array([-5, 2, 4, 900], np.int32), np.array([-7, 0, 5, 2, 77, 1, 3, 1], np.int32)
    D = upload(gpu, np.zeros((8, 24), np.float32))
    gpu.EXPERTS.grouped_gemm(upload(gpu, a), upload(gpu, w), D, upload(gpu, offsets), rows=8, groups=3, n=24, k=16, d_type=np.float32, gather=upload(gpu, gather), a_rows=6)
    exact, _ = ref.grouped(a.astype(float), w.astype(float).transpose(0, 2, 1), np.array([0, 2, 4, 8]), np.clip(gather, 0, 5), np.zeros((8, 24)))
    assert np.array_equal(D.to_host().reshape(8, 24), exact)
    falling = np.array([6, 2, 8, 1], np.int32)  # groups 0 and 2 have no rows then
    D = upload(gpu, np.full((8, 24), 99, np.float32))
    gpu.EXPERTS.grouped_gemm(upload(gpu, a), upload(gpu, w), D, upload(gpu, falling), rows=8, groups=3, n=24, k=16, d_type=np.float32, gather=upload(gpu, gather), a_rows=6)
    got = D.to_host().reshape(8, 24)
    assert np.all(got[:2] == 99)
    D = upload(gpu, np.full((3, 16, 24), 99, np.float32))
    gpu.EXPERTS.grouped_wgrad(upload(gpu, a), upload(gpu, rng.integers(-2, 3, (6, 24)).astype(np.float16)), D, upload(gpu, np.array([3, 1, 2, 99], np.int32)), rows=6, groups=3,
                              m=16, n=24)
    assert not D.to_host()[:16 * 24].any()


# ------------------------------------------------------------------------------------- joining the answers

@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,top,n,pitch,gated", [(1, 1, 1, 0, True), (3, 2, 7, 0, True), (16, 4, 512, 0, True), (5, 9, 2056, 8, True), (33, 8, 4096, 0, False), (70, 5, 100, 4, True), (9, 3, 2048, 3, False)])
def test_combine_and_its_gradient(gpu, tokens, top, n, pitch, gated, kind):
    kind, rng = KINDS[kind], np.random.default_rng(tokens + n)
    rows = tokens * top + 3
    h, dy = kind.load(kind.store(rng.normal(size=(rows, n)))), kind.load(kind.store(rng.normal(size=(tokens, n))))
    gates = rng.random((tokens, top)).astype(np.float32)
    place = rng.permutation(rows)[:tokens * top].reshape(tokens, top).astype(np.int32)
    place[rng.random((tokens, top)) < 0.2] = -1
    if tokens > 3:
        place[2] = -1
        place[3, 0] = rows + 5
    h_stored = _padded(kind, h, n + pitch)
    unplaced = np.setdiff1d(np.arange(rows), place)
    h_stored[unplaced] = 0x7FC0 if kind.name == "bf16" else np.nan
    Y, dH, dg = upload(gpu, np.full((tokens, n + pitch), 9, kind.dtype)), upload(gpu, np.full((rows, n + pitch), 9, kind.dtype)), upload(gpu, np.full((tokens, top), 7, np.float32))
    H, G, at = upload(gpu, h_stored), upload(gpu, gates) if gated else None, upload(gpu, place)
    sizes = dict(tokens=tokens, top=top, n=n, rows=rows, dtype=kind.marker(gpu), gates=G, ldh=n + pitch, ldy=n + pitch)
    gpu.EXPERTS.combine(H, at, Y, **sizes)
    gpu.EXPERTS.combine_grad(upload(gpu, _padded(kind, dy, n + pitch)), H, at, dH, dg, lddh=n + pitch, **sizes)
    g64 = gates.astype(np.float64) if gated else np.ones((tokens, top))
    has = (place >= 0) & (place < rows)
    answers = np.where(has[..., None], h[np.where(has, place, 0)], 0.0)
    y, got = Y.to_host().reshape(tokens, n + pitch), dH.to_host().reshape(rows, n + pitch)
    assert np.all(y[:, n:] == 9) and np.all(got[:, n:] == 9) and np.all(got[unplaced] == 9)
    _check(kind.load(y[:, :n]), (g64[..., None] * answers).sum(1), (g64[..., None] * np.abs(answers)).sum(1), top, kind)
    want = g64[has][:, None] * np.repeat(np.arange(tokens), top).reshape(tokens, top)[has][:, None] * 0 + g64[has][:, None] * dy[np.nonzero(has)[0]]
    _check(kind.load(got[place[has], :n]), want, np.abs(want), 1, kind)
    _check(dg.to_host().reshape(tokens, top).astype(np.float64), (answers * dy[:, None]).sum(2), np.abs(answers * dy[:, None]).sum(2), n, KINDS["f32"])
    assert not dg.to_host().reshape(tokens, top)[~has].any()
    dH2 = upload(gpu, np.full((rows, n + pitch), 9, kind.dtype))
    gpu.EXPERTS.combine_grad(upload(gpu, _padded(kind, dy, n + pitch)), None, at, dH2, None, lddh=n + pitch, **sizes)
    assert np.array_equal(dH2.to_host(), dH.to_host())


# ------------------------------------------------------------------------------------- microscaled 4-bit matrices

@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,k,pitch", [(1, 1, 0), (3, 32, 0), (2, 33, 0), (5, 250, 6), (4, 256, 0), (7, 1000, 8), (64, 520, 1), (33, 2048, 0)])
def test_mxfp4_quantize_and_back(gpu, rows, k, pitch, kind):
    Q, kind, rng = gpu.MXFP4, KINDS[kind], np.random.default_rng(rows + k)
    x = rng.normal(size=(rows, k)) * np.exp(rng.normal(size=(rows, 1)) * 3)
    x = kind.load(kind.store(np.where(rng.random((rows, k)) < 0.2, np.round(x * 4) / 4, x)))  # (quarters: ties)
    x[rng.random((rows, k)) < 0.1] = 0.0
    if k > 64:
        x[0, 32:64] = 0.0
        x[-1, 40] = -0.0
    blocks = -(-k // 32)
    ldq, lds = 16 * blocks + (32 if pitch else 0), rows + rows % 2 + (4 if pitch else 0)
    codes, scales = upload(gpu, np.full((rows, ldq), 0xAB, np.uint8)), upload(gpu, np.full((-(-blocks // 8), lds, 8), 0xAB, np.uint8))
    Q.quantize(upload(gpu, _padded(kind, x, k + pitch)), codes, scales, rows=rows, k=k, dtype=kind.marker(gpu), ld=k + pitch, ldq=ldq, lds=lds)
    want_codes, want_scales, value = ref.quantize(x)
    got = codes.to_host().reshape(rows, ldq)
    assert np.array_equal(got[:, :16 * blocks], want_codes) and np.all(got[:, 16 * blocks:] == 0xAB)
    got = scales.to_host().reshape(-1, lds, 8)
    assert np.array_equal(got[:, :rows].transpose(1, 0, 2).reshape(rows, -1)[:, :blocks], want_scales)
    for out in ("bf16", "f32", "f16"):
        okind = KINDS[out]
        back = upload(gpu, np.full((rows, k + pitch), 9, okind.dtype))
        Q.dequantize(codes, scales, back, rows=rows, k=k, dtype=okind.marker(gpu), ldq=ldq, lds=lds, ld=k + pitch)
        back = back.to_host().reshape(rows, k + pitch)
        assert np.all(back[:, k:] == 9)
        assert np.array_equal(okind.load(back[:, :k]), value.astype(np.float16).astype(np.float64) if out == "f16" else value)


def test_mxfp4_extremes(gpu):
    """Float32's range: subnormals, the largest, infinities and NaN, each block by itself."""
    Q = gpu.MXFP4
    tiny, big = np.float32(1e-45), np.finfo(np.float32).max
    x = np.zeros((12, 64), np.float32)
    for r, v in enumerate((tiny, 2.0 ** -149 * 3, 2.0 ** -127, 2.0 ** -126, 2.0 ** -125, 2.0 ** -124 * 1.9, big, -big, np.inf, -np.inf, np.nan, 7.0)):
        x[r, 3], x[r, 9], x[r, 40] = v, 0.3 * v if np.isfinite(v) else 1.0, r
    codes, scales, back = upload(gpu, np.zeros((12, 32), np.uint8)), upload(gpu, np.zeros((1, 12, 8), np.uint8)), upload(gpu, np.zeros((12, 64), np.float32))
    Q.quantize(upload(gpu, x), codes, scales, rows=12, k=64, dtype=np.float32)
    Q.dequantize(codes, scales, back, rows=12, k=64)
    with np.errstate(invalid="ignore"):
        want_codes, want_scales, value = ref.quantize(x.astype(np.float64))
    got_scales = scales.to_host().reshape(12, 8)
    assert np.array_equal(got_scales[:, :2], want_scales) and not got_scales[:, 2:].any()
    fine = want_scales[:, 0] != 255
    assert np.array_equal(codes.to_host().reshape(12, 32)[fine], want_codes[fine])
    back = back.to_host().reshape(12, 64)
    assert np.array_equal(np.isnan(back), np.isnan(value)) and np.array_equal(back[fine], value[fine].astype(np.float32))


def _random_mxfp4(rng, rows, k, spread=3, blocks_of_nan=0):
    """Any codes, scales of a few powers of two around 1; what lies beyond k is zero, the scales' padding stands for NaN."""
    blocks = -(-k // 32)
    codes = rng.integers(0, 256, (rows, 16 * blocks)).astype(np.uint8)
    value = np.stack([codes & 15, codes >> 4], -1).reshape(rows, -1)
    value[:, k:] = 0
    codes = (value[:, 0::2] | value[:, 1::2] << 4).astype(np.uint8)
    scales = rng.integers(127 - spread, 127 + spread + 1, (rows, blocks)).astype(np.uint8)
    x = np.where(value & 8, -1.0, 1.0) * ref.E2M1[value & 7] * np.exp2(np.repeat(scales.astype(float), 32, 1) - 127)
    return codes, scales, x[:, :k]


@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("m,n,k,pad", [(1, 1, 1, 0), (1, 64, 32, 0), (5, 37, 100, 0), (16, 256, 256, 16), (33, 130, 992, 32), (130, 258, 288, 0), (300, 520, 1025, 16), (257, 264, 4096, 0), (64, 96, 65, 0)])
def test_mxfp4_gemm(gpu, m, n, k, pad, out):
    Q, okind, rng = gpu.MXFP4, KINDS[out], np.random.default_rng(m + n + k)
    a, b = _random_mxfp4(rng, m, k), _random_mxfp4(rng, n, k)
    pitch = 16 * -(-k // 32) + pad
    lds_a, lds_b = m + m % 2 + pad, n + n % 2 + pad
    D = upload(gpu, np.full((m, n + pad), 9, okind.dtype))
    args = []
    for (codes, scales, _), lds in ((a, lds_a), (b, lds_b)):
        args += [upload(gpu, ref.packed(codes, pitch, 0xFF)), upload(gpu, ref.panels(scales, lds, 255))]
    Q.gemm(*args, D, m=m, n=n, k=k, d_type=okind.marker(gpu), lda=pitch, ldb=pitch, lds_a=lds_a, lds_b=lds_b, ldd=n + pad)
    got = D.to_host().reshape(m, n + pad)
    assert np.all(got[:, n:] == 9)
    _check(okind.load(got[:, :n]), a[2] @ b[2].T, np.abs(a[2]) @ np.abs(b[2]).T, k, okind)


@pytest.mark.parametrize("epilogue", [None, "gated_silu"])
@pytest.mark.parametrize("rows,groups,n,k", [(1, 1, 2, 32), (7, 3, 38, 96), (70, 5, 256, 544), (64, 64, 64, 512), (260, 3, 264, 320), (600, 130, 40, 64), (1000, 4, 512, 256)])
def test_mxfp4_grouped_gemm(gpu, rows, groups, n, k, epilogue):
    Q, rng, okind = gpu.MXFP4, np.random.default_rng(rows + n), KINDS["f32"]
    offsets = _sizes_of(groups, rows, rng, 0.3)
    if groups > 1 and rows > 20:
        offsets = np.clip(offsets, 3, rows - 2)
    a_rows = max(1, rows // 2)
    gather = rng.integers(0, a_rows, rows).astype(np.int32) if rows % 2 == 0 else None
    a = _random_mxfp4(rng, a_rows if gather is not None else rows, k, 1)
    w = [_random_mxfp4(rng, n, k, 1) for _ in range(groups)]
    width = n if epilogue is None else n // 2
    D = upload(gpu, np.full((rows, width), 99, np.float32))
    Q.grouped_gemm(upload(gpu, a[0]), upload(gpu, ref.panels(a[1], fill=255)), upload(gpu, np.stack([x[0] for x in w])),
                   upload(gpu, np.stack([ref.panels(x[1], fill=255) for x in w])), D, upload(gpu, offsets), rows=rows, groups=groups, n=n, k=k, d_type=np.float32,
                   gather=None if gather is None else upload(gpu, gather), a_rows=len(a[2]), epilogue=epilogue)
    got = D.to_host().reshape(rows, width).astype(np.float64)
    exact, size = ref.grouped(a[2], np.stack([x[2].T for x in w]), offsets, gather, np.zeros((rows, n)))
    inside = (np.arange(rows) >= offsets[0]) & (np.arange(rows) < offsets[-1])
    assert np.all(got[~inside] == 99)
    if epilogue is None:
        _check(got[inside], exact[inside], size[inside], k, okind)
    else:
        with np.errstate(over="ignore"):
            want = ref.gated(exact)
        error = (k + 2) * 2.0 ** -24 * (1.1 * size[:, 0::2] * np.abs(exact[:, 1::2]) + np.abs(exact[:, 0::2]) * size[:, 1::2])
        assert np.all(np.abs(got - want)[inside] <= (error + 64 * 2.0 ** -23 * (1 + np.abs(exact[:, 0::2])) * np.abs(want) + 2.0 ** -25)[inside])


@pytest.mark.parametrize("rows,groups,n,k", [(4000, 1, 4088, 600), (2900, 3, 4096, 1000), (1000, 4, 2056, 328), (500, 12, 1032, 2080), (16, 1, 4096, 1120)])
def test_mxfp4_grouped_gemm_large(gpu, rows, groups, n, k):
    """Whole numbers of magnitude 0 to 2 and scales of 1, 2 and 4: exact in Float32."""
    Q, rng = gpu.MXFP4, np.random.default_rng(rows)
    offsets = _large_groups(groups, rows)
    a_rows = rows // 2 + 7
    gather = rng.integers(0, a_rows, rows).astype(np.int32)

    def matrix(rows):
        blocks = -(-k // 32)
        value = rng.choice(np.array([0, 2, 4, 8 + 2, 8 + 4], np.uint8), (rows, 32 * blocks))
        value[:, k:] = 0
        scales = rng.integers(127, 130, (rows, blocks)).astype(np.uint8)
        x = np.where(value & 8, -1, 1) * ref.E2M1[value & 7] * np.exp2(np.repeat(scales.astype(np.float32), 32, 1) - 127)
        return (value[:, 0::2] | value[:, 1::2] << 4).astype(np.uint8), ref.panels(scales, fill=255), x[:, :k].astype(np.float32)

    a, w = matrix(a_rows), [matrix(n) for _ in range(groups)]
    D = upload(gpu, np.full((rows, n), 99, np.float32))
    Q.grouped_gemm(upload(gpu, a[0]), upload(gpu, a[1]), upload(gpu, np.stack([x[0] for x in w])), upload(gpu, np.stack([x[1] for x in w])), D, upload(gpu, offsets), rows=rows,
                   groups=groups, n=n, k=k, d_type=np.float32, gather=upload(gpu, gather), a_rows=a_rows)
    got = D.to_host().reshape(rows, n)
    for g in range(groups):
        r = slice(offsets[g], offsets[g + 1])
        assert np.array_equal(got[r], a[2][gather[r]] @ w[g][2].T), g
    assert np.all(got[:offsets[0]] == 99) and np.all(got[offsets[-1]:] == 99)


def test_mxfp4_scales_that_stand_for_nan(gpu):
    """A block with an infinity makes its row's and column's results NaN and no others."""
    Q, rng = gpu.MXFP4, np.random.default_rng(3)
    x, y = rng.normal(size=(6, 320)).astype(np.float32), rng.normal(size=(5, 320)).astype(np.float32)
    x[2, 300] = np.inf
    ops = []
    for v in (x, y):
        codes, scales = upload(gpu, np.zeros(Q.codes_bytes(len(v), 320), np.uint8)), upload(gpu, np.zeros(Q.scales_bytes(len(v), 320), np.uint8))
        Q.quantize(upload(gpu, v), codes, scales, rows=len(v), k=320, dtype=np.float32)
        ops += [codes, scales]
    D = upload(gpu, np.zeros((6, 5), np.float32))
    Q.gemm(*ops, D, m=6, n=5, k=320, d_type=np.float32)
    got = D.to_host().reshape(6, 5)
    assert np.isnan(got[2]).all() and np.isfinite(np.delete(got, 2, 0)).all()


def test_calls_on_a_stream_of_their_own(gpu):
    """The same results from work that is queued on another stream than the default one."""
    E, rng = gpu.EXPERTS, np.random.default_rng(4)
    s = gpu.Stream()
    z, x, w = rng.normal(size=(300, 16)).astype(np.float32), rng.normal(size=(300, 64)).astype(np.float16), rng.normal(size=(16, 72, 64)).astype(np.float16)
    outs = []
    for stream in (None, s):
        i32 = lambda n: upload(gpu, np.zeros(n, np.int32))  # noqa: E731
        chosen, gates, offsets, rows, place = i32(600), upload(gpu, np.zeros(600, np.float32)), i32(17), i32(600), i32(600)
        ws = upload(gpu, np.zeros(max(16, E.route_workspace(300, 16, 2)), np.uint8))
        H, Y = upload(gpu, np.zeros((600, 72), np.float16)), upload(gpu, np.zeros((300, 72), np.float16))
        dz, dx, dw = upload(gpu, z), upload(gpu, x), upload(gpu, w)
        gpu.synchronize()
        E.route(dz, chosen, gates, offsets, rows, place, tokens=300, experts=16, top=2, workspace=ws, stream=stream)
        E.grouped_gemm(dx, dw, H, offsets, rows=600, groups=16, n=72, k=64, gather=rows, a_rows=300, stream=stream)
        E.combine(H, place, Y, tokens=300, top=2, n=72, rows=600, gates=gates, stream=stream)
        gpu.synchronize(stream)
        outs.append(Y.to_host())
    assert np.array_equal(*outs) and outs[0].any()
