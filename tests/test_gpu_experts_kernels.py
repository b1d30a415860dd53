"""Each kernel behind the experts' operators at the sizes and layouts where it can go wrong, on whole numbers whose results are exact."""
import numpy as np
import pytest

import experts_oracle as ref
from experts_oracle import KINDS, upload
from test_gpu_experts import _sizes_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,groups,n,k", [(2000, 3, 584, 544), (900, 5, 198, 288), (4000, 2, 4088, 800), (1500, 3, 1411, 320), (60, 6, 200, 512), (10500, 70, 520, 300)])
def test_mxfp4_grouped_gemm_panels_of_all_groups(gpu, rows, groups, n, k):
    """Every group's matrix in the same panels, one behind the other, widths that no tile divides; the last panel ends with the last group."""
    Q, rng = gpu.MXFP4, np.random.default_rng(n)
    own, blocks = n + n % 2, -(-k // 32)
    offsets = _sizes_of(groups, rows, rng, 0.0)
    value = rng.choice(np.array([0, 2, 4, 8 + 2, 8 + 4], np.uint8), (rows + groups * own, 32 * blocks))
    value[:, k:] = 0
    scales = rng.integers(127, 130, (rows + groups * own, blocks)).astype(np.uint8)
    x = (np.where(value & 8, -1, 1) * ref.E2M1[value & 7] * np.exp2(np.repeat(scales.astype(np.float32), 32, 1) - 127))[:, :k].astype(np.float32)
    codes = (value[:, 0::2] | value[:, 1::2] << 4).astype(np.uint8)
    D = upload(gpu, np.full((rows, n), 99, np.float32))
    Q.grouped_gemm(upload(gpu, codes[:rows]), upload(gpu, ref.panels(scales[:rows], fill=255)), upload(gpu, codes[rows:]), upload(gpu, ref.panels(scales[rows:], fill=255)), D,
                   upload(gpu, offsets), rows=rows, groups=groups, n=n, k=k, d_type=np.float32, lds_w=groups * own, stride_w=own * codes.shape[1], stride_ws=8 * own)
    got, w = D.to_host().reshape(rows, n), x[rows:].reshape(groups, own, k)[:, :n]
    for g in range(groups):
        r = slice(offsets[g], offsets[g + 1])
        assert np.array_equal(got[r], x[r] @ w[g].T), g


@pytest.mark.parametrize("kind", ["f16", "mxfp4"])
def test_many_groups_without_rows(gpu, kind):
    """65536 groups, ten rows, wide weights: memory for all of them, and numbers in those that have rows."""
    groups, n, k, E, Q, rng = 65536, 2056, 32, gpu.EXPERTS, gpu.MXFP4, np.random.default_rng(3)
    used, lib = np.array([0, 1, 4097, 30000, 65535]), gpu._lib.load()
    sizes = np.zeros(groups, np.int64)
    sizes[used] = [1, 3, 1, 3, 2]
    offsets = upload(gpu, np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32))
    a, w = rng.integers(-2, 3, (10, k)).astype(np.float16), rng.integers(-2, 3, (len(used), n, k)).astype(np.float16)
    D = upload(gpu, np.full((10, n), 99, np.float32))

    def spread(parts):
        parts = np.ascontiguousarray(parts).reshape(len(used), -1).view(np.uint8)
        out = gpu.DeviceArray.undef(np.uint8, groups * parts.shape[1])
        for g, part in zip(used, parts):
            assert lib.miw_memcpy_h2d(out.ptr + int(g) * parts.shape[1], part.ctypes.data, part.nbytes) == 0
        return out

    if kind == "f16":
        E.grouped_gemm(upload(gpu, a), spread(w), D, offsets, rows=10, groups=groups, n=n, k=k, d_type=np.float32)
    else:
        quantized = [ref.quantize(x.astype(float)) for x in (a, *w)]
        assert all(np.array_equal(q[2], x) for q, x in zip(quantized, (a, *w)))
        Q.grouped_gemm(upload(gpu, quantized[0][0]), upload(gpu, ref.panels(quantized[0][1])), spread([q[0] for q in quantized[1:]]), spread([ref.panels(q[1]) for q in quantized[1:]]), D,
                       offsets, rows=10, groups=groups, n=n, k=k, d_type=np.float32)
    got, at = D.to_host().reshape(10, n), 0
    for g, x in zip(used, w):
        for _ in range(sizes[g]):
            assert np.array_equal(got[at], x.astype(float) @ a[at].astype(float)), (g, at)
            at += 1


def test_route_and_its_gradient_of_2_to_25_tokens(gpu):
    """More tokens than one pass of the grid: a batch of tokens over and over gives that batch's results over and over."""
    E, rng = gpu.EXPERTS, np.random.default_rng(8)
    part, times, experts, top = 1 << 15, 1 << 10, 5, 2
    z, dg = rng.normal(size=(part, experts)).astype(np.float16), rng.normal(size=(part, top)).astype(np.float32)
    out = []
    for n, more in ((1, 0), (times, 7)):
        tokens = part * n + more
        repeat = lambda a: upload(gpu, np.concatenate([np.tile(a, (n, 1)), a[:more]]))  # noqa: E731
        new = lambda T, *shape: gpu.DeviceArray.undef(T, int(np.prod(shape)))  # noqa: E731
        sizes = dict(tokens=tokens, experts=experts, top=top, dtype=np.float16, over_all=True)
        Z, chosen, gates, offsets, rows, place = repeat(z), new(np.int32, tokens, top), new(np.float32, tokens, top), new(np.int32, experts + 1), new(np.int32, tokens, top), new(np.int32, tokens, top)
        dz = new(np.float16, tokens, experts)
        E.route(Z, chosen, gates, offsets, rows, place, workspace=new(np.uint8, E.route_workspace(tokens, experts, top)), **sizes)
        E.route_grad(Z, chosen, gates, repeat(dg), dz, **sizes)
        out.append([v.to_host() for v in (chosen, gates, dz)] + [offsets.to_host(), place.to_host()])
    small, large = out
    for s, l in zip(small[:3], large[:3]):
        assert np.array_equal(l[:len(s) * times].reshape(times, -1), np.broadcast_to(s, (times, len(s)))) and np.array_equal(l[len(s) * times:], s[:len(l) - len(s) * times])
    # the sorted position of each choice: those of its expert from the first on, in the order of tokens
    chosen, offsets, place = large[0], large[3], large[4]
    for e in range(experts):
        assert np.array_equal(place[chosen == e], np.arange(offsets[e], offsets[e + 1]))
    assert offsets[0] == 0 and offsets[-1] == len(chosen)


@pytest.mark.parametrize("experts", [8, 300])
def test_route_takes_infinity_for_the_largest_float(gpu, experts):
    """+inf counts as the largest finite Float32: the two are equal, and the lower expert goes first."""
    E, top = gpu.EXPERTS, 4
    most = np.finfo(np.float32).max
    z = np.zeros((3, experts), np.float32)
    z[0, [1, 3, 5]] = most, np.inf, most
    z[1, [0, experts - 1]] = np.inf, most
    z[2, [2, experts - 2]] = most, np.inf
    want = ref.route(z.astype(np.float64), top, False)
    for over_all in (False, True):
        out = [upload(gpu, np.zeros(n, t)) for n, t in ((3 * top, np.int32), (3 * top, np.float32), (experts + 1, np.int32), (3 * top, np.int32), (3 * top, np.int32))]
        E.route(upload(gpu, z), *out, tokens=3, experts=experts, top=top, over_all=over_all)
        assert np.array_equal(out[0].to_host().reshape(3, top), want[0])
        assert np.allclose(out[1].to_host().reshape(3, top), want[1], rtol=1e-6, atol=0)


# Units of 2^-24 of a gate: exp is off by at most one unit in the last place (2) of the numerator and of each summand (2), the sum takes at
# most sixteen registers' and four lanes' additions (20), the quotient is rounded once (1).  The differences of these logits are exact.
GATE = 25 * 2.0 ** -24


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("experts", [8, 120, 700])
@pytest.mark.parametrize("over_all", [False, True])
def test_small_gates_keep_their_bits(gpu, experts, kind, over_all):
    """Logits as far as 84 below the largest: gates of 10^-36 are as precise as gates of one half."""
    kind, rng = KINDS[kind], np.random.default_rng(experts)
    tokens, top, E = 40, 8, gpu.EXPERTS
    # multiples of 1/2 that every type holds; eight of them above the others
    z = np.full((tokens, experts), -45.0)
    z[:, :8] = rng.integers(-88, 81, (tokens, 8)) / 2
    z[:, 0] = 40.0
    out = [upload(gpu, np.zeros(n, t)) for n, t in ((tokens * top, np.int32), (tokens * top, np.float32), (experts + 1, np.int32), (tokens * top, np.int32), (tokens * top, np.int32))]
    Z, dgates, dz = upload(gpu, kind.store(z)), np.zeros((tokens, top), np.float32), upload(gpu, np.zeros((tokens, experts), kind.dtype))
    E.route(Z, *out, tokens=tokens, experts=experts, top=top, dtype=kind.marker(gpu), over_all=over_all)
    chosen, gates = (v.to_host().reshape(tokens, top) for v in out[:2])
    want = ref.route(z, top, over_all)
    assert np.array_equal(chosen, want[0])
    far = np.abs(gates - want[1]) / want[1]
    assert far.max() <= GATE, far.max() * 2.0 ** 24
    # the gradient from the largest choice alone: minus the product of two gates for every other one, in Float32 two gates' errors, a sum of sixteen
    # products and three roundings
    dgates[:, 0] = 1.0
    E.route_grad(Z, out[0], out[1], upload(gpu, dgates), dz, tokens=tokens, experts=experts, top=top, dtype=kind.marker(gpu), over_all=over_all)
    exact = ref.route_grad(z, want[0], dgates.astype(np.float64), over_all)
    others = (z < 40) & (exact != 0)
    far = np.abs(kind.load(dz.to_host().reshape(tokens, experts)) - exact)[others] - kind.roundoff * 1.01 * np.abs(exact[others])
    assert np.all(far <= (2 * GATE + 8 * 2.0 ** -24) * np.abs(exact[others]) + (2.0 ** -25 if kind.name == "f16" else 0.0))
