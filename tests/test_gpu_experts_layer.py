"""The experts' layer of the examples on the GPU: serving in 16 and 4 bits and a training step against the same layer in 64
bits; and the activation between its products by itself.

Tolerances of the layer.  Every stage rounds to Float16 (relative 2^-11) what it stores; an answer passes at most six such
roundings (x to y: Z, A, H, Y; backwards: dH, dA, dZ, dX_rows, dX and those that the forward pass left in Z, A, H), each of
which moves the result, in the norm, by at most 2^-11 times a factor that stays below 4 for matrices of this distribution
(normal entries of variance 1 / k keep the norm, the gated activation has a slope below 1.1 per unit of its inputs, which are
of order 1).  12 * 4 * 2^-11 = 0.024 in the norm bounds them all."""
import importlib.util
import os

import numpy as np
import pytest

import experts_oracle as ref
from experts_oracle import KINDS, upload

LAYER = 12 * 4 * 2.0 ** -11


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cudanative.jl_amd", "examples", "experts_layer.py")
    spec = importlib.util.spec_from_file_location("experts_layer_example", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _gated_grad(z, da):
    u, v = z[..., 0::2], z[..., 1::2]
    s = 1 / (1 + np.exp(-u))
    dz = np.empty(z.shape)
    dz[..., 0::2], dz[..., 1::2] = da * v * s * (1 + u * (1 - s)), da * u * s
    return dz


class Layer64:
    def __init__(self, w1, w2, top):
        self.w1, self.w2, self.top = w1, w2, top

    def forward(self, x, logits):
        self.x, self.logits = x, logits
        self.chosen, self.gates, _, _, _ = ref.route(logits.astype(np.float64), self.top, False)
        y = np.zeros((len(x), self.w2.shape[1]))
        for t in range(len(x)):
            for j, e in enumerate(self.chosen[t]):
                if e >= 0:
                    y[t] += self.gates[t, j] * (self.w2[e] @ ref.gated(self.w1[e] @ x[t]))
        return y

    def backward(self, dy):
        dx, dw1, dw2, dg = np.zeros(self.x.shape), np.zeros(self.w1.shape), np.zeros(self.w2.shape), np.zeros(self.gates.shape)
        for t in range(len(dy)):
            for j, e in enumerate(self.chosen[t]):
                if e < 0:
                    continue
                z = self.w1[e] @ self.x[t]
                a = ref.gated(z)
                dg[t, j] = dy[t] @ (self.w2[e] @ a)
                dh = self.gates[t, j] * dy[t]
                dw2[e] += np.outer(dh, a)
                dz = _gated_grad(z, self.w2[e].T @ dh)
                dw1[e] += np.outer(dz, self.x[t])
                dx[t] += self.w1[e].T @ dz
        return dx, ref.route_grad(self.logits.astype(np.float64), self.chosen, dg, False), dw1, dw2


def _inputs(tokens, experts, width, hidden, masked):
    rng = np.random.default_rng(tokens + width)
    w1 = (rng.normal(size=(experts, 2 * hidden, width)) / width ** 0.5).astype(np.float16)
    w2 = (rng.normal(size=(experts, width, hidden)) / hidden ** 0.5).astype(np.float16)
    x, dy = rng.normal(size=(tokens, width)).astype(np.float16), rng.normal(size=(tokens, width)).astype(np.float16)
    logits = rng.normal(size=(tokens, experts)).astype(np.float32)
    logits[:, experts - 1] = -np.inf  # an expert without rows
    if masked:
        logits[0] = -np.inf  # a token without experts
        logits[1, 1:] = -np.inf
    return w1, w2, x, dy, logits


def _far(got, want):
    """Distance in the norm; exact zeros (the gradient of a softmax over one choice) have to be met."""
    if not want.any():
        return 0.0 if not got.any() else np.inf
    return np.linalg.norm(got.astype(np.float64).reshape(want.shape) - want) / np.linalg.norm(want)


SIZES = [(2, 4, 1, 16, 8, False), (16, 8, 2, 128, 64, True), (77, 5, 3, 200, 72, True), (130, 3, 2, 256, 128, False), (9, 4, 2, 34, 10, True)]


def test_gradients_of_the_layer_in_64_bits_against_differences():
    w1, w2, x, dy, logits = (v.astype(np.float64) for v in _inputs(3, 4, 6, 5, False))
    logits = np.where(np.isinf(logits), -9.0, logits)
    layer, h = Layer64(w1, w2, 2), 1e-5
    layer.forward(x, logits)
    got = layer.backward(dy)
    for i, v in enumerate((x, logits, w1, w2)):
        want = np.zeros(v.size)
        for at in range(v.size):
            old = v.flat[at]
            v.flat[at] = old + h
            up = (layer.forward(x, logits) * dy).sum()
            v.flat[at] = old - h
            down = (layer.forward(x, logits) * dy).sum()
            v.flat[at] = old
            want[at] = (up - down) / (2 * h)
        # (differences of second order: an error of h^2 times a third derivative of order 1 to 10, and 1e-16 / h of cancellation)
        assert np.allclose(got[i].ravel(), want, rtol=1e-6, atol=1e-7), i


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,top,width,hidden,masked", SIZES)
def test_training_step(gpu, example, tokens, experts, top, width, hidden, masked):
    w1, w2, x, dy, logits = _inputs(tokens, experts, width, hidden, masked)
    layer = example.ExpertsLayer(gpu, upload(gpu, w1), upload(gpu, w2), tokens=tokens, experts=experts, top=top, width=width, hidden=hidden)
    layer.prepare_training()
    X, Z, dY = upload(gpu, x), upload(gpu, logits), upload(gpu, dy)
    plain = Layer64(w1.astype(np.float64), w2.astype(np.float64), top)
    y = plain.forward(x.astype(np.float64), logits)
    served = layer.serve(X, Z, tokens=tokens).to_host()
    assert _far(served, y) <= LAYER
    assert _far(layer.forward(X, Z, tokens=tokens).to_host(), y) <= LAYER
    want = plain.backward(dy.astype(np.float64))
    for got, exact in zip(layer.backward(X, Z, dY, tokens=tokens), want):
        got = got.to_host()
        assert np.isfinite(got).all() and _far(got, exact) <= LAYER
    if masked:
        assert not served.reshape(tokens, width)[0].any() and not layer.dX.to_host().reshape(tokens, width)[0].any()
    assert not layer.dW1.to_host().reshape(w1.shape)[experts - 1].any()
    # a second batch's gradients on top of the first's
    layer.forward(X, Z, tokens=tokens)
    layer.backward(X, Z, dY, tokens=tokens, accumulate=True)
    assert _far(layer.dW1.to_host(), 2 * want[2]) <= LAYER and _far(layer.dW2.to_host(), 2 * want[3]) <= LAYER


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,top,width,hidden,masked", SIZES)
def test_serving_in_4_bits(gpu, example, tokens, experts, top, width, hidden, masked):
    """Against the 64-bit layer on weights and activations that were rounded to 4 bits; the activations between the products
    are taken from the GPU, since a value at the edge between two codes may fall on either side."""
    w1, w2, x, dy, logits = _inputs(tokens, experts, width, hidden, masked)
    layer = example.ExpertsLayer(gpu, upload(gpu, w1), upload(gpu, w2), tokens=tokens, experts=experts, top=top, width=width, hidden=hidden)
    layer.pack()
    got = layer.serve_mxfp4(upload(gpu, x), upload(gpu, logits), tokens=tokens).to_host()
    w1q, w2q = (ref.quantize(w.reshape(-1, w.shape[2]).astype(np.float64))[2].reshape(w.shape) for w in (w1, w2))
    xq = ref.quantize(x.astype(np.float64))[2]
    chosen, gates, offsets, rows, place = ref.route(logits.astype(np.float64), top, False)
    a, y = layer.A.to_host().reshape(-1, hidden), np.zeros((tokens, width))
    aq = ref.quantize(a.astype(np.float64))[2]
    exact_a = np.zeros(a.shape)
    for e in range(experts):
        for r in range(offsets[e], offsets[e + 1]):
            exact_a[r] = ref.gated(w1q[e] @ xq[rows[r]])
    assert _far(a, exact_a) <= LAYER
    for t in range(tokens):
        for j, e in enumerate(chosen[t]):
            if e >= 0:
                y[t] += gates[t, j] * (w2q[e] @ aq[place[t, j]])
    assert _far(got, y) <= LAYER


# Float32 of the activation between its load and its rounding: some ten operations of relative error 2^-24 each, exp's own
# error of |u| 2^-24 for the scaled argument (|u| at most 100 before s or 1 - s vanishes) on top, and 1 + u (1 - s) cancels
# near its zero at u = -1.28, where the terms are below 1.3: an absolute error of 2^-16 of |da v| covers all.
@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("rows,n,pitch,odd", [(1, 2, 0, 0), (5, 6, 0, 0), (3, 8, 0, 0), (70, 64, 8, 0), (33, 100, 4, 0), (7, 2064, 0, 0), (300, 512, 0, 1), (2, 4096, 16, 0)])
def test_gated_silu_and_its_gradient(gpu, rows, n, pitch, odd, kind):
    kind, rng, E = KINDS[kind], np.random.default_rng(rows + n), gpu.EXPERTS
    z, da = kind.load(kind.store(4 * rng.normal(size=(rows, n)))), kind.load(kind.store(rng.normal(size=(rows, n // 2))))
    z[0, 0], z[-1, n - 2] = -300.0, 60.0
    ldz, lda = n + pitch, n // 2 + pitch // 2

    def padded(a, pitch):
        out = np.full((rows, pitch), 9, kind.dtype)
        out[:, :a.shape[1]] = kind.store(a)
        return np.concatenate([np.zeros(odd, kind.dtype), out.reshape(-1)])

    Z, dA = upload(gpu, padded(z, ldz)), upload(gpu, padded(da, lda))
    A, dZ = upload(gpu, padded(0 * da, lda)), upload(gpu, padded(0 * z, ldz))
    at = lambda v: v.ptr + 2 * odd  # noqa: E731
    sizes = dict(rows=rows, n=n, dtype=kind.marker(gpu), ldz=ldz)
    E.gated_silu(at(Z), at(A), lda=lda, **sizes)
    E.gated_silu_grad(at(Z), at(dA), at(dZ), ldda=lda, lddz=ldz, **sizes)
    a, dz = A.to_host()[odd:].reshape(rows, lda), dZ.to_host()[odd:].reshape(rows, ldz)
    assert np.all(a[:, n // 2:] == 9) and np.all(dz[:, n:] == 9)
    with np.errstate(over="ignore"):
        want, dwant = ref.gated(z), _gated_grad(z, da)
    assert np.all(np.abs(kind.load(a[:, :n // 2]) - want) <= 1.01 * kind.roundoff * np.abs(want) + 2.0 ** -16 * np.abs(want) + 2.0 ** -25)
    scale = np.repeat(np.abs(da), 2, 1) * np.maximum(np.abs(z[:, np.arange(n) ^ 1]), np.abs(z))
    assert np.all(np.abs(kind.load(dz[:, :n]) - dwant) <= 1.01 * kind.roundoff * np.abs(dwant) + 2.0 ** -16 * scale + 2.0 ** -25)
    E.gated_silu_grad(at(Z), at(dA), at(Z), ldda=lda, lddz=ldz, **sizes)  # in place
    assert np.array_equal(Z.to_host()[odd:].reshape(rows, ldz)[:, :n], dz[:, :n])


def test_gated_silu_refusals(miw):
    E, L, P = miw.EXPERTS, miw._lib, 1 << 20
    ok = dict(rows=4, n=8)

    def refused(code, call, *args, **kw):
        with pytest.raises(miw.MIWError) as e:
            call(*args, **kw)
        assert e.value.code == code, e.value

    for call, count in ((E.gated_silu, 2), (E.gated_silu_grad, 3)):
        for i in range(count):
            refused(L.ERR_NULL_POINTER, call, *[None if i == j else P * (1 + j) for j in range(count)], **ok)
            refused(L.ERR_MISALIGNED, call, *[P + 1 if i == j else P * (1 + j) for j in range(count)], **ok)
        args = [P * (1 + j) for j in range(count)]
        for bad in (dict(rows=-1), dict(n=0), dict(n=7), dict(n=1 << 27)):
            refused(L.ERR_INVALID_SHAPE, call, *args, **{**ok, **bad})
        refused(L.ERR_INVALID_VALUE, call, *args, **ok, ldz=7)
        refused(L.ERR_INVALID_TYPE, call, *args, **ok, dtype=np.float32)
        call(*[None] * count, **{**ok, "rows": 0})
    refused(L.ERR_INVALID_VALUE, E.gated_silu, P, 2 * P, **ok, lda=3)
    refused(L.ERR_INVALID_VALUE, E.gated_silu_grad, P, 2 * P, 3 * P, **ok, ldda=3)
    refused(L.ERR_INVALID_VALUE, E.gated_silu_grad, P, 2 * P, 3 * P, **ok, lddz=7)
    refused(L.ERR_INVALID_VALUE, E.gated_silu_grad, P, 2 * P, P, **ok, ldz=8, lddz=16)


def test_addresses_that_are_no_plain_integers(miw):
    """numpy's integers and typed pointers are addresses too; other numbers are not.  (Nothing is launched for no rows, and a
    null address is looked at first.)"""
    E, L = miw.EXPERTS, miw._lib
    E.gated_silu(np.int64(1 << 20), np.uint64(1 << 21), rows=0, n=8)
    null, typed = miw.DevicePtr(np.float16, 0), miw.DevicePtr(np.float16, 1 << 20)
    for Z, A in ((null, typed), (typed, null), (np.int64(0), typed)):
        with pytest.raises(miw.MIWError) as e:
            E.gated_silu(Z, A, rows=4, n=8)
        assert e.value.code == L.ERR_NULL_POINTER
    with pytest.raises(TypeError):
        E.gated_silu(1.5, 1 << 20, rows=4, n=8)
    with pytest.raises(TypeError):
        E.gated_silu("a", 1 << 20, rows=4, n=8, dtype="no type")
