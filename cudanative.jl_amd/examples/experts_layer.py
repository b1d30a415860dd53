"""A feed-forward layer of experts on the library's operators: serving in 16, 8 and 4 bits, and training steps with a loss over a vocabulary.

Every token goes to `top` of `experts` pairs of matrices: Z = x W1 (gates and values side by side), A = silu(gate) * value,
H = A W2, and its answers are joined by the router's weights.

    route -> grouped_gemm (gated) -> grouped_gemm -> combine                               serve
    quantize -> grouped_gemm (gated) -> quantize -> grouped_gemm -> combine                serve_mxfp4, weights in 4 bits
    the same in 8 bits                                                                     serve_fp8
    combine_grad -> grouped_gemm, grouped_wgrad -> gated_silu_grad -> the same -> combine -> route_grad     backward

With prepare_training(fp8=True) the four products that make rows take 8-bit operands, the weights' in blocks of 128 x 128, so that the codes of W1 and W2 and of
their transposes stand for the same values; gradients to the weights stay products of 16 bits.  Of the columns before the activation 8 bits are kept.

Nothing waits for the device between the first call and the last; all buffers are the layer's own, allocated once.

    python cudanative.jl_amd/examples/experts_layer.py [tokens]
"""
import os
import sys
import time

import numpy as np


class ExpertsLayer:
    """W1: experts x 2 hidden x width (rows 2c and 2c + 1: gate and value of hidden unit c), W2: experts x width x hidden, both
    Float16 and on the device; at most `tokens` tokens a call."""

    def __init__(self, pkg, W1, W2, *, tokens, experts, top, width, hidden):
        self.pkg, self.W1, self.W2 = pkg, W1, W2
        self.experts, self.top, self.width, self.hidden, self.tokens = experts, top, width, hidden, tokens
        E, rows = pkg.EXPERTS, tokens * top
        new = pkg.DeviceArray.undef
        self.chosen, self.gates, self.offsets = new(np.int32, rows), new(np.float32, rows), new(np.int32, experts + 1)
        self.rows, self.place = new(np.int32, rows), new(np.int32, rows)
        self.workspace = new(np.uint8, max(16, E.route_workspace(tokens, experts, top)))
        self.A, self.H, self.Y = self._half(rows * hidden), self._half(rows * width), self._half(tokens * width)
        self.packed = None

    def _half(self, n):
        # Rows that belong to no expert are not written by the products and are read by the conversions.
        a = self.pkg.DeviceArray.undef(np.float16, n)
        a.fill_bytes(0)
        return a

    def _route(self, logits, tokens, stream):
        self.pkg.EXPERTS.route(logits, self.chosen, self.gates, self.offsets, self.rows, self.place, tokens=tokens, experts=self.experts,
                               top=self.top, workspace=self.workspace, stream=stream)

    def _join(self, tokens, stream):
        self.pkg.EXPERTS.combine(self.H, self.place, self.Y, tokens=tokens, top=self.top, n=self.width, rows=tokens * self.top, gates=self.gates,
                                 stream=stream)
        return self.Y

    def serve(self, x, logits, *, tokens, stream=None):
        """x: tokens x width Float16, logits: tokens x experts Float32; the answers, tokens x width."""
        E, rows = self.pkg.EXPERTS, tokens * self.top
        self._route(logits, tokens, stream)
        E.grouped_gemm(x, self.W1, self.A, self.offsets, rows=rows, groups=self.experts, n=2 * self.hidden, k=self.width, gather=self.rows,
                       a_rows=tokens, epilogue=E.GATED_SILU, stream=stream)
        E.grouped_gemm(self.A, self.W2, self.H, self.offsets, rows=rows, groups=self.experts, n=self.width, k=self.hidden, stream=stream)
        return self._join(tokens, stream)

    # ---- weights and activations in 4 bits

    def pack(self, stream=None):
        """Both weights in 4 bits, once.  All experts' matrices lie one behind the other in each panel of scales, every one on an even row;
        where their rows are even in number they are one tall matrix to the quantisation."""
        Q, new = self.pkg.MXFP4, self.pkg.DeviceArray.undef
        self.packed = []
        for W, n, k in ((self.W1, 2 * self.hidden, self.width), (self.W2, self.width, self.hidden)):
            own = n + n % 2
            lds, at_once, first = self.experts * own, self.experts if own == n else 1, getattr(W, "ptr", W)
            codes, scales = new(np.uint8, Q.codes_bytes(self.experts * n, k)), new(np.uint8, Q.scales_bytes(lds, k))
            for e in range(0, self.experts, at_once):
                Q.quantize(first + 2 * e * n * k, codes.ptr + Q.codes_bytes(e * n, k), scales.ptr + 8 * e * own, rows=at_once * n, k=k, lds=lds, stream=stream)
            self.packed.append((codes, scales, dict(n=n, k=k, lds_w=lds, stride_ws=8 * own)))
        self.x4 = new(np.uint8, Q.codes_bytes(self.tokens, self.width)), new(np.uint8, Q.scales_bytes(self.tokens, self.width))
        rows = self.tokens * self.top
        self.a4 = new(np.uint8, Q.codes_bytes(rows, self.hidden)), new(np.uint8, Q.scales_bytes(rows, self.hidden))

    def serve_mxfp4(self, x, logits, *, tokens, stream=None):
        """serve with weights and activations in 4 bits (after pack)."""
        Q, rows = self.pkg.MXFP4, tokens * self.top
        (w1, s1, sizes1), (w2, s2, sizes2) = self.packed
        self._route(logits, tokens, stream)
        Q.quantize(x, *self.x4, rows=tokens, k=self.width, stream=stream)
        Q.grouped_gemm(*self.x4, w1, s1, self.A, self.offsets, rows=rows, groups=self.experts, gather=self.rows, a_rows=tokens,
                       epilogue=self.pkg.EXPERTS.GATED_SILU, stream=stream, **sizes1)
        Q.quantize(self.A, *self.a4, rows=rows, k=self.hidden, stream=stream)
        Q.grouped_gemm(*self.a4, w2, s2, self.H, self.offsets, rows=rows, groups=self.experts, stream=stream, **sizes2)
        return self._join(tokens, stream)

    # ---- weights and activations in 8 bits

    def _codes(self, rows, k):
        Q, new = self.pkg.FP8, self.pkg.DeviceArray.undef
        return new(np.uint8, Q.codes_bytes(rows, k)), new(np.uint8, Q.scales_bytes(rows, k))

    def pack_fp8(self, stream=None):
        """Both weights in 8 bits, as they lie and turned (for the gradients to the rows); after every change of the weights."""
        Q, wmma = self.pkg.FP8, self.pkg.WMMA
        if getattr(self, "packed8", None) is None:
            rows = self.tokens * self.top
            self.x8, self.a8 = self._codes(self.tokens, self.width), self._codes(rows, self.hidden)
            self.packed8 = []
            for W, n, k in ((self.W1, 2 * self.hidden, self.width), (self.W2, self.width, self.hidden)):
                for rows, columns, layout in ((n, k, wmma.RowMajor), (k, n, wmma.ColMajor)):
                    each = Q.codes_bytes(rows, columns), Q.scales_bytes(rows, columns)
                    codes, scales = (self.pkg.DeviceArray.undef(np.uint8, self.experts * b) for b in each)
                    self.packed8.append((W, codes, scales, layout, each, dict(n=rows, k=columns)))
        for W, codes, scales, layout, each, sizes in self.packed8:
            n, k, first = sizes["n"], sizes["k"], getattr(W, "ptr", W)
            for e in range(self.experts):
                Q.quantize(first + 2 * e * n * k, codes.ptr + e * each[0], scales.ptr + e * each[1], rows=n, k=k, block_rows=128, x_layout=layout, stream=stream)

    def _product8(self, operand, which, D, tokens, stream, **kw):
        _, codes, scales, _, _, sizes = self.packed8[which]
        self.pkg.FP8.grouped_gemm(*operand, codes, scales, D, self.offsets, rows=tokens * self.top, groups=self.experts, stream=stream, **sizes, **kw)

    def serve_fp8(self, x, logits, *, tokens, stream=None):
        """serve with weights and activations in 8 bits (after pack_fp8)."""
        Q = self.pkg.FP8
        self._route(logits, tokens, stream)
        Q.quantize(x, *self.x8, rows=tokens, k=self.width, stream=stream)
        self._product8(self.x8, 0, self.A, tokens, stream, gather=self.rows, a_rows=tokens, epilogue=self.pkg.EXPERTS.GATED_SILU)
        Q.quantize(self.A, *self.a8, rows=tokens * self.top, k=self.hidden, stream=stream)
        self._product8(self.a8, 2, self.H, tokens, stream)
        return self._join(tokens, stream)

    # ---- training

    def prepare_training(self, fp8=False):
        rows, new = self.tokens * self.top, self.pkg.DeviceArray.undef
        self.fp8 = fp8
        if fp8:
            self.pack_fp8()
            self.kept, self.dh8, self.dz8 = self._codes(rows, 2 * self.hidden), self._codes(rows, self.width), self._codes(rows, 2 * self.hidden)
        self.Z, self.dH, self.dA, self.dX_rows, self.dX = (self._half(n) for n in (rows * 2 * self.hidden, rows * self.width, rows * self.hidden,
                                                                                     rows * self.width, self.tokens * self.width))
        self.dgates, self.dlogits = new(np.float32, rows), new(np.float32, self.tokens * self.experts)
        self.dW1, self.dW2 = new(np.float32, self.experts * 2 * self.hidden * self.width), new(np.float32, self.experts * self.width * self.hidden)

    def forward(self, x, logits, *, tokens, stream=None):
        """serve, with the columns before the activation kept for backward."""
        E, rows = self.pkg.EXPERTS, tokens * self.top
        self._route(logits, tokens, stream)
        if self.fp8:
            Q = self.pkg.FP8
            Q.quantize(x, *self.x8, rows=tokens, k=self.width, stream=stream)
            self._product8(self.x8, 0, self.Z, tokens, stream, gather=self.rows, a_rows=tokens)
            Q.gated_silu(self.Z, self.A, *self.kept, rows=rows, n=2 * self.hidden, stream=stream)
            Q.quantize(self.A, *self.a8, rows=rows, k=self.hidden, stream=stream)
            self._product8(self.a8, 2, self.H, tokens, stream)
            return self._join(tokens, stream)
        E.grouped_gemm(x, self.W1, self.Z, self.offsets, rows=rows, groups=self.experts, n=2 * self.hidden, k=self.width, gather=self.rows,
                       a_rows=tokens, stream=stream)
        E.gated_silu(self.Z, self.A, rows=rows, n=2 * self.hidden, stream=stream)
        E.grouped_gemm(self.A, self.W2, self.H, self.offsets, rows=rows, groups=self.experts, n=self.width, k=self.hidden, stream=stream)
        return self._join(tokens, stream)

    def backward(self, x, logits, dY, *, tokens, accumulate=False, stream=None):
        """From dY (tokens x width, the gradient to the answers): dX, dlogits, and the weights' gradients in Float32 (accumulate: added to those of earlier calls)."""
        E, rows, RowMajor = self.pkg.EXPERTS, tokens * self.top, self.pkg.WMMA.RowMajor
        both = dict(rows=rows, groups=self.experts, stream=stream)
        E.combine_grad(dY, self.H, self.place, self.dH, self.dgates, tokens=tokens, top=self.top, n=self.width, rows=rows, gates=self.gates, stream=stream)
        E.route_grad(logits, self.chosen, self.gates, self.dgates, self.dlogits, tokens=tokens, experts=self.experts, top=self.top, stream=stream)
        dZ = self.Z  # in its place
        if self.fp8:
            # Gradients have the range of e5m2.  The activation that the gradient to W2 multiplies is made again from the 8 bits that were kept.
            Q = self.pkg.FP8
            Q.quantize(self.dH, *self.dh8, rows=rows, k=self.width, format=Q.E5M2, stream=stream)
            self._product8(self.dh8, 3, self.dA, tokens, stream, a_format=Q.E5M2)
            Q.gated_silu_grad(*self.kept, self.dA, dZ, A=self.A, rows=rows, n=2 * self.hidden, stream=stream)
            Q.quantize(dZ, *self.dz8, rows=rows, k=2 * self.hidden, format=Q.E5M2, stream=stream)
            self._product8(self.dz8, 1, self.dX_rows, tokens, stream, a_format=Q.E5M2)
        else:
            E.grouped_gemm(self.dH, self.W2, self.dA, self.offsets, n=self.hidden, k=self.width, w_layout=RowMajor, **both)
            E.gated_silu_grad(self.Z, self.dA, dZ, rows=rows, n=2 * self.hidden, stream=stream)
            E.grouped_gemm(dZ, self.W1, self.dX_rows, self.offsets, n=self.width, k=2 * self.hidden, w_layout=RowMajor, **both)
        E.grouped_wgrad(self.dH, self.A, self.dW2, self.offsets, m=self.width, n=self.hidden, accumulate=accumulate, **both)
        E.grouped_wgrad(dZ, x, self.dW1, self.offsets, m=2 * self.hidden, n=self.width, gather=self.rows, b_rows=tokens, accumulate=accumulate, **both)
        E.combine(self.dX_rows, self.place, self.dX, tokens=tokens, top=self.top, n=self.width, rows=rows, stream=stream)
        return self.dX, self.dlogits, self.dW1, self.dW2


class Vocabulary:
    """What a model ends in: the loss of its answers' scores over a vocabulary of vectors W (vocabulary x width, Float16, on the device), for at most `tokens` tokens
    a call.  Scores are never stored."""

    def __init__(self, pkg, W, *, tokens, vocabulary, width):
        self.pkg, self.W, self.sizes, new = pkg, W, dict(vocabulary=vocabulary, width=width), pkg.DeviceArray.undef
        self.losses, self.lse, self.dX, self.dW = new(np.float32, tokens), new(np.float32, tokens), new(np.float16, tokens * width), new(np.float32, vocabulary * width)
        self.workspace = new(np.uint8, max(16, pkg.LOSS.cross_entropy_workspace(tokens, vocabulary, width, grad=True)))

    def forward(self, X, targets, *, tokens, stream=None):
        """Losses of the tokens (Float32); targets outside the vocabulary do not count."""
        self.pkg.LOSS.cross_entropy(X, self.W, targets, self.losses, self.lse, tokens=tokens, workspace=self.workspace, stream=stream, **self.sizes)
        return self.losses

    def backward(self, X, targets, dlosses, *, tokens, accumulate=False, stream=None):
        """From dlosses (Float32): the gradients to X and to W (in Float32; accumulate: added to those of earlier calls)."""
        self.pkg.LOSS.cross_entropy_grad(X, self.W, targets, self.lse, dlosses, self.dX, self.dW, dw_type=np.float32, tokens=tokens, accumulate=accumulate, workspace=self.workspace,
                                         stream=stream, **self.sizes)
        return self.dX, self.dW


def main(tokens=256, experts=16, top=2, width=1024, hidden=512, vocabulary=16384):
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
    from __graft_entry__ import load_package
    pkg = load_package()
    pkg.init(0)
    rng = np.random.default_rng(0)

    def upload(shape, scale, T=np.float16):
        return pkg.DeviceArray((scale * rng.standard_normal(shape, np.float32)).astype(T).reshape(-1))

    sizes = dict(tokens=tokens, experts=experts, top=top, width=width, hidden=hidden)
    W1, W2 = upload((experts, 2 * hidden, width), width ** -0.5), upload((experts, width, hidden), hidden ** -0.5)
    layer, layer8 = ExpertsLayer(pkg, W1, W2, **sizes), ExpertsLayer(pkg, W1, W2, **sizes)
    words = Vocabulary(pkg, upload((vocabulary, width), width ** -0.5), tokens=tokens, vocabulary=vocabulary, width=width)
    x, logits = upload((tokens, width), 1.0), upload((tokens, experts), 1.0, np.float32)
    targets = pkg.DeviceArray(rng.integers(0, vocabulary, tokens).astype(np.int32))
    dlosses = pkg.DeviceArray(np.full(tokens, 1.0 / tokens, np.float32))  # of the mean
    layer.pack()
    layer.pack_fp8()
    layer.prepare_training()
    layer8.prepare_training(fp8=True)

    def step(layer):
        y = layer.forward(x, logits, tokens=tokens)
        words.forward(y, targets, tokens=tokens)
        dy, _ = words.backward(y, targets, dlosses, tokens=tokens)
        layer.backward(x, logits, dy, tokens=tokens)

    def host(a):
        return a.to_host().astype(np.float64)

    print("%d tokens, %d of %d experts, %d -> %d -> %d, %d words" % (tokens, top, experts, width, hidden, width, vocabulary))
    served = host(layer.serve(x, logits, tokens=tokens))
    for bits, call in ((8, layer.serve_fp8), (4, layer.serve_mxfp4)):
        print("%d-bit answers differ from the 16-bit ones by %.3f of their norm" % (bits, np.linalg.norm(host(call(x, logits, tokens=tokens)) - served) / np.linalg.norm(served)))
    for name, call in (("serving", lambda: layer.serve(x, logits, tokens=tokens)), ("serving, 8 bits", lambda: layer.serve_fp8(x, logits, tokens=tokens)),
                       ("serving, 4 bits", lambda: layer.serve_mxfp4(x, logits, tokens=tokens)), ("training step", lambda: step(layer)), ("training, 8 bits", lambda: step(layer8))):
        call()
        pkg.synchronize()
        t0 = time.perf_counter()
        for _ in range(20):
            call()
        pkg.synchronize()
        print("%-16s %8.1f us" % (name, (time.perf_counter() - t0) / 20 * 1e6))
    print("mean loss %.3f" % host(words.losses).mean())


if __name__ == "__main__":
    main(*map(int, sys.argv[1:2]))
