"""A feed-forward layer of experts on the library's operators: serving in 16 and in 4 bits, and a training step.

Every token goes to `top` of `experts` pairs of matrices: Z = x W1 (gates and values side by side), A = silu(gate) * value,
H = A W2, and its answers are joined by the router's weights.

    route -> grouped_gemm (gated) -> grouped_gemm -> combine                               serve
    quantize -> grouped_gemm (gated) -> quantize -> grouped_gemm -> combine                serve_mxfp4, weights in 4 bits
    combine_grad -> grouped_gemm, grouped_wgrad -> gated_silu_grad -> the same -> combine -> route_grad     backward

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

    # ---- training

    def prepare_training(self):
        rows, new = self.tokens * self.top, self.pkg.DeviceArray.undef
        self.Z, self.dH, self.dA, self.dX_rows, self.dX = (self._half(n) for n in (rows * 2 * self.hidden, rows * self.width, rows * self.hidden,
                                                                                     rows * self.width, self.tokens * self.width))
        self.dgates, self.dlogits = new(np.float32, rows), new(np.float32, self.tokens * self.experts)
        self.dW1, self.dW2 = new(np.float32, self.experts * 2 * self.hidden * self.width), new(np.float32, self.experts * self.width * self.hidden)

    def forward(self, x, logits, *, tokens, stream=None):
        """serve, with the columns before the activation kept for backward."""
        E, rows = self.pkg.EXPERTS, tokens * self.top
        self._route(logits, tokens, stream)
        E.grouped_gemm(x, self.W1, self.Z, self.offsets, rows=rows, groups=self.experts, n=2 * self.hidden, k=self.width, gather=self.rows,
                       a_rows=tokens, stream=stream)
        E.gated_silu(self.Z, self.A, rows=rows, n=2 * self.hidden, stream=stream)
        E.grouped_gemm(self.A, self.W2, self.H, self.offsets, rows=rows, groups=self.experts, n=self.width, k=self.hidden, stream=stream)
        return self._join(tokens, stream)

    def backward(self, x, logits, dY, *, tokens, accumulate=False, stream=None):
        """From dY (tokens x width): dX, dlogits, and the weights' gradients in Float32 (accumulate: added to those of earlier calls)."""
        E, rows, RowMajor = self.pkg.EXPERTS, tokens * self.top, self.pkg.WMMA.RowMajor
        both = dict(rows=rows, groups=self.experts, stream=stream)
        E.combine_grad(dY, self.H, self.place, self.dH, self.dgates, tokens=tokens, top=self.top, n=self.width, rows=rows, gates=self.gates, stream=stream)
        E.route_grad(logits, self.chosen, self.gates, self.dgates, self.dlogits, tokens=tokens, experts=self.experts, top=self.top, stream=stream)
        E.grouped_gemm(self.dH, self.W2, self.dA, self.offsets, n=self.hidden, k=self.width, w_layout=RowMajor, **both)
        E.grouped_wgrad(self.dH, self.A, self.dW2, self.offsets, m=self.width, n=self.hidden, accumulate=accumulate, **both)
        dZ = self.Z  # in its place
        E.gated_silu_grad(self.Z, self.dA, dZ, rows=rows, n=2 * self.hidden, stream=stream)
        E.grouped_gemm(dZ, self.W1, self.dX_rows, self.offsets, n=self.width, k=2 * self.hidden, w_layout=RowMajor, **both)
        E.grouped_wgrad(dZ, x, self.dW1, self.offsets, m=2 * self.hidden, n=self.width, gather=self.rows, b_rows=tokens, accumulate=accumulate, **both)
        E.combine(self.dX_rows, self.place, self.dX, tokens=tokens, top=self.top, n=self.width, rows=rows, stream=stream)
        return self.dX, self.dlogits, self.dW1, self.dW2


def main(tokens=256, experts=16, top=2, width=1024, hidden=512):
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
    from __graft_entry__ import load_package
    pkg = load_package()
    pkg.init(0)
    rng = np.random.default_rng(0)

    def upload(shape, scale, T=np.float16):
        return pkg.DeviceArray((scale * rng.standard_normal(shape, np.float32)).astype(T).reshape(-1))

    layer = ExpertsLayer(pkg, upload((experts, 2 * hidden, width), width ** -0.5), upload((experts, width, hidden), hidden ** -0.5), tokens=tokens,
                         experts=experts, top=top, width=width, hidden=hidden)
    x, logits, dY = upload((tokens, width), 1.0), upload((tokens, experts), 1.0, np.float32), upload((tokens, width), 1.0)
    layer.pack()
    layer.prepare_training()

    def step():
        layer.forward(x, logits, tokens=tokens)
        layer.backward(x, logits, dY, tokens=tokens)

    served = layer.serve(x, logits, tokens=tokens).to_host().astype(np.float64)
    packed = layer.serve_mxfp4(x, logits, tokens=tokens).to_host().astype(np.float64)
    print("%d tokens, %d of %d experts, %d -> %d -> %d" % (tokens, top, experts, width, hidden, width))
    print("4-bit answers differ from the 16-bit ones by %.3f of their norm" % (np.linalg.norm(packed - served) / np.linalg.norm(served)))
    for name, call in (("serving", lambda: layer.serve(x, logits, tokens=tokens)), ("serving, 4 bits", lambda: layer.serve_mxfp4(x, logits, tokens=tokens)),
                       ("training step", step)):
        call()
        pkg.synchronize()
        t0 = time.perf_counter()
        for _ in range(20):
            call()
        pkg.synchronize()
        print("%-16s %8.1f us" % (name, (time.perf_counter() - t0) / 20 * 1e6))


if __name__ == "__main__":
    main(*map(int, sys.argv[1:2]))
