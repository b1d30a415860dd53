"""The experts' operators captured in a HIP graph: every replay, with other inputs in the same buffers and eager work between, gives the eager
calls' bits."""
import ctypes
import re

import numpy as np
import pytest

from experts_oracle import upload
from test_gpu_experts_layer import example  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


class Graph:
    """A graph of what `body(stream)` queues, through the HIP runtime that the library has loaded."""

    def __init__(self, gpu, body):
        with open("/proc/self/maps") as maps:
            self.hip = ctypes.CDLL(re.search(r"/\S*libamdhip64\S*", maps.read()).group())
        self.gpu, self.stream = gpu, gpu.Stream()
        at, graph, self.exec = ctypes.c_void_p(self.stream.handle), ctypes.c_void_p(), ctypes.c_void_p()
        self._call("hipStreamBeginCapture", at, 0)
        body(self.stream)
        self._call("hipStreamEndCapture", at, ctypes.byref(graph))
        self._call("hipGraphInstantiate", ctypes.byref(self.exec), graph, None, None, ctypes.c_size_t(0))
        self._call("hipGraphDestroy", graph)

    def _call(self, name, *args):
        rc = getattr(self.hip, name)(*args)
        assert rc == 0, (name, rc)

    def replay(self):
        self._call("hipGraphLaunch", self.exec, ctypes.c_void_p(self.stream.handle))
        self.gpu.synchronize(self.stream)

    def close(self):
        self._call("hipGraphExecDestroy", self.exec)


# Tokens on both sides of the routing's one launch; few and many rows an expert; sums and widths with remainders.
@pytest.mark.parametrize("tokens,experts,top,width,hidden", [(16, 8, 2, 136, 72), (300, 16, 2, 264, 200), (2000, 4, 2, 520, 264), (300, 5, 2, 36, 18)])
def test_layer(gpu, example, tokens, experts, top, width, hidden):  # noqa: F811
    rng = np.random.default_rng(tokens)
    half = lambda *shape: rng.normal(size=shape).astype(np.float16)  # noqa: E731
    layer = example.ExpertsLayer(gpu, upload(gpu, half(experts, 2 * hidden, width) / np.float16(width ** 0.5)), upload(gpu, half(experts, width, hidden) / np.float16(hidden ** 0.5)),
                                 tokens=tokens, experts=experts, top=top, width=width, hidden=hidden)
    layer.pack()
    layer.prepare_training()
    x, dy, logits = upload(gpu, half(tokens, width)), upload(gpu, half(tokens, width)), upload(gpu, rng.normal(size=(tokens, experts)).astype(np.float32))
    packed = gpu.DeviceArray.undef(np.float16, tokens * width)
    kept = gpu.DeviceArray.undef(np.float32, tokens * width)
    Q = gpu.MXFP4

    def body(stream):
        layer.serve_mxfp4(x, logits, tokens=tokens, stream=stream)
        gpu.EXPERTS.combine(layer.H, layer.place, packed, tokens=tokens, top=top, n=width, rows=tokens * top, gates=layer.gates, stream=stream)
        Q.dequantize(*layer.x4, kept, rows=tokens, k=width, stream=stream)
        layer.forward(x, logits, tokens=tokens, stream=stream)
        layer.backward(x, logits, dy, tokens=tokens, stream=stream)

    results = (packed, kept, layer.Y, layer.dX, layer.dlogits, layer.dW1, layer.dW2, layer.offsets, layer.rows, layer.place)
    gpu.synchronize()
    graph = Graph(gpu, body)
    for turn in range(4):
        new = half(tokens, width).reshape(-1), rng.normal(size=tokens * experts).astype(np.float32), half(tokens, width).reshape(-1)
        for buffer, values in zip((x, logits, dy), new):
            buffer.copy_from(values)
        for r in results:
            r.fill_bytes(turn + 1)
        gpu.synchronize()
        graph.replay()
        got = [r.to_host() for r in results]
        for r in results:
            r.fill_bytes(turn + 9)
        body(None)
        gpu.synchronize()
        for i, (a, b) in enumerate(zip(got, results)):
            b = b.to_host()
            assert b.any() and np.array_equal(a.view(np.uint8), b.view(np.uint8)), (turn, i)
    graph.close()


def test_dense_product_in_4_bits(gpu):
    Q, rng = gpu.MXFP4, np.random.default_rng(2)
    m, n, k = 200, 264, 1100
    X, Y = upload(gpu, rng.normal(size=(m, k)).astype(np.float16)), upload(gpu, rng.normal(size=(n, k)).astype(np.float16))
    codes = [gpu.DeviceArray.undef(np.uint8, f(rows, k)) for rows in (m, n) for f in (Q.codes_bytes, Q.scales_bytes)]
    D = gpu.DeviceArray.undef(np.float16, m * n)

    def body(stream):
        Q.quantize(X, *codes[:2], rows=m, k=k, stream=stream)
        Q.quantize(Y, *codes[2:], rows=n, k=k, stream=stream)
        Q.gemm(*codes, D, m=m, n=n, k=k, stream=stream)

    gpu.synchronize()
    graph = Graph(gpu, body)
    for _ in range(3):
        X.copy_from(rng.normal(size=m * k).astype(np.float16))
        D.fill_bytes(1)
        gpu.synchronize()
        graph.replay()
        got = D.to_host()
        D.fill_bytes(2)
        body(None)
        gpu.synchronize()
        assert got.any() and np.array_equal(got, D.to_host())
    graph.close()
