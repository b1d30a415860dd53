"""The experts' layer of the examples at sizes that are not those of its first call, or not even."""
import numpy as np
import pytest

import test_gpu_experts_layer as layer_tests
from experts_oracle import upload
from test_gpu_experts_layer import example  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def test_calls_of_fewer_tokens_than_the_layer_was_made_for(gpu, example):  # noqa: F811
    """Every call up to the most tokens: the answers are those of a layer made for that many."""
    rng = np.random.default_rng(7)
    w1, w2 = (upload(gpu, rng.normal(size=s).astype(np.float16)) for s in ((16, 2 * 24, 40), (16, 40, 24)))
    x, logits, dy = upload(gpu, rng.normal(size=(5000, 40)).astype(np.float16)), upload(gpu, rng.normal(size=(5000, 16)).astype(np.float32)), upload(gpu, rng.normal(size=(5000, 40)).astype(np.float16))
    sizes = dict(experts=16, top=2, width=40, hidden=24)
    layer = example.ExpertsLayer(gpu, w1, w2, tokens=5000, **sizes)
    layer.pack()
    layer.prepare_training()
    for tokens in (5000, 4096, 65, 64, 4097, 1):
        own = example.ExpertsLayer(gpu, w1, w2, tokens=tokens, **sizes)
        own.pack()
        own.prepare_training()
        for call in ("serve", "serve_mxfp4", "forward"):
            got, want = (getattr(a, call)(x, logits, tokens=tokens).to_host()[:tokens * 40] for a in (layer, own))
            assert got.any() and np.array_equal(got, want), (tokens, call)
        for got, want in zip(layer.backward(x, logits, dy, tokens=tokens), own.backward(x, logits, dy, tokens=tokens)):
            want = want.to_host()
            assert np.array_equal(got.to_host()[:len(want)], want), tokens


# Widths of an odd number of columns, whose matrices of 4-bit weights start on even rows of their panels; few and many rows an expert.
@pytest.mark.parametrize("tokens,experts,top,width,hidden", [(9, 4, 2, 35, 11), (70, 3, 2, 301, 145), (400, 5, 2, 129, 67)])
def test_odd_widths(gpu, example, tokens, experts, top, width, hidden):  # noqa: F811
    layer_tests.test_serving_in_4_bits(gpu, example, tokens, experts, top, width, hidden, True)
    layer_tests.test_training_step(gpu, example, tokens, experts, top, width, hidden, True)
