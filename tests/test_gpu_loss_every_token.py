"""lse of every token, with a target in the vocabulary or without: on every kernel that makes scores, with rows and vectors far apart, and in the experts' layer.

Tolerances are those that test_gpu_loss derives for lse, which do not depend on the target; all else is compared as there."""
import numpy as np
import pytest

import loss_oracle as ref
import test_gpu_fp8_far as far
import test_gpu_fp8_layer as layer
from experts_oracle import KINDS, upload
from loss_choice import loss_kernels
from test_gpu_experts_layer import SIZES, example  # noqa: F401 (a fixture)
from test_gpu_loss import _check, _make, _space

pytestmark = pytest.mark.gpu


def _check_lse(got, x, w):
    lse, z = ref.log_sums(x, w), np.abs(x @ w.T).max(1)
    off = (w.shape[1] + 2) * 2.0 ** -24 * (np.abs(x) @ np.abs(w).T).max(1) + 2.0 ** -22 * z + 2.0 ** -20 + 2.0 ** -24 * 200 + 2.0 ** -23 * np.abs(lse)
    assert np.all(np.abs(got - lse) <= off), (np.abs(got - lse) - off).max()


def _check_all(got, x, w, targets, *rest, **kw):
    """_check with lse of every token."""
    _check_lse(got[1], x, w)
    some = (targets >= 0) & (targets < len(w))
    _check([got[0], np.where(some, got[1], 0.0)] + list(got[2:]), x, w, targets, *rest, **kw)


def _scores(gpu, x, w, targets, kind):
    tokens, sizes = len(x), dict(tokens=len(x), vocabulary=len(w), width=x.shape[1])
    losses, lse = (upload(gpu, np.full(tokens, 7.0, np.float32)) for _ in range(2))
    gpu.LOSS.cross_entropy(upload(gpu, kind.store(x)), upload(gpu, kind.store(w)), upload(gpu, targets), losses, lse, dtype=kind.marker(gpu), workspace=_space(gpu, *sizes.values()), **sizes)
    return losses.to_host().astype(np.float64), lse.to_host().astype(np.float64)


# Every kernel that makes scores; 64 and 65 tokens.
@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("ignored", [0.3, 1.1])
@pytest.mark.parametrize("tokens,vocabulary,width,kernel", [(1, 1, 1, "plain"), (10, 33000, 64, "narrow 1 2 2"), (16, 4200, 4200, "narrow 1 2 4"), (20, 1000, 64, "narrow 2 1 8"), (64, 500, 72, "narrow 2 1 8"),
                                                            (65, 500, 72, "128x64"), (300, 1000, 64, "128x64"), (50, 33000, 64, "256x128"), (1500, 3000, 2008, "256x128"), (2050, 1000, 520, "128x128"),
                                                            (2050, 4200, 64, "256x256"), (100, 500, 65, "plain")])
def test_every_kernel(gpu, tokens, vocabulary, width, kernel, ignored, kind):
    assert loss_kernels(gpu, tokens, vocabulary, width)[0] == kernel
    kind = KINDS[kind]
    x, w, targets, _ = _make(tokens + vocabulary, tokens, vocabulary, width, kind, ignored)
    some = (targets >= 0) & (targets < vocabulary)
    assert ignored < 1 or not some.any()
    losses, lse = _scores(gpu, x, w, targets, kind)
    _check_all([losses, lse], x, w, targets, None, kind)
    # lse is the same, to the bit, whatever the targets are
    every = _scores(gpu, x, w, np.arange(tokens, dtype=np.int32) % vocabulary, kind)[1]
    assert np.array_equal(every, lse) and (some.all() or lse[~some].any())


def test_padding_that_nobody_filled(gpu):
    """NaN and infinities in rows without a target reach nothing; the same in a row with one are seen."""
    kind = KINDS["f16"]
    x, w, targets, _ = _make(1, 200, 700, 64, kind, 0.0)
    x[[3, 60, 61, 150]], targets[[3, 60, 150]] = np.nan, [-1, 700, -2 ** 31]
    x[150, 1:] = np.inf
    losses, lse = _scores(gpu, x, w, targets, kind)
    assert not lse[[3, 60, 150]].any() and not losses[[3, 60, 150]].any() and np.isnan(lse[61]) and np.isnan(losses[61])
    others = np.delete(np.arange(200), [3, 60, 61, 150])
    _check_all([losses[others], lse[others]], x[others], w, targets[others], None, kind)


@pytest.mark.parametrize("tokens,vocabulary,ldw", [(90, 300, 64), (20, 1100, 1 << 21), (90, 80, 1 << 25)])
def test_far_apart(gpu, monkeypatch, tokens, vocabulary, ldw):
    monkeypatch.setattr(far, "_check", _check_all)
    far.test_loss(gpu, tokens, vocabulary, ldw)


@pytest.mark.parametrize("vocabulary,width", [(1100, 64), (5000, 4104), (700, 2008)])
def test_few_tokens_apart(gpu, monkeypatch, vocabulary, width):
    monkeypatch.setattr(far, "_check", _check_all)
    far.test_loss_of_few_tokens_apart(gpu, vocabulary, width)


@pytest.mark.parametrize("vocabulary", [300, 2051])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("tokens,experts,top,width,hidden,masked", SIZES)
def test_training_step(gpu, example, monkeypatch, tokens, experts, top, width, hidden, masked, fp8, vocabulary):  # noqa: F811
    monkeypatch.setattr(layer, "check_loss", _check_all)
    layer.test_training_step_with_the_loss(gpu, example, tokens, experts, top, width, hidden, masked, fp8, vocabulary)
