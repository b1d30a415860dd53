"""Losses of confident tokens keep their digits: far below 1, where lse and the target's score agree in all that Float32 has of them.

A row of X picks one of the vectors' columns, so that scores are Float16 numbers and exact.  Then an exponential is off by the rounding of its argument, |z - largest| 2^-24
of it, and the instruction's two units, 2^-23; a sum of positive terms by 200 roundings of 2^-24 (test_gpu_loss) and four more for each join's factors; log1p by two units.
All are relative, and so is the bound: (2 |z - largest| + 300) 2^-24 for terms that count, those within 80 of the largest (vocabularies are below e^11)."""
import numpy as np
import pytest

from experts_oracle import KINDS, upload
from loss_choice import loss_kernels
from test_gpu_loss import _space

pytestmark = pytest.mark.gpu

HEIGHTS = [0.0, 3.0, 12.0, 20.0, 30.0, 40.0, 60.0]  # of the largest score over the others' mean; 0: the two largest are equal


def _exact(z, targets):
    """log(1 + sum over the others of exp(z - z_target)), with no difference of large numbers."""
    t = np.arange(len(z))
    goal = z[t, targets][:, None]
    over = z.max(1, keepdims=True) - goal
    each = np.exp(z - goal - over)
    each[t, targets] = 0.0
    others, over = each.sum(1), over[:, 0]
    return np.where(over == 0, np.log1p(others), over + np.log(others + np.exp(-over)))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,vocabulary,width,kernel", [(7, 33000, 64, "narrow 1 2 2"), (14, 4200, 4200, "narrow 1 2 4"), (21, 1000, 64, "narrow 2 1 8"), (300, 1000, 64, "128x64"), (50, 33000, 64, "256x128"),
                                                            (2050, 1000, 520, "128x128"), (2050, 4200, 64, "256x256"), (100, 500, 65, "plain")])
def test_small_losses(gpu, tokens, vocabulary, width, kernel, kind):
    assert loss_kernels(gpu, tokens, vocabulary, width)[0] == kernel
    kind, rng = KINDS[kind], np.random.default_rng(vocabulary)
    w = rng.normal(size=(vocabulary, width))
    w[:, :7] = np.round(w[:, :7] * 16) / 16
    top = rng.permutation(vocabulary)[:7]
    w[top, np.arange(7)] = np.maximum(w[:, :7].max(0), HEIGHTS)
    w[(top[0] + 100) % vocabulary, 0] = w[top[0], 0]
    x, column = np.zeros((tokens, width)), np.arange(tokens) % 7
    x[np.arange(tokens), column] = 1.0
    w = kind.load(kind.store(w))
    # most tokens' target is the largest score, some of the later ones' another word
    targets = np.where(rng.random(tokens) < np.where(np.arange(tokens) < 7, 1.0, 0.7), top[column], rng.integers(0, vocabulary, tokens)).astype(np.int32)
    losses, lse = (upload(gpu, np.full(tokens, 7.0, np.float32)) for _ in range(2))
    gpu.LOSS.cross_entropy(upload(gpu, kind.store(x)), upload(gpu, kind.store(w)), upload(gpu, targets), losses, lse, tokens=tokens, vocabulary=vocabulary, width=width, dtype=kind.marker(gpu),
                           workspace=_space(gpu, tokens, vocabulary, width))
    z = x @ w.T
    want, got = _exact(z, targets), losses.to_host().astype(np.float64)
    assert want.min() < 1e-20 and (want < 1e-5).sum() >= 3
    assert np.all(np.abs(got - want) <= (2 * 80 + 300) * 2.0 ** -24 * want), (np.abs(got - want) / want).max()
    assert np.all(got > 0)
    most = z.max(1)
    assert np.all(np.abs(lse.to_host() - most - np.log(np.exp(z - most[:, None]).sum(1))) <= (2 * 80 + 300) * 2.0 ** -24 + 2.0 ** -23 * (most + 12))
