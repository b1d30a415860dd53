"""The loss's gradients over several pieces of the vocabulary on the kernels of large sizes, and where the library itself cuts the vocabulary, by value.
Tolerances: test_gpu_loss."""
import numpy as np
import pytest

from experts_oracle import KINDS
from loss_choice import piece_kernels
from test_gpu_loss import _check, _make, _run

pytestmark = pytest.mark.gpu

# Tokens, vocabulary, width, piece; of each piece columns and the kernels of probabilities, rows' and vectors' gradients.  Last pieces are shorter, whole and of one column.
PIECES = [(2000, 9000, 2008, 6000, [(6016, "256x256", "2 x 256x128", "dense"), (2984, "256x128", "2 x 256x128", "dense")]),
          (2000, 6017, 2008, 6016, [(6016, "256x256", "2 x 256x128", "dense"), (1, "128x64", "2 x 256x128", "dense")]),
          (2050, 1100, 4104, 500, [(512, "128x64", "1 x 256x256", "128x64"), (512, "128x64", "1 x 256x256", "128x64"), (76, "128x64", "1 x 256x256", "128x64")]),
          (2050, 2000, 520, 1000, [(1024, "128x128", "2 x 128x128", "128x64"), (976, "128x128", "2 x 128x128", "128x64")]),
          (1500, 6016, 2008, 3000, [(3008, "256x128", "2 x 256x128", "128x128"), (3008, "256x128", "2 x 256x128", "128x128")]),
          (6000, 300, 264, 100, [(128, "128x64", "1 x 128x128", "128x64"), (128, "128x64", "1 x 128x128", "128x64"), (44, "128x64", "1 x 128x128", "128x64")])]


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("added", [False, True])
@pytest.mark.parametrize("tokens,vocabulary,width,piece,kernels", PIECES)
def test_pieces_on_large_kernels(gpu, tokens, vocabulary, width, piece, kernels, added, kind):
    assert piece_kernels(gpu, tokens, vocabulary, width, piece) == kernels
    kind = KINDS[kind]
    x, w, targets, share = _make(vocabulary + width, tokens, vocabulary, width, kind, 0.1)
    before = np.random.default_rng(1).integers(-4, 5, (vocabulary, width)) / 64.0 if added else None
    for dw in ("f32", "own") if added else ("f32",):
        _check(_run(gpu, x, w, targets, share, kind, dw, 0, piece, before), x, w, targets, share, kind, dw, before)


# More than 2^27 scores: the library's own pieces.
@pytest.mark.parametrize("tokens,vocabulary,width,kind,kernels", [(12000, 20000, 264, "f16", [(10048, "256x256", "2 x 256x256", "128x64"), (9952, "256x256", "2 x 256x256", "128x64")]),
                                                                  (9000, 17000, 1032, "bf16", [(8512, "256x256", "1 x 256x256", "dense"), (8488, "256x256", "1 x 256x256", "dense")])])
def test_pieces_of_the_librarys_choice(gpu, tokens, vocabulary, width, kind, kernels):
    assert tokens * vocabulary > 1 << 27 and piece_kernels(gpu, tokens, vocabulary, width) == kernels
    kind, rng = KINDS[kind], np.random.default_rng(1)
    x, w, targets, share = _make(tokens, tokens, vocabulary, width, kind, 0.1)
    got = _run(gpu, x, w, targets, share, kind, "f32")
    some = np.flatnonzero((targets >= 0) & (targets < vocabulary))
    assert np.all(got[2][np.setdiff1d(np.arange(tokens), some)] == 0)
    # The rows' gradients of some tokens
    rows = rng.choice(some, 150, replace=False)
    _check([got[0][rows], got[1][rows], None, None], x[rows], w, targets[rows], share[rows], kind, "f32")
    scale = np.abs(share[some]).max()
    z, size = x[rows] @ w.T, np.abs(x[rows]) @ np.abs(w).T
    exact, bound = _products(z, size, _lse(z), size.max(1), np.abs(z).max(1), targets[rows], np.arange(vocabulary), share[rows], scale, width, kind)
    want = exact @ w
    bound = bound @ np.abs(w) + (vocabulary + 10) * 2.0 ** -24 * (np.abs(exact) @ np.abs(w)) + kind.roundoff * 1.01 * np.abs(want) + 2.0 ** -25
    assert np.all(np.abs(got[2][rows] - want) <= bound), (np.abs(got[2][rows] - want) - bound).max()
    # and the vectors' of some words, at both ends of the pieces and between
    first = kernels[0][0]
    words = np.unique([0, 1, first - 1, first, first + 1, vocabulary - 2, vocabulary - 1, *targets[some[:40]], *rng.integers(0, vocabulary, 60)])
    lse, largest, high = np.empty(len(some)), np.empty(len(some)), np.empty(len(some))
    for i in range(0, len(some), 1000):
        part = some[i:i + 1000]
        z = x[part] @ w.T
        lse[i:i + 1000], high[i:i + 1000], largest[i:i + 1000] = _lse(z), np.abs(z).max(1), (np.abs(x[part]) @ np.abs(w).T).max(1)
    exact, bound = _products(x[some] @ w[words].T, np.abs(x[some]) @ np.abs(w[words]).T, lse, largest, high, targets[some], words, share[some], scale, width, kind)
    want = exact.T @ x[some]
    bound = bound.T @ np.abs(x[some]) + (tokens + 10) * 2.0 ** -24 * (np.abs(exact).T @ np.abs(x[some])) + 2.0 ** -23 * np.abs(want) + 2.0 ** -25
    assert np.all(np.abs(got[3][words] - want) <= bound), (np.abs(got[3][words] - want) - bound).max()


def _lse(z):
    most = z.max(1)
    return most + np.log(np.exp(z - most[:, None]).sum(1))


def _products(z, size, lse, largest, high, targets, words, share, scale, width, kind):
    """share (softmax - [target]) of some tokens and words, and how far the stored ones may be off.  largest, high: of a token's sums of magnitudes and of its scores' size over all words."""
    share, E = share.astype(np.float64)[:, None], (width + 2) * 2.0 ** -24
    soft, goal = np.exp(z - lse[:, None]), words[None, :] == targets[:, None]
    p = share * (soft - goal)
    off = (E * largest + 2.0 ** -22 * high + 2.0 ** -20 + 2.0 ** -24 * 200)[:, None]
    bound = (E * size + 2 * off + 2.0 ** -22 * (1 + np.abs(z))) * (soft + np.where(goal, 1.0, 0.0)) * np.abs(share) + kind.roundoff * np.abs(p) * 1.01
    return p, bound + (2.0 ** -38 * scale if kind.name == "f16" else 0.0)
