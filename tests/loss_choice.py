"""Which kernels the loss runs on, by the library's own rules."""
import ctypes

from grouped_choice import TILES, _Choice, _GroupedParams


class _Cut(ctypes.Structure):
    _fields_ = [("slices", ctypes.c_int), ("tile", ctypes.c_int)]


def _rule(miw, symbol, result, *args):
    f = getattr(ctypes.CDLL(miw._lib.LIB_PATH), symbol)
    f.restype, f.argtypes = result, args
    return f


def sum_is_dense(miw, p, cus=256):
    return _rule(miw, "_ZN3miw17loss_sum_is_denseERKNS_14grouped_paramsEi", ctypes.c_bool, ctypes.POINTER(_GroupedParams), ctypes.c_int)(ctypes.byref(p), cus)


def piece(miw, tokens, vocabulary, asked=0):
    return _rule(miw, "_ZN3miw10loss_pieceElll", ctypes.c_int64, *[ctypes.c_int64] * 3)(tokens, vocabulary, asked)


def _name(c):
    return "plain" if c.kernel == 0 else "narrow %d %d %d" % (c.rows, c.weights, c.waves) if c.kernel == 1 else TILES[c.tile]


def loss_kernels(miw, tokens, vocabulary, width, cus=256):
    """The kernels of dense, aligned operands' scores, rows' gradients (with the slices) and vectors' gradients, for a vocabulary in one piece."""
    scores = _rule(miw, "_ZN3miw16choose_loss_rowsERKNS_14grouped_paramsEi", _Choice, ctypes.POINTER(_GroupedParams), ctypes.c_int)
    grouped = _rule(miw, "_ZN3miw14choose_groupedERKNS_14grouped_paramsEbbi", _Choice, ctypes.POINTER(_GroupedParams), ctypes.c_bool, ctypes.c_bool, ctypes.c_int)
    columns = piece(miw, tokens, vocabulary)
    assert columns >= vocabulary
    vector = width % 8 == 0
    p = _GroupedParams(groups=1, rows=tokens, source_rows=tokens, I=vocabulary, K=width, ldx=2 * width, ldy=2 * width, x_k_major=1, vector=vector)
    names = [_name(scores(ctypes.byref(p), cus))]
    p = _GroupedParams(groups=1, rows=tokens, source_rows=tokens, I=width, K=vocabulary, ldx=2 * width, ldy=2 * columns, vector=vector)
    cut = _rule(miw, "_ZN3miw13cut_loss_rowsEllli", _Cut, ctypes.c_long, ctypes.c_long, ctypes.c_long, ctypes.c_int)(tokens, width, vocabulary, cus)
    plain = grouped(ctypes.byref(p), False, False, cus).kernel == 0
    names += ["%d x %s" % (cut.slices, "plain" if plain else TILES[cut.tile])]
    p = _GroupedParams(groups=1, rows=tokens, source_rows=tokens, I=width, J=vocabulary + 7 & -8, ldx=2 * width, ldy=2 * columns, vector=vector)
    return names + ["dense" if sum_is_dense(miw, p, cus) else _name(grouped(ctypes.byref(p), False, True, cus))]


def score_run(miw, tokens, vocabulary, width, vector=True, cus=256):
    """Tokens that scores are made of at a time, and the slices of the vocabulary that each of them has statistics of."""
    class Slices(ctypes.Structure):
        _fields_ = [("width", ctypes.c_int), ("count", ctypes.c_int)]

    p = _GroupedParams(groups=1, rows=tokens, source_rows=tokens, I=vocabulary, K=width, ldx=2 * width, ldy=2 * width, x_k_major=1, vector=vector)
    run = _rule(miw, "_ZN3miw8loss_runENS_14grouped_paramsEi", ctypes.c_long, _GroupedParams, ctypes.c_int)(p, cus)
    p.rows = p.source_rows = run
    return run, _rule(miw, "_ZN3miw17loss_score_slicesERKNS_14grouped_paramsEi", Slices, ctypes.POINTER(_GroupedParams), ctypes.c_int)(ctypes.byref(p), cus).count


def piece_kernels(miw, tokens, vocabulary, width, asked=0, cus=256):
    """For each piece of the vocabulary, its columns and the kernels of its probabilities, rows' gradients (with the slices) and vectors' gradients, of dense, aligned operands."""
    scores = _rule(miw, "_ZN3miw16choose_loss_rowsERKNS_14grouped_paramsEi", _Choice, ctypes.POINTER(_GroupedParams), ctypes.c_int)
    grouped = _rule(miw, "_ZN3miw14choose_groupedERKNS_14grouped_paramsEbbi", _Choice, ctypes.POINTER(_GroupedParams), ctypes.c_bool, ctypes.c_bool, ctypes.c_int)
    columns = piece(miw, tokens, vocabulary, asked)
    longest = min(columns, vocabulary)
    cut = _rule(miw, "_ZN3miw13cut_loss_rowsEllli", _Cut, ctypes.c_long, ctypes.c_long, ctypes.c_long, ctypes.c_int)(tokens, width, longest, cus)

    def sums(n):
        return _GroupedParams(groups=1, rows=tokens, source_rows=tokens, I=width, J=n + 7 & -8, ldx=2 * width, ldy=2 * columns, vector=1)

    dense, out = sum_is_dense(miw, sums(longest), cus), []  # (of the first piece, and so of all)
    for n in [min(columns, vocabulary - first) for first in range(0, vocabulary, columns)]:
        p = _GroupedParams(groups=1, rows=tokens, source_rows=tokens, I=n, K=width, ldx=2 * width, ldy=2 * width, x_k_major=1, vector=1)
        out.append((n, _name(scores(ctypes.byref(p), cus)), "%d x %s" % (cut.slices, TILES[cut.tile]), "dense" if dense else _name(grouped(ctypes.byref(sums(n)), False, True, cus))))
    return out
