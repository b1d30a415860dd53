"""Softmax cross entropy over a large vocabulary, and its gradient, without storing the scores.

The scores are the product of X (tokens x width, what a model ends in) and W (vocabulary x width).  `cross_entropy` sums their
exponentials up where they are made; `cross_entropy_grad` makes them again, a piece of the vocabulary at a time.  A token whose
target is outside the vocabulary (-1, say) does not count: it has an lse, a loss of 0 and no part in the gradient.

No counterpart in the reference; the products are the chain of mma calls of docs/src/device/wmma.md:51-52.  Arrays are
DeviceArrays or raw device addresses; matrices are row-major, a pitch of 0 means dense.  All calls are asynchronous on `stream`.
"""
import ctypes

from .experts import TYPE_CODES, _library, call
from .gemm import _stream
from .wmma import Float16


def cross_entropy_workspace(tokens, vocabulary, width, *, grad=False, piece=0):
    """Bytes of workspace that cross_entropy needs for these sizes, or, with grad, both it and cross_entropy_grad."""
    n = ctypes.c_size_t()
    call(_library.miw_cross_entropy_workspace, tokens, vocabulary, width, 1 if grad else 0, piece, ctypes.byref(n))
    return n.value


def cross_entropy(X, W, targets, losses, lse, *, tokens, vocabulary, width, dtype=Float16, ldx=0, ldw=0, workspace, stream=None):
    """losses[t] = lse[t] - X[t] . W[targets[t]] with lse[t] = log(sum over v of exp(X[t] . W[v])); Float32.  Losses are 0 for
    tokens that do not count, and so is their lse where their row of X makes it no number.  targets: Int32.  workspace: a DeviceArray of cross_entropy_workspace bytes."""
    call(_library.miw_cross_entropy, TYPE_CODES[dtype], tokens, vocabulary, width, ldx, ldw, X, W, targets, losses, lse, workspace,
         0 if workspace is None else workspace.nbytes, None if stream is None else _stream(stream))


def cross_entropy_grad(X, W, targets, lse, dlosses, dX, dW, *, tokens, vocabulary, width, dtype=Float16, dw_type=None, ldx=0, ldw=0, lddx=0, lddw=0, piece=0,
                       accumulate=False, workspace, stream=None):
    """The gradients to X (of its type) and to W (dw_type: of their type or Float32) from those to the losses; None: not computed.
    lse is cross_entropy's.  piece: columns of the vocabulary at a time (0: the library's choice), which the workspace has to be
    made for.  accumulate: added to what dW holds."""
    call(_library.miw_cross_entropy_grad, TYPE_CODES[dtype], TYPE_CODES[dtype if dw_type is None else dw_type], 1 if accumulate else 0, tokens, vocabulary, width,
         ldx, ldw, lddx, lddw, piece, X, W, targets, lse, dlosses, dX, dW, workspace, 0 if workspace is None else workspace.nbytes,
         None if stream is None else _stream(stream))
