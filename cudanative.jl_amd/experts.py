"""A layer of experts: routing, products grouped by expert, the join of the answers, and the gradients.

Every token goes to a few of many matrices.  `route` chooses them and sorts the rows by expert, `grouped_gemm` multiplies
each expert's rows by its matrix, `combine` joins a token's answers by its gates; `route_grad`, `grouped_wgrad`,
`gated_silu_grad` and `combine_grad` are the way back.  How many rows an expert has stays on the device: nothing here waits for it.

No counterpart in the reference; the products are the chain of mma calls of docs/src/device/wmma.md:51-52 on ragged
rows.  Arrays are DeviceArrays or raw device addresses; matrices are row-major, a pitch or stride of 0 means dense.  All
calls are asynchronous on `stream`.
"""
import ctypes
import operator

import numpy as np

from . import _lib
from .gemm import _layout_code, _stream
from .wmma import ColMajor, Float16, Float32


_library = _lib.load()


class BFloat16:
    """Element type of the experts' operators and the 4-bit conversions that numpy has no name for."""


GATED_SILU = "gated_silu"


class _TypeCodes(dict):
    def __missing__(self, T):
        code = None
        try:
            code = None if T is None else self.get(np.dtype(T).type)
        except TypeError:
            pass
        if code is None:
            raise TypeError("element types here are Float16, BFloat16 and Float32")
        return code


TYPE_CODES = _TypeCodes({np.float16: _lib.F16, np.float32: _lib.F32, BFloat16: _lib.BF16})


def _plain(x):
    return x if x is None or hasattr(x, "_as_parameter_") else operator.index(x)


def call(entry, *arguments):
    """A call is a few microseconds in all: whole numbers, None and DeviceArrays go to ctypes as they are, and only what it does not
    take for an address (numpy's integers) is made plain."""
    try:
        rc = entry(*arguments)
    except ctypes.ArgumentError:
        rc = entry(*map(_plain, arguments))
    if rc:
        _lib.check(rc)


def epilogue_code(epilogue):
    if epilogue is None:
        return _lib.EPILOGUE_NONE
    if epilogue != GATED_SILU:
        raise ValueError("epilogue is None or GATED_SILU")
    return _lib.EPILOGUE_GATED_SILU


def route_workspace(tokens, experts, top):
    """Bytes of workspace that route needs for these sizes (0: none)."""
    n = ctypes.c_size_t()
    call(_library.miw_route_workspace, tokens, experts, top, ctypes.byref(n))
    return n.value


def route(logits, chosen, gates, offsets, rows, place, *, tokens, experts, top, dtype=Float32, ld=0, over_all=False, workspace=None, stream=None):
    """The `top` largest of each token's logits (ties to the lowest expert; -inf and NaN never), their softmax, and the
    order of the rows by expert.

    Int32 and Float32 arrays, written here: chosen [tokens, top] (-1: none), gates [tokens, top] (softmax over the chosen, or
    over all logits with over_all), offsets [experts + 1], rows [tokens * top] (the token at each sorted position), place [tokens,
    top] (the sorted position of each choice, or -1).  workspace: a DeviceArray of route_workspace bytes, where that is not 0."""
    call(_library.miw_route, TYPE_CODES[dtype], tokens, experts, top, ld, 1 if over_all else 0, logits, chosen, gates, offsets,
         rows, place, workspace, 0 if workspace is None else workspace.nbytes, None if stream is None else _stream(stream))


def route_grad(logits, chosen, gates, dgates, dlogits, *, tokens, experts, top, dtype=Float32, ld=0, ldd=0, over_all=False, stream=None):
    """The gradient to the logits from the gradient to the gates; writes all of dlogits [tokens, experts]."""
    call(_library.miw_route_grad, TYPE_CODES[dtype], tokens, experts, top, ld, ldd, 1 if over_all else 0, logits, chosen, gates,
         dgates, dlogits, None if stream is None else _stream(stream))


def grouped_gemm(A, W, D, offsets, *, rows, groups, n, k, dtype=Float16, d_type=None, w_layout=ColMajor, gather=None, a_rows=0, lda=0, ldw=0, stride_w=0,
                 ldd=0, epilogue=None, stream=None):
    """D[r] = A[gather[r]] * W_g for the sorted positions offsets[g] <= r < offsets[g + 1] of each group g (gather None: A[r]).

    W_g is k x n: n x k in memory with w_layout ColMajor, k x n with RowMajor.  a_rows: rows of A, needed with gather.  D has
    `dtype` elements or Float32 ones; its rows outside the groups are not touched.  epilogue GATED_SILU: D is n / 2 wide,
    column c of it silu(column 2c) * (column 2c + 1)."""
    call(_library.miw_grouped_gemm, TYPE_CODES[dtype], TYPE_CODES[dtype if d_type is None else d_type], _layout_code(w_layout), epilogue_code(epilogue),
         rows, groups, n, k, lda, ldw, stride_w, ldd, a_rows, A, W, D, offsets, gather,
         None if stream is None else _stream(stream))


def grouped_wgrad(A, B, D, offsets, *, rows, groups, m, n, dtype=Float16, d_type=Float32, gather=None, b_rows=0, lda=0, ldb=0, ldd=0, stride_d=0,
                  accumulate=False, stream=None):
    """D_g (m x n) = sum over the sorted positions r of group g of A[r]^T * B[gather[r]]; zeros for a group without rows.
    accumulate: added to D."""
    call(_library.miw_grouped_wgrad, TYPE_CODES[dtype], TYPE_CODES[d_type], 1 if accumulate else 0, rows, groups, m, n, lda, ldb, ldd, stride_d, b_rows,
         A, B, D, offsets, gather, None if stream is None else _stream(stream))


def gated_silu(Z, A, *, rows, n, dtype=Float16, ldz=0, lda=0, stream=None):
    """A (rows x n / 2) = silu(columns 2c) * (columns 2c + 1) of Z (rows x n): what the epilogue GATED_SILU does, from stored columns."""
    call(_library.miw_gated_silu, TYPE_CODES[dtype], rows, n, ldz, lda, Z, A, None if stream is None else _stream(stream))


def gated_silu_grad(Z, dA, dZ, *, rows, n, dtype=Float16, ldz=0, ldda=0, lddz=0, stream=None):
    """The gradient to Z from the one to A; dZ may be Z."""
    call(_library.miw_gated_silu_grad, TYPE_CODES[dtype], rows, n, ldz, ldda, lddz, Z, dA, dZ, None if stream is None else _stream(stream))


def combine(H, place, Y, *, tokens, top, n, rows, dtype=Float16, gates=None, ldh=0, ldy=0, stream=None):
    """Y[t] = sum over j of gates[t, j] * H[place[t, j]] (gates None: 1; a place outside 0 .. rows - 1 adds nothing)."""
    call(_library.miw_combine, TYPE_CODES[dtype], tokens, top, n, rows, ldh, ldy, H, gates, place, Y, None if stream is None else _stream(stream))


def combine_grad(dY, H, place, dH, dgates, *, tokens, top, n, rows, dtype=Float16, gates=None, ldy=0, ldh=0, lddh=0, stream=None):
    """dH[place[t, j]] = gates[t, j] * dY[t] and dgates[t, j] = dY[t] . H[place[t, j]] (dgates None: not computed, H not read)."""
    call(_library.miw_combine_grad, TYPE_CODES[dtype], tokens, top, n, rows, ldy, ldh, lddh, dY, H, gates, place, dH,
         dgates, None if stream is None else _stream(stream))
