"""8-bit floating point: matrices of e4m3 or e5m2 values with one e8m0 scale for 128 along k, their products, and the gated
activation that keeps its input in this form for the backward pass.

A rows x k matrix is two byte arrays.  codes: one value to a byte, rows of 128 * ceil(k / 128) bytes.  scales: panels of four
blocks (512 values of k), ceil(k / 512) x (rows rounded up to a multiple of 4) x 4 bytes.  `codes_bytes` and `scales_bytes` say
how much memory they take.  A last block's values beyond k are zeros: `quantize` writes them, products count on them.

No counterpart in the reference.  Arrays are DeviceArrays or raw device addresses; a pitch or stride of 0 means dense.  All
calls are asynchronous on `stream`.
"""
from . import _lib
from .experts import TYPE_CODES, _library, call, epilogue_code
from .gemm import _layout_code, _stream
from .wmma import Float16, Float32, RowMajor

E4M3, E5M2 = "e4m3", "e5m2"
_FORMATS = {E4M3: _lib.E4M3, E5M2: _lib.E5M2}


def _format_code(format):
    try:
        return _FORMATS[format]
    except (KeyError, TypeError):
        raise ValueError("a format of codes is E4M3 or E5M2") from None


def codes_bytes(rows, k):
    return rows * ((k + 127) // 128 * 128)


def scales_bytes(rows, k):
    return (k + 511) // 512 * ((rows + 3) // 4 * 4) * 4


def quantize(X, codes, scales, *, rows, k, dtype=Float16, format=E4M3, block_rows=1, x_layout=RowMajor, ld=0, ldq=0, lds=0, stream=None):
    """X (rows x k, Float16, BFloat16 or Float32; k x rows in memory with x_layout ColMajor) into codes and scales: the smallest power
    of two that brings a block's largest magnitude within the format, nearest code, ties to even; a block that holds an infinity or a
    NaN gets the scale that stands for NaN.  block_rows 128: one scale for 128 rows and 128 of k, so that a matrix and its transpose
    have the same codes."""
    call(_library.miw_fp8_quantize, TYPE_CODES[dtype], _format_code(format), _layout_code(x_layout), block_rows, rows, k, ld, ldq, lds, X, codes, scales,
         None if stream is None else _stream(stream))


def dequantize(codes, scales, X, *, rows, k, dtype=Float32, format=E4M3, ldq=0, lds=0, ld=0, stream=None):
    """What codes and scales stand for, as Float16, BFloat16 or Float32."""
    call(_library.miw_fp8_dequantize, TYPE_CODES[dtype], _format_code(format), rows, k, ldq, lds, ld, codes, scales, X,
         None if stream is None else _stream(stream))


def gemm(A, A_scales, B, B_scales, D, *, m, n, k, d_type=Float16, a_format=E4M3, lda=0, lds_a=0, ldb=0, lds_b=0, ldd=0, epilogue=None, stream=None):
    """D (m x n, row-major) = A * B^T with A m x k in a_format and B n x k in E4M3.  With d_type Float32 all bits of the products are summed up
    in Float32; for results of 16 bits the matrix cores cut products off 13 bits below the largest of their eight, which is twice as fast."""
    call(_library.miw_fp8_gemm, TYPE_CODES[d_type], _format_code(a_format), epilogue_code(epilogue), m, n, k, lda, lds_a, ldb, lds_b, ldd, A, A_scales, B,
         B_scales, D, None if stream is None else _stream(stream))


def grouped_gemm(A, A_scales, W, W_scales, D, offsets, *, rows, groups, n, k, d_type=Float16, a_format=E4M3, gather=None, a_rows=0, lda=0, lds_a=0, ldw=0,
                 lds_w=0, stride_w=0, stride_ws=0, ldd=0, epilogue=None, stream=None):
    """EXPERTS.grouped_gemm with A in a_format and the groups' n x k matrices W in E4M3; strides from group to group in bytes."""
    call(_library.miw_fp8_grouped_gemm, TYPE_CODES[d_type], _format_code(a_format), epilogue_code(epilogue), rows, groups, n, k, lda, lds_a, ldw, lds_w,
         stride_w, stride_ws, ldd, a_rows, A, A_scales, W, W_scales, D, offsets, gather, None if stream is None else _stream(stream))


def gated_silu(Z, A, codes, scales, *, rows, n, dtype=Float16, ldz=0, lda=0, ldq=0, lds=0, stream=None):
    """EXPERTS.gated_silu that also writes Z (rows x n) as codes (E4M3) and scales, which is all that the backward pass needs of it."""
    call(_library.miw_fp8_gated_silu, TYPE_CODES[dtype], rows, n, ldz, lda, ldq, lds, Z, A, codes, scales, None if stream is None else _stream(stream))


def gated_silu_grad(codes, scales, dA, dZ, *, rows, n, dtype=Float16, A=None, ldq=0, lds=0, ldda=0, lddz=0, lda=0, stream=None):
    """The gradient to Z from the one to A, with what was kept of Z.  A: where given, the activation of the same values (it may be dA)."""
    call(_library.miw_fp8_gated_silu_grad, TYPE_CODES[dtype], rows, n, ldq, lds, ldda, lddz, lda, codes, scales, dA, dZ, A,
         None if stream is None else _stream(stream))
