"""Microscaled 4-bit floating point: matrices of e2m1 values with one e8m0 scale for 32 along k, and their products.

A rows x k matrix is two byte arrays.  codes: two values to a byte, the one of the lower k in the low half, rows of 16 *
ceil(k / 32) bytes.  scales: panels of eight blocks (256 values of k), ceil(k / 256) x (rows rounded up to an even number) x 8
bytes.  `codes_bytes` and `scales_bytes` say how much memory they take.  A last block's values beyond k are zeros: `quantize` writes them, products count on them.

No counterpart in the reference.  Arrays are DeviceArrays or raw device addresses; a pitch or stride of 0 means dense.  All
calls are asynchronous on `stream`.
"""
from .experts import TYPE_CODES, _library, call, epilogue_code
from .gemm import _stream
from .wmma import Float16, Float32


def codes_bytes(rows, k):
    return rows * ((k + 31) // 32 * 16)


def scales_bytes(rows, k):
    return (k + 255) // 256 * (rows + rows % 2) * 8


def quantize(X, codes, scales, *, rows, k, dtype=Float16, ld=0, ldq=0, lds=0, stream=None):
    """X (rows x k, Float16, BFloat16 or Float32) into codes and scales: scale 2^(floor(log2(largest magnitude)) - 2), nearest
    code, ties to even; a block that holds an infinity or a NaN gets the scale that stands for NaN."""
    call(_library.miw_mxfp4_quantize, TYPE_CODES[dtype], rows, k, ld, ldq, lds, X, codes, scales, None if stream is None else _stream(stream))


def dequantize(codes, scales, X, *, rows, k, dtype=Float32, ldq=0, lds=0, ld=0, stream=None):
    """What codes and scales stand for, as Float16, BFloat16 (exact) or Float32."""
    call(_library.miw_mxfp4_dequantize, TYPE_CODES[dtype], rows, k, ldq, lds, ld, codes, scales, X, None if stream is None else _stream(stream))


def gemm(A, A_scales, B, B_scales, D, *, m, n, k, d_type=Float16, lda=0, lds_a=0, ldb=0, lds_b=0, ldd=0, epilogue=None, stream=None):
    """D (m x n, row-major) = A * B^T with A m x k and B n x k in 4 bits and Float32 sums."""
    call(_library.miw_mxfp4_gemm, TYPE_CODES[d_type], epilogue_code(epilogue), m, n, k, lda, lds_a, ldb, lds_b, ldd, A, A_scales, B,
         B_scales, D, None if stream is None else _stream(stream))


def grouped_gemm(A, A_scales, W, W_scales, D, offsets, *, rows, groups, n, k, d_type=Float16, gather=None, a_rows=0, lda=0, lds_a=0, ldw=0, lds_w=0,
                 stride_w=0, stride_ws=0, ldd=0, epilogue=None, stream=None):
    """EXPERTS.grouped_gemm with A and the groups' n x k matrices W in 4 bits; strides from group to group in bytes."""
    call(_library.miw_mxfp4_grouped_gemm, TYPE_CODES[d_type], epilogue_code(epilogue), rows, groups, n, k, lda, lds_a, ldw, lds_w, stride_w, stride_ws,
         ldd, a_rows, A, A_scales, W, W_scales, D, offsets, gather,
         None if stream is None else _stream(stream))
