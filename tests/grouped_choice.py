"""Which kernel runs a product grouped by expert, by the library's own rule."""
import ctypes


class _GroupedParams(ctypes.Structure):
    """grouped_params of csrc/experts.hpp."""
    _fields_ = ([(x, ctypes.c_void_p) for x in ("X", "Y", "xs", "ys", "offsets", "gather", "D")] +
                [(x, ctypes.c_int) for x in ("groups", "rows", "source_rows", "I", "J", "K")] +
                [(x, ctypes.c_long) for x in ("ldx", "ldy", "ldd", "sx", "sd", "sxs", "lxs", "lys")] +
                [(x, ctypes.c_int) for x in ("x_k_major", "gated", "accumulate", "vector", "d_vector", "most_tiles")])


class _Choice(ctypes.Structure):
    _fields_ = [(x, ctypes.c_int) for x in ("kernel", "rows", "weights", "waves", "tile")] + [("workgroups", ctypes.c_long)]


TILES = ("256x256", "256x128", "128x128", "128x64")


def grouped_kernel(miw, *, rows, groups, n, k=0, m=0, layout="col", mxfp4=False, vector=True, a_rows=0, cus=256):
    """(name, workgroups, threads of one) for dense operands.  m: a ragged sum of m x n.  Names: "plain"; "narrow" with the 16-row tiles of rows and of
    weights and the wavefronts; "tile" with its extents."""
    lib = ctypes.CDLL(miw._lib.LIB_PATH)
    f = lib._ZN3miw14choose_groupedERKNS_14grouped_paramsEbbi
    f.restype, f.argtypes = _Choice, [ctypes.POINTER(_GroupedParams), ctypes.c_bool, ctypes.c_bool, ctypes.c_int]
    row = (k + 31) // 32 * 16 if mxfp4 else 2 * k
    p = _GroupedParams(groups=groups, rows=rows, source_rows=a_rows or rows, I=n, J=m, K=k, vector=vector and (mxfp4 or n % 8 == 0 or layout == "col") and (mxfp4 or (m or k) % 8 == 0),
                       x_k_major=layout == "col" and not m)
    p.ldx, p.ldy = (2 * n, 2 * m) if m else (row if layout == "col" else 2 * n, row)
    c = f(ctypes.byref(p), mxfp4, m > 0, cus)
    if c.kernel == 0:
        return "plain", 0, 0
    if c.kernel == 1:
        return "narrow %d %d %d" % (c.rows, c.weights, c.waves), c.workgroups, 64 * c.waves
    return "tile " + TILES[c.tile], c.workgroups, 512
