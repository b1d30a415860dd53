"""What the Python entries take for a stream, and the Julia ones for a workspace; no GPU needed."""
import ctypes
import os

import numpy as np
import pytest

from conftest import ROOT

P = 1 << 20  # an address that nothing looks at


def test_typed_pointers_are_no_streams(miw):
    """An array or a typed pointer in a stream's place is refused before the library sees it."""
    typed, desc, E = miw.DevicePtr(np.float16, P), miw.GEMM.make_desc(16, 16, 16), miw.EXPERTS
    for call in (lambda: miw.synchronize(typed), lambda: miw.GEMM.gemm(P, P, P, P, desc, stream=typed), lambda: miw.GEMM.gemm_bench(P, P, P, P, desc, stream=typed),
                 lambda: E.combine(P, P, P, tokens=4, top=2, n=8, rows=8, stream=typed), lambda: miw.cuda(lambda: None, threads=64, stream=typed)):
        with pytest.raises(ctypes.ArgumentError):
            call()


def test_julias_routing_knows_the_size_of_its_workspace():
    """A DeviceBuffer that is given as workspace needs no size beside it (the library refuses one of no bytes)."""
    text = open(os.path.join(ROOT, "cudanative.jl_amd", "julia", "MIWMMA.jl")).read()
    assert "workspace=nothing, workspace_bytes::Integer=buffer_bytes(workspace)" in text
    assert "buffer_bytes(::Nothing) = 0" in text and "buffer_bytes(a::DeviceBuffer{T}) where {T} = length(a) * sizeof(T)" in text
