"""Functions of the grouped products' kernels and dispatch that also run on the host: addresses and choices of kernels, without a GPU."""
import os
import re
import shutil
import subprocess

import pytest

from grouped_choice import grouped_kernel

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SCALES = """
#include "grouped_tile.hpp"
#include <cstdio>
// Matrices of n rows each, one behind the other in each panel of lds rows of scales (the last one's rows end where the panel ends, or `more`
// rows before that): the bytes that a tile's loads of scales touch in the last panel of the last matrix.
int main()
{
    for (long n : {1l, 2l, 38l, 130l, 192l, 1087l, 1088l, 2879l, 2880l})
        for (long matrices : {1l, 2l, 5l})
            for (long more : {0l, 2l, 300l})
                for (int bi : {128, 256}) {
                    const long own = n + n % 2, lds = matrices * own + more, base = (matrices - 1) * own;
                    for (long i0 = 0; i0 < n; i0 += bi)
                        for (int part = 0; part < bi / 128; part++)
                            for (int lane = 0; lane < 64; lane++) {
                                const long row = miw::scale_pair((int)i0, part, lane, (int)n), wanted = i0 + 128 * part + 2 * lane;
                                if (row < 0 || row % 2 || base + row + 2 > matrices * own || (wanted < n && row != wanted)) {
                                    std::printf("%ld matrices of %ld rows, panels of %ld, tile of %d at %ld: part %d, lane %d reads rows %ld and %ld", matrices, n, lds, bi, i0, part, lane,
                                                base + row, base + row + 1);
                                    return 1;
                                }
                            }
                }
    return 0;
}
"""


def _run(tmp_path, source):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    src, exe = tmp_path / "host.hip", tmp_path / "host"
    src.write_text(source)
    r = subprocess.run([hipcc, "--offload-arch=gfx950", "-O1", "-std=c++20", "-Wno-inline-asm", "-I" + os.path.join(ROOT, "cudanative.jl_amd", "csrc"),
                        "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", str(src), "-o", str(exe)], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


def test_loads_of_scales_stay_inside_their_matrix(tmp_path):
    """4-bit matrices that lie one behind the other in panels: no load of the last one's scales goes beyond its rows."""
    _run(tmp_path, SCALES)


@pytest.mark.parametrize("experts", [1, 16, 1024])
def test_route_workspace_never_falls_as_tokens_grow(miw, experts):
    """What suffices for the most tokens of a program suffices for all its calls."""
    need = [miw.EXPERTS.route_workspace(t, experts, 1) for t in [*range(0, 20000), *(1 << b for b in range(15, 31))]]
    assert not any(need[:65]) and need[65] > 0
    assert all(a <= b for a, b in zip(need, need[1:]))


# Sizes up to what the entries accept, and matrices that a GPU's memory holds.
GROUPS, WIDTHS, DEPTHS, ROWS = (1, 3, 64, 1024, 8192, 65536), (8, 64, 336, 2016, 2056, 8192, 32768), (8, 32, 64, 2048, 16384), (1, 10, 700, 65536, 600000)


@pytest.mark.parametrize("kind", ["16 bits", "4 bits", "sum"])
def test_the_kernel_that_is_chosen_can_be_launched(miw, kind):
    seen = set()
    for groups in GROUPS:
        for n in WIDTHS:
            for k in DEPTHS:
                for rows in ROWS:
                    if groups * n * (n if kind == "sum" else k) > 1 << 37 or rows * max(n, k) > 1 << 37:
                        continue
                    tiles = -(-n // 256) * (min(groups, rows) + rows // 256 if kind != "sum" else groups * -(-n // 256))
                    if kind != "16 bits" and tiles >= (1 << 23) - 8:  # (refused)
                        continue
                    sizes = dict(m=n, n=n) if kind == "sum" else dict(n=n, k=k, layout="col")
                    name, workgroups, threads = grouped_kernel(miw, rows=rows, groups=groups, mxfp4=kind == "4 bits", **sizes)
                    seen.add(name)
                    walks = name.startswith("tile") and kind == "16 bits"
                    assert workgroups < 1 << 30 if walks else workgroups * threads < 1 << 32, (kind, groups, n, k, rows, name, workgroups)
    assert len(seen) > 3, seen


def test_many_groups_of_few_rows(miw):
    """As many groups as the products take, nearly all of them without rows."""
    for mxfp4 in (False, True):
        for n in (2016, 2056, 4096, 65536):
            name, workgroups, threads = grouped_kernel(miw, rows=10, groups=65536, n=n, k=64, mxfp4=mxfp4)
            assert workgroups * threads < 1 << 32, (n, name, workgroups)


def _instances(miw, kernel):
    """Template arguments of a kernel's instances in the library (those with a 16-bit type of results have names that nm may not take apart)."""
    nm = shutil.which("nm")
    if nm is None:
        pytest.skip("no nm")
    names = subprocess.run([nm, "-C", miw._lib.LIB_PATH], capture_output=True, text=True, check=True).stdout
    return {tuple(x.strip() for x in args.split(",")) for args in re.findall(r"__device_stub__%s<(.*)>\(" % kernel, names)}


def _chosen(miw, **form):
    return {grouped_kernel(miw, rows=rows, groups=groups, n=n, k=k, **form)[0]
            for groups in (1, 3, 8, 16, 64, 128) for n in (64, 256, 336, 1024, 2048, 4096) for k in (32, 512, 2048, 8192) for rows in (1, 24, 64, 100, 500, 1000, 3000, 16384, 65536)}


@pytest.mark.parametrize("op,mxfp4", [("op_f16", False), ("op_bf16", False), ("op_mxfp4", True)])
def test_every_grouped_kernel_of_the_library_is_chosen_for_some_product(miw, op, mxfp4):
    chosen = _chosen(miw, mxfp4=mxfp4)
    forms = {"narrow %s %s %s" % a[1:4] for a in _instances(miw, "k_grouped_narrow") if a[0].endswith(op)}
    assert forms == {c for c in chosen if c.startswith("narrow")}
    tiles = {a[1:3] + (a[7],) for a in _instances(miw, "k_grouped_tile") if a[0].endswith(op)}  # (extents and form)
    reached = {("col", c) for c in chosen}
    if not mxfp4:
        reached |= {("row", c) for c in _chosen(miw, layout="row")}
        reached |= {("sum", c) for c in {grouped_kernel(miw, rows=rows, groups=groups, n=n, m=m)[0] for groups in (1, 8, 64) for n in (64, 336, 1024, 4096) for m in (64, 1024, 4096)
                                         for rows in (1, 100, 1000, 16384)}}
    assert tiles == {tuple(c.split()[1].split("x")) + ({"col": "0", "row": "1", "sum": "3" if c == "tile 256x128" else "2"}[form],) for form, c in reached if c.startswith("tile")}


def test_every_routing_kernel_of_the_library_is_launched_for_some_experts(miw):
    """Sixteen lanes a token hold 16 experts a register up to 256 experts, a wavefront 64 beyond."""
    forms = {a[1:3] for a in _instances(miw, "k_route_choose")}
    assert forms == {("4", "true"), ("8", "true"), ("16", "true"), ("16", "false")}
