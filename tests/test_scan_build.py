"""The gated recurrence as it is built: how its rows are cut into waves and tiles, and that no kernel of it keeps its rows anywhere but in registers."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def lib():
    import os
    from tensoflow_amd import lib as L
    if not os.path.exists(L.LIB_PATH):
        import __graft_entry__ as ge
        ge.build()
    return L.load()


class Geo(C.Structure):
    _fields_ = [(k, C.c_int) for k in ("V", "CL", "W", "LP", "hs", "parts", "slabs", "nw")] + [("shared", C.c_bool), ("tile_rows", C.c_int64), ("tiles", C.c_int64)]


def geometry(lib, n, d, g, x_type):
    from tensoflow_amd import lib as L
    f = C.CDLL(L.LIB_PATH)["_ZN6tfscan8geometryERK11TfGatedScan"]
    f.restype, f.argtypes = Geo, [C.POINTER(L.TfGatedScan)]
    return f(C.byref(L.TfGatedScan(n, 1, d, g, d, g, x_type, x_type, 0, 0, 0)))


@pytest.mark.parametrize("d,g", [(1, 1), (4, 1), (7, 7), (30, 3), (64, 64), (96, 2), (260, 260), (600, 1), (4096, 32), (65521, 65521)])
@pytest.mark.parametrize("x_type", [0, 2])
def test_no_wave_without_rows(lib, d, g, x_type):
    """Rows that fit the waves of one workgroup are one tile, of no more waves than they need; beyond that a tile is full."""
    for n in [1, 2, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 500, 513, 1000, 1025, 2048, 2049, 5000, 40000]:
        t = geometry(lib, n, d, g, x_type)
        wave = 64 // t.CL * 8
        most = 4 if x_type == 0 or d < 64 else 8
        assert t.tile_rows == t.nw * wave and t.tiles == -(-n // t.tile_rows)
        if n <= most * wave:
            assert t.tiles == 1 and t.nw in (1, 2, 4, 8) and (t.nw == 1 or n > t.nw // 2 * wave), (n, t.nw)
        else:
            assert t.nw == 1 or t.tiles * t.slabs >= 512, (n, t.nw)


# ---------------------------------------------------------------------------------------------- registers
REMARK = "a.hip:1:1: remark: {} [-Rpass-analysis=kernel-resource-usage]\n"


def report(**kernels):
    out = "a.hip:1:1: warning: something else\n"
    for name, (spill, scratch, dynamic) in kernels.items():
        for line in (f"Function Name: {name}", "    TotalSGPRs: 106", "    VGPRs: 128", "    AGPRs: 0", f"    ScratchSize [bytes/lane]: {scratch}", f"    Dynamic Stack: {dynamic}",
                     "    Occupancy [waves/SIMD]: 4", "    SGPRs Spill: 104", f"    VGPRs Spill: {spill}", "    LDS Size [bytes/block]: 80"):
            out += REMARK.format(line)
    return out


@pytest.mark.parametrize("kernels,word", [
    (dict(a=(0, 0, "False"), b=(0, 0, "False")), None), (dict(a=(0, 0, "False"), b=(63, 252, "False")), "b: VGPRs Spill 63"),
    (dict(a=(0, 48, "False"), b=(0, 0, "False")), "a: ScratchSize [bytes/lane] 48"), (dict(a=(0, 0, "True")), "a: Dynamic Stack True"), ({}, "no kernel")])
def test_spilled_vector_registers_end_the_build(tmp_path, kernels, word):
    import os
    import subprocess
    import sys
    from tensoflow_amd import lib as L
    path = tmp_path / "a.usage"
    path.write_text(report(**kernels))
    run = subprocess.run([sys.executable, os.path.join(os.path.dirname(L.__file__), "csrc", "no_spills.py"), str(path)], capture_output=True, text=True)
    assert (run.returncode == 0) == (word is None) and "something else" in run.stderr and (word is None or word in run.stderr)


@pytest.mark.parametrize("source", ["scan_fwd", "scan_bwd", "scan", "segment"])
def test_the_build_looks_for_spills(source):
    import os
    import subprocess
    from tensoflow_amd import lib as L
    csrc = os.path.join(os.path.dirname(L.__file__), "csrc")
    plan = subprocess.run(["make", "-n", "-B", "-C", csrc, f"{source}.o"], capture_output=True, text=True, check=True).stdout
    assert "-Rpass-analysis=kernel-resource-usage" in plan and f"no_spills.py {source}.usage" in plan
