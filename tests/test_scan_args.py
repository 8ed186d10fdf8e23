"""Packed sequences on the CPU: the oracle against closed forms, and the refusals of the entry points (checked on the host before any launch)."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import recurrence as rec


@pytest.fixture(scope="module")
def lib():
    import os
    from tensoflow_amd import lib as L
    if not os.path.exists(L.LIB_PATH):
        import __graft_entry__ as ge
        ge.build()
    return L.load()


def test_oracle_closed_forms():
    """A constant decay is a geometric sum, an alpha gate run backwards the transmittance-weighted sum; gradients against central differences."""
    off = [0, 4, 4, 9]
    y = rec.scan(np.full((9, 1), 0.5), np.ones((9, 2)), off, None)["y"]
    assert np.allclose(y[:4, 0], 2 - 0.5 ** np.arange(4)) and np.allclose(y[4:, 1], 2 - 0.5 ** np.arange(5))
    r = np.random.RandomState(0)
    al, v = r.rand(9, 1), r.randn(9, 3)
    out = rec.scan(al, v, off, None, "alpha", True)
    for s in range(3):
        T, want = 1.0, np.zeros(3)
        for i in range(off[s], off[s + 1]):
            want += T * al[i, 0] * v[i]
            T *= 1 - al[i, 0]
        assert np.allclose(out["final"][s], want)
    h0, gy, gf = r.randn(3, 4), r.randn(9, 4), r.randn(3, 4)
    x = r.randn(9, 4)
    for form in ("decay", "log", "alpha"):
        for reverse in (False, True):
            gate = -r.rand(9, 2) if form == "log" else r.rand(9, 2)
            got = rec.scan(gate, x, off, h0, form, reverse, gy, gf)

            def value(gate, x, h0):
                w = rec.scan(gate, x, off, h0, form, reverse)
                return (w["y"] * gy).sum() + (w["final"] * gf).sum()
            for k, t in enumerate((gate, x, h0)):
                d = r.randn(*t.shape)
                args = [gate, x, h0]
                hi, lo = list(args), list(args)
                hi[k], lo[k] = t + 1e-6 * d, t - 1e-6 * d
                num = (value(*hi) - value(*lo)) / 2e-6
                ana = (got[("g_gate", "g_x", "g_h0")[k]] * d).sum()
                assert abs(num - ana) < 1e-6 * (1 + abs(ana)), (form, reverse, k)


def test_oracle_tables():
    o, i, p, b, t, s = rec.tables([2, 0, 3], 6, 2, [7, 1, 4], 2)
    assert o.tolist() == [0, 2, 2, 5] and i.tolist() == [0, 0, 2, 2, 2, -1] and p.tolist() == [0, 1, 0, 1, 2, -1] and b.tolist() == [0b101]
    assert t.tolist() == [[7, -1], [-1, -1], [1, 4]] and s.tolist() == [14, 15, 2, 3, 8, -1]


def desc(**kw):
    from tensoflow_amd import lib as L
    d = dict(n_rows=8, n_segments=2, ld_x=4, ld_gate=2, channels=4, gates=2, x_type=0, gate_type=0, form=0, reverse=0, zero_rest=0)
    d.update(kw)
    return L.TfGatedScan(*[d[k] for k, _ in L.TfGatedScan._fields_])


def test_cabi_refusals(lib):
    a = C.addressof((C.c_int64 * 64)())
    err = lambda: lib.tf_last_error()
    # tables
    tab = lambda lengths=a, r=2, n=8, off=a, idx=a, pos=a, st=a, br=0, free=None, nf=0, mb=0, bt=None, sl=None, ws=None, nw=0: \
        lib.tf_segment_tables(lengths, r, n, off, idx, pos, st, br, free, nf, mb, bt, sl, ws, nw, None)
    assert tab(r=-1) == -2 and tab(n=-1) == -2 and tab(br=-1) == -2 and tab(off=None) == -1 and tab(lengths=None) == -1
    assert tab(n=1 << 60) == -2 and b"too many" in err()
    assert tab(bt=a) == -1 and b"without a block size" in err()
    assert tab(r=2049) == -2 and b"workspace" in err() and tab(r=2049, br=4, free=a, nf=2, mb=2, bt=a, sl=a, ws=a, nw=2050) == -2 and b"workspace" in err()
    assert tab(st=None) == -1 and b"need starts" in err() and tab(br=4, free=a, nf=2, mb=2, bt=a, sl=a, idx=None) == -1 and b"need an index" in err()
    assert tab(br=1 << 31, free=a, nf=2, mb=2, bt=a, sl=a) == -2 and b"blocks too large" in err()
    assert tab(br=4, free=a, nf=2, mb=1 << 40, bt=a, sl=a, ws=a, nw=2) == -2 and b"too large" in err()
    assert tab(br=4, nf=2, mb=2, bt=a, sl=a, ws=a, nw=2) == -1 and tab(br=4, free=a, nf=2, mb=2, sl=a, ws=a, nw=2) == -1
    assert lib.tf_segment_from_index(a, -1, 2, a, a, None) == -2 and lib.tf_segment_from_index(None, 4, 2, a, a, None) == -1
    assert lib.tf_segment_from_index(a, 4, 2, None, a, None) == -1
    # scan
    big = 1 << 30
    fwd = lambda d, gate=a, x=a, off=a, idx=a, st=a, y=a, nw=big: lib.tf_gated_scan_fwd(C.byref(d), gate, x, off, idx, st, None, y, None, None, a, nw, None)
    bwd = lambda d, gate=a, x=a, off=a, idx=a, st=a, nw=big, ws=a: lib.tf_gated_scan_bwd(C.byref(d), gate, x, off, idx, st, None, a, a, None, a, a, None, ws, nw, None)
    for run in (fwd, bwd):
        assert run(desc(n_rows=-1)) == -2 and run(desc(n_segments=-1)) == -2 and run(desc(channels=0)) == -2 and run(desc(gates=3)) == -2 and run(desc(gates=0)) == -2
        assert run(desc(channels=1 << 20, gates=1)) == -2 and run(desc(ld_x=-4)) == -2 and run(desc(n_rows=1 << 40)) == -2
        assert run(desc(x_type=3)) == -1 and run(desc(x_type=0, gate_type=1)) == -1 and run(desc(x_type=1, gate_type=2)) == -1 and run(desc(form=3)) == -1
        assert run(desc(n_rows=100, ld_x=5)) == -1 and run(desc(), x=a + 4) == -1 and b"aligned" in err() and run(desc(gates=4, ld_gate=5)) == -1
        assert run(desc(), gate=None) == -1 and run(desc(), x=None) == -1 and run(desc(), off=None) == -1
    assert fwd(desc(), y=None) == -1 and fwd(desc(), y=a + 4) == -1 and fwd(desc(n_rows=100000), nw=0) == -2 and b"workspace" in err()
    assert lib.tf_gated_scan_fwd(None, a, a, a, a, a, None, a, None, None, a, big, None) == -1 and b"null descriptor" in err()
    # step
    step = lambda d, gate=a, x=a, slots=a, ns=4, state=a, y=a: lib.tf_gated_step(C.byref(d), gate, x, slots, ns, state, y, None)
    assert step(desc(n_rows=0)) == 0 and step(desc(n_rows=8193)) == -2 and step(desc(), ns=-1) == -2 and step(desc(), slots=None) == -1 and step(desc(), state=None) == -1
    assert step(desc(), y=None) == -1 and step(desc(form=-1)) == -1


def test_wrappers_refuse_the_cpu_and_wrong_shapes():
    from tensoflow_amd import ops
    z = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t)
    tab = ops.SegmentTables(4, 1, z(2, t=torch.int64), None, None, z(1, t=torch.int64))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.segment_tables(z(3, t=torch.int64), 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.segment_tables_from_index(z(3, t=torch.int64), 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.gated_scan(z(4, 1), z(4, 2), tab)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.gated_step(z(4, 2), z(4, t=torch.int64), z(4, 1), z(4, 2))
    with pytest.raises(RuntimeError, match=r"\[R\]"):
        ops.segment_tables(z(3, 3, t=torch.int64), 4)
    desc_of = lambda gate, x, form="decay": ops._scan_desc(gate, x, 1, form, False, 0)
    d, n, c = desc_of(z(4, 2), z(4, 2, 3))
    assert (n, c, d.gates, d.ld_x, d.ld_gate) == (4, 6, 2, 6, 2)
    d, n, c = desc_of(z(4, 9)[:, 1:3], z(5, 4, 7)[1, :, 2:6])
    assert (n, c, d.gates, d.ld_x, d.ld_gate) == (4, 4, 2, 7, 9)
    assert desc_of(z(4), z(4, 3))[0].gates == 1 and desc_of(z(2).expand(4, 2), z(4, 4))[0].ld_gate == 0
    for gate, x, form, word in ((z(4, 3), z(4, 4), "decay", "does not go"), (z(3, 2), z(4, 4), "decay", "does not go"), (z(4, 2), z(4, 4), "exp", "form"),
                                (z(4, 2, t=torch.float64), z(4, 4), "decay", "float32, float16"), (z(4, 2, t=torch.float16), z(4, 4), "decay", "must be"),
                                (z(4, 2), z(4, 4, t=torch.int32), "decay", "float32, float16"), (z(4, 2), z(4, 8)[:, ::2], "decay", "contiguous"),
                                (z(4, 1).expand(4, 2), z(4, 4), "decay", "contiguous"), (z(4), z(4), "decay", "x must be"), (z(4, 2), z(4, 0), "decay", "does not go")):
        with pytest.raises(RuntimeError, match=word):
            desc_of(gate, x, form)
    with pytest.raises(RuntimeError, match="h0 must be"):
        ops._state(z(3, 4), 2, 4, "h0")
