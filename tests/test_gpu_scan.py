"""Packed sequences on the GPU (segment tables, gated linear recurrence, one-token form) against their step-by-step evaluation in 64 bits
(oracle/recurrence.py).  Tolerances: the oracle's worst-case bound of an fp32 evaluation, plus half a step of the result's type."""
import numpy as np
import pytest
import torch

from oracle import recurrence as rec

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected but no GPU is visible")
    return torch.device("cuda:0")


def near(got, want, tol, name):
    """|got - want| <= tol + half a step of got's type (subnormals: half the smallest one)."""
    t = got.dtype
    got, want, tol = got.detach().double().cpu().numpy().reshape(want.shape), want, np.broadcast_to(tol, want.shape)
    eps, tiny = torch.finfo(t).eps, torch.finfo(t).tiny
    room = 1.001 * tol + (np.abs(want) + tol) * (eps / 2) + (tiny * eps / 2 if t != torch.float32 else 1e-37)
    bad = ~(np.abs(got - want) <= room)
    assert not bad.any(), (name, int(bad.sum()), bad.size, np.argwhere(bad)[:3].tolist(), got[bad][:3], want[bad][:3], room[bad][:3])


def lengths_of(kind, seed=0):
    g = np.random.RandomState(seed)
    return {
        "one": [1], "row": [0, 0, 1, 0], "ones": [1] * 131, "none": [0, 0, 0], "long": [1500], "two": [700, 801], "word": [63, 1, 64, 65, 127, 0, 128, 1],
        "ragged": g.randint(0, 40, 60).tolist(), "mixed": [0, 0, 5, 900, 0, 1, 1, 300, 0] + [0] * 300 + [33, 0], "holes": (g.randint(0, 3, 200) * g.randint(0, 9, 200)).tolist(),
        "tile": [256, 256, 512, 32, 2048], "off": [255, 257, 31, 33, 2047, 2049],
    }[kind]


def inputs(n, d, g, t, gt, form, seed, gen_dev="cpu"):
    r = torch.Generator().manual_seed(seed)
    z = torch.randn(n, g, generator=r)
    gate = {"decay": lambda: torch.sigmoid(1.5 * z + 2), "log": lambda: -torch.nn.functional.softplus(1.5 * z - 2), "alpha": lambda: torch.sigmoid(3 * z - 3)}[form]()
    return gate.to(TYPES[gt]), torch.randn(n, d, generator=r).to(TYPES[t])


def d64(t):
    return None if t is None else t.detach().double().cpu().numpy()


# ---------------------------------------------------------------------------------------------- tables
@pytest.mark.parametrize("extra", [0, 7, 200])
@pytest.mark.parametrize("kind", ["one", "row", "ones", "none", "long", "word", "ragged", "mixed", "holes", "off"])
def test_tables(dev, kind, extra):
    from tensoflow_amd import ops
    ln = lengths_of(kind)
    n = sum(ln) + extra
    t = ops.segment_tables(torch.tensor(ln, device=dev), n)
    offsets, index, position, bits = rec.tables(ln, n)
    assert np.array_equal(t.offsets.cpu().numpy(), offsets) and np.array_equal(t.index.cpu().numpy(), index)
    assert np.array_equal(t.position.cpu().numpy(), position) and np.array_equal(t.starts.cpu().numpy().view(np.uint64), bits)
    if extra == 0:
        whole = ops.segment_tables(torch.tensor(ln, device=dev), index=False, position=False)
        assert whole.n_rows == n and whole.index is None and whole.position is None and torch.equal(whole.starts, t.starts)
    head = index[: sum(ln)]
    u = ops.segment_tables_from_index(torch.from_numpy(head).to(dev), len(ln))
    o2, _, _, b2 = rec.tables(ln, len(head))
    assert np.array_equal(u.offsets.cpu().numpy(), o2) and np.array_equal(u.starts.cpu().numpy().view(np.uint64), b2)


@pytest.mark.parametrize("n", [0, 10, 300])
def test_tables_of_bad_lengths(dev, n):
    """Negative lengths count as none; what goes beyond n_rows is cut."""
    from tensoflow_amd import ops
    ln = [5, -3, 0, 100, -(1 << 62), 1 << 62, 4]
    t = ops.segment_tables(torch.tensor(ln, device=dev), n, block_rows=8, free_blocks=torch.arange(400, dtype=torch.int32, device=dev), max_blocks=9)
    want = rec.tables(ln, n, 8, np.arange(400), 9)
    for got, w in zip((t.offsets, t.index, t.position, t.starts, t.block_table, t.slots), want):
        assert np.array_equal(got.cpu().numpy().view(w.dtype), w)


def test_tables_without_segments(dev):
    from tensoflow_amd import ops
    assert ops.segment_offsets(torch.zeros(0, dtype=torch.int64, device=dev)).tolist() == [0]
    assert ops.segment_offsets(torch.tensor([3, -1, 0, 4], device=dev)).tolist() == [0, 3, 3, 3, 7]
    t = ops.segment_tables(torch.zeros(0, dtype=torch.int64, device=dev), 70)
    assert t.offsets.tolist() == [0] and t.index.eq(-1).all() and t.position.eq(-1).all() and t.starts.eq(0).all()


@pytest.mark.parametrize("block,n_free,width", [(1, 5000, 700), (16, 5000, 128), (16, 20, 128), (100, 40, 3), (64, 0, 5), (7, 500, 0)])
def test_blocks(dev, block, n_free, width):
    from tensoflow_amd import ops
    ln = lengths_of("mixed") + lengths_of("ragged")
    n = sum(ln) + 9
    free = torch.randperm(n_free, generator=torch.Generator().manual_seed(1)).int()
    t = ops.segment_tables(torch.tensor(ln, device=dev), n, block_rows=block, free_blocks=free.to(dev), max_blocks=width)
    want = rec.tables(ln, n, block, free.numpy(), width)
    assert np.array_equal(t.block_table.cpu().numpy(), want[4]) and np.array_equal(t.slots.cpu().numpy(), want[5])


@pytest.mark.parametrize("r,n", [(1023, 5000), (1024, 3), (4097, 100000), (70001, 200000), (300000, 250), (1100000, 3000001)])
def test_tables_of_many(dev, r, n):
    """Against torch on the host: longer lists than the step-by-step form is made for, runs of a hundred thousand empty segments among them."""
    from tensoflow_amd import ops
    g = torch.Generator().manual_seed(r)
    w = torch.rand(r, generator=g) ** 2 * (torch.rand(r, generator=g) > 0.3)
    w[r // 5: r // 2] = 0
    cut = (w.double().cumsum(0) / w.double().sum() * n).round().long()
    ln = torch.diff(cut, prepend=torch.zeros(1, dtype=torch.int64))
    t = ops.segment_tables(ln.to(dev), n, block_rows=16, free_blocks=torch.arange(n // 16 + r, dtype=torch.int32, device=dev), max_blocks=2)
    index = torch.repeat_interleave(torch.arange(r), ln)
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), ln.cumsum(0)])
    assert torch.equal(t.offsets.cpu(), offsets) and torch.equal(t.index.cpu(), index) and torch.equal(t.position.cpu(), torch.arange(n) - offsets[index])
    nb = (ln + 15) // 16
    at = (nb.cumsum(0) - nb)[:, None] + torch.arange(2)
    assert torch.equal(t.block_table.cpu(), torch.where(torch.arange(2) < nb[:, None], at, -1).int())
    u = ops.segment_tables_from_index(t.index, r)
    assert torch.equal(u.offsets, t.offsets) and torch.equal(u.starts, t.starts)


# ---------------------------------------------------------------------------------------------- scan
SHAPES = [(1, 1), (2, 1), (3, 1), (4, 1), (4, 4), (7, 7), (10, 1), (12, 4), (15, 5), (33, 1), (64, 64), (66, 22), (96, 2), (130, 130), (200, 2), (256, 1), (260, 260)]


def run_case(dev, ln, d, g, t, gt, form, reverse, h0=True, extra=0, seed=0, gy=True, gf=True):
    from tensoflow_amd import ops
    n, R = sum(ln) + extra, len(ln)
    gate, x = inputs(n, d, g, t, gt, form, seed)
    r = torch.Generator().manual_seed(seed + 1)
    h = torch.randn(R, d, generator=r) if h0 else None
    G = torch.randn(n, d, generator=r).to(TYPES[t]) if gy else None
    Gf = torch.randn(R, d, generator=r) if gf else None
    c = lambda v: None if v is None else v.to(dev)
    tab = ops.segment_tables(torch.tensor(ln, device=dev), n)
    y, final, carry = ops.gated_scan(c(gate), c(x), tab, c(h), form, reverse, want_final=True, want_carry=True)
    want = rec.scan(d64(gate), d64(x), rec.tables(ln, n)[0], d64(h), form, reverse, d64(G), d64(Gf))
    near(y, want["y"], want["y_tol"], "y")
    near(final, want["final"], want["final_tol"], "final")
    y2, none = ops.gated_scan(c(gate), c(x), tab, c(h), form, reverse)
    assert none is None and torch.equal(y2, y)
    if gy or gf:
        gg, gx, gh = ops.gated_scan_bwd(c(gate), c(x), tab, carry, c(G), c(Gf), c(h), form, reverse)
        near(gg, want["g_gate"], want["g_gate_tol"], "g_gate")
        near(gx, want["g_x"], want["g_x_tol"], "g_x")
        near(gh, want["g_h0"], want["g_h0_tol"], "g_h0")


@pytest.mark.parametrize("d,g", SHAPES)
def test_scan_shapes(dev, d, g):
    k = SHAPES.index((d, g))
    run_case(dev, lengths_of("ragged", k), d, g, "f32", "f32", ("decay", "log", "alpha")[k % 3], k % 2 == 1, seed=k)
    run_case(dev, lengths_of("word"), d, g, "bf16", ("bf16", "f32")[k % 2], ("alpha", "decay", "log")[k % 3], k % 2 == 0, seed=k + 100, extra=5)


@pytest.mark.parametrize("form", ["decay", "log", "alpha"])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("t,gt", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
def test_scan_types_and_forms(dev, t, gt, form, reverse):
    run_case(dev, lengths_of("mixed"), 24, 24, t, gt, form, reverse, seed=3)
    run_case(dev, lengths_of("two"), 40, 5, t, gt, form, reverse, seed=4, extra=70)


@pytest.mark.parametrize("kind", ["one", "row", "ones", "none", "long", "two", "word", "ragged", "mixed", "holes", "tile", "off"])
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_lengths(dev, kind, reverse):
    for k, (d, g) in enumerate([(3, 1), (16, 16), (80, 1)]):
        run_case(dev, lengths_of(kind), d, g, "f32", "f32", ("alpha", "log", "decay")[k], reverse, h0=k != 1, extra=(0, 130, 3)[k], seed=k)


@pytest.mark.parametrize("gy,gf,h0", [(True, False, False), (False, True, True), (True, True, False)])
def test_scan_missing_gradients(dev, gy, gf, h0):
    run_case(dev, lengths_of("mixed"), 20, 4, "f32", "f32", "log", False, h0=h0, gy=gy, gf=gf)
    run_case(dev, lengths_of("mixed"), 3, 1, "f16", "f32", "alpha", True, h0=h0, gy=gy, gf=gf)


@pytest.mark.parametrize("d,g,t", [(1, 1, "f32"), (8, 1, "f32"), (512, 512, "bf16"), (384, 3, "f16"), (600, 1, "bf16"), (1030, 2, "f32"), (2048, 16, "bf16")])
def test_scan_long(dev, d, g, t):
    """Sequences over many pieces, alone and beside short ones."""
    run_case(dev, [5000, 3, 0, 1200], d, g, t, "f32", "decay", False, seed=d)
    run_case(dev, [1, 4100], d, g, t, "f32", "log", True, seed=d + 1, extra=1)


@pytest.mark.parametrize("d,g,t,gt", [(387, 387, "f32", "f32"), (387, 3, "bf16", "f32"), (259, 1, "f16", "f16"), (514, 514, "bf16", "bf16"), (514, 257, "f32", "f32"),
                                      (63, 63, "bf16", "f32"), (60, 60, "f16", "f16"), (62, 31, "bf16", "f32"), (774, 2, "bf16", "bf16")])
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_odd_widths(dev, d, g, t, gt, reverse):
    """Every width of a lane's vector, one workgroup and several across the channels, heads across workgroups, short rows of two types."""
    for k, form in enumerate(("decay", "log", "alpha")):
        run_case(dev, [70, 0, 3, 300, 1, 1, 140], d, g, t, gt, form, reverse, seed=d + k, extra=3 * k)


@pytest.mark.parametrize("d,n,reverse", [(1, 3000001, False), (3, 1200007, True), (8, 400003, False), (64, 70001, True), (520, 9001, False)])
def test_scan_many_tiles_exactly(dev, d, n, reverse):
    """Decays of 1 and small whole numbers: every sum is exact in 24 bits in any order, so thousands of tiles have to give the running sums to the bit."""
    from tensoflow_amd import ops
    g = torch.Generator(device=dev).manual_seed(d)
    cut = n // 3
    ln = [cut, 0, 1, n - cut - 1]
    x = torch.randint(-2, 3, (n, d), device=dev, generator=g).float()
    gy = torch.randint(-2, 3, (n, d), device=dev, generator=g).float()
    one = torch.ones(n, 1, device=dev)
    tab = ops.segment_tables(torch.tensor(ln, device=dev), n)
    sums = lambda v, back: torch.cat([(s.flip(0) if back else s).double().cumsum(0).flip([0] if back else []) for s in v.split([cut, 1, n - cut - 1])])
    y, final, carry = ops.gated_scan(one, x, tab, None, "decay", reverse, want_final=True, want_carry=True)
    want, lam = sums(x, reverse), sums(gy, not reverse)
    assert float(want.abs().max()) < 2 ** 24 and float(lam.abs().max()) < 2 ** 24
    assert torch.equal(y.double(), want)
    ends = [0, cut, cut + 1] if reverse else [cut - 1, cut, n - 1]
    assert torch.equal(final[[0, 2, 3]].double(), want[ends]) and bool((final[1] == 0).all())
    gg, gx, gh = ops.gated_scan_bwd(one, x, tab, carry, gy, None, None, "decay", reverse)
    assert torch.equal(gx.double(), lam)
    ends = [cut - 1, cut, n - 1] if reverse else [0, cut, cut + 1]
    assert torch.equal(gh[[0, 2, 3]].double(), lam[ends]) and bool((gh[1] == 0).all())
    before = want - x.double()
    part = lam * before
    # each product is rounded once and at most d - 1 sums of theirs follow
    assert bool(((gg.double() - part.sum(1, keepdim=True)).abs() <= d * 2.0 ** -24 * part.abs().sum(1, keepdim=True)).all())


def test_scan_without_segments(dev):
    from tensoflow_amd import ops
    tab = ops.segment_tables(torch.zeros(0, dtype=torch.int64, device=dev), 300)
    for d, gates in ((3, 1), (300, 300)):
        x, gate = torch.full((300, d), float("nan"), device=dev), torch.full((300, gates), float("nan"), device=dev)
        y, final, carry = ops.gated_scan(gate, x, tab, torch.zeros(0, d, device=dev), want_final=True, want_carry=True)
        assert bool((y == 0).all()) and final.shape == (0, d)
        gg, gx, gh = ops.gated_scan_bwd(gate, x, tab, carry, x, final, torch.zeros(0, d, device=dev))
        assert bool((gg == 0).all()) and bool((gx == 0).all()) and gh.shape == (0, d)


def test_scan_does_not_cross_segments(dev):
    """A neighbour's NaN, inf or overflow stays there: a first step selects its own state, it does not multiply the last one by 0."""
    from tensoflow_amd import ops
    for d, g in ((3, 1), (64, 64), (256, 2)):
        for reverse in (False, True):
            ln = [300, 400, 0, 1, 700]
            n = sum(ln)
            gate, x = inputs(n, d, g, "f32", "f32", "decay", 5)
            gy, h0 = torch.randn(n, d, generator=torch.Generator().manual_seed(2)), torch.zeros(5, d)
            want = rec.scan(d64(gate), d64(x), rec.tables(ln, n)[0], d64(h0), "decay", reverse, d64(gy), None)
            keep = torch.ones(n, dtype=torch.bool)
            keep[300:700] = False
            x[350], x[400], gate[500], gy[450], h0[1] = float("nan"), float("inf"), float("inf"), float("nan"), float("-inf")
            tab = ops.segment_tables(torch.tensor(ln, device=dev), n)
            y, final, carry = ops.gated_scan(gate.to(dev), x.to(dev), tab, h0.to(dev), "decay", reverse, want_final=True, want_carry=True)
            gg, gx, gh = ops.gated_scan_bwd(gate.to(dev), x.to(dev), tab, carry, gy.to(dev), None, h0.to(dev), "decay", reverse)
            k = keep.numpy()
            near(y[keep.to(dev)], want["y"][k], want["y_tol"][k], "y")
            near(gx[keep.to(dev)], want["g_x"][k], want["g_x_tol"][k], "g_x")
            near(gg[keep.to(dev)], want["g_gate"][k], want["g_gate_tol"][k], "g_gate")
            rows = [0, 2, 3, 4]
            near(final[rows], want["final"][rows], want["final_tol"][rows], "final")
            near(gh[rows], want["g_h0"][rows], want["g_h0_tol"][rows], "g_h0")
            assert not bool(torch.isfinite(final[1]).any())


def test_scan_first_step_with_an_infinite_decay(dev):
    """a h0 + b at a segment's first row as the formula has it, for short rows and long ones."""
    from tensoflow_amd import ops
    for d, g in ((4, 1), (40, 40), (256, 2)):
        ln = [20, 30, 41]
        gate, x = inputs(91, d, g, "f32", "f32", "decay", 3)
        h0 = torch.ones(3, d)
        gate[20] = float("inf")
        h0[1, 0] = -1.0
        y, _ = ops.gated_scan(gate.to(dev), x.to(dev), ops.segment_tables(torch.tensor(ln, device=dev), 91), h0.to(dev))
        assert bool(torch.isinf(y[20]).all()) and float(y[20, 0]) < 0 < float(y[20, 1]) and bool(torch.isfinite(y[:20]).all()) and bool(torch.isfinite(y[50:]).all())


def test_scan_leaves_the_rest(dev):
    from tensoflow_amd import ops
    ln, n, d = [5, 0, 60], 200, 12
    gate, x = inputs(n, d, 1, "f16", "f16", "alpha", 1)
    x[65:], gate[65:] = float("nan"), float("nan")
    tab = ops.segment_tables(torch.tensor(ln, device=dev), n)
    out = torch.full((n, d), 7.0, dtype=torch.float16, device=dev)
    y, _ = ops.gated_scan(gate.to(dev), x.to(dev), tab, form="alpha", out=out)
    z, _, carry = ops.gated_scan(gate.to(dev), x.to(dev), tab, form="alpha", want_carry=True)
    assert y is out and bool((y[65:] == 7).all()) and torch.equal(y[:65], z[:65]) and bool((z[65:] == 0).all())
    gg, gx, _ = ops.gated_scan_bwd(gate.to(dev), x.to(dev), tab, carry, torch.full_like(x, float("nan")).to(dev).index_fill_(0, torch.arange(65, device=dev), 1.0), None,
                                   form="alpha", need_h0=False)
    assert bool((gg[65:] == 0).all()) and bool((gx[65:] == 0).all()) and bool(torch.isfinite(gx).all()) and bool(torch.isfinite(gg).all())


def test_scan_from_an_index_with_foreign_rows(dev):
    """Rows in front of the first segment and behind the last one."""
    from tensoflow_amd import ops
    index = torch.tensor([-1] * 70 + [0] * 3 + [2] * 100 + [5] * 40 + [7] * 90)
    n, d = len(index), 20
    gate, x = inputs(n, d, 20, "f32", "f32", "decay", 2)
    gy = torch.randn(n, d, generator=torch.Generator().manual_seed(2))
    tab = ops.segment_tables_from_index(index.to(dev), 6)
    assert tab.offsets.tolist() == [70, 73, 73, 173, 173, 173, 213]
    for reverse in (False, True):
        want = rec.scan(d64(gate), d64(x), tab.offsets.tolist(), None, "decay", reverse, d64(gy), None)
        y, final, carry = ops.gated_scan(gate.to(dev), x.to(dev), tab, None, "decay", reverse, want_final=True, want_carry=True)
        gg, gx, gh = ops.gated_scan_bwd(gate.to(dev), x.to(dev), tab, carry, gy.to(dev), None, None, "decay", reverse)
        for got, k in ((y, "y"), (final, "final"), (gg, "g_gate"), (gx, "g_x"), (gh, "g_h0")):
            near(got, want[k], want[k + "_tol"], k)


def test_scan_of_garbage_tables_stays_in_bounds(dev):
    """Unsorted indexes and lengths from elsewhere give some numbers, and read and write nothing outside."""
    from tensoflow_amd import ops
    n, d = 500, 16
    gate, x = inputs(n, d, 4, "f32", "f32", "log", 2)
    r = torch.Generator().manual_seed(1)
    for index in (torch.randint(-5, 40, (n,), generator=r), torch.randint(-2 ** 62, 2 ** 62, (n,), generator=r)):
        tab = ops.segment_tables_from_index(index.to(dev), 30)
        assert int(tab.offsets.min()) >= 0 and int(tab.offsets.max()) <= n
        y, final, carry = ops.gated_scan(gate.to(dev), x.to(dev), tab, torch.zeros(30, d, device=dev), "log", want_final=True, want_carry=True)
        g = ops.gated_scan_bwd(gate.to(dev), x.to(dev), tab, carry, x.to(dev), final, torch.zeros(30, d, device=dev), "log")
        assert y.shape == x.shape and g[2].shape == (30, d)
    torch.cuda.synchronize()


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("off", [0, 1, 3])
def test_scan_strides_and_alignment(dev, t, off):
    """Column slices of a wider projection, rows of one gate for all, heads as a third dimension."""
    from tensoflow_amd import ops
    ln = lengths_of("two")
    n = sum(ln)
    for d, g in ((3, 1), (12, 4), (128, 128), (136, 2)):
        gate, x = inputs(n, d, g, t, t, "decay", 7)
        tab = ops.segment_tables(torch.tensor(ln, device=dev), n)
        a, _ = ops.gated_scan(gate.to(dev), x.to(dev), tab)
        both = torch.randn(n, off + d + 5 + g + 2, device=dev).to(TYPES[t])
        both[:, off:off + d], both[:, off + d + 5:off + d + 5 + g] = x.to(dev), gate.to(dev)
        xs, gs = both[:, off:off + d], both[:, off + d + 5:off + d + 5 + g]
        b, _, carry = ops.gated_scan(gs, xs, tab, want_carry=True)
        assert torch.equal(a, b)
        gy = torch.randn(n * d + off, device=dev).to(TYPES[t])[off:].view(n, d)
        plain = ops.gated_scan_bwd(gate.to(dev), x.to(dev), tab, carry, gy.clone(), None)
        for p, q in zip(plain, ops.gated_scan_bwd(gs, xs, tab, carry, gy, None)):
            assert torch.equal(p, q)
        room = torch.full((n * d + 7 + off,), 3.0, dtype=x.dtype, device=dev)
        o, _ = ops.gated_scan(gs, xs, tab, out=room[off:off + n * d].view(n, d))
        assert torch.equal(o, a) and torch.equal(room[off:off + n * d].view(n, d), a) and bool((room[off + n * d:] == 3).all()) and bool((room[:off] == 3).all())
        c, _ = ops.gated_scan(gate.to(dev).view(n, g), x.to(dev).view(n, g, d // g), tab)
        assert c.shape == (n, g, d // g) and torch.equal(c.view(n, d), a)
        row = gate[:1].to(dev).expand(n, g)
        e, _ = ops.gated_scan(row, x.to(dev), tab)
        f, _ = ops.gated_scan(row.contiguous(), x.to(dev), tab)
        assert torch.equal(e, f)
    one = torch.randn(n, device=dev)
    p, _ = ops.gated_scan(one.sigmoid(), torch.ones(n, 6, device=dev), tab)
    q, _ = ops.gated_scan(one.sigmoid()[:, None], torch.ones(n, 6, device=dev), tab)
    assert torch.equal(p, q)


def test_scan_repeats_bit_by_bit(dev):
    from tensoflow_amd import ops
    for d, g, ln in ((1024, 8, [6000, 5, 900]), (3, 1, [40] * 3000 + [9000])):
        n = sum(ln)
        gate, x = inputs(n, d, g, "f32", "f32", "decay", 1)
        gate, x, tab = gate.to(dev), x.to(dev), ops.segment_tables(torch.tensor(ln, device=dev), n)
        ref = None
        for _ in range(5):
            y, f, c = ops.gated_scan(gate, x, tab, want_final=True, want_carry=True)
            got = (y, f, *ops.gated_scan_bwd(gate, x, tab, c, x, f))
            ref = ref or got
            assert all(torch.equal(p, q) for p, q in zip(ref, got))


def test_scan_is_the_composite(dev):
    """Back-to-front blending of a ray's samples is its weighted sum: the recurrence's end state against tf_composite_fwd, and its alpha
    gradient against tf_composite_bwd, on the same packed rays."""
    from tensoflow_amd import autograd, ops
    g = torch.Generator().manual_seed(4)
    ln = torch.randint(0, 130, (500,), generator=g)
    n = int(ln.sum())
    tab = ops.segment_tables(ln.to(dev))
    alpha = torch.sigmoid(3 * torch.randn(n, generator=g) - 3).to(dev).requires_grad_()
    vals = torch.rand(n, 5, generator=g).to(dev).requires_grad_()
    w, acc, out = autograd.CompositeFn.apply(alpha, vals, tab.index, 500)
    y, final = autograd.gated_scan(alpha, vals, tab, form="alpha", reverse=True)
    go = torch.randn(500, 5, generator=g).to(dev)
    # both are convex sums of values in [0, 1]: 130 steps of 3 roundings of 2^-24 each, and the same for the other
    assert float((final - out).detach().abs().max()) < 2 * 130 * 3 * 2 ** -24
    ga, gv = torch.autograd.grad(out, (alpha, vals), go)
    sa, sv = torch.autograd.grad(final, (alpha, vals), go)
    want = rec.scan(d64(alpha)[:, None], d64(vals), tab.offsets.tolist(), None, "alpha", True, None, d64(go))
    near(sa, want["g_gate"][:, 0], want["g_gate_tol"][:, 0], "alpha")
    near(sv, want["g_x"], want["g_x_tol"], "values")
    assert float((gv - sv).abs().max()) < 1e-4 and float((ga - sa).abs().max()) < 1e-3 * float(sa.abs().max())


# ---------------------------------------------------------------------------------------------- autograd
def test_autograd_against_differences(dev):
    """The directional derivative of a random functional, central differences of the 64-bit evaluation: off by the differences' own h^2."""
    from tensoflow_amd import autograd, ops
    ln = [40, 0, 1, 90]
    n, d, g = sum(ln), 12, 3
    for form in ("decay", "log", "alpha"):
        for reverse in (False, True):
            gate, x = inputs(n, d, g, "f32", "f32", form, 9)
            r = torch.Generator().manual_seed(10)
            h0, cy, cf = torch.randn(4, d, generator=r), torch.randn(n, d, generator=r), torch.randn(4, d, generator=r)
            dg, dx, dh = [torch.randn(t.shape, generator=r) for t in (gate, x, h0)]
            off = rec.tables(ln, n)[0]

            def value(e):
                w = rec.scan(d64(gate) + e * d64(dg), d64(x) + e * d64(dx), off, d64(h0) + e * d64(dh), form, reverse)
                return float((w["y"] * d64(cy)).sum() + (w["final"] * d64(cf)).sum())
            e = 1e-5
            want = (value(e) - value(-e)) / (2 * e)
            leaves = [t.to(dev).requires_grad_() for t in (gate, x, h0)]
            tab = ops.segment_tables(torch.tensor(ln, device=dev))
            y, final = autograd.gated_scan(leaves[0], leaves[1], tab, leaves[2], form, reverse)
            ((y * cy.to(dev)).sum() + (final * cf.to(dev)).sum()).backward()
            terms = [(t.grad.double().cpu() * v.double()) for t, v in zip(leaves, (dg, dx, dh))]
            got, size = sum(float(t.sum()) for t in terms), sum(float(t.abs().sum()) for t in terms)
            assert abs(got - want) < 1e-5 * size, (form, reverse, got, want, size)     # 2^-24 x ~100 steps of the terms' sizes, and e^2


def test_autograd_of_views_and_broadcasts(dev):
    from tensoflow_amd import autograd, ops
    ln = [30, 50]
    tab = ops.segment_tables(torch.tensor(ln, device=dev))
    base = torch.rand(4, device=dev, requires_grad=True)
    x = torch.randn(24, 80, device=dev, requires_grad=True)
    y, f = autograd.gated_scan(base.expand(80, 4), x.t(), tab)                        # a gate for all rows; channels across the rows
    gb, gx = torch.autograd.grad(y.sum() + f.sum(), (base, x))
    full = base.detach().expand(80, 4).contiguous().requires_grad_()
    xc = x.detach().t().contiguous().requires_grad_()
    y2, f2 = autograd.gated_scan(full, xc, tab)
    gfull, gxc = torch.autograd.grad(y2.sum() + f2.sum(), (full, xc))
    assert torch.equal(y, y2) and torch.allclose(gb, gfull.sum(0), rtol=1e-5) and torch.equal(gx, gxc.t())
    z, zf = autograd.gated_scan(torch.rand(0, 4, device=dev), torch.rand(0, 24, device=dev, requires_grad=True), ops.segment_tables(torch.zeros(2, dtype=torch.int64, device=dev)))
    assert z.shape == (0, 24) and zf.eq(0).all()
    only = autograd.gated_scan(full, xc.detach(), tab)[1]                             # the gate alone wants a gradient, of the end state alone
    assert torch.autograd.grad(only.sum(), full)[0].shape == (80, 4)


def test_autograd_of_rounded_outputs(dev):
    """y in bf16 is rounded, the gradients are those of the unrounded states."""
    from tensoflow_amd import autograd, ops
    ln = [700, 801]
    n = sum(ln)
    gate, x = inputs(n, 256, 2, "bf16", "f32", "decay", 12)
    gy = torch.randn(n, 256, generator=torch.Generator().manual_seed(1)).bfloat16()
    a, b = gate.to(dev).requires_grad_(), x.to(dev).requires_grad_()
    y, _ = autograd.gated_scan(a, b, ops.segment_tables(torch.tensor(ln, device=dev)))
    ga, gx = torch.autograd.grad(y, (a, b), gy.to(dev))
    want = rec.scan(d64(gate), d64(x), [0, 700, 1501], None, "decay", False, d64(gy), None)
    near(ga, want["g_gate"], want["g_gate_tol"], "g_gate")
    near(gx, want["g_x"], want["g_x_tol"], "g_x")


# ---------------------------------------------------------------------------------------------- one token
@pytest.mark.parametrize("b,d,g,t,gt", [(1, 1, 1, "f32", "f32"), (1, 2048, 2048, "bf16", "bf16"), (5, 10, 2, "f16", "f32"), (33, 96, 1, "bf16", "f32"), (256, 130, 130, "f32", "f32"),
                                        (300, 4, 4, "f16", "f16"), (64, 515, 5, "bf16", "bf16")])
@pytest.mark.parametrize("form", ["decay", "log", "alpha"])
def test_step(dev, b, d, g, t, gt, form):
    from tensoflow_amd import ops
    S = b + 20
    gate, x = inputs(b, d, g, t, gt, form, b)
    r = torch.Generator().manual_seed(b)
    pool, slots = torch.randn(S, d, generator=r), torch.randperm(S, generator=r)[:b]
    if b > 4:
        slots[1], slots[3], slots[b - 1], slots[b // 2] = -1, slots[0], slots[0], S        # padding, one sequence three times, out of the pool
    state = pool.to(dev)
    y = ops.gated_step(state, slots.to(dev), gate.to(dev), x.to(dev), form)
    want, after, written = rec.step(d64(pool), slots.numpy(), d64(gate), d64(x), form)
    # at most three steps of four roundings (exp: its own two, and its argument's) of sums that never pass 4 (1 + |h| + |x|)
    tol = 2.0 ** -24 * 3 * 16 * (1 + np.abs(after).max())
    near(y, want, tol * written[:, None], "y")
    near(state, after, tol * (d64(pool) != after), "state")
    out = torch.full((b, d), 3.0, dtype=x.dtype, device=dev)
    ops.gated_step(pool.to(dev), slots.to(dev), gate.to(dev), x.to(dev), form, out=out)
    w = torch.from_numpy(written).to(dev)
    assert torch.equal(out[w], y[w]) and bool((out[~w] == 3).all()) and bool((y[~w] == 0).all())


def test_step_of_many_rows(dev):
    """Beyond what one launch takes, a slot's rows in two launches among them."""
    from tensoflow_amd import ops
    b, d, S = 9000, 8, 10000
    gate, x = inputs(b, d, 2, "f32", "f32", "decay", 1)
    r = torch.Generator().manual_seed(3)
    pool, slots = torch.randn(S, d, generator=r), torch.randperm(S, generator=r)[:b]
    slots[8999], slots[5000], slots[8500] = slots[17], -1, slots[8400]
    state = pool.to(dev)
    y = ops.gated_step(state, slots.to(dev), gate.to(dev), x.to(dev))
    want, after, written = rec.step(d64(pool), slots.numpy(), d64(gate), d64(x), "decay")
    near(y, want, 2.0 ** -24 * 3 * 16 * (1 + np.abs(after).max()) * written[:, None], "y")
    near(state, after, 2.0 ** -24 * 3 * 16 * (1 + np.abs(after).max()) * (d64(pool) != after), "state")


def test_step_after_step_is_the_scan(dev):
    """Ragged prompts through the scan, their end states into the pool, then tokens one by one: the states of the scan over the whole."""
    from tensoflow_amd import ops
    b, d, T = 6, 128, 9
    prompts = [17, 1, 0, 300, 64, 65]
    whole = [n + T for n in prompts]
    n = sum(whole)
    gate, x = inputs(n, d, 4, "f32", "f32", "log", 8)
    off = rec.tables(whole, n)[0]
    head = torch.cat([torch.arange(off[s], off[s] + prompts[s]) for s in range(b)])
    want = rec.scan(d64(gate), d64(x), off, None, "log", False)
    gate, x = gate.to(dev), x.to(dev)
    tab = ops.segment_tables(torch.tensor(prompts, device=dev), len(head))
    _, final = ops.gated_scan(gate[head.to(dev)], x[head.to(dev)], tab, form="log", want_final=True)
    pool = torch.full((20, d), float("nan"), device=dev)
    slots = torch.tensor([3, 19, 0, 7, 8, 1], device=dev)
    pool[slots] = final
    for k in range(T):
        rows = torch.tensor([off[s] + prompts[s] + k for s in range(b)])
        y = ops.gated_step(pool, slots, gate[rows.to(dev)], x[rows.to(dev)], form="log")
        near(y, want["y"][rows.numpy()], want["y_tol"][rows.numpy()], f"token {k}")
    near(pool[slots], want["final"], want["final_tol"], "final")


# ---------------------------------------------------------------------------------------------- streams and graphs
def test_step_strides(dev):
    """Column slices of a fused projection, at even and odd places."""
    from tensoflow_amd import ops
    for b, d in ((3, 40), (80, 1024)):
        for off in (0, 1, 4):
            both = torch.randn(b, 2 * d + 9, device=dev).bfloat16()
            x, g = both[:, off:off + d], both[:, off + d:off + 2 * d].sigmoid()
            wide = torch.zeros(b, 2 * d + 9, device=dev, dtype=torch.bfloat16)
            wide[:, off + 1:off + 1 + d] = g
            s1, slots = torch.randn(b + 5, d, device=dev), torch.randperm(b + 5, device=dev)[:b].contiguous()
            s2 = s1.clone()
            assert torch.equal(ops.gated_step(s1, slots, wide[:, off + 1:off + 1 + d], x), ops.gated_step(s2, slots, g.contiguous(), x.contiguous())) and torch.equal(s1, s2)


def test_scan_on_other_streams(dev):
    from tensoflow_amd import ops
    ln = [4000, 7, 900]
    n = sum(ln)
    gate, x = inputs(n, 512, 512, "bf16", "f32", "log", 1)
    gate, x, lens = gate.to(dev), x.to(dev), torch.tensor(ln, device=dev)
    ref, _ = ops.gated_scan(gate, x, ops.segment_tables(lens, n), form="log")
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for k in range(6):                                     # two streams at once, tables and scan on each
        with torch.cuda.stream(side[k % 2]):
            got.append(ops.gated_scan(gate, x, ops.segment_tables(lens, n), form="log")[0])
    torch.cuda.synchronize()
    assert all(torch.equal(ref, y) for y in got)


def test_scan_in_a_graph(dev):
    """Tables, scan, its backward and a step captured together and replayed on new inputs, eager work and synchronisations between the replays."""
    from tensoflow_amd import autograd, ops
    ln = [3000, 0, 40, 1500]
    n, d, g = sum(ln), 256, 2
    lens = torch.tensor(ln, device=dev)
    gate, x = [t.to(dev) for t in inputs(n, d, g, "f32", "f32", "decay", 1)]
    gy = torch.randn(n, d, device=dev)
    pool, slots = torch.randn(8, d, device=dev), torch.tensor([2, 5, 2, 7], device=dev)
    keep = pool.clone()

    def work(gate, x):
        a, b = gate.detach().requires_grad_(), x.detach().requires_grad_()
        tab = ops.segment_tables(lens, n)
        y, final = autograd.gated_scan(a, b, tab)
        ga, gx = torch.autograd.grad((y, final), (a, b), (gy, final.detach()))
        z = ops.gated_step(pool, slots, gate[:4], x[:4])
        return y.detach(), final.detach(), ga, gx, z, tab.index

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            work(gate, x)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):                                     # two graphs of the same work, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = work(gate, x)
        graphs.append((graph, out))
    for k in range(6):
        new_gate, new_x = inputs(n, d, g, "f32", "f32", "decay", 20 + k)
        gate.copy_(new_gate.to(dev))
        x.copy_(new_x.to(dev))
        pool.copy_(keep)
        graph, out = graphs[k % 2]
        graph.replay()
        torch.cuda.synchronize()
        after = pool.clone()
        pool.copy_(keep)
        for p, q in zip(work(gate, x), out):
            assert torch.equal(p, q), k
        assert torch.equal(pool, after)


# ---------------------------------------------------------------------------------------------- in the march
def test_march_to_running_colour(golden, dev):
    """The operators as a renderer uses them: packed samples of the fixed-step sampler, tables of their rays, opacities of the field, then the
    running back-to-front blend; its end is what render_core composites."""
    from conftest import AABB
    from tensoflow_amd import march, ops
    g = golden("march_r32")
    f = march.SdfField(g.sd, AABB, [32, 32, 32], 3, device=dev)
    o, d = g["rays_o"].to(dev), g["dirs"].to(dev)
    near_, far_ = march.near_far_from_sphere(o, d)
    t0, t1, ridx = march.march_uniform(f, o, d, near_, far_, n_steps=64)
    rn = o.shape[0]
    tab = ops.segment_tables_from_index(ridx, rn)
    radii, cos = g["radiis"].to(dev), g["rays_cos"].to(dev)
    out = march.render_core(f, o, d, radii, cos, t0, t1, ridx, float(g["base_radii"]), 20.0, 0.5)
    ones = torch.ones(len(ridx), 1, device=dev)
    y, final = ops.gated_scan(out["alpha"], torch.cat([ones, out["grad"]], -1).contiguous(), tab, form="alpha", reverse=True, want_final=True)
    longest = int(torch.diff(tab.offsets).max())
    # the opacity is a convex sum of ones, the normals' sum that of gradients: two evaluations of `longest` steps, 3 roundings each
    room = 2 * 3 * longest * 2 ** -24
    assert float((final[:, :1] - out["acc"]).abs().max()) < room
    _, _, ref = ops.composite(out["alpha"], ridx, out["grad"].contiguous(), rn)
    assert float((final[:, 1:] - ref).abs().max()) < room * max(1.0, float(out["grad"].abs().max()))
    first = tab.offsets[:-1][torch.diff(tab.offsets) > 0]
    assert torch.equal(y[first], final[torch.diff(tab.offsets) > 0])
