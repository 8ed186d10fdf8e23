"""Packed sequences: tables of more segments than one workgroup sums by itself, steps of many channels, and every kernel of the scan, against
their step-by-step evaluation in 64 bits (oracle/recurrence.py)."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import recurrence as rec
from test_gpu_scan import TYPES, d64, inputs, lengths_of, near, run_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected but no GPU is visible")
    return torch.device("cuda:0")


# ---------------------------------------------------------------------------------------------- tables
def many(kind):
    """Over 2048 lengths."""
    g = np.random.RandomState(5)
    return {
        "short": lengths_of("mixed") + g.randint(0, 5, 4000).tolist() + lengths_of("off"),
        "empty": [0] * 3000 + [3] + [0] * 2500 + lengths_of("ragged") + [0] * 900,
        "ones": [1] * 2049,
        "bad": [5, -3, 0, 100] + g.randint(-4, 4, 3000).tolist() + [-(1 << 62), 1 << 62, 4] + [1 << 62] * 5 + [2] * 100,
    }[kind]


def rows_in(ln):
    return sum(n for n in ln if 0 < n < 1 << 40)


def same(got, want):
    for t, w in zip((got.offsets, got.index, got.position, got.starts, got.block_table, got.slots), want):
        assert t is None or np.array_equal(t.cpu().numpy().view(w.dtype), w)


@pytest.mark.parametrize("kind", ["short", "empty", "ones", "bad"])
@pytest.mark.parametrize("extra", [-40, 0, 7, 200])
def test_tables_of_many_segments(dev, kind, extra):
    """Rows behind the last segment, lengths that go beyond the rows, negative ones; one table or the other left out."""
    from tensoflow_amd import ops
    ln = many(kind)
    n = rows_in(ln) + extra
    lens, want = torch.tensor(ln, device=dev), rec.tables(ln, n)
    same(ops.segment_tables(lens, n), want)
    for index, position in ((True, False), (False, True), (False, False)):
        t = ops.segment_tables(lens, n, index=index, position=position)
        assert (t.index is not None, t.position is not None) == (index, position)
        same(t, want)


@pytest.mark.parametrize("kind,extra", [("short", 9), ("empty", 0), ("bad", -30), ("ones", 70)])
@pytest.mark.parametrize("block,n_free,width", [(1, 20000, 70), (16, 9000, 20), (16, 300, 20), (100, 2500, 1), (64, 0, 5), (7, 9000, 0), (7, 9000, 200)])
def test_blocks_of_many_segments(dev, kind, extra, block, n_free, width):
    from tensoflow_amd import ops
    ln = many(kind)
    n = rows_in(ln) + extra
    free = torch.randperm(n_free, generator=torch.Generator().manual_seed(1)).int()
    t = ops.segment_tables(torch.tensor(ln, device=dev), n, block_rows=block, free_blocks=free.to(dev), max_blocks=width)
    same(t, rec.tables(ln, n, block, free.numpy(), width))


def test_tables_at_odd_addresses(dev):
    """8 bytes off a 16-byte border: rows are stored one by one; what stands around them stays."""
    from tensoflow_amd import lib as L
    ln = many("short")
    n, R, B, free = rows_in(ln) + 5, len(ln), 16, torch.arange(20000, dtype=torch.int32, device=dev)
    want = rec.tables(ln, n, B, free.cpu().numpy(), 9)
    lens, lib = torch.tensor(ln, device=dev), L.load()
    new = lambda k: torch.full((k + 2,), 77, dtype=torch.int64, device=dev)
    off, idx, pos, st, sl = new(R + 1), new(n), new(n), new((n + 63) // 64), new(n)
    bt = torch.full((R * 9 + 2,), 77, dtype=torch.int32, device=dev)
    nw = lib.tf_segment_workspace_words(R, B)
    work = torch.empty(nw, dtype=torch.int64, device=dev)
    at = lambda t: C.c_void_p(t.data_ptr() + t.element_size())
    L.check(lib.tf_segment_tables(lens.data_ptr(), R, n, at(off), at(idx), at(pos), at(st), B, free.data_ptr(), len(free), 9, at(bt), at(sl), work.data_ptr(), nw,
                                  torch.cuda.current_stream().cuda_stream), "tf_segment_tables")
    for t, w in zip((off, idx, pos, st, bt, sl), want):
        assert np.array_equal(t[1:-1].cpu().numpy().view(w.dtype), w.reshape(-1)) and int(t[0]) == 77 and int(t[-1]) == 77


# ---------------------------------------------------------------------------------------------- one token
@pytest.mark.parametrize("t,gt", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("form", ["decay", "log", "alpha"])
def test_step_of_wide_batches(dev, t, gt, form):
    """Four channels a lane, gates of their own and of heads; padding, rows of one slot, slots outside the pool."""
    from tensoflow_amd import ops
    for b, d, g in ((70, 1024, 1024), (70, 1024, 8), (257, 300, 3), (257, 300, 300)):
        gate, x = inputs(b, d, g, t, gt, form, b + g)
        r = torch.Generator().manual_seed(b)
        pool, slots = torch.randn(b + 20, d, generator=r), torch.randperm(b + 20, generator=r)[:b]
        slots[1], slots[3], slots[b - 1], slots[b // 2], slots[7] = -1, slots[0], slots[0], b + 20, 1 << 40
        state = pool.to(dev)
        y = ops.gated_step(state, slots.to(dev), gate.to(dev), x.to(dev), form)
        want, after, written = rec.step(d64(pool), slots.numpy(), d64(gate), d64(x), form)
        # at most three steps of four roundings (exp: its own two, and its argument's) of sums that never pass 4 (1 + |h| + |x|)
        tol = 2.0 ** -24 * 3 * 16 * (1 + np.abs(after).max())
        near(y, want, tol * written[:, None], "y")
        near(state, after, tol * (d64(pool) != after), "state")


# ---------------------------------------------------------------------------------------------- every kernel
# (own or shared gates, channels a lane, a wave across the channels): widths that take it; heads of a power of two, of pieces, alone and side by side
WIDTHS = {
    (False, 1, False): [(7, 7), (1, 1)], (False, 2, False): [(14, 14), (2, 2)], (False, 3, False): [(15, 15), (3, 3)], (False, 4, False): [(20, 20), (128, 128)],
    (False, 1, True): [(65, 65)], (False, 2, True): [(130, 130)], (False, 3, True): [(195, 195)], (False, 4, True): [(260, 260)],
    (True, 1, False): [(15, 3), (5, 1)], (True, 2, False): [(30, 3), (2, 1)], (True, 3, False): [(27, 3), (3, 1)], (True, 4, False): [(96, 3), (4, 1)],
    (True, 1, True): [(74, 2), (77, 1)], (True, 2, True): [(148, 2), (154, 1)], (True, 3, True): [(222, 2), (231, 1)], (True, 4, True): [(256, 1), (260, 1)],
}


@pytest.mark.parametrize("t,gt", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("shared,v,wide", list(WIDTHS))
def test_scan_every_kernel(dev, t, gt, shared, v, wide):
    """Each instantiation of both directions: all gate forms, both ways, many tiles of one wave and one tile of several, with and without a start state."""
    for d, g in WIDTHS[shared, v, wide]:
        for k, form in enumerate(("decay", "log", "alpha")):
            for reverse in (False, True):
                run_case(dev, [37, 0, 150, 1, 1, 200, 2, 3], d, g, t, gt, form, reverse, h0=k != 1 or reverse, extra=11 * (k == 2), seed=d + k)
                run_case(dev, [3, 1, 0, 19, 5], d, g, t, gt, form, reverse, h0=k != 0 or reverse, extra=2 * k, seed=d + k)


@pytest.mark.parametrize("t,gt", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("d,g", [(512, 512), (512, 2), (516, 1), (250, 250), (60, 60), (60, 20)])
def test_scan_tiles_of_several_waves_exactly(dev, t, gt, d, g):
    """Decays of 1 and small whole numbers: every sum is exact in 24 bits in any order, so what is rounded once has to agree to the bit."""
    from tensoflow_amd import ops
    n = {512: 16500, 516: 16500, 250: 33000, 60: 160001}[d]
    r = torch.Generator(device=dev).manual_seed(d)
    cut = n // 3
    ln = [cut, 0, 1, n - cut - 1]
    x = torch.randint(-2, 3, (n, d), device=dev, generator=r).to(TYPES[t])
    gy = torch.randint(-2, 3, (n, d), device=dev, generator=r).to(TYPES[t])
    one = torch.ones(n, g, device=dev, dtype=TYPES[gt])
    tab = ops.segment_tables(torch.tensor(ln, device=dev), n)
    sums = lambda v, back: torch.cat([(s.flip(0) if back else s).double().cumsum(0).flip([0] if back else []) for s in v.split([cut, 1, n - cut - 1])])
    for reverse in (False, True):
        y, final, carry = ops.gated_scan(one, x, tab, None, "decay", reverse, want_final=True, want_carry=True)
        want, lam = sums(x, reverse), sums(gy, not reverse)
        assert float(want.abs().max()) < 60000 and float(lam.abs().max()) < 60000
        ends = [0, cut, cut + 1] if reverse else [cut - 1, cut, n - 1]
        assert torch.equal(y, want.to(y.dtype)) and torch.equal(final[[0, 2, 3]].double(), want[ends]) and bool((final[1] == 0).all())
        gg, gx, gh = ops.gated_scan_bwd(one, x, tab, carry, gy, None, None, "decay", reverse)
        ends = [cut - 1, cut, n - 1] if reverse else [0, cut, cut + 1]
        assert torch.equal(gx, lam.to(gx.dtype)) and torch.equal(gh[[0, 2, 3]].double(), lam[ends]) and bool((gh[1] == 0).all())
        part = (lam * (want - x.double())).view(n, g, d // g)
        # each product is rounded once, at most d / g - 1 sums of theirs follow, and the result is rounded to its type
        room, whole = (d // g) * 2.0 ** -24 * part.abs().sum(2), part.sum(2)
        half = torch.finfo(gg.dtype).eps / 2
        off = (gg.double() - whole).abs()
        inside = torch.isfinite(gg) if gt == "f16" else torch.ones_like(gg, dtype=torch.bool)
        assert bool((off <= room + (whole.abs() + room) * half)[inside].all())
        assert bool((whole.abs() + room >= 65504)[~inside].all())
