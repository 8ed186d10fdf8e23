"""Packed sequences: what the documentation of the operators allows and promises at their edges (shapes of gradients, second derivatives, first steps,
tensors changed between the passes, sums beyond 64 bits)."""
import numpy as np
import pytest
import torch

from oracle import recurrence as rec
from test_gpu_scan import d64, inputs, near

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.fail("GPU test collected but no GPU is visible")
    return torch.device("cuda:0")


def test_sums_beyond_64_bits(dev):
    """Lengths whose plain sum leaves 63 bits are cut like any others."""
    from tensoflow_amd import ops
    most, r = 1 << 38, (1 << 25) + 4099
    off = ops.segment_offsets(torch.full((r,), 1 << 62, dtype=torch.int64, device=dev))
    assert int(off[0]) == 0 and bool((off[1:] == most).all())


def test_block_counts_beyond_64_bits(dev):
    import ctypes as C
    from tensoflow_amd import lib as L
    most, r = 1 << 38, (1 << 25) + 4099
    lib, new = L.load(), lambda k, t=torch.int64: torch.full((k,), 5, dtype=t, device=dev)
    lens, off, table, free = new(r).fill_(1 << 62), new(r + 1), new(2 * r, torch.int32), torch.arange(3, dtype=torch.int32, device=dev)
    nw = lib.tf_segment_workspace_words(r, 1)
    work = new(nw)
    L.check(lib.tf_segment_tables(lens.data_ptr(), r, most, off.data_ptr(), None, None, None, 1, free.data_ptr(), 3, 2, table.data_ptr(), None, work.data_ptr(), nw,
                                  C.c_void_p(torch.cuda.current_stream().cuda_stream)), "tf_segment_tables")
    assert int(off[0]) == 0 and bool((off[1:] == most).all()) and table[:4].tolist() == [0, 1, -1, -1] and bool((table[2:] == -1).all())


@pytest.mark.parametrize("flat", [True, False])
def test_heads_with_a_start_state(dev, flat):
    """x [N, H, P] with h0 [R, C] or [R, H, P]: each gradient in its input's shape."""
    from tensoflow_amd import autograd, ops
    ln, h, p = [30, 0, 41], 4, 5
    n = sum(ln)
    gate, x = inputs(n, h * p, h, "f32", "f32", "decay", 3)
    r = torch.Generator().manual_seed(1)
    h0, gy, gf = torch.randn(3, h * p, generator=r), torch.randn(n, h * p, generator=r), torch.randn(3, h * p, generator=r)
    want = rec.scan(d64(gate), d64(x), rec.tables(ln, n)[0], d64(h0), "decay", False, d64(gy), d64(gf))
    leaves = [t.to(dev).requires_grad_() for t in (gate, x.view(n, h, p), h0 if flat else h0.view(3, h, p))]
    tab = ops.segment_tables(torch.tensor(ln, device=dev), n)
    y, final = autograd.gated_scan(leaves[0], leaves[1], tab, leaves[2])
    assert y.shape == (n, h, p) and final.shape == (3, h, p)
    got = torch.autograd.grad((y, final), leaves, (gy.to(dev).view(n, h, p), gf.to(dev).view(3, h, p)))
    for g, leaf, k in zip(got, leaves, ("g_gate", "g_x", "g_h0")):
        assert g.shape == leaf.shape
        near(g, want[k], want[k + "_tol"], k)
    _, _, carry = ops.gated_scan(leaves[0].detach(), leaves[1].detach(), tab, leaves[2].detach(), want_carry=True)
    gh = ops.gated_scan_bwd(leaves[0].detach(), leaves[1].detach(), tab, carry, None, gf.to(dev), leaves[2].detach())[2]
    assert gh.shape == leaves[2].shape
    assert ops.gated_scan_bwd(leaves[0].detach(), leaves[1].detach(), tab, carry, None, gf.to(dev))[2].shape == (3, h, p)


def test_second_derivative_is_refused(dev):
    """A gradient taken with create_graph is the same; what depends on it through the recurrence raises, it is not left out of a sum."""
    from tensoflow_amd import autograd, ops
    tab = ops.segment_tables(torch.tensor([20, 3], device=dev))
    for k in range(3):
        leaves = [torch.rand(23, 2, device=dev), torch.randn(23, 4, device=dev), torch.randn(2, 4, device=dev)]
        leaves[k].requires_grad_()
        y, final = autograd.gated_scan(leaves[0], leaves[1], tab, leaves[2])
        plain, = torch.autograd.grad(y.sum() + final.sum(), leaves[k], retain_graph=True)
        g, = torch.autograd.grad(y.sum() + final.sum(), leaves[k], create_graph=True)
        assert torch.equal(g, plain) and g.requires_grad == (k == 0)
        loss = (g ** 2).sum() + (leaves[k] ** 2).sum()
        if k == 0:
            with pytest.raises(RuntimeError, match="differentiated once"):
                loss.backward()
        else:                                                                         # y is linear in x and h0: that part of the derivative is 0
            loss.backward()
            assert torch.equal(leaves[k].grad, 2 * leaves[k].detach())
    leaves = [torch.rand(23, 2, device=dev, requires_grad=True), torch.randn(23, 4, device=dev, requires_grad=True), torch.randn(2, 4, device=dev, requires_grad=True)]
    y, final = autograd.gated_scan(leaves[0], leaves[1], tab, leaves[2])
    grads = torch.autograd.grad(y.sum() + final.sum(), leaves, create_graph=True)
    for a, b in ((0, 0), (0, 1), (0, 2), (1, 0), (2, 0)):                             # the gate's gradient depends on all three, the others on the gate
        with pytest.raises(RuntimeError, match="differentiated once"):
            torch.autograd.grad(grads[a].sum(), leaves[b], retain_graph=True)
    assert torch.autograd.grad(grads[1].sum() + leaves[1].sum(), leaves[1])[0].eq(1).all()
    weight = torch.rand(23, 4, device=dev, requires_grad=True)                       # a gradient with respect to what comes from behind
    x = torch.randn(23, 4, device=dev, requires_grad=True)
    y, _ = autograd.gated_scan(torch.rand(23, 2, device=dev), x, tab)
    g, = torch.autograd.grad((y * weight).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated once"):
        torch.autograd.grad(g.sum(), weight)
    loss = (autograd.gated_scan(torch.rand(23, 2, device=dev), x, tab)[0]).sum() + (weight ** 3).sum()
    gw, gx = torch.autograd.grad(loss, (weight, x), create_graph=True)                # and where nothing asks for it, nothing is refused
    gw.sum().backward()
    assert torch.allclose(weight.grad, 6 * weight) and gx.shape == x.shape


def test_changes_between_the_passes_are_seen(dev):
    """A pool stepped in place, an `out` and the tables count as changed: a backward pass that needs what they held raises."""
    from tensoflow_amd import autograd, ops
    changed = "modified by an inplace operation"
    lens = torch.tensor([20, 3], device=dev)
    gate, x, pool = torch.rand(23, 2, device=dev), torch.randn(23, 4, device=dev), torch.randn(2, 4, device=dev)

    def forward():
        tab = ops.segment_tables(lens)
        leaf, data = gate.clone().requires_grad_(), x.clone()
        return tab, leaf, data, autograd.gated_scan(leaf, data, tab, pool)[0].sum()
    tab, leaf, data, loss = forward()
    torch.autograd.grad(loss, leaf)
    _, leaf, _, loss = forward()
    ops.gated_step(pool, torch.tensor([1], device=dev), gate[:1], x[:1])
    with pytest.raises(RuntimeError, match=changed):
        torch.autograd.grad(loss, leaf)
    tab, leaf, data, loss = forward()
    ops.gated_scan(gate, x, tab, out=data)
    with pytest.raises(RuntimeError, match=changed):
        torch.autograd.grad(loss, leaf)
    _, leaf, data, loss = forward()
    ops.gated_step(pool.clone(), torch.tensor([1], device=dev), gate[:1], x[:1], out=data[2:3])
    with pytest.raises(RuntimeError, match=changed):
        torch.autograd.grad(loss, leaf)
    for name in ("offsets", "index", "starts"):
        tab, leaf, _, loss = forward()
        getattr(tab, name).add_(0)
        with pytest.raises(RuntimeError, match=changed):
            torch.autograd.grad(loss, leaf)
    data = x.clone().requires_grad_()                                                 # x's gradient does not depend on the start state
    want, = torch.autograd.grad(autograd.gated_scan(gate, data, tab, pool)[0].sum(), data)
    loss = autograd.gated_scan(gate, data, tab, pool)[0].sum()
    ops.gated_step(pool, torch.tensor([1], device=dev), gate[:1], x[:1])
    assert torch.equal(torch.autograd.grad(loss, data)[0], want)
    with torch.inference_mode():                                                      # tensors without a count of their changes
        state = torch.zeros(2, 4, device=dev)
        ops.gated_step(state, torch.tensor([1, 0], device=dev), gate[:2], x[:2])
        ops.gated_scan(gate, x, ops.segment_tables(lens), out=torch.empty(23, 4, device=dev))


@pytest.mark.parametrize("t,gt", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("d,g", [(4, 1), (10, 1), (12, 12), (40, 40), (40, 10), (256, 2), (260, 260)])
def test_first_steps_without_a_start_state(dev, d, g, t, gt):
    """No h0 is an h0 of zeros, also where a first row's decay is infinite or NaN: a 0 + b in every kernel and in both passes."""
    from tensoflow_amd import ops
    ln = [20, 30, 41, 9]
    n = sum(ln)
    for form in ("decay", "log"):
        for reverse in (False, True):
            gate, x = inputs(n, d, g, t, gt, form, d)
            gy = torch.randn(n, d, generator=torch.Generator().manual_seed(2)).to(x.dtype)
            first = [19, 49, 90, 99] if reverse else [0, 20, 50, 91]
            gate[first[1]], gate[first[2]] = float("inf"), float("nan")
            off = rec.tables(ln, n)[0]
            with np.errstate(invalid="ignore"):
                want = rec.scan(d64(gate), d64(x), off, None, form, reverse, d64(gy), None)
            tab = ops.segment_tables(torch.tensor(ln, device=dev), n)
            res = []
            for h0 in (None, torch.zeros(4, d, device=dev)):
                y, final, carry = ops.gated_scan(gate.to(dev), x.to(dev), tab, h0, form, reverse, want_final=True, want_carry=True)
                res.append((y, final, *ops.gated_scan_bwd(gate.to(dev), x.to(dev), tab, carry, gy.to(dev), None, h0, form, reverse)))
            for a, b, k in zip(*res, ("y", "final", "g_gate", "g_x", "g_h0")):
                assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0.0), b.nan_to_num(0.0)), k
                fine = np.isfinite(want[k])
                assert np.array_equal(a.isfinite().cpu().numpy(), fine), (k, form, reverse)
                near(a[torch.from_numpy(fine).to(dev)], want[k][fine], want[k + "_tol"][fine], k)
