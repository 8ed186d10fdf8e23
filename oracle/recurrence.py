"""Packed sequences in 64 bits, step by step: segment tables, the gated linear recurrence with its gradients, its one-token form, and worst-case
bounds of an fp32 evaluation of it (the oracle of tf_segment_tables, tf_gated_scan_* and tf_gated_step)."""
import numpy as np


def tables(lengths, n_rows, block_rows=0, free_blocks=None, max_blocks=0):
    """offsets, index, position, start bits [, block_table, slots] row by row."""
    lengths = [min(max(int(n), 0), n_rows) for n in lengths]
    offsets, index, position = [0], np.full(n_rows, -1, np.int64), np.full(n_rows, -1, np.int64)
    table, slots, taken = np.full((len(lengths), max_blocks), -1, np.int32), np.full(n_rows, -1, np.int64), 0
    for s, n in enumerate(lengths):
        lo, hi = offsets[-1], min(offsets[-1] + n, n_rows)
        offsets.append(hi)
        index[lo:hi], position[lo:hi] = s, np.arange(hi - lo)
        if block_rows:
            for c in range(-(-n // block_rows)):
                if c < max_blocks and taken < len(free_blocks):
                    table[s, c] = free_blocks[taken]
                taken += 1
            for i in range(lo, hi):
                c = (i - lo) // block_rows
                if c < max_blocks and table[s, c] >= 0:
                    slots[i] = int(table[s, c]) * block_rows + (i - lo) % block_rows
    bits = np.zeros((n_rows + 63) // 64, np.uint64)
    for i in np.nonzero(position == 0)[0].tolist():
        bits[i // 64] |= np.uint64(1) << np.uint64(i % 64)
    out = (np.array(offsets, np.int64), index, position, bits)
    return out + ((table, slots) if block_rows else ())


def _terms(gate, x, form):
    g = np.repeat(gate, x.shape[1] // gate.shape[1], axis=1)
    a = {"decay": lambda: g, "log": lambda: np.exp(g), "alpha": lambda: 1.0 - g}[form]()
    return g, a, (g * x if form == "alpha" else x)


def scan(gate, x, offsets, h0=None, form="decay", reverse=False, gy=None, g_final=None):
    """gate [N, G], x [N, D], h0 [R, D] float64 -> dict: y, final, and with gy / g_final also g_gate, g_x, g_h0.  Every entry k has `k_tol`: how far an
    fp32 evaluation in any order of the additions may be from it before the result is rounded to its type.  A contribution that came d steps ago
    has been through at most 2 d + 64 roundings (a product and a sum for each step; 64: within and across the pieces that a parallel scan
    joins) of half a step each, exp(g) another 2 for each step and 2 |g| (the argument's own rounding)."""
    u = 2.0 ** -24
    N, D = x.shape
    R = len(offsets) - 1
    g, a, b = _terms(gate, x, form)
    per = np.full_like(a, 2.0) if form != "log" else 4.0 + 2.0 * np.abs(g)
    per = per + (1.0 if form == "alpha" else 0.0)                                          # 1 - g is rounded too
    out = {k: np.zeros((N, D)) for k in ("y", "y_tol", "before", "before_tol", "lam", "lam_tol")}
    out["final"], out["final_tol"] = np.zeros((R, D)), np.zeros((R, D))
    out["g_h0"], out["g_h0_tol"] = np.zeros((R, D)), np.zeros((R, D))
    for s in range(R):
        rows = range(offsets[s], offsets[s + 1])
        rows = rows[::-1] if reverse else rows
        h = h0[s].copy() if h0 is not None else np.zeros(D)
        m, w = np.abs(h), np.zeros(D)                          # sum of |contributions|, and of |contributions| x roundings that came with the steps
        for i in rows:
            out["before"][i], out["before_tol"][i] = h, u * (w + 64 * m)
            h = a[i] * h + b[i]
            w = np.abs(a[i]) * (w + per[i] * m)
            m = np.abs(a[i]) * m + np.abs(b[i])
            out["y"][i], out["y_tol"][i] = h, u * (w + 64 * m)
        out["final"][s], out["final_tol"][s] = h, u * (w + 64 * m) if len(rows) else 0.0
        if gy is None and g_final is None:
            continue
        l = g_final[s].copy() if g_final is not None else np.zeros(D)
        m, w = np.abs(l), np.zeros(D)
        for i in rows[::-1]:
            if gy is not None:
                l = l + gy[i]
                m = m + np.abs(gy[i])
            out["lam"][i], out["lam_tol"][i] = l, u * (w + 64 * m)
            l = a[i] * l
            w = np.abs(a[i]) * (w + per[i] * m)
            m = np.abs(a[i]) * m
        out["g_h0"][s], out["g_h0_tol"][s] = l, u * (w + 64 * m) if len(rows) else 0.0
    if gy is None and g_final is None:
        return out
    lam, lt, hb, ht = out["lam"], out["lam_tol"], out["before"], out["before_tol"]
    if form == "alpha":
        out["g_x"], out["g_x_tol"] = g * lam, np.abs(g) * (lt + 2 * u * np.abs(lam))
        part, left = lam * (x - hb), np.abs(x - hb)
        tol = left * lt + (np.abs(lam) + lt) * (ht + u * (np.abs(x) + np.abs(hb)))
    else:
        out["g_x"], out["g_x_tol"] = lam, lt
        scale = np.abs(a) if form == "log" else 1.0
        part = lam * hb * (a if form == "log" else 1.0)
        tol = scale * (np.abs(hb) * lt + (np.abs(lam) + lt) * ht) + (np.abs(part) * u * (4 + 2 * np.abs(g)) if form == "log" else 0.0)
    P = D // gate.shape[1]
    fold = lambda v: v.reshape(N, gate.shape[1], P).sum(-1)
    out["g_gate"] = fold(part)
    out["g_gate_tol"] = fold(tol) + u * (P + 4) * fold(np.abs(part))                        # the sum over the head, in any order
    return out


def step(state, slots, gate, x, form="decay"):
    """-> (y, state afterwards, written rows): row after row, as they stand."""
    state = state.copy()
    _, a, b = _terms(gate, x, form)
    y, written = np.zeros_like(x), np.zeros(len(slots), bool)
    for r, s in enumerate(np.asarray(slots).tolist()):
        if 0 <= s < len(state):
            state[s] = a[r] * state[s] + b[r]
            y[r], written[r] = state[s], True
    return y, state, written
