"""The sequence operators from their formulas, in 64 bits on the CPU, with bounds on what 32-bit arithmetic and one rounding of
each result may be off.  numpy in, numpy out; written apart from the kernels.

A result stored with a step of `eps` relative to its value is off by at most eps / 2 of it; everything before that is held in
32 bits or more, with a relative error of U = 2^-24 per operation.  The bounds count operations, each a little generously."""
import numpy as np
import torch

U = 2.0 ** -24
HALF_STEP = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# below the smallest normal number steps no longer shrink with the value
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def f64(t):
    return None if t is None else t.detach().cpu().double().numpy()


def check(what, got, ref, dtype, slack):
    """|got - ref| <= half a step of ref + slack, elementwise; infinities and NaN in the same places."""
    got = f64(got)
    assert got.shape == ref.shape, f"{what}: shape {got.shape}, expected {ref.shape}"
    if not ref.size:
        return
    fine = np.isfinite(ref)
    assert np.array_equal(fine, np.isfinite(got)), f"{what}: infinities or NaN in other places"
    bound = HALF_STEP[dtype] * np.abs(np.where(fine, ref, 0)) + TINY[dtype] + np.broadcast_to(slack, ref.shape)
    err = np.where(fine, np.abs(np.where(fine, got, 0) - np.where(fine, ref, 0)), 0)
    worst = np.unravel_index(np.argmax(err - bound), err.shape)
    assert (err <= bound).all(), (f"{what}{worst}: {got[worst]!r}, expected {ref[worst]!r}: off by {err[worst]:.3g}, allowed {bound[worst]:.3g}; "
                                  f"{np.mean(err > bound):.3g} of the values are outside")


def logistic(g):
    t = np.exp(-np.abs(g))
    big = 1 / (1 + t)
    return np.where(g < 0, t * big, big), np.where(g < 0, big, t * big)


def ranges(rows, sequences, steps=None, offsets=None, lengths=None):
    if offsets is not None:
        return [(int(offsets[s]), int(offsets[s + 1])) for s in range(sequences)]
    return [(s * steps, s * steps + (int(lengths[s]) if lengths is not None else steps)) for s in range(sequences)]


def recurrence(x, g, form, spans, initial=None, dy=None, dlast=None):
    """x [rows, channels], g of x's shape or [channels] -> dict; with dy / dlast the gradients as well.  Entries ending in
    _slack: what 32-bit arithmetic may be off."""
    rows, c = x.shape
    n = len(spans)
    one = g.ndim == 1
    a, k = logistic(g) if form == "gate" else (g, np.ones_like(g))
    dk = a * k if form == "gate" else None
    y, before, lam = (np.zeros((rows, c)) for _ in range(3))
    dx, dg = np.zeros((rows, c)), np.zeros((rows, c))
    state, dinitial = np.zeros((n, c)), np.zeros((n, c))
    for s, (b, e) in enumerate(spans):
        h = np.zeros(c) if initial is None else initial[s].copy()
        for t in range(b, e):
            at, kt = (a, k) if one else (a[t], k[t])
            before[t] = h
            h = at * h + kt * x[t]
            y[t] = h
        state[s] = h
        if dy is not None or dlast is not None:
            m = np.zeros(c) if dlast is None else dlast[s].copy()
            for t in range(e - 1, b - 1, -1):
                at, kt = (a, k) if one else (a[t], k[t])
                lam[t] = m + (0 if dy is None else dy[t])
                dx[t] = kt * lam[t]
                dg[t] = lam[t] * (before[t] - x[t]) * (dk if one else dk[t]) if form == "gate" else lam[t] * before[t]
                m = at * lam[t]
            dinitial[s] = m
    live = np.zeros(rows, bool)
    for b, e in spans:
        live[b:e] = True
    a_live = np.abs(a if one else a[live])
    longest = max([e - b for b, e in spans], default=0)
    keep = a_live.max() if a_live.size else 0.0
    # an error made at a step stays for about 1 / (1 - |a|) steps (all of them where |a| >= 1): that many can add up
    memory = min(longest, 1 / max(1 - keep, 1e-9)) + 1
    top = lambda *v: max([np.abs(t[np.isfinite(t)]).max() if t is not None and np.isfinite(t).any() else 0.0 for t in v])  # noqa: E731
    h_top = top(y, before, None if initial is None else initial, x[live] if form == "gate" else None)
    l_top = top(lam)
    ops = 12   # of a step: the logistic function (6, one of them exp with two), the update, the composition of pieces
    h_slack, l_slack = ops * memory * U * h_top, ops * memory * U * l_top
    out = {"y": y, "state": state, "y_slack": h_slack, "state_slack": h_slack}
    if dy is not None or dlast is not None:
        reach = top(before - x if form == "gate" else before) * (0.25 if form == "gate" else 1.0)
        g_slack = l_slack * reach + h_slack * l_top * (2 if form == "gate" else 1) + ops * U * np.abs(dg)
        out.update(dx=dx, dinitial=dinitial, dx_slack=l_slack + ops * U * np.abs(dx), dinitial_slack=l_slack)
        if one:
            out.update(dg=dg.sum(0), dg_slack=g_slack.sum(0) + rows * U * np.abs(dg).sum(0))
        else:
            out.update(dg=dg, dg_slack=g_slack)
    return out


def block_norm(x, gate=None, residual=None, post=None, scale=None, pre=None, eps=1e-6, dh=None, dn=None):
    rows, c = x.shape
    one = np.ones(c)
    rs1 = 1 / np.sqrt((x * x).mean(1, keepdims=True) + eps) if post is not None else np.ones((rows, 1))
    w1 = one if post is None else post
    xh = x * rs1
    u = xh * w1
    f, k = logistic(gate) if gate is not None else (None, None)
    silu, dsilu = (gate * f, f * (1 + gate * k)) if gate is not None else (np.ones_like(x), None)
    v = u * silu
    sc = one if scale is None else scale
    h = v * sc + (0 if residual is None else residual)
    # a sum of c squares by 64 lanes or more at a time, then a tree; its root's relative error is half of that
    ops = 24 + c / 64
    h_abs = np.abs(v * sc) + (0 if residual is None else np.abs(residual))
    out = {"h": h, "h_slack": ops * U * h_abs}
    rs2 = None
    if pre is not None:
        rs2 = 1 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
        hh = h * rs2
        # an error of h goes into its own norm as well
        rel = (h_abs * h_abs).mean(1, keepdims=True) * rs2 * rs2
        out.update(n=hh * pre, n_slack=ops * U * np.abs(pre) * rs2 * h_abs * (2 + rel))
    if dh is None and dn is None:
        return out
    d = np.zeros_like(x) if dh is None else dh
    d_abs = np.abs(d)
    if pre is not None and dn is not None:
        q = dn * pre
        mean = (q * hh).mean(1, keepdims=True)
        d = d + rs2 * (q - hh * mean)
        ah = h_abs * rs2
        d_abs = d_abs + rs2 * (np.abs(q) + ah * (np.abs(q) * ah).mean(1, keepdims=True)) * (2 + rel)
        out.update(dpre=(dn * hh).sum(0), dpre_slack=(ops + rows / 64) * U * (np.abs(dn) * ah * (2 + rel)).sum(0))
    elif pre is not None:
        out.update(dpre=np.zeros(c), dpre_slack=0.0)
    ops *= 2
    dv = d * sc
    du = dv * silu
    out.update(dresidual=d, dresidual_slack=ops * U * d_abs,
               dscale=(d * v).sum(0), dscale_slack=(ops + rows / 64) * U * (d_abs * np.abs(v)).sum(0))
    if gate is not None:
        out.update(dgate=dv * u * dsilu, dgate_slack=ops * U * d_abs * np.abs(sc * u) * (np.abs(f) * (1 + np.abs(gate) * k)))
    if post is not None:
        p = du * w1
        out["dx"] = rs1 * (p - xh * (p * xh).mean(1, keepdims=True))
        p_abs = d_abs * np.abs(sc * silu * w1)
        out["dx_slack"] = ops * U * rs1 * (p_abs + np.abs(xh) * (p_abs * np.abs(xh)).mean(1, keepdims=True)) * 2
        out.update(dpost=(du * xh).sum(0), dpost_slack=(ops + rows / 64) * U * (d_abs * np.abs(sc * silu * xh)).sum(0))
    else:
        out["dx"], out["dx_slack"] = du, ops * U * d_abs * np.abs(sc * silu)
    return out


def embedding(ids, table, scale=1.0, padding=None, dout=None):
    vocab, c = table.shape
    flat = ids.reshape(-1)
    inside = (flat >= 0) & (flat < vocab)
    e = np.where(inside[:, None], table[np.where(inside, flat, 0)], 0) * scale
    out = {"e": e.reshape(*ids.shape, c), "e_slack": 2 * U * np.abs(e).reshape(*ids.shape, c)}
    if dout is not None:
        d = dout.reshape(-1, c)
        take = inside if padding is None else inside & (flat != padding)
        sums, mags, count = np.zeros((vocab, c)), np.zeros((vocab, c)), np.zeros(vocab)
        np.add.at(sums, flat[take], d[take])
        np.add.at(mags, flat[take], np.abs(d[take]))
        np.add.at(count, flat[take], 1)
        out.update(dtable=sums * scale, dtable_slack=(count[:, None] + 2) * U * mags * abs(scale))
    return out
