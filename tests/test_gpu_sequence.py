"""The sequence operators (dali_amd.sequence) on the device against their formulas in 64 bits (tests/sequence_reference.py, whose
bounds count the roundings), at the sizes, lengths, types and layouts where they can go wrong."""
import os

import numpy as np
import pytest
import torch

from dali_amd import sequence
from tests import sequence_reference as R

pytestmark = pytest.mark.gpu

if os.environ.get("DALI_AMD_HIPEMU"):   # the kernels on the CPU model: its "device" tensors are torch's CPU tensors
    sequence._HOST_MEMORY = True

BF, HF, F = torch.bfloat16, torch.float16, torch.float32


def rand(seed, *shape, dtype=F, scale=1.0, shift=0.0):
    v = np.random.default_rng(seed).normal(shift, scale, shape)
    return torch.from_numpy(v).to(dtype).cuda()


def leaf(t):
    return None if t is None else t.detach().requires_grad_(True)


# ------------------------------------------------------------------ linear recurrence
def run_recurrence(x, g, form, spans, initial, train, **kw):
    """One call with checks of everything it returns; (y, state, gradients)."""
    rows, c = x.numel() // x.shape[-1], x.shape[-1]
    if not train:
        y, state = sequence.linear_recurrence(x, g, form=form, initial_state=initial, **kw)
        grads, dy, dlast = {}, None, None
    else:
        leaves = [leaf(x), leaf(g), leaf(initial)]
        # leaves keep their own strides: views of a wider tensor are passed as such
        y, state = sequence.linear_recurrence(leaves[0], leaves[1], form=form, initial_state=leaves[2], **kw)
        dy, dlast = rand(91, *y.shape, dtype=y.dtype), rand(92, *state.shape)
        names = [n for n, t in zip(("dx", "dg", "dinitial"), leaves) if t is not None]
        got = torch.autograd.grad((y, state), [t for t in leaves if t is not None], (dy, dlast))
        grads = dict(zip(names, got))
    flat = lambda t: None if t is None else R.f64(t).reshape(rows, c)  # noqa: E731
    ref = R.recurrence(flat(x), R.f64(g) if g.dim() == 1 else flat(g), form, spans, R.f64(initial),
                       flat(dy), R.f64(dlast))
    assert y.dtype == x.dtype and state.dtype == F and y.shape == x.shape
    R.check("y", y.reshape(rows, c), ref["y"], x.dtype, ref["y_slack"])
    R.check("state", state, ref["state"], F, ref["state_slack"])
    for n, t in grads.items():
        want = {"dx": x, "dg": g, "dinitial": initial}[n]
        assert t.dtype == want.dtype and t.shape == want.shape
        R.check(n, t.reshape(ref[n].shape), ref[n], t.dtype, ref[n + "_slack"])
    return y, state, grads


def decays(seed, form, *shape, dtype=F):
    g = rand(seed, *shape, scale=1.5, shift=2.0)
    return (g if form == "gate" else torch.sigmoid(g.clamp(max=4.0))).to(dtype)


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("form", ["decay", "gate"])
@pytest.mark.parametrize("dtype,gdtype", [(F, F), (BF, BF), (BF, F), (HF, HF), (HF, F)])
@pytest.mark.parametrize("batch,steps,channels", [(2, 300, 64), (3, 1, 40), (1, 513, 24), (5, 7, 33), (2, 256, 8)])
def test_recurrence_dense(batch, steps, channels, dtype, gdtype, form, train):
    x = rand(1, batch, steps, channels, dtype=dtype)
    g = decays(2, form, batch, steps, channels, dtype=gdtype)
    h0 = rand(3, batch, channels)
    spans = R.ranges(batch * steps, batch, steps)
    run_recurrence(x, g, form, spans, h0, train)


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("lens,head,tail", [([5, 0, 1, 300, 2, 0, 0, 259, 1, 1, 64], 0, 0), ([1], 0, 0), ([0], 0, 3), ([0, 0], 0, 0), ([40, 8], 3, 17),
                                            ([1] * 70, 0, 0), ([255, 257, 256, 511], 1, 0), ([9, 0, 700, 0], 0, 300)])
@pytest.mark.parametrize("dtype,channels", [(BF, 72), (F, 37)])
def test_recurrence_packed(dtype, channels, lens, head, tail, index, train):
    """Sequences of every length, empty ones among them, and rows of none in front and behind, which hold NaN and infinities."""
    offsets = torch.from_numpy(np.cumsum([head] + lens)).to(index).cuda()
    rows = head + sum(lens) + tail
    x, g = rand(4, rows, channels, dtype=dtype), decays(5, "gate", rows, channels, dtype=dtype)
    for t in (x, g):
        t[:head], t[rows - tail:] = float("nan"), float("inf")
    h0 = rand(6, len(lens), channels)
    spans = R.ranges(rows, len(lens), offsets=offsets.cpu().tolist())
    run_recurrence(x, g, "gate", spans, h0, train, offsets=offsets)


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_recurrence_padded_batch(index, train):
    """lengths: what the padding holds is used by nothing."""
    lengths = torch.tensor([17, 0, 330, 1, 329], dtype=index).cuda()
    x, g = rand(7, 5, 330, 48, dtype=HF), decays(8, "decay", 5, 330, 48, dtype=HF)
    for b, n in enumerate(lengths.cpu().tolist()):
        x[b, n:], g[b, n:] = float("nan"), float("inf")
    spans = R.ranges(5 * 330, 5, 330, lengths=lengths.cpu().tolist())
    run_recurrence(x, g, "decay", spans, rand(9, 5, 48), train, lengths=lengths)


@pytest.mark.parametrize("form", ["decay", "gate"])
@pytest.mark.parametrize("dtype,channels", [(F, 80), (BF, 31), (HF, 136)])
@pytest.mark.parametrize("packed", [False, True])
def test_recurrence_decay_per_channel(packed, dtype, channels, form):
    """The same decay at every step: its gradient is a sum over all rows."""
    g = decays(10, form, channels)
    if packed:
        lens = [300, 0, 41, 1, 600]
        offsets = torch.from_numpy(np.cumsum([0] + lens)).int().cuda()
        spans = R.ranges(942, 5, offsets=offsets.cpu().tolist())
        run_recurrence(rand(11, 942, channels, dtype=dtype), g, form, spans, None, True, offsets=offsets)
    else:
        run_recurrence(rand(11, 3, 270, channels, dtype=dtype), g.to(dtype), form, R.ranges(810, 3, 270), rand(12, 3, channels), True)


@pytest.mark.parametrize("logit", [9.0, 14.0, 30.0, -30.0])
def test_recurrence_gates_near_their_ends(logit):
    """A gate that holds for thousands of steps moves by 1 - f per step: that difference has to keep its digits.  A constant input
    and constant gates, where errors of one sign would add up."""
    x, g = torch.full((1, 3000, 16), 0.75).cuda(), torch.full((1, 3000, 16), logit).cuda()
    run_recurrence(x, g, "gate", [(0, 3000)], None, True)
    run_recurrence(x, g[0, 0].contiguous(), "gate", [(0, 3000)], None, True)


def test_recurrence_long_and_split():
    """A long sequence with few channels, and several that begin and end inside the pieces it would be cut into."""
    x, g = rand(13, 1, 20011, 16), decays(14, "gate", 1, 20011, 16)
    run_recurrence(x, g, "gate", [(0, 20011)], rand(15, 1, 16), True)
    lens = [9000, 1, 0, 7001, 513, 3]
    offsets = torch.from_numpy(np.cumsum([0] + lens)).cuda()
    run_recurrence(rand(16, sum(lens), 16, dtype=BF), decays(17, "decay", sum(lens), 16), "decay", R.ranges(0, 6, offsets=offsets.cpu().tolist()),
                   rand(18, 6, 16), True, offsets=offsets)


def test_recurrence_infinities_stay_in_their_sequence_and_channel():
    lens = [100, 300, 5]
    offsets = torch.from_numpy(np.cumsum([0] + lens)).int().cuda()
    x, g = rand(19, 405, 24), decays(20, "decay", 405, 24)
    x[50, 3], x[120, 5] = float("inf"), float("nan")
    y, state = sequence.linear_recurrence(x, g, offsets=offsets)
    bad = ~torch.isfinite(y.cpu())
    want = torch.zeros(405, 24, dtype=torch.bool)
    want[50:100, 3] = True
    want[120:400, 5] = True
    assert torch.equal(bad, want)
    assert torch.equal(~torch.isfinite(state.cpu()), torch.stack([want[99], want[399], want[404]]))


@pytest.mark.parametrize("dtype,shift", [(BF, 0), (BF, 1), (F, 0), (F, 3)])
def test_recurrence_strided_views(dtype, shift):
    """x and decay as slices of one wide projection, gradients as slices of something wider, aligned and not."""
    wide = rand(21, 3, 290, 2 * 56 + 9, dtype=dtype)
    x, g = wide[..., shift:shift + 56], wide[..., shift + 56:shift + 112]
    spans = R.ranges(3 * 290, 3, 290)
    y, state, _ = run_recurrence(x, g, "gate", spans, None, False)
    a, b = leaf(x), leaf(g)
    assert a.stride() == x.stride()
    z, s = sequence.linear_recurrence(a, b, form="gate")
    dy = rand(22, 3, 290, 56 + 9, dtype=dtype)[..., shift:shift + 56]
    dx, dg = torch.autograd.grad(z, (a, b), dy)
    ref = R.recurrence(R.f64(x).reshape(-1, 56), R.f64(g).reshape(-1, 56), "gate", spans, None, R.f64(dy).reshape(-1, 56))
    R.check("dx", dx.reshape(-1, 56), ref["dx"], dtype, ref["dx_slack"])
    R.check("dg", dg.reshape(-1, 56), ref["dg"], dtype, ref["dg_slack"])
    assert torch.equal(z, y) and torch.equal(s, state)
    # time and batch exchanged, channels apart: a view, and a copy
    swapped = x.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(sequence.linear_recurrence(swapped, g, form="gate")[0], y)
    apart = x.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(sequence.linear_recurrence(apart, g, form="gate")[0], y)


def test_recurrence_gradients_of_one_output_or_input():
    x, g, h0 = rand(23, 2, 70, 40), decays(24, "gate", 2, 70, 40), rand(25, 2, 40)
    spans = R.ranges(140, 2, 70)
    for use in ("y", "state"):
        a, b, c = leaf(x), leaf(g), leaf(h0)
        y, state = sequence.linear_recurrence(a, b, form="gate", initial_state=c)
        dy, dl = (rand(26, 2, 70, 40), None) if use == "y" else (None, rand(27, 2, 40))
        got = torch.autograd.grad(y if use == "y" else state, (a, b, c), dy if use == "y" else dl)
        ref = R.recurrence(R.f64(x).reshape(140, 40), R.f64(g).reshape(140, 40), "gate", spans, R.f64(h0),
                           None if dy is None else R.f64(dy).reshape(140, 40), R.f64(dl))
        for n, t in zip(("dx", "dg", "dinitial"), got):
            R.check(n, t.reshape(ref[n].shape), ref[n], F, ref[n + "_slack"])
    a = leaf(g)
    y, _ = sequence.linear_recurrence(x, a, form="gate")
    y.sum().backward()          # an expanded gradient: every stride of it is zero
    ref = R.recurrence(R.f64(x).reshape(140, 40), R.f64(g).reshape(140, 40), "gate", spans, None, np.ones((140, 40)))
    R.check("dg", a.grad.reshape(140, 40), ref["dg"], F, ref["dg_slack"])


@pytest.mark.parametrize("form", ["decay", "gate"])
def test_recurrence_gradient_against_differences(form):
    """Along a random direction, from the formula's values at two near points in 64 bits."""
    x, g, h0 = rand(28, 1, 90, 16), decays(29, form, 1, 90, 16), rand(30, 1, 16)
    dy, dl = rand(31, 1, 90, 16), rand(32, 1, 16)
    a, b, c = leaf(x), leaf(g), leaf(h0)
    y, state = sequence.linear_recurrence(a, b, form=form, initial_state=c)
    got = [R.f64(t) for t in torch.autograd.grad((y, state), (a, b, c), (dy, dl))]
    rng = np.random.default_rng(33)
    at = [R.f64(t) for t in (x, g, h0)]
    way = [rng.normal(size=v.shape) for v in at]

    def value(step):
        p = [v + step * d for v, d in zip(at, way)]
        ref = R.recurrence(p[0][0], p[1][0], form, [(0, 90)], p[2])
        return float((ref["y"] * R.f64(dy)[0]).sum() + (ref["state"] * R.f64(dl)).sum())
    slope = (value(1e-5) - value(-1e-5)) / 2e-5
    along = sum(float((u * d).sum()) for u, d in zip(got, way))
    # the difference's own error is of the order of 1e-10 of the terms, the gradient's of 2^-24 of each of 3000 terms
    size = sum(float(np.abs(u * d).sum()) for u, d in zip(got, way))
    assert abs(slope - along) <= 64 * R.U * size, (slope, along)


@pytest.mark.parametrize("dtype", [BF, F])
def test_recurrence_state_in_place_step_by_step(dtype):
    """One token at a time with the state updated in place gives what one call gives, up to rounding."""
    x, g = rand(34, 6, 20, 72, dtype=dtype), decays(35, "gate", 6, 20, 72, dtype=dtype)
    state = torch.zeros(6, 72).cuda()
    steps = []
    for t in range(20):
        y, s = sequence.linear_recurrence(x[:, t:t + 1], g[:, t:t + 1], form="gate", initial_state=state, final_state=state)
        assert s is state
        steps.append(y)
    ref = R.recurrence(R.f64(x).reshape(120, 72), R.f64(g).reshape(120, 72), "gate", R.ranges(120, 6, 20))
    R.check("y", torch.cat(steps, 1).reshape(120, 72), ref["y"], dtype, ref["y_slack"])
    R.check("state", state, ref["state"], F, ref["state_slack"])
    # in place over many steps as well, and split in two calls
    half = torch.zeros(6, 72).cuda()
    for lo, hi in ((0, 13), (13, 20)):
        sequence.linear_recurrence(x[:, lo:hi], g[:, lo:hi], form="gate", initial_state=half, final_state=half)
    R.check("state", half, ref["state"], F, ref["state_slack"])


@pytest.mark.parametrize("lens", [[40, 1, 300, 0, 7, 90], [2000, 3, 700]])
def test_recurrence_state_in_place_packed(lens):
    """The final states are written over the initial ones, of sequences that share a tile of rows and that span several."""
    offsets = torch.from_numpy(np.cumsum([0] + lens)).int().cuda()
    x, g = rand(42, sum(lens), 64, dtype=BF), decays(43, "gate", sum(lens), 64, dtype=BF)
    state = rand(44, len(lens), 64)
    spans = R.ranges(0, len(lens), offsets=offsets.cpu().tolist())
    ref = R.recurrence(R.f64(x), R.f64(g), "gate", spans, R.f64(state))
    y, s = sequence.linear_recurrence(x, g, form="gate", initial_state=state, offsets=offsets, final_state=state)
    assert s is state
    R.check("y", y, ref["y"], BF, ref["y_slack"])
    R.check("state", state, ref["state"], F, ref["state_slack"])


def test_recurrence_offsets_out_of_range_are_clamped():
    """Nothing outside the tensors is read or written, whatever the offsets say: rows behind stay as they were."""
    big = rand(36, 64 + 300, 40)
    x = big[:300]
    before = big[300:].clone()
    offsets = torch.tensor([-5, 100, 100, 1 << 40, 1 << 41]).cuda()
    y, state = sequence.linear_recurrence(x, decays(37, "decay", 300, 40), offsets=offsets)
    ref = R.recurrence(R.f64(x), R.f64(decays(37, "decay", 300, 40)), "decay", [(0, 100), (100, 100), (100, 300), (300, 300)])
    R.check("y", y, ref["y"], F, ref["y_slack"])
    R.check("state", state, ref["state"], F, ref["state_slack"])
    assert torch.equal(big[300:], before)


def test_recurrence_same_inputs_same_bits():
    x, g = rand(38, 4, 700, 80, dtype=BF), decays(39, "gate", 80)
    runs = []
    for _ in range(2):
        a, b = leaf(x), leaf(g)
        y, s = sequence.linear_recurrence(a, b, form="gate")
        runs.append([y, s, *torch.autograd.grad((y, s), (a, b), (x, s.detach()))])
    assert all(torch.equal(u, v) for u, v in zip(*runs))


# ------------------------------------------------------------------ norms around a block
PARTS = ["post", "gate", "residual", "scale", "pre"]
COMBINATIONS = [PARTS, ["pre"], ["post"], ["post", "gate"], ["residual", "pre"], ["residual", "scale"], ["gate"], ["post", "residual", "scale", "pre"],
                ["gate", "residual", "pre"], []]


def norm_inputs(parts, rows, c, dtype, rdtype, wdtype, seed=40):
    t = {"x": rand(seed, rows, c, dtype=dtype, scale=1.7), "gate": rand(seed + 1, rows, c, dtype=dtype, scale=2.0),
         "residual": rand(seed + 2, rows, c, dtype=rdtype, scale=2.0), "post": rand(seed + 3, c, dtype=wdtype, scale=0.3, shift=1.0),
         "scale": rand(seed + 4, c, dtype=wdtype, scale=0.5), "pre": rand(seed + 5, c, dtype=wdtype, scale=0.3, shift=1.0)}
    return {k: v if k == "x" or k in parts else None for k, v in t.items()}


def call_norm(t, **kw):
    return sequence.block_norm(t["x"], gate=t["gate"], residual=t["residual"], post_weight=t["post"], scale=t["scale"], pre_weight=t["pre"], **kw)


def run_norm(t, eps=1e-6, train=True, use=("h", "n")):
    shape, c = t["x"].shape, t["x"].shape[-1]
    t = {k: leaf(v) if train else v for k, v in t.items()}
    h, n = call_norm(t, eps=eps)
    hdtype = t["x"].dtype if t["residual"] is None else t["residual"].dtype
    assert h.dtype == hdtype and h.shape == shape and (n is None) == (t["pre"] is None)
    dh = rand(50, *shape, dtype=hdtype) if train and "h" in use else None
    dn = rand(51, *shape, dtype=t["x"].dtype) if train and "n" in use and n is not None else None
    f = {k: R.f64(v) if v is None or v.dim() == 1 else R.f64(v).reshape(-1, c) for k, v in t.items()}
    flat = lambda v: None if v is None else R.f64(v).reshape(-1, c)  # noqa: E731
    ref = R.block_norm(f["x"], f["gate"], f["residual"], f["post"], f["scale"], f["pre"], eps, flat(dh), flat(dn))
    R.check("hidden", h.reshape(-1, c), ref["h"], hdtype, ref["h_slack"])
    if n is not None:
        assert n.dtype == t["x"].dtype and n.shape == shape
        R.check("normed", n.reshape(-1, c), ref["n"], n.dtype, ref["n_slack"])
    if train and (dh is not None or dn is not None):
        have = [k for k in t if t[k] is not None]
        outs = [o for o, d in ((h, dh), (n, dn)) if d is not None]
        got = torch.autograd.grad(outs, [t[k] for k in have], [d for d in (dh, dn) if d is not None], allow_unused=True)
        names = {"x": "dx", "gate": "dgate", "residual": "dresidual", "post": "dpost", "scale": "dscale", "pre": "dpre"}
        for k, v in zip(have, got):
            assert v.dtype == t[k].dtype and v.shape == t[k].shape
            R.check(names[k], v.reshape(ref[names[k]].shape), ref[names[k]], v.dtype, ref[names[k] + "_slack"])
    return h, n


@pytest.mark.parametrize("parts", COMBINATIONS, ids="-".join)
@pytest.mark.parametrize("dtype,rdtype,wdtype", [(BF, F, BF), (BF, BF, F), (F, F, F), (HF, HF, HF)])
def test_block_norm_parts_and_types(dtype, rdtype, wdtype, parts):
    run_norm(norm_inputs(parts, 37, 136, dtype, rdtype, wdtype))
    run_norm(norm_inputs(parts, 5, 136, dtype, rdtype, wdtype), train=False)


@pytest.mark.parametrize("rows,channels", [(1, 1), (3, 7), (130, 80), (65, 512), (9, 513), (4, 1111), (7, 2048), (2, 4096), (3, 5000), (2, 8192), (2, 16384),
                                           (1, 16383), (600, 64), (2050, 8)])
@pytest.mark.parametrize("dtype", [BF, F])
def test_block_norm_sizes(rows, channels, dtype):
    run_norm(norm_inputs(PARTS, rows, channels, dtype, F, dtype))


@pytest.mark.parametrize("rows,channels", [(4095, 300), (4096, 257), (4097, 511), (4098, 513), (4099, 1001), (4097, 1111), (4101, 1280)])
@pytest.mark.parametrize("dtype,rdtype", [(BF, F), (HF, HF)])
def test_block_norm_many_rows(rows, channels, dtype, rdtype):
    """Rows that a wave has to itself, and their number just below."""
    run_norm(norm_inputs(PARTS, rows, channels, dtype, rdtype, dtype), train=False)


def test_block_norm_many_rows_with_gradients():
    run_norm(norm_inputs(PARTS, 4097, 300, BF, F, BF))
    run_norm(norm_inputs(("post", "gate"), 4099, 301, HF, HF, HF))


@pytest.mark.parametrize("use", [("h",), ("n",)])
def test_block_norm_gradient_of_one_output(use):
    run_norm(norm_inputs(PARTS, 19, 200, BF, F, F), use=use)


def test_block_norm_shapes_and_strides():
    t = norm_inputs(PARTS, 24, 96, BF, BF, BF)
    h, n = run_norm(t)
    cube = {k: v if v is None or v.dim() == 1 else v.view(2, 3, 4, 96) for k, v in t.items()}
    h4, n4 = run_norm(cube)
    assert h4.shape == (2, 3, 4, 96) and torch.equal(h4.view(24, 96), h) and torch.equal(n4.view(24, 96), n)
    for shift in (0, 1):       # slices of one wide projection, aligned and not
        wide = torch.zeros(24, 2 * 96 + 5, dtype=BF).cuda()
        wide[:, shift:shift + 96], wide[:, shift + 96:shift + 192] = t["x"], t["gate"]
        s = dict(t, x=wide[:, shift:shift + 96], gate=wide[:, shift + 96:shift + 192])
        hs, ns = run_norm(s)
        assert torch.equal(hs, h) and torch.equal(ns, n)
    flipped = dict(t, x=t["x"].t().contiguous().t())
    hf, _ = call_norm(flipped)
    assert torch.equal(hf, h)
    vector = {k: v if v is None or v.dim() == 1 else v[0] for k, v in t.items()}
    hv, nv = call_norm(vector)
    assert hv.shape == (96,) and torch.equal(hv, h[0]) and torch.equal(nv, n[0])


def test_block_norm_zero_rows_infinities_and_large_values():
    t = norm_inputs(["post", "pre"], 6, 300, F, F, F)
    t["x"][1] = 0                                  # rstd = 1 / sqrt(eps)
    t["x"][2] *= 1e15                              # its square is within 32 bits, and so is the sum
    t["x"][3, 7] = float("inf")
    t["x"][4, 9] = float("nan")
    h, n = call_norm(t)
    h, n = h.cpu(), n.cpu()
    assert (h[1] == 0).all() and (n[1] == 0).all() and torch.isfinite(h[[0, 1, 2, 5]]).all()
    assert torch.isnan(h[4]).all() and torch.isnan(h[3, 7])
    fine = {k: v if v is None or v.dim() == 1 else v[[0, 1, 2, 5]] for k, v in t.items()}
    run_norm(fine, train=False)


def test_block_norm_gradient_against_differences():
    t = norm_inputs(PARTS, 5, 48, F, F, F)
    live = {k: leaf(v) for k, v in t.items()}
    h, n = call_norm(live)
    dh, dn = rand(52, 5, 48), rand(53, 5, 48)
    got = [R.f64(g) for g in torch.autograd.grad((h, n), list(live.values()), (dh, dn))]
    at = [R.f64(v) for v in t.values()]
    rng = np.random.default_rng(54)
    way = [rng.normal(size=v.shape) for v in at]

    def value(step):
        p = dict(zip(t, [v + step * d for v, d in zip(at, way)]))
        ref = R.block_norm(p["x"], p["gate"], p["residual"], p["post"], p["scale"], p["pre"])
        return float((ref["h"] * R.f64(dh)).sum() + (ref["n"] * R.f64(dn)).sum())
    slope = (value(1e-5) - value(-1e-5)) / 2e-5
    along = sum(float((g * d).sum()) for g, d in zip(got, way))
    size = sum(float(np.abs(g * d).sum()) for g, d in zip(got, way))
    assert abs(slope - along) <= 128 * R.U * size, (slope, along)


def test_block_norm_no_rows():
    t = norm_inputs(PARTS, 0, 64, BF, F, BF)
    live = {k: leaf(v) for k, v in t.items()}
    h, n = call_norm(live)
    assert h.shape == (0, 64) and n.shape == (0, 64)
    g = torch.autograd.grad((h.sum(), n.sum()), list(live.values()))
    assert all((v == 0).all() for v in g)


# ------------------------------------------------------------------ embedding lookup
def run_embedding(ids, table, train=True, **kw):
    tab = leaf(table) if train else table
    e = sequence.embedding_lookup(ids, tab, **kw)
    assert e.shape == (*ids.shape, table.shape[1]) and e.dtype == kw.get("dtype", table.dtype)
    scale, pad = kw.get("scale", 1.0), kw.get("padding_idx")
    pad = None if pad is None else pad % table.shape[0]
    d = rand(60, *e.shape, dtype=e.dtype) if train else None
    ref = R.embedding(ids.cpu().numpy(), R.f64(table), float(np.float32(scale)), pad, R.f64(d))
    R.check("e", e, ref["e"], e.dtype, ref["e_slack"])
    if train:
        dt, = torch.autograd.grad(e, tab, d)
        assert dt.dtype == table.dtype
        R.check("dtable", dt, ref["dtable"], dt.dtype, ref["dtable_slack"])
        return e, dt
    return e, None


def tokens(seed, vocab, *shape, dtype=torch.int64):
    """Frequent ones and rare ones: 1 / rank."""
    u = np.random.default_rng(seed).random(shape)
    return torch.from_numpy(np.minimum(np.exp(u * np.log(vocab + 1)).astype(np.int64) - 1, vocab - 1)).to(dtype).cuda()


@pytest.mark.parametrize("dtype,out", [(BF, BF), (F, F), (HF, HF), (F, BF), (BF, F)])
@pytest.mark.parametrize("count,vocab,channels", [(1, 1, 1), (300, 50, 64), (1000, 7, 40), (64, 2000, 136), (5000, 300, 33), (257, 70000, 8)])
def test_embedding_sizes_and_types(count, vocab, channels, dtype, out):
    run_embedding(tokens(61, vocab, count), rand(62, vocab, channels, dtype=dtype), scale=2.5, dtype=out)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_embedding_padding_and_ids_outside(index):
    ids = tokens(63, 90, 7, 60, dtype=index)
    ids[0, :5] = torch.tensor([-1, 90, 2 ** 31 - 1, -2 ** 31, 89], dtype=index).cuda()
    table = rand(64, 90, 48)
    e, dt = run_embedding(ids, table, padding_idx=3, scale=0.5)
    assert (e[0, :4] == 0).all() and (dt[3] == 0).all()
    e2, dt2 = run_embedding(ids, table, padding_idx=-87, scale=0.5)
    assert torch.equal(e, e2) and torch.equal(dt, dt2)


@pytest.mark.parametrize("count", [4096, 4097, 20000])
def test_embedding_one_token_everywhere(count):
    """A padding token or a frequent word: one row of the table takes nearly every gradient."""
    ids = torch.full((count,), 5).cuda()
    ids[::97] = 2
    ids[1] = 6
    run_embedding(ids, rand(65, 9, 72, dtype=BF))
    run_embedding(torch.full((count,), 8).cuda(), rand(66, 9, 24))


def test_embedding_shapes_and_strides():
    table = rand(67, 40, 64, dtype=HF)
    ids = tokens(68, 40, 6, 10)
    e, dt = run_embedding(ids, table)
    run_embedding(ids.t(), table)
    run_embedding(ids[:, ::3], table)
    run_embedding(ids[0, 0], table)
    wide = torch.zeros(40, 64 + 7, dtype=HF).cuda()
    for shift in (0, 3):
        wide[:, shift:shift + 64] = table
        e2, dt2 = run_embedding(ids, wide[:, shift:shift + 64])
        assert torch.equal(e, e2) and torch.equal(dt, dt2)
    run_embedding(ids, table.t().contiguous().t())
    run_embedding(tokens(69, 40, 0), table)
    tab = leaf(table)
    sequence.embedding_lookup(ids, tab).sum().backward()
    ref = R.embedding(ids.cpu().numpy(), R.f64(table), dout=np.ones((6, 10, 64)))
    R.check("dtable", tab.grad, ref["dtable"], HF, ref["dtable_slack"])


def test_embedding_same_inputs_same_bits():
    ids, table = tokens(70, 200, 6000), rand(71, 200, 40)
    d = rand(72, 6000, 40)
    got = []
    for _ in range(3):
        tab = leaf(table)
        got.append(torch.autograd.grad(sequence.embedding_lookup(ids, tab), tab, d)[0])
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


# ------------------------------------------------------------------ together
def layer(p, ids, offsets, state, step=None):
    """Token rows -> norm -> gated recurrence -> norm, gate, scaled residual and the norm behind, as a layer uses them."""
    e = sequence.embedding_lookup(ids, p["table"], scale=4.0)
    h, n = sequence.block_norm(e, pre_weight=p["w_in"])
    kw = {"offsets": offsets} if step is None else {}
    x = n if step is None else n.unsqueeze(1)
    g = (n * p["slope"]) if step is None else (n * p["slope"]).unsqueeze(1)
    y, state = sequence.linear_recurrence(x, g, form="gate", initial_state=state, **kw)
    y = y if step is None else y.squeeze(1)
    h, n = sequence.block_norm(y, gate=n, residual=h, post_weight=p["w_post"], scale=p["s"], pre_weight=p["w_out"])
    return h, n, state


def layer_parameters(c=48, vocab=60, dtype=F):
    return {"table": rand(80, vocab, c, dtype=dtype), "w_in": rand(81, c, dtype=dtype, scale=0.2, shift=1), "slope": rand(82, c, dtype=dtype, shift=1),
            "w_post": rand(83, c, dtype=dtype, scale=0.2, shift=1), "s": rand(84, c, dtype=dtype, scale=0.3), "w_out": rand(85, c, dtype=dtype, scale=0.2, shift=1)}


def test_together_training_step_against_64_bits():
    p = {k: leaf(v) for k, v in layer_parameters().items()}
    lens = [30, 1, 0, 77]
    ids = tokens(86, 60, 108)
    offsets = torch.tensor([0, 30, 31, 31, 108]).cuda()
    h, n, state = layer(p, ids, offsets, None)
    dn = rand(87, 108, 48)
    got = dict(zip(p, torch.autograd.grad(n, list(p.values()), dn)))
    # the same in 64 bits, with automatic differentiation of plain operations
    q = {k: v.detach().cpu().double().requires_grad_(True) for k, v in p.items()}
    norm = lambda z, w: z / torch.sqrt((z * z).mean(-1, keepdim=True) + 1e-6) * w  # noqa: E731
    e = q["table"][ids.cpu()] * 4.0
    m = norm(e, q["w_in"])
    f = torch.sigmoid(m * q["slope"])
    rows = []
    for s, k in enumerate(lens):
        c = torch.zeros(48, dtype=torch.float64)
        for t in range(sum(lens[:s]), sum(lens[:s + 1])):
            c = f[t] * c + (1 - f[t]) * m[t]
            rows.append(c)
    hh = e + q["s"] * (norm(torch.stack(rows), q["w_post"]) * torch.nn.functional.silu(m))
    nn = norm(hh, q["w_out"])
    want = dict(zip(q, torch.autograd.grad(nn, list(q.values()), dn.cpu().double())))
    # a chain of about 200 operations in 32 bits: their errors relative to the largest of the values
    assert np.abs(R.f64(h) - hh.detach().numpy()).max() <= 200 * R.U * hh.abs().max().item()
    assert np.abs(R.f64(n) - nn.detach().numpy()).max() <= 200 * R.U * nn.abs().max().item()
    for k in p:
        # sums over 108 rows, of terms as large as the largest gradient times a few
        assert np.abs(R.f64(got[k]) - want[k].numpy()).max() <= 108 * 20 * R.U * max(1.0, want[k].abs().max().item()), k


def test_together_decoding_equals_prompt():
    """All tokens in one packed call, and one token at a time for every sequence with its state."""
    p = layer_parameters(dtype=BF)
    ids = tokens(88, 60, 3, 12)
    offsets = torch.tensor([0, 12, 24, 36], dtype=torch.int32).cuda()
    h, n, state = layer(p, ids.reshape(-1), offsets, None)
    s = None
    for t in range(12):
        ht, nt, s = layer(p, ids[:, t], None, s, step=t)
        # the recurrence's output is rounded once either way; its 32-bit value differs by a few roundings, which moves a
        # bf16 value by a step at most, and what follows by a few of them
        assert (nt.float() - n.view(3, 12, 48)[:, t].float()).abs().max() <= 4 * 2 ** -7 * n.float().abs().max()
    assert np.abs(R.f64(s) - R.f64(state)).max() <= 500 * R.U * max(1.0, float(state.abs().max()))
