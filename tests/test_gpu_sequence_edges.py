"""The sequence operators where their inputs are at an end of their range or their work at the end of a piece: excluded tokens behind
the last real one, gates that are wide open or shut, states that share memory.  Bounds are derived beside each test from half a
step of each type and 2^-24 per operation in 32 bits."""
import ctypes as C
import os

import numpy as np
import pytest
import torch
import torch._decomp.decompositions_for_jvp  # noqa: F401  (what make_dual would load where torch's factories are patched)
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from dali_amd import _capi as capi
from dali_amd import sequence
from tests import sequence_reference as R
from tests.test_gpu_sequence import BF, F, HF, decays, leaf, rand, run_recurrence

MODEL = bool(os.environ.get("DALI_AMD_HIPEMU"))
pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ embedding: tokens that take no part
def embedding_gradient(ids, dout, vocab, padding=-1, dtype=F):
    """The table's gradient through the C entries, into memory that holds NaN."""
    lib, channels = capi.kernels(), dout.shape[1]
    dtable = torch.full((vocab, channels), float("nan"), dtype=dtype).cuda()
    names = {F: capi.FLOAT, BF: capi.BFLOAT16, HF: capi.FLOAT16}
    a = capi.EmbeddingArgs(ids=ids.data_ptr(), table=dtable.data_ptr(), dout=dout.data_ptr(), dtable=dtable.data_ptr(), tokens=ids.numel(), vocab=vocab,
                           padding=padding, table_row=channels, dout_row=dout.stride(0), channels=channels, dtype=names[dtype],
                           out_dtype=names[dout.dtype], index_dtype=capi.INT64 if ids.dtype == torch.int64 else capi.INT32, scale=1.0)
    plan = capi.EmbeddingPlan()
    capi.check(lib.daliamdEmbeddingSetup(C.byref(a), C.byref(plan)))
    ws = torch.empty(plan.backward_workspace_bytes, dtype=torch.uint8).cuda()
    capi.check(lib.daliamdEmbeddingBackwardRun(C.c_void_p(torch.cuda.current_stream().cuda_stream), C.byref(a), C.c_void_p(ws.data_ptr()), C.c_size_t(ws.numel())))
    torch.cuda.synchronize()
    return dtable


@pytest.mark.parametrize("behind", ["outside", "padding"])
@pytest.mark.parametrize("count", [16384, 32768])
def test_embedding_every_row_is_written_whatever_excluded_tokens_are_behind(count, behind):
    """More than 1024 channels: chunks of 16 sorted tokens from 16384 on, of 32 from 32768 on.  The last real tokens end at every place
    of a chunk, the highest id's run begins in it, is one token or several, and excluded tokens fill the rest of it and chunks behind.
    Gradients are small whole numbers: their sums are exact."""
    channels, vocab, highest = 1025, 120, 100
    rng = np.random.default_rng(1)
    dout = torch.from_numpy(rng.integers(-3, 4, (count, channels)).astype(np.float32)).to(BF).cuda()
    host = dout.cpu().float()
    start = count // 2
    places = (0, 1, 8, 9, 16, 24, 31) if MODEL else range(33)
    for place in places:
        for run in (1, 5, 40):
            real = start + place
            ids = torch.full((count,), -1 if behind == "outside" else 7, dtype=torch.int64)
            ids[:real] = torch.from_numpy(rng.integers(8, highest, real))
            ids[real - run:real] = highest
            got = embedding_gradient(ids.cuda(), dout, vocab, padding=-1 if behind == "outside" else 7).cpu()
            want = torch.zeros(vocab, channels).index_add_(0, ids[:real], host[:real])
            assert torch.equal(got, want), (place, run, (got != want).any(1).nonzero().flatten().tolist())


# ------------------------------------------------------------------ gates at the ends of their type
def ends(dtype):
    return [float("-inf"), float("inf"), torch.finfo(dtype).min, torch.finfo(dtype).max]


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("dtype,gdtype", [(F, F), (BF, BF), (BF, F), (HF, HF), (HF, F)])
@pytest.mark.parametrize("steps", [1, 3, 300])
def test_recurrence_gates_at_the_ends_of_their_type(steps, dtype, gdtype, train):
    """f is 0 at -infinity and at the lowest value, 1 at the other end: no value of a gate makes a NaN."""
    x, g = rand(500, 2, steps, 24, dtype=dtype), decays(501, "gate", 2, steps, 24, dtype=gdtype)
    pick = np.random.default_rng(502).integers(0, 8, g.shape)
    for k, v in enumerate(ends(gdtype)):
        g[torch.from_numpy(pick == k).cuda()] = v
    run_recurrence(x, g, "gate", R.ranges(2 * steps, 2, steps), rand(503, 2, 24), train)


@pytest.mark.parametrize("dtype", [F, BF, HF])
def test_recurrence_gates_per_channel_at_the_ends_of_their_type(dtype):
    g = decays(504, "gate", 24, dtype=dtype)
    g[:4] = torch.tensor(ends(dtype), dtype=dtype)
    run_recurrence(rand(505, 2, 300, 24, dtype=dtype), g, "gate", R.ranges(600, 2, 300), rand(506, 2, 24), True)


@pytest.mark.parametrize("dtype", [F, BF, HF])
@pytest.mark.parametrize("post", [False, True])
def test_block_norm_gates_at_the_ends_of_their_type(post, dtype):
    """g silu'(g) and silu(g) at the lowest and the largest value, the former with the norm in front as well (with the latter its sums
    would not fit); at infinity the product is infinite."""
    gate = rand(510, 5, 40, dtype=dtype)
    gate[1, 3], gate[2] = torch.finfo(dtype).min, torch.finfo(dtype).min
    if not post:
        gate[3, ::2], gate[4, 7] = torch.finfo(dtype).max, torch.finfo(dtype).max
    x, dh = (rand(511 + k, 5, 40, scale=0.2).clamp(-0.9, 0.9).to(dtype) for k in (0, 1))
    w = rand(513, 40, dtype=dtype) if post else None
    leaves = [leaf(x), leaf(gate)]
    h, _ = sequence.block_norm(leaves[0], gate=leaves[1], post_weight=w)
    dx, dgate = torch.autograd.grad(h, leaves, dh)
    ref = R.block_norm(R.f64(x), R.f64(gate), post=R.f64(w), dh=R.f64(dh))
    R.check("hidden", h, ref["h"], dtype, ref["h_slack"])
    R.check("dx", dx, ref["dx"], dtype, ref["dx_slack"])
    R.check("dgate", dgate, ref["dgate"], dtype, ref["dgate_slack"])
    gate[4, 9] = float("inf")
    h, _ = sequence.block_norm(x, gate=gate)
    assert torch.isinf(h[4, 9]) and torch.signbit(h[4, 9]) == torch.signbit(x[4, 9]) and not torch.isnan(h).any()


# ------------------------------------------------------------------ what would not see the kernels
def calls():
    """name: (a function of tensors that have a derivative, the tensors)"""
    ids = torch.tensor([3, 0, 3]).cuda()
    x, g, w = rand(520, 2, 5, 8), rand(521, 2, 5, 8), rand(522, 8)
    return {
        "linear_recurrence": (lambda x, g, h: sequence.linear_recurrence(x, g, form="gate", initial_state=h)[0], [x, g, rand(523, 2, 8)]),
        "block_norm": (lambda x, g, r, w1, s, w2: sequence.block_norm(x, gate=g, residual=r, post_weight=w1, scale=s, pre_weight=w2)[1],
                       [x, g, rand(524, 2, 5, 8), w, rand(525, 8), rand(526, 8)]),
        "embedding_lookup": (lambda table: sequence.embedding_lookup(ids, table), [rand(527, 6, 8)]),
    }


@pytest.mark.parametrize("op", ["linear_recurrence", "block_norm", "embedding_lookup"])
def test_forward_mode_is_refused(op):
    """A tangent would be lost without a word: its place in the result is not computed."""
    f, tensors = calls()[op]
    want = f(*tensors)
    for k in range(len(tensors)):
        for leaf_too in (False, True):
            for grad in (False, True):
                with forward_ad.dual_level(), torch.set_grad_enabled(grad):
                    args = [t.clone().requires_grad_(leaf_too) for t in tensors]
                    args[k] = forward_ad.make_dual(args[k], torch.ones_like(args[k]))
                    with pytest.raises(RuntimeError, match=f"{op} has no forward-mode derivative"):
                        f(*args)
    assert torch.equal(f(*tensors), want)
    # ... and so for the gradient's gradients along a tangent
    leaves = [leaf(t) for t in tensors]
    out = f(*leaves)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match=f"{op} has no forward-mode derivative"):
            torch.autograd.grad(out, leaves, forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out)))


@pytest.mark.parametrize("op", ["linear_recurrence", "block_norm", "embedding_lookup"])
@pytest.mark.parametrize("leaf_too", [False, True])
def test_tracing_is_refused(op, leaf_too):
    """A trace would hold the outputs' allocation and not the kernels."""
    f, tensors = calls()[op]
    want = f(*tensors)
    args = tuple(t.clone().requires_grad_(leaf_too) for t in tensors)
    with pytest.raises(RuntimeError, match=f"{op} cannot be traced"):
        torch.jit.trace(f, args, check_trace=False)
    for pre_dispatch in (False, True):
        with pytest.raises(RuntimeError, match=f"{op} cannot be traced"):
            make_fx(f, pre_dispatch=pre_dispatch)(*args)
    assert torch.equal(f(*tensors), want)
    leaves = [leaf(t) for t in tensors]
    out = f(*leaves)
    with pytest.raises(RuntimeError, match=f"{op} cannot be traced"):
        make_fx(lambda d: torch.autograd.grad(out, leaves, d))(torch.ones_like(out))


# ------------------------------------------------------------------ negated in name only
def negated(t):
    """-t as torch holds the imaginary part of a conjugate: the memory of t and a mark."""
    return torch._neg_view(t)


def test_views_that_are_negated_in_name_only():
    """Every tensor of a call, and the gradients that a backward pass is given."""
    x, g, h0 = rand(530, 2, 9, 8), rand(531, 2, 9, 8), rand(532, 2, 8)
    dy, dlast = rand(533, 2, 9, 8), rand(534, 2, 8)
    lengths, offsets = torch.tensor([9, 4]).cuda(), torch.tensor([0, 5, 18]).cuda()

    def recurrence(form, *t, **kw):
        leaves = [leaf(v) for v in t[:3]]
        y, state = sequence.linear_recurrence(leaves[0], leaves[1], form=form, initial_state=leaves[2], **kw)
        return (y, state) + torch.autograd.grad((y, state), leaves, t[3:])

    t = (x, g, h0, dy, dlast)
    for form, kw in (("gate", {"lengths": lengths}), ("decay", {})):
        want = recurrence(form, *t, **kw)
        got = recurrence(form, *[negated(-v) for v in t], **{k: negated(-v) for k, v in kw.items()})
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    flat = [v.reshape(18, 8) for v in (x, g)]
    want = sequence.linear_recurrence(*flat, offsets=offsets, form="gate")
    got = sequence.linear_recurrence(*[negated(-v) for v in flat], offsets=negated(-offsets), form="gate")
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    per_channel = sequence.linear_recurrence(x, g[0, 0], form="gate")[0]
    assert torch.equal(sequence.linear_recurrence(x, negated(-g[0, 0]), form="gate")[0], per_channel)
    # one channel: the imaginary part of a conjugate as a program gets it
    z = torch.complex(rand(535, 3, 7, 1), rand(536, 3, 7, 1))
    imaginary = z.conj().imag
    assert imaginary.is_neg()
    assert torch.equal(sequence.linear_recurrence(imaginary, x[0, :1, 0])[0], sequence.linear_recurrence(-z.imag.contiguous(), x[0, :1, 0])[0])

    def norm(*t):
        leaves = [leaf(v) for v in t[:6]]
        out = sequence.block_norm(leaves[0], gate=leaves[1], residual=leaves[2], post_weight=leaves[3], scale=leaves[4], pre_weight=leaves[5])
        return out + torch.autograd.grad(out, leaves, t[6:])

    t = [rand(540 + k, 5, 24) for k in range(3)] + [rand(543 + k, 24) for k in range(3)] + [rand(546 + k, 5, 24) for k in range(2)]
    assert all(torch.equal(a, b) for a, b in zip(norm(*[negated(-v) for v in t]), norm(*t)))

    def embedding(ids, table, d):
        table = leaf(table)
        e = sequence.embedding_lookup(ids, table)
        return e, torch.autograd.grad(e, table, d)[0]

    t = (torch.tensor([1, 0, 3, 1]).cuda(), rand(550, 4, 24), rand(551, 4, 24))
    assert all(torch.equal(a, b) for a, b in zip(embedding(*[negated(-v) for v in t]), embedding(*t)))


def test_a_state_that_is_negated_in_name_only_is_not_written():
    x, state = rand(552, 2, 3, 8), negated(torch.zeros(2, 8).cuda())
    with pytest.raises(ValueError, match="final_state"):
        sequence.linear_recurrence(x, x, final_state=state)


# ------------------------------------------------------------------ gates of all sizes, element by element
def elementwise(x, g, spans, initial, dy, dlast, per_step):
    """The gate form in 64 bits with a bound for each element by itself.  H and L are the same sums of absolute values: what a state or a
    gradient is made of.  A step's arithmetic is off by per_step 2^-24 of what it adds up, and passes on f of the error it is given; the
    pieces that a sequence is cut into are joined by 16 further roundings, each of such a sum."""
    rows, c = x.shape
    one = g.ndim == 1
    f, k = R.logistic(g)
    at = (lambda t: f) if one else (lambda t: f[t])
    kt = (lambda t: k) if one else (lambda t: k[t])
    out = R.recurrence(x, g, "gate", spans, initial, dy, dlast)
    e = {n: np.zeros((rows, c)) for n in ("y", "dx", "dg")}
    e["state"], e["dinitial"] = np.zeros((len(spans), c)), np.zeros((len(spans), c))
    u, join = per_step * R.U, 16 * R.U
    for s, (b, end) in enumerate(spans):
        h = np.zeros(c) if initial is None else np.abs(initial[s])
        err, before = np.zeros(c), []
        for t in range(b, end):
            before.append((h, err + join * h))
            grown = at(t) * h + kt(t) * np.abs(x[t])
            h, err = grown, at(t) * err + u * grown
            e["y"][t] = err + join * h
        e["state"][s] = err + join * h
        m, err = np.abs(dlast[s]), np.zeros(c)
        for t in range(end - 1, b - 1, -1):
            l = m + np.abs(dy[t])   # noqa: E741
            err = err + u * l
            seen = err + join * l
            hb, eb = before[t - b]
            e["dx"][t] = kt(t) * (seen + u * l)
            reach = hb + np.abs(x[t])
            e["dg"][t] = at(t) * kt(t) * (seen * reach + l * (eb + u * reach))
            m, err = at(t) * l, at(t) * (err + u * l)
        e["dinitial"][s] = err + join * m
    if one:   # a sum over the rows in 32 bits
        terms = np.zeros((rows, c))
        for b, end in spans:
            m = np.abs(dlast[spans.index((b, end))])
            for t in range(end - 1, b - 1, -1):
                l = m + np.abs(dy[t])   # noqa: E741
                terms[t] = f * k * l * np.abs(np.abs(x[t]) + (np.abs(out["y"][t - 1]) if t > b else np.abs(initial[spans.index((b, end))])))
                m = f * l
        e["dg"] = e["dg"].sum(0) + (32 + rows / 256) * R.U * terms.sum(0)
    return out, e


@pytest.mark.parametrize("dtype,gdtype", [(F, F), (BF, BF), (BF, F), (HF, HF), (F, "per channel")])
@pytest.mark.parametrize("low,high", [(-40, -4), (-40, 40), (3, 12), (-2, 2)])
@pytest.mark.parametrize("batch,steps", [(2, 300), (3, 3), (1, 1100)])
def test_recurrence_gates_of_all_sizes(batch, steps, low, high, dtype, gdtype):
    """A gate that is nearly shut leaves f of the state in front, as exactly as one that is nearly open leaves 1 - f of the input: x is
    large at some steps and small at others, and each result is compared with what it is made of, not with the largest one."""
    c, rows = 24, batch * steps
    rng = np.random.default_rng(560)
    one = gdtype == "per channel"
    gdtype = F if one else gdtype
    spread = 2 if dtype == HF else 5       # (float16 ends at 65504)
    wide = lambda *shape: torch.from_numpy(rng.normal(size=shape) * 10.0 ** rng.uniform(-spread, spread, shape))  # noqa: E731
    x = wide(batch, steps, c).clamp(-1e4, 1e4).to(dtype).cuda()
    g = torch.from_numpy(rng.uniform(low, high, (c,) if one else (batch, steps, c))).to(gdtype).cuda()
    h0, dy, dlast = wide(batch, c).float().cuda(), rand(561, batch, steps, c, dtype=dtype), rand(562, batch, c)
    leaves = [leaf(t) for t in (x, g, h0)]
    y, state = sequence.linear_recurrence(leaves[0], leaves[1], form="gate", initial_state=leaves[2])
    dx, dg, dinitial = torch.autograd.grad((y, state), leaves, (dy, dlast))
    flat = lambda t: R.f64(t).reshape(rows, c)  # noqa: E731
    # 12: the logistic function (exp with two, 1 + t, its reciprocal, their product), the step, a product of two; 16-bit gates leave out
    # the rounding of g log2(e), which is |g| 2^-24 of the power
    per_step = 12 + (0 if gdtype == F else max(abs(low), abs(high)))
    ref, e = elementwise(flat(x), R.f64(g) if one else flat(g), R.ranges(rows, batch, steps), R.f64(h0), flat(dy), R.f64(dlast), per_step)
    # (2^-126: a power below the smallest normal number may be taken for 0; times what it multiplies, at most 1e8)
    for name, got, t in (("y", y, dtype), ("state", state, F), ("dx", dx, dtype), ("dg", dg, gdtype), ("dinitial", dinitial, F)):
        R.check(name, got.reshape(ref[name].shape), ref[name], t, e[name] + 2.0 ** -99)
    # and without gradients, where a thread goes through a few steps by itself
    z, last = sequence.linear_recurrence(x, g, form="gate", initial_state=h0)
    R.check("y", z.reshape(rows, c), ref["y"], dtype, e["y"] + 2.0 ** -99)
    R.check("state", last, ref["state"], F, e["state"] + 2.0 ** -99)


@pytest.mark.parametrize("dtype,gdtype", [(F, F), (BF, BF), (HF, F)])
@pytest.mark.parametrize("low,high", [(-40, -4), (-40, 40)])
def test_recurrence_gates_of_all_sizes_packed(low, high, dtype, gdtype):
    """Sequences that begin and end inside the pieces, none, one and many steps long."""
    c, lens = 40, [5, 0, 300, 1, 257, 40, 0, 3]
    rows, rng = sum(lens), np.random.default_rng(565)
    ends = np.cumsum([0] + lens)
    x = torch.from_numpy(rng.normal(size=(rows, c)) * 10.0 ** rng.uniform(-2, 2, (rows, c))).to(dtype).cuda()
    g = torch.from_numpy(rng.uniform(low, high, (rows, c))).to(gdtype).cuda()
    h0, dy, dlast = rand(566, len(lens), c, scale=100.0), rand(567, rows, c, dtype=dtype), rand(568, len(lens), c)
    leaves = [leaf(t) for t in (x, g, h0)]
    y, state = sequence.linear_recurrence(leaves[0], leaves[1], form="gate", initial_state=leaves[2], offsets=torch.from_numpy(ends).cuda())
    dx, dg, dinitial = torch.autograd.grad((y, state), leaves, (dy, dlast))
    per_step = 12 + (0 if gdtype == F else max(abs(low), abs(high)))
    ref, e = elementwise(R.f64(x), R.f64(g), list(zip(ends[:-1], ends[1:])), R.f64(h0), R.f64(dy), R.f64(dlast), per_step)
    for name, got, t in (("y", y, dtype), ("state", state, F), ("dx", dx, dtype), ("dg", dg, gdtype), ("dinitial", dinitial, F)):
        R.check(name, got, ref[name], t, e[name] + 2.0 ** -99)


# ------------------------------------------------------------------ decays of more than 1
@pytest.mark.parametrize("one", [False, True])
@pytest.mark.parametrize("decay", [100.0, -3e38])
@pytest.mark.parametrize("steps", [7, 512, 1800])
def test_recurrence_large_decays_of_a_state_that_is_zero(steps, decay, one):
    """A state of 0 stays 0 under any decay, however large the product of many of them; in both directions of time."""
    x, g = torch.zeros(2, steps, 24).cuda(), torch.full((24,) if one else (2, steps, 24), decay).cuda()
    x[:, -1 if one else -2] = rand(570, 2, 24)
    if not one:
        g[0, steps // 3, ::2], g[1, 3, ::3] = 0.0, 0.0     # (a product of infinity and 0 is none either)
        g[:, -1] = 0.5
    leaves = [leaf(x), leaf(g)]
    y, state = sequence.linear_recurrence(*leaves)
    dy = torch.zeros_like(y)
    dy[:, 0] = rand(571, 2, 24)
    dx, dg = torch.autograd.grad((y, state), leaves, (dy, torch.zeros_like(state)))
    ref = R.recurrence(R.f64(x).reshape(-1, 24), R.f64(g) if one else R.f64(g).reshape(-1, 24), "decay", R.ranges(2 * steps, 2, steps), None,
                       R.f64(dy).reshape(-1, 24), np.zeros((2, 24)))
    for name, got in (("y", y), ("state", state), ("dx", dx), ("dg", dg)):
        want = ref[name]
        assert np.isfinite(want).all()
        # a product or two of numbers that are not 0, and nothing added to them
        R.check(name, got.reshape(want.shape), want, F, 4 * R.U * np.abs(want))


# ------------------------------------------------------------------ states that share memory
@pytest.mark.parametrize("shift", [-1, 0, 1, 3])
@pytest.mark.parametrize("steps", [1, 4, 5, 300])
def test_recurrence_states_that_overlap(steps, shift):
    """The final states in the memory of the initial ones, or some rows off it: what is read is what was there before the call."""
    n, c = 40, 72
    x, g = rand(580, n, steps, c, dtype=BF), decays(581, "gate", n, steps, c, dtype=BF)
    memory = rand(582, n + 4, c)
    start = max(-shift, 0)
    initial = memory[start:start + n].clone()
    want, last = sequence.linear_recurrence(x, g, form="gate", initial_state=initial)
    rest = memory.clone()
    rest[start + shift:start + shift + n] = last
    y, state = sequence.linear_recurrence(x, g, form="gate", initial_state=memory[start:start + n], final_state=memory[start + shift:start + shift + n])
    assert torch.equal(y, want) and torch.equal(state, last) and torch.equal(memory, rest)


@pytest.mark.parametrize("steps", [1, 4, 5, 300])
def test_recurrence_workspace_does_not_depend_on_what_setup_names(steps):
    """C entries: the sizes that Setup gives without the tensors suffice for every Run over the same states."""
    n, c, lib = 6, 40, capi.kernels()
    x, g, state = rand(583, n, steps, c), decays(584, "gate", n, steps, c), rand(585, n, c)
    before = state.clone()
    a, plan = capi.RecurrenceArgs(), capi.RecurrencePlan()
    a.seq.rows, a.seq.steps, a.seq.sequences = n * steps, steps, n
    a.x_row, a.x_seq, a.decay_row, a.decay_seq = c, steps * c, c, steps * c
    a.channels, a.dtype, a.decay_dtype, a.form = c, capi.FLOAT, capi.FLOAT, capi.RECURRENCE_GATE
    a.initial = a.final_state = state.data_ptr()
    capi.check(lib.daliamdRecurrenceSetup(C.byref(a), C.byref(plan)))
    y, ws = torch.empty_like(x), torch.empty(max(plan.forward_workspace_bytes, 16), dtype=torch.uint8).cuda()
    saved = torch.empty(max(plan.saved_bytes, 16), dtype=torch.uint8).cuda()
    a.x, a.decay, a.y, a.saved = x.data_ptr(), g.data_ptr(), y.data_ptr(), saved.data_ptr()
    capi.check(lib.daliamdRecurrenceRun(C.c_void_p(torch.cuda.current_stream().cuda_stream), C.byref(a), C.c_void_p(ws.data_ptr()),
                                        C.c_size_t(plan.forward_workspace_bytes)))
    torch.cuda.synchronize()
    want, last = sequence.linear_recurrence(x, g, form="gate", initial_state=before)
    assert torch.equal(y, want) and torch.equal(state, last)


# ------------------------------------------------------------------ embedding: a table that changes before the backward pass
def test_embedding_table_changed_before_the_backward_pass():
    """The gradient does not depend on the table's values: an optimizer may have stepped, as with torch's own lookup."""
    ids, d = torch.tensor([3, 1, 3, 0]).cuda(), rand(590, 4, 24, dtype=BF)
    table = leaf(rand(591, 5, 24, dtype=BF))
    want, = torch.autograd.grad(sequence.embedding_lookup(ids, table, scale=2.0, padding_idx=1), table, d)
    e = sequence.embedding_lookup(ids, table, scale=2.0, padding_idx=1)
    with torch.no_grad():
        table += 1
    got, = torch.autograd.grad(e, table, d)
    assert got.dtype == BF and torch.equal(got, want)
    # the ids are read: to change them is an error
    e = sequence.embedding_lookup(ids, table)
    ids += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(e, table, d)


# ------------------------------------------------------------------ more threads than one launch may have (2^32)
@pytest.fixture
def enough_memory():
    def need(gigabytes):
        if MODEL or torch.cuda.mem_get_info()[0] < gigabytes * 2 ** 30:
            pytest.skip("not enough memory on the device")
    if not MODEL:
        torch.cuda.empty_cache()
    yield need
    if not MODEL:
        torch.cuda.empty_cache()


def test_embedding_of_as_many_tokens_as_there_may_be(enough_memory):
    """2^31 - 1 tokens of one channel: the lookup, and the join of 2^26 chunks of 32 sorted tokens.  Counts are exact in 32 bits."""
    enough_memory(90)
    count, vocab = 2 ** 31 - 1, 300
    ids = torch.empty(count, dtype=torch.int32, device="cuda").random_(0, vocab)
    table = leaf(torch.arange(vocab).to(F).view(-1, 1).cuda())
    e = sequence.embedding_lookup(ids, table, dtype=HF)
    for first in range(0, count, 2 ** 28):
        assert torch.equal(e[first:first + 2 ** 28, 0], ids[first:first + 2 ** 28].to(HF))
    counts = torch.zeros(vocab, dtype=torch.int64, device="cuda")
    for first in range(0, count, 2 ** 28):
        counts += torch.bincount(ids[first:first + 2 ** 28], minlength=vocab)
    assert int(counts.max()) < 2 ** 24
    got, = torch.autograd.grad(e, table, torch.ones_like(e))
    assert torch.equal(got[:, 0].long(), counts)


def test_embedding_of_a_table_of_more_rows_than_one_launch_fills(enough_memory):
    enough_memory(40)
    vocab = 2 ** 30 + 1000
    table = torch.empty(vocab, 2, dtype=HF, device="cuda").fill_(1).requires_grad_(True)
    rows = torch.tensor([0, 63, 64, 2 ** 29, 2 ** 30 - 64, 2 ** 30 - 1, 2 ** 30, vocab - 1]).cuda()
    ids = rows.repeat(700)
    got, = torch.autograd.grad(sequence.embedding_lookup(ids, table), table, torch.ones(ids.numel(), 2, dtype=HF, device="cuda"))
    assert (got[rows] == 700).all()
    got[rows] = 0
    assert not got.any()


def test_recurrence_of_more_sequences_than_one_launch_steps_through(enough_memory):
    """One step of 1.45e9 sequences of 5 channels: a thread has two channels, so three threads each."""
    enough_memory(130)
    n = 1_450_000_000
    x = torch.empty(n, 1, 5, device="cuda").fill_(0.25)
    x[-1] = 3.0
    x[::1_000_003] = -1.0
    g = torch.tensor([0.0, 1.0, -1.0, 0.5, 2.0]).cuda()
    y, state = sequence.linear_recurrence(x, g)
    assert torch.equal(y, x) and torch.equal(state, x[:, 0])


def test_recurrence_of_more_short_sequences_than_tiles_of_their_own(enough_memory):
    """8 400 000 sequences of 129 steps, of which a tile of 256 rows would have one: sums of -1, 0 and 1 with changing sign, exact in
    every type; in both directions of time."""
    enough_memory(60)
    n, steps = 8_400_000, 129
    x, dy = (torch.empty(n, steps, 1, dtype=BF, device="cuda") for _ in range(2))
    for t in (x, dy):
        t.random_(-1, 2)
    a = torch.tensor([-1.0], device="cuda")
    xs = leaf(x)
    y, state = sequence.linear_recurrence(xs, a)
    dx, = torch.autograd.grad(y, xs, dy)
    sign = (1 - 2 * (torch.arange(steps, device="cuda") % 2)).to(torch.int32).view(1, steps)
    for first in range(0, n, 2 ** 20):
        part = slice(first, first + 2 ** 20)
        v = x[part, :, 0].to(torch.int32) * sign
        want = torch.cumsum(v, 1).to(torch.int32) * sign
        assert torch.equal(y[part, :, 0].to(torch.int32), want) and torch.equal(state[part, 0].to(torch.int32), want[:, -1])
        d = (dy[part, :, 0].to(torch.int32) * sign).flip(1)
        assert torch.equal(dx[part, :, 0].to(torch.int32), (torch.cumsum(d, 1).to(torch.int32)).flip(1) * sign)


def test_recurrence_gradient_per_channel_is_a_sum_over_many_rows(enough_memory):
    """2^28 rows, of which 256 at a time are added up in 32 bits (at most 8 + 2 + 8 roundings), those sums in 64, and the result is rounded
    once.  With a decay of 0 a state is the input itself, and a term of the sum one product."""
    enough_memory(30)
    torch.manual_seed(2)
    x, dy = (torch.empty(2 ** 13, 2 ** 15, 4, device="cuda").uniform_(0, 1) for _ in range(2))
    a = leaf(torch.zeros(4).cuda())
    y, _ = sequence.linear_recurrence(x, a)
    got, = torch.autograd.grad(y, a, dy)
    want = torch.zeros(4, dtype=torch.float64, device="cuda")
    for s in range(0, 2 ** 13, 32):
        want += (x[s:s + 32, :-1].double() * dy[s:s + 32, 1:].double()).sum((0, 1))
    assert ((got.double() - want).abs() <= 20 * R.U * want).all(), (got.double() / want - 1).abs() / R.U


def test_more_rows_and_channels_than_one_launch_may_have_are_refused():
    lib, plan = capi.kernels(), capi.RecurrencePlan()
    a = capi.RecurrenceArgs()
    a.seq.rows = a.seq.steps = 0x7fff0000
    a.seq.sequences, a.channels, a.dtype, a.decay_dtype = 1, 32, capi.FLOAT, capi.FLOAT
    assert lib.daliamdRecurrenceSetup(C.byref(a), C.byref(plan)) == 0
    a.channels = 33
    assert lib.daliamdRecurrenceSetup(C.byref(a), C.byref(plan)) == 3
    b, plan_b = capi.EmbeddingArgs(tokens=2 ** 31 - 1, vocab=9, channels=1024, dtype=capi.FLOAT, out_dtype=capi.FLOAT, index_dtype=capi.INT64), capi.EmbeddingPlan()
    assert lib.daliamdEmbeddingSetup(C.byref(b), C.byref(plan_b)) == 3
    b.channels = 64
    assert lib.daliamdEmbeddingSetup(C.byref(b), C.byref(plan_b)) == 0
