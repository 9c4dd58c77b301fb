"""The sequence operators as a program uses them: captured into graphs and replayed, on other streams and from other threads, two calls
at once, behind a pipeline, and with tensors of more than 2^31 elements.  What a call computes is checked in
test_gpu_sequence.py; equal inputs give equal bits, so most tests here compare with another call."""
import os
import threading

import numpy as np
import pytest
import torch

from dali_amd import sequence
from tests import sequence_reference as R
from tests.test_gpu_sequence import BF, F, HF, decays, layer, layer_parameters, leaf, rand, tokens

MODEL = bool(os.environ.get("DALI_AMD_HIPEMU"))
pytestmark = pytest.mark.gpu
device_only = pytest.mark.skipif(MODEL, reason="graphs, streams and the size of the device's memory are not on the CPU model")


def same(got, want):
    assert len(got) == len(want)
    for k, (g, w) in enumerate(zip(got, want)):
        assert g.shape == w.shape and torch.equal(g, w), f"result {k} differs in {(g != w).sum()} of {g.numel()} values"


# ------------------------------------------------------------------ graphs
class Captured:
    """f's results for inputs copied into the captured ones."""

    def __init__(self, f, inputs, pool=None):
        self.inputs = [t.clone() for t in inputs]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f(*self.inputs)
        torch.cuda.current_stream().wait_stream(side)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, pool=pool):
            self.outputs = f(*self.inputs)

    def __call__(self, *inputs):
        for mine, t in zip(self.inputs, inputs):
            mine.copy_(t)
        self.graph.replay()
        return [t.clone() for t in self.outputs]


def recurrence_step(x, g, dy, dlast, offsets):
    x, g = leaf(x), leaf(g)
    y, state = sequence.linear_recurrence(x, g, form="gate", offsets=offsets)
    return (y.detach(), state.detach()) + torch.autograd.grad((y, state), (x, g), (dy, dlast))


def norm_step(x, gate, residual, w, dh, dn):
    leaves = [leaf(t) for t in (x, gate, residual, w)]
    h, n = sequence.block_norm(leaves[0], gate=leaves[1], residual=leaves[2], post_weight=leaves[3], scale=leaves[3], pre_weight=leaves[3])
    return (h.detach(), n.detach()) + torch.autograd.grad((h, n), leaves, (dh, dn))


def embedding_step(ids, table, de):
    table = leaf(table)
    e = sequence.embedding_lookup(ids, table, scale=3.0, padding_idx=1)
    return (e.detach(),) + torch.autograd.grad(e, table, de)


def recurrence_inputs(seed, rows=3001, c=200, dtype=BF):
    offsets = torch.from_numpy(np.sort(np.random.default_rng(seed).integers(0, rows + 1, 9))).cuda()
    return (rand(seed, rows, c, dtype=dtype), decays(seed + 1, "gate", rows, c, dtype=dtype), rand(seed + 2, rows, c, dtype=dtype),
            rand(seed + 3, 8, c), offsets)


def norm_inputs(seed, rows=700, c=1000):
    return [rand(seed + k, rows, c, dtype=BF) for k in range(3)] + [rand(seed + 3, c, dtype=BF)] + [rand(seed + k, rows, c, dtype=BF) for k in (4, 5)]


def embedding_inputs(seed, count=5000, vocab=300, c=96):
    return tokens(seed, vocab, count), rand(seed + 1, vocab, c), rand(seed + 2, count, c)


STEPS = {"recurrence": (recurrence_step, recurrence_inputs), "norm": (norm_step, norm_inputs), "embedding": (embedding_step, embedding_inputs)}


@device_only
@pytest.mark.parametrize("op", list(STEPS))
def test_captured_training_step_replays(op):
    step, inputs = STEPS[op]
    captured = Captured(step, inputs(100))
    for k in range(4):
        new = inputs(110 + 10 * k)
        got = captured(*new)
        torch.cuda.synchronize()
        same(got, step(*new))           # (eager work between the replays)
        rand(5, 1000, 1000).sum().item()


@device_only
def test_captured_graphs_of_one_pool():
    """Workspaces of both graphs lie in the same memory."""
    a_in, b_in = recurrence_inputs(200), embedding_inputs(210)
    a = Captured(recurrence_step, a_in)
    b = Captured(embedding_step, b_in, pool=a.graph.pool())
    c = Captured(recurrence_step, recurrence_inputs(220, rows=5000), pool=a.graph.pool())
    for k in range(3):
        for captured, step, new in ((a, recurrence_step, recurrence_inputs(230 + 10 * k)), (b, embedding_step, embedding_inputs(231 + 10 * k)),
                                    (c, recurrence_step, recurrence_inputs(232 + 10 * k, rows=5000))):
            got = captured(*new)
            same(got, step(*new))


@device_only
def test_captured_decoding_updates_its_state():
    """One token per replay, the state updated in place, ids read by the device."""
    p = layer_parameters(dtype=BF)
    state, ids, ids_all = torch.zeros(3, 48).cuda(), tokens(240, 60, 3), tokens(241, 60, 3, 6)

    def step(ids):
        e = sequence.embedding_lookup(ids, p["table"], scale=4.0)
        _, n = sequence.block_norm(e, pre_weight=p["w_in"])
        y, _ = sequence.linear_recurrence(n.unsqueeze(1), (n * p["slope"]).unsqueeze(1), form="gate", initial_state=state, final_state=state)
        return (y,)

    captured = Captured(step, [ids])
    state.zero_()
    got = [captured(ids_all[:, t].contiguous())[0] for t in range(6)]
    end = state.clone()
    state.zero_()
    for t in range(6):
        same([got[t]], step(ids_all[:, t].contiguous()))
    assert torch.equal(end, state)


@device_only
def test_captured_layer_as_a_whole():
    p = {k: v for k, v in layer_parameters().items()}
    names = list(p)
    offsets = torch.tensor([0, 30, 31, 31, 108]).cuda()

    def step(ids, dn, *values):
        q = {k: leaf(v) for k, v in zip(names, values)}
        h, n, state = layer(q, ids, offsets, None)
        return (h.detach(), n.detach(), state.detach()) + torch.autograd.grad(n, list(q.values()), dn)

    captured = Captured(step, [tokens(250, 60, 108), rand(251, 108, 48)] + list(p.values()))
    for k in range(3):
        new = [tokens(252 + k, 60, 108), rand(256 + k, 108, 48)] + [v + 0.01 * k for v in p.values()]
        same(captured(*new), step(*new))


# ------------------------------------------------------------------ streams and threads
@device_only
@pytest.mark.parametrize("op", list(STEPS))
def test_on_another_stream(op):
    step, inputs = STEPS[op]
    new = inputs(300)
    want = step(*new)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*new)
    side.synchronize()
    same(got, want)


@pytest.mark.skipif(MODEL or torch.cuda.device_count() < 2, reason="needs a second device")
@pytest.mark.parametrize("op", list(STEPS))
def test_on_a_device_that_is_not_the_current_one(op):
    step, inputs = STEPS[op]
    new = inputs(305)
    same([t.cpu() for t in step(*[t.to("cuda:1") for t in new])], [t.cpu() for t in step(*new)])
    assert torch.cuda.current_device() == 0


@device_only
def test_two_calls_at_once():
    """Workgroups of both chains share the compute units; neither waits for the other."""
    new = [recurrence_inputs(310, rows=20000, c=512), recurrence_inputs(320, rows=30000, c=300, dtype=HF)]
    want = [recurrence_step(*n) for n in new]
    streams = [torch.cuda.Stream() for _ in new]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(recurrence_step(*new[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for g in got[k]:
            same(g, want[k])


@device_only
def test_from_two_threads():
    new = {op: inputs(330) for op, (_, inputs) in STEPS.items()}
    want = {op: STEPS[op][0](*new[op]) for op in STEPS}
    torch.cuda.synchronize()
    got, errors = {}, []

    def work(op):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[op] = STEPS[op][0](*new[op])
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(op,)) for op in STEPS]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for op in STEPS:
        same(got[op], want[op])


# ------------------------------------------------------------------ autograd's rules
@pytest.mark.parametrize("op", list(STEPS))
def test_differentiated_twice_raises(op):
    if op == "recurrence":
        v = leaf(rand(340, 2, 9, 8))
        out = sequence.linear_recurrence(v, v.detach().sigmoid())[0]
    elif op == "norm":
        v = leaf(rand(341, 4, 16))
        out = sequence.block_norm(v, pre_weight=torch.ones(16).to(v.device))[1]
    else:
        v = leaf(rand(342, 7, 8))
        out = sequence.embedding_lookup(tokens(343, 7, 5), v)
    g, = torch.autograd.grad(out.sum(), v, create_graph=True)
    assert not torch.isnan(g).any()
    with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
        torch.autograd.grad(g.sum(), v, allow_unused=True, retain_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
        (out.sum() + g.pow(2).sum()).backward()


def test_state_written_in_place_under_a_backward_pass_raises():
    x, g, state = leaf(rand(350, 2, 5, 8)), rand(351, 2, 5, 8), rand(352, 2, 8)
    y, _ = sequence.linear_recurrence(x, g, form="gate", initial_state=state)
    with torch.no_grad():
        sequence.linear_recurrence(x, g, form="gate", initial_state=state, final_state=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_inference_mode():
    x, g = rand(353, 2, 300, 8), rand(354, 2, 300, 8)
    y, _ = sequence.linear_recurrence(x, g, form="gate")
    with torch.inference_mode():
        state = torch.zeros(2, 8).to(x.device)
        z, last = sequence.linear_recurrence(x, g, form="gate", initial_state=state, final_state=state)
        assert torch.equal(y, z) and last.data_ptr() == state.data_ptr()
        h, n = sequence.block_norm(x, pre_weight=torch.ones(8).to(x.device))
        e = sequence.embedding_lookup(tokens(355, 2, 3), x[:, 0])
    assert n.shape == x.shape and e.shape == (3, 8)


@pytest.mark.parametrize("op", list(STEPS))
def test_gradients_of_broadcast_inputs(op):
    """An expanded input (stride 0) gets the sum of its places' gradients; an expanded gradient is read as such."""
    if op == "recurrence":
        small = leaf(decays(360, "gate", 1, 1, 24))
        x = rand(361, 3, 40, 24)
        y, _ = sequence.linear_recurrence(x, small.expand(3, 40, 24), form="gate")
        got, = torch.autograd.grad(y.sum(), small)
        full = leaf(small.expand(3, 40, 24).contiguous())
        z, _ = sequence.linear_recurrence(x, full, form="gate")
        want, = torch.autograd.grad(z, full, torch.ones_like(z))
        assert torch.equal(y, z)
        terms = 120
    elif op == "norm":
        small = leaf(rand(362, 1, 40))
        x = rand(363, 50, 40)
        h, _ = sequence.block_norm(x, gate=small.expand(50, 40))
        got, = torch.autograd.grad(h.sum(), small)
        full = leaf(small.expand(50, 40).contiguous())
        h2, _ = sequence.block_norm(x, gate=full)
        want, = torch.autograd.grad(h2, full, torch.ones_like(h2))
        assert torch.equal(h, h2)
        terms = 50
    else:
        small = leaf(rand(364, 1, 16))
        ids = tokens(365, 9, 200)
        e = sequence.embedding_lookup(ids, small.expand(9, 16))
        got, = torch.autograd.grad(e.sum(), small)
        full = leaf(small.expand(9, 16).contiguous())
        e2 = sequence.embedding_lookup(ids, full)
        want, = torch.autograd.grad(e2, full, torch.ones_like(e2))
        assert torch.equal(e, e2)
        terms = 9
    want = want.double().reshape(-1, want.shape[-1])
    # the same numbers added up by torch, in 32 bits
    assert ((got.double().reshape(-1) - want.sum(0)).abs() <= terms * R.U * want.abs().sum(0)).all()


# ------------------------------------------------------------------ more than 2^31 elements
@device_only
def test_recurrence_of_more_than_2_31_elements():
    c, rows = 32768, 66001                       # 2.16e9 elements
    g = decays(400, "gate", c)
    x = torch.empty(rows, c, dtype=BF, device="cuda").fill_(0.5)
    x[-700:] = rand(401, 700, c, dtype=BF)
    offsets = torch.tensor([0, rows - 700, rows - 1, rows]).cuda()
    y, state = sequence.linear_recurrence(x, g, form="gate", offsets=offsets)
    tail = torch.tensor([0, 699, 700]).cuda()
    want, last = sequence.linear_recurrence(x[-700:], g, form="gate", offsets=tail)
    # (the tiles lie elsewhere in the sequence: other sums in 32 bits, rounded to bf16 at most one step apart)
    assert ((y[-700:].float() - want.float()).abs() <= 2 ** -7 * want.float().abs() + 1e-5).all()
    assert ((state[1:] - last).abs() <= 800 * R.U * (1 + last.abs())).all()
    assert ((y[60000:rows - 700:997].float() - 0.5).abs() <= 2 ** -8).all()    # the mean of a constant
    del y, want
    xs, dy = leaf(x), torch.zeros(rows, c, dtype=BF, device="cuda")
    dy[-1] = 1
    y, _ = sequence.linear_recurrence(xs, g, form="gate", offsets=offsets)
    dx, = torch.autograd.grad(y, xs, dy)
    k = 1 / (1 + torch.exp(g.double()))
    assert ((dx[-1].double() - k).abs() <= (2 ** -8 + 20 * R.U) * k).all() and not dx[:-1].any()


@device_only
def test_norm_of_more_than_2_31_elements():
    c, rows = 16384, 132000
    x = torch.empty(rows, c, dtype=BF, device="cuda").fill_(2.0)
    x[-3:] = rand(410, 3, c, dtype=BF)
    w = rand(411, c, dtype=BF)
    h, n = sequence.block_norm(x, pre_weight=w)
    same([h[-3:], n[-3:]], sequence.block_norm(x[-3:], pre_weight=w))
    assert torch.equal(n[131000], n[0])
    del h
    xs = leaf(x)
    _, m = sequence.block_norm(xs, pre_weight=w)
    dn = torch.zeros_like(m)
    dn[-3:] = 1
    dx, = torch.autograd.grad(m, xs, dn)
    ys = leaf(x[-3:])
    want, = torch.autograd.grad(sequence.block_norm(ys, pre_weight=w)[1], ys, dn[-3:])
    same([dx[-3:]], [want])
    assert not dx[:-3].any()


@device_only
def test_embedding_of_more_than_2_31_elements():
    c, vocab = 16384, 132000
    table = torch.zeros(vocab, c, dtype=BF, device="cuda")
    table[-2:] = rand(420, 2, c, dtype=BF)
    ids = torch.tensor([vocab - 1, 0, vocab - 2, vocab - 1]).cuda()
    e = sequence.embedding_lookup(ids, table)
    assert torch.equal(e[0], table[-1]) and torch.equal(e[2], table[-2]) and torch.equal(e[3], table[-1]) and not e[1].any()
    many = torch.zeros(vocab, dtype=torch.int64, device="cuda")
    many[-1] = vocab - 1
    e = sequence.embedding_lookup(many, table)       # a result of as many elements
    assert torch.equal(e[-1], table[-1]) and not e[:-1].any()
    del e
    ts, de = leaf(table), rand(421, 4, c, dtype=BF)
    d, = torch.autograd.grad(sequence.embedding_lookup(ids, ts), ts, de)
    sums = de[0].double() + de[3].double()
    assert ((d[-1].double() - sums).abs() <= (2 ** -8 + 2 * R.U) * sums.abs()).all()
    assert torch.equal(d[-2], de[2]) and torch.equal(d[0], de[1]) and not d[1:-2].any()


# ------------------------------------------------------------------ behind a pipeline
def test_behind_a_pipeline():
    """Ragged mel frames of a pipeline, packed, smoothed along time by a learned gate per mel channel and normalised."""
    from dali_amd import fn
    from dali_amd.pipeline import Pipeline
    from dali_amd.plugin.pytorch import block_norm, linear_recurrence, packed_rows

    rng = np.random.default_rng(430)
    audio = [rng.normal(0, 0.3, n).astype(np.float32) for n in (4000, 16000, 700, 9111)]
    pipe = Pipeline(batch_size=4, num_threads=2, device_id=0)
    with pipe:
        a = fn.external_source(source=lambda: audio, name="audio")
        spec = fn.spectrogram(a.gpu(), nfft=512, window_length=400, window_step=160)
        pipe.set_outputs(fn.to_decibels(fn.mel_filter_bank(spec, nfilter=80, sample_rate=16000.0), cutoff_db=-80.0))
    pipe.build()
    for _ in range(2):
        mel, = pipe.run()
        parts = [np.asarray(mel[k].as_cpu()) for k in range(4)]
        x, offsets = packed_rows(mel, axis=1)
        if MODEL:
            x, offsets = x.cpu(), offsets.cpu()
        ends = np.cumsum([0] + [p.shape[1] for p in parts])
        assert offsets.tolist() == ends.tolist() and x.shape == (ends[-1], 80)
        assert np.array_equal(x.cpu().numpy(), np.concatenate([p.T for p in parts]))
        logits, w = leaf(rand(431, 80, shift=1.0)), leaf(rand(432, 80))
        y, state = linear_recurrence(x, logits, form="gate", offsets=offsets)
        h, n = block_norm(y, pre_weight=w)
        dn = rand(433, *n.shape)
        dlogits, dw = torch.autograd.grad(n, (logits, w), dn)
        spans = list(zip(ends[:-1], ends[1:]))
        ref = R.recurrence(R.f64(x), R.f64(logits), "gate", spans)
        R.check("y", y, ref["y"], F, ref["y_slack"])
        R.check("state", state, ref["state"], F, ref["state_slack"])
        yy = torch.from_numpy(ref["y"])
        normed = yy / torch.sqrt((yy * yy).mean(-1, keepdim=True) + 1e-6)
        err = ref["y_slack"].max() if np.ndim(ref["y_slack"]) else ref["y_slack"]
        rms = np.sqrt((ref["y"] ** 2).mean(-1)).min()
        # what y may be off moves a row by at most that, and its norm by as much again
        bound = (100 * R.U * normed.abs().max() + 2 * (err + R.U * np.abs(ref["y"]).max()) / rms) * w.detach().cpu().double().abs().max()
        assert (n.detach().cpu().double() - normed * w.detach().cpu().double()).abs().max() <= bound
        assert torch.isfinite(dlogits).all() and torch.isfinite(dw).all() and dlogits.any() and dw.any()
