"""Cases of the sequence operators (dali_amd.sequence): linear recurrence, block norm, embedding lookup.

`own` False: the operators in elementary torch operations; `own` True: the calls of a user of dali_amd.sequence."""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ITEM = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


def listed():
    return [
        # one token for each running request, the state of each in hand
        {"name": "recurrence step", "op": "recurrence", "pass": "forward", "form": "gate", "dtype": "bf16", "gate_dtype": "bf16", "seqs": 96,
         "rows": 96, "channels": 2048, "ragged": False, "per_channel": False, "initial": True},
        # prompts of very different lengths, packed back to back
        {"name": "recurrence prompts", "op": "recurrence", "pass": "forward", "form": "gate", "dtype": "bf16", "gate_dtype": "bf16", "seqs": 21,
         "rows": 20011, "channels": 1536, "ragged": True, "per_channel": False, "initial": True},
        # one long recording: few channels, the work has to be split along time
        {"name": "recurrence long", "op": "recurrence", "pass": "forward", "form": "decay", "dtype": "f16", "gate_dtype": "f32", "seqs": 1,
         "rows": 65536, "channels": 512, "ragged": False, "per_channel": False, "initial": False},
        # learned smoothing of 80 mel channels over a batch of 64 utterances, a training step
        {"name": "recurrence mel frames", "op": "recurrence", "pass": "train", "form": "gate", "dtype": "f32", "gate_dtype": "f32", "seqs": 64,
         "rows": 56111, "channels": 80, "ragged": True, "per_channel": True, "initial": True},
        # a layer's training step
        {"name": "recurrence training", "op": "recurrence", "pass": "train", "form": "gate", "dtype": "bf16", "gate_dtype": "bf16", "seqs": 8,
         "rows": 32768, "channels": 2048, "ragged": False, "per_channel": False, "initial": False},
        # one token for each running request, every part in use
        {"name": "norm step", "op": "norm", "pass": "forward", "dtype": "bf16", "residual_dtype": "bf16", "rows": 48, "channels": 4096,
         "post": True, "gate": True, "residual": True, "scale": True, "pre": True},
        # the gated output norm of a block of an odd width
        {"name": "norm gated odd", "op": "norm", "pass": "train", "dtype": "f16", "residual_dtype": "f16", "rows": 5003, "channels": 1111,
         "post": True, "gate": True, "residual": False, "scale": False, "pre": False},
        # between two blocks of a layer, residual stream in 32 bits, a training step
        {"name": "norm training", "op": "norm", "pass": "train", "dtype": "bf16", "residual_dtype": "f32", "rows": 32768, "channels": 2048,
         "post": True, "gate": True, "residual": True, "scale": True, "pre": True},
        # one token for each running request
        {"name": "embedding step", "op": "embedding", "pass": "forward", "dtype": "bf16", "tokens": 96, "vocab": 32000, "channels": 2048,
         "padding": False},
        # the tokens of a large batch
        {"name": "embedding batch", "op": "embedding", "pass": "forward", "dtype": "bf16", "tokens": 131072, "vocab": 64000, "channels": 2048,
         "padding": False},
        # characters or words of short texts, padded to one length
        {"name": "embedding odd", "op": "embedding", "pass": "train", "dtype": "f32", "tokens": 4095, "vocab": 5003, "channels": 300,
         "padding": True},
        # a training step's tokens, frequent ones thousands of times
        {"name": "embedding training", "op": "embedding", "pass": "train", "dtype": "bf16", "tokens": 65536, "vocab": 48000, "channels": 1024,
         "padding": False},
    ]


def _spread(rng, low, high):
    """A whole number between the two, even in its logarithm; every other one odd."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return min(high, max(low, v | 1 if rng.random() < 0.5 else v))


def draw(rng):
    op = rng.choice(["recurrence", "norm", "embedding"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "recurrence":
        channels = _spread(rng, 40, 4096)
        rows = _spread(rng, 16, min(131072, (1 << 25) // channels))
        seqs = min(_spread(rng, 1, 128), rows)
        ragged = rng.random() < 0.6
        per_channel = rng.random() < 0.25
        return {"op": op, "pass": rng.choice(["forward", "train"]), "form": rng.choice(["gate", "gate", "decay"]), "dtype": dtype,
                "gate_dtype": "f32" if per_channel else rng.choice([dtype, dtype, "f32"]), "seqs": seqs,
                "rows": rows if ragged else rows // seqs * seqs, "channels": channels, "ragged": ragged, "per_channel": per_channel,
                "initial": rng.random() < 0.5}
    if op == "norm":
        channels = _spread(rng, 40, 8192)
        case = {"op": op, "pass": rng.choice(["forward", "train"]), "dtype": dtype, "residual_dtype": rng.choice([dtype, "f32"]),
                "rows": _spread(rng, 8, (1 << 25) // channels), "channels": channels}
        case.update({k: rng.random() < 0.6 for k in ("post", "gate", "residual", "scale")})
        case["pre"] = rng.random() < 0.6 or not (case["post"] or case["gate"] or case["residual"] or case["scale"])
        if not case["residual"]:
            case["residual_dtype"] = dtype
        return case
    channels = _spread(rng, 40, 4096)
    return {"op": op, "pass": rng.choice(["forward", "train"]), "dtype": dtype, "tokens": _spread(rng, 16, min(131072, (1 << 26) // channels)),
            "vocab": _spread(rng, 30, min(128000, (1 << 26) // channels)), "channels": channels, "padding": rng.random() < 0.3}


def _lengths(case, seed):
    """The sequences' lengths: equal ones, or spread over a factor of ten around their mean."""
    rows, seqs = case["rows"], case["seqs"]
    if not case["ragged"]:
        return np.full(seqs, rows // seqs, np.int64)
    w = np.exp(np.random.RandomState(seed % (1 << 31)).normal(0, 0.7, seqs))
    ends = np.floor(np.cumsum(w) / w.sum() * rows + 0.5).astype(np.int64)
    ends[-1] = rows
    return np.diff(ends, prepend=0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["dtype"]]
    train = case["pass"] == "train"

    def normal(*shape, dtype=dt, scale=1.0, shift=0.0):
        return (torch.randn(shape, device="cuda", generator=gen) * scale + shift).to(dtype)

    s = dict(case)
    c = case["channels"]
    if case["op"] == "recurrence":
        lengths = _lengths(case, seed)
        shape = (case["rows"], c) if case["ragged"] else (case["seqs"], case["rows"] // case["seqs"], c)
        gate_dt = TYPES[case["gate_dtype"]]
        s["longest"] = int(lengths.max())
        s["x"] = normal(*shape)
        logits = normal(*((c,) if case["per_channel"] else shape), dtype=torch.float32, scale=1.2, shift=3.0)
        # decays stay away from 1, where their own rounding to few bits would be all that is seen
        s["gate"] = (logits if case["form"] == "gate" else torch.sigmoid(logits.clamp(max=5.0))).to(gate_dt)
        s["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)).cuda()
        s["state"] = normal(case["seqs"], c, dtype=torch.float32) if case["initial"] else None
        s["dy"] = normal(*shape) if train else None
        s["dlast"] = normal(case["seqs"], c, dtype=torch.float32) if train else None
        s["leaves"] = [s["x"], s["gate"]] + ([s["state"]] if case["initial"] else [])
    elif case["op"] == "norm":
        rdt = TYPES[case["residual_dtype"]]
        s["x"] = normal(case["rows"], c, scale=1.7)
        s["g"] = normal(case["rows"], c) if case["gate"] else None
        s["r"] = normal(case["rows"], c, dtype=rdt, scale=2.0) if case["residual"] else None
        s["w_post"] = normal(c, scale=0.2, shift=1.0) if case["post"] else None
        s["s"] = normal(c, scale=0.1, shift=0.3) if case["scale"] else None
        s["w_pre"] = normal(c, scale=0.2, shift=1.0) if case["pre"] else None
        s["dh"] = normal(case["rows"], c, dtype=rdt) if train else None
        s["dn"] = normal(case["rows"], c) if train and case["pre"] else None
        s["leaves"] = [t for t in (s["x"], s["g"], s["r"], s["w_post"], s["s"], s["w_pre"]) if t is not None]
    else:
        u = torch.rand(case["tokens"], device="cuda", generator=gen)
        # frequency falls with the rank, as words' does
        s["ids"] = (torch.exp(u.double() * math.log(case["vocab"])) - 1).long().clamp(0, case["vocab"] - 1)
        s["factor"] = math.sqrt(c)
        s["pad"] = None
        if case["padding"]:
            s["pad"] = case["vocab"] - 1
            s["ids"][torch.rand(case["tokens"], device="cuda", generator=gen) < 0.3] = s["pad"]
        s["table"] = normal(case["vocab"], c, scale=0.05)
        s["dy"] = normal(case["tokens"], c) if train else None
        s["leaves"] = [s["table"]]
    if train:
        for t in s["leaves"]:
            t.requires_grad_(True)
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------------

def _scan(a, b, longest):
    """h_t = a_t h_{t-1} + b_t along dim 0, by doubling: after a step each row holds the composition of twice as many."""
    d = 1
    while d < longest:
        b = torch.cat([b[:d], b[d:] + a[d:] * b[:-d]])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def _plain_recurrence(s):
    dt, gdt = s["x"].dtype, s["gate"].dtype
    # a decay of one channel is the same at every step: what its rounding in 32 bits is off adds up over the steps
    wide = torch.float64 if s["per_channel"] else torch.float32
    c, rows, seqs = s["channels"], s["rows"], s["seqs"]
    x = s["x"].detach().to(wide).reshape(rows, c)
    g = s["gate"].detach().to(wide)
    g = g.reshape(-1, c).expand(rows, c)
    off = s["offsets"].long()
    live = off[1:] > off[:-1]
    first, last = off[:-1][live], off[1:][live] - 1
    if s["form"] == "gate":
        a, k = 1 / (1 + torch.exp(-g)), 1 / (1 + torch.exp(g))
        b = k * x
    else:
        a, k, b = g, None, x.clone()
    h0 = torch.zeros(seqs, c, device=x.device, dtype=wide) if s["state"] is None else s["state"].detach().to(wide)
    b = b.index_add(0, first, a[first] * h0[live])
    cut = a.clone()
    cut[first] = 0
    y = _scan(cut, b, s["longest"])
    state = h0.clone()
    state[live] = y[last]
    out = {"y": y.to(dt).reshape(s["x"].shape), "state": state.float()}
    if s["pass"] == "train":
        dy = s["dy"].to(wide).reshape(rows, c).index_add(0, last, s["dlast"].to(wide)[live])
        nxt = torch.cat([a[1:], a[:1]])
        nxt[last] = 0
        lam = _scan(nxt.flip(0), dy.flip(0), s["longest"]).flip(0)
        before = torch.cat([y[:1], y[:-1]])
        before[first] = h0[live]
        if s["form"] == "gate":
            dx, dg = k * lam, lam * (before - x) * a * k
        else:
            dx, dg = lam, lam * before
        out["dx"] = dx.to(dt).reshape(s["x"].shape)
        out["dgate"] = (dg.double().sum(0) if s["per_channel"] else dg).to(gdt).reshape(s["gate"].shape)
        if s["state"] is not None:
            dinit = s["dlast"].to(wide).clone()
            dinit[live] = (a * lam)[first]
            out["dinitial"] = dinit.float()
    return out


def _plain_norm(s):
    dt = s["x"].dtype
    f = {k: None if s[k] is None else s[k].detach().float() for k in ("x", "g", "r", "w_post", "s", "w_pre", "dh", "dn")}
    x = f["x"]
    u, rs1, xh = x, None, None
    if f["w_post"] is not None:
        rs1 = 1 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)
        xh = x * rs1
        u = xh * f["w_post"]
    sig = None if f["g"] is None else 1 / (1 + torch.exp(-f["g"]))
    v = u if sig is None else u * f["g"] * sig
    h = v if f["s"] is None else v * f["s"]
    h = h if f["r"] is None else h + f["r"]
    out = {"h": h.to(TYPES[s["residual_dtype"]])}
    dr = f["dh"]
    if f["w_pre"] is not None:
        rs2 = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
        hh = h * rs2
        out["n"] = (hh * f["w_pre"]).to(dt)
        if s["pass"] == "train":
            d = f["dn"] * f["w_pre"]
            dr = dr + rs2 * (d - hh * (d * hh).mean(1, keepdim=True))
            out["dw_pre"] = (f["dn"] * hh).double().sum(0).to(dt)
    if s["pass"] == "train":
        if f["r"] is not None:
            out["dr"] = dr.to(s["r"].dtype)
        dv = dr
        if f["s"] is not None:
            out["ds"] = (dr * v).double().sum(0).to(dt)
            dv = dr * f["s"]
        du = dv
        if sig is not None:
            out["dg"] = (dv * u * sig * (1 + f["g"] * (1 - sig))).to(dt)
            du = dv * f["g"] * sig
        dx = du
        if rs1 is not None:
            out["dw_post"] = (du * xh).double().sum(0).to(dt)
            d = du * f["w_post"]
            dx = rs1 * (d - xh * (d * xh).mean(1, keepdim=True))
        out["dx"] = dx.to(dt)
    return out


def _plain_embedding(s):
    table, ids = s["table"].detach(), s["ids"]
    out = {"e": (table[ids].float() * s["factor"]).to(table.dtype)}
    if s["pass"] == "train":
        d = s["dy"].float() * s["factor"]
        if s["pad"] is not None:
            d = d * (ids != s["pad"]).unsqueeze(1)
        out["dtable"] = torch.zeros(table.shape, device=table.device).index_add_(0, ids, d).to(table.dtype)
    return out


# ---- the framework's operators -----------------------------------------------------------------------------------------

def _own_recurrence(s):
    from dali_amd import sequence
    y, state = sequence.linear_recurrence(s["x"], s["gate"], form=s["form"], initial_state=s["state"],
                                          offsets=s["offsets"] if s["ragged"] else None)
    out = {"y": y, "state": state}
    if s["pass"] == "train":
        out.update(zip(("dx", "dgate", "dinitial"), torch.autograd.grad((y, state), s["leaves"], (s["dy"], s["dlast"]))))
    return out


def _own_norm(s):
    from dali_amd import sequence
    h, n = sequence.block_norm(s["x"], gate=s["g"], residual=s["r"], post_weight=s["w_post"], scale=s["s"], pre_weight=s["w_pre"], eps=EPS)
    out = {"h": h}
    if n is not None:
        out["n"] = n
    if s["pass"] == "train":
        names = [k for k, t in zip(("dx", "dg", "dr", "dw_post", "ds", "dw_pre"), (s["x"], s["g"], s["r"], s["w_post"], s["s"], s["w_pre"]))
                 if t is not None]
        outs, grads = ((h, n), (s["dh"], s["dn"])) if n is not None else ((h,), (s["dh"],))
        out.update(zip(names, torch.autograd.grad(outs, s["leaves"], grads)))
    return out


def _own_embedding(s):
    from dali_amd import sequence
    e = sequence.embedding_lookup(s["ids"], s["table"], scale=s["factor"], padding_idx=s["pad"])
    out = {"e": e}
    if s["pass"] == "train":
        out["dtable"], = torch.autograd.grad((e,), s["leaves"], (s["dy"],))
    return out


def run(state):
    if own:
        return {"recurrence": _own_recurrence, "norm": _own_norm, "embedding": _own_embedding}[state["op"]](state)
    with torch.no_grad():
        return {"recurrence": _plain_recurrence, "norm": _plain_norm, "embedding": _plain_embedding}[state["op"]](state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------

def work(case):
    c, e, train = case["channels"], ITEM[case["dtype"]], case["pass"] == "train"
    if case["op"] == "recurrence":
        n, ge = case["rows"] * c, ITEM[case["gate_dtype"]]
        gate = c * 4 if case["per_channel"] else n * ge
        states = case["seqs"] * c * 4
        b = n * e * 2 + gate + states * (2 if case["initial"] else 1)
        if train:
            b += n * e * 2 + gate + states * (2 if case["initial"] else 1)
        return {"bytes": b, "flops": n * ((6 if case["form"] == "gate" else 2) + (14 if train else 0))}
    if case["op"] == "norm":
        n, re = case["rows"] * c, ITEM[case["residual_dtype"]]
        parts = 1 + case["gate"]
        b = n * (e * parts + re * (1 + case["residual"]) + e * case["pre"])
        if train:
            b += n * (re * (1 + case["residual"]) + e * case["pre"] + e * parts)
        return {"bytes": b, "flops": n * (4 * case["post"] + 6 * case["gate"] + case["residual"] + case["scale"] + 4 * case["pre"]) * (3 if train else 1)}
    t, v = case["tokens"], case["vocab"]
    rank = np.arange(1, v + 1, dtype=np.float64)
    p = np.log((rank + 1) / rank) / math.log(v + 1)
    touched = float(np.sum(-np.expm1(t * np.log1p(-p)))) if v > 1 else 1.0
    b = t * 8 + touched * c * e + t * c * e
    if train:
        b += t * c * e + v * c * e
    return {"bytes": b, "flops": t * c * (3 if train else 1)}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def _exact_recurrence(s):
    """Step by step along time, all sequences at once; rows of a sequence that has ended are left alone."""
    c, seqs = s["channels"], s["seqs"]
    x = s["x"].detach().double().reshape(-1, c)
    g = s["gate"].detach().double().reshape(-1, c)
    keep, take = (torch.sigmoid(g), torch.sigmoid(-g)) if s["form"] == "gate" else (g, torch.ones_like(g))
    one = s["per_channel"]
    off = s["offsets"].long()
    begin, length = off[:-1], off[1:] - off[:-1]
    order = torch.argsort(length, descending=True)
    sizes = length[order].cpu().numpy()
    counts = np.searchsorted(-sizes, -np.arange(s["longest"]), side="left")
    h = torch.zeros(seqs, c, device=x.device, dtype=torch.float64) if s["state"] is None else s["state"].detach().double()[order]
    y, before = torch.empty_like(x), torch.empty_like(x)
    start = begin[order]
    for t, k in enumerate(counts):
        at = start[:k] + t
        before[at] = h[:k]
        h[:k] = (keep if one else keep[at]) * h[:k] + (take if one else take[at]) * x[at]
        y[at] = h[:k]
    back = torch.argsort(order)
    out = {"y": y.reshape(s["x"].shape), "state": h[back]}
    if s["pass"] == "train":
        dy = s["dy"].double().reshape(-1, c)
        lam, dx = s["dlast"].double()[order], torch.empty_like(x)
        dg = torch.empty_like(x)
        for t in range(s["longest"] - 1, -1, -1):
            k = counts[t]
            at = start[:k] + t
            f, i = (keep, take) if one else (keep[at], take[at])
            lam[:k] += dy[at]
            dx[at] = i * lam[:k]
            dg[at] = lam[:k] * (before[at] - x[at]) * f * i if s["form"] == "gate" else lam[:k] * before[at]
            lam[:k] *= f
        out["dx"] = dx.reshape(s["x"].shape)
        out["dgate"] = dg.sum(0) if one else dg.reshape(s["gate"].shape)
        if s["state"] is not None:
            out["dinitial"] = lam[back]
    return out


def _exact_norm(s):
    """The forward formula in 64 bits, its gradients by automatic differentiation."""
    names = {"x": "dx", "g": "dg", "r": "dr", "w_post": "dw_post", "s": "ds", "w_pre": "dw_pre"}
    f = {k: None if s[k] is None else s[k].detach().double().requires_grad_(s["pass"] == "train") for k in names}
    z = f["x"]
    if f["w_post"] is not None:
        z = f["w_post"] * z * torch.rsqrt(z.pow(2).mean(-1, keepdim=True) + EPS)
    if f["g"] is not None:
        z = z * (f["g"] * torch.sigmoid(f["g"]))
    if f["s"] is not None:
        z = f["s"] * z
    if f["r"] is not None:
        z = f["r"] + z
    out, outs, grads = {"h": z.detach()}, [z], [s["dh"]]
    if f["w_pre"] is not None:
        n = f["w_pre"] * z * torch.rsqrt(z.pow(2).mean(-1, keepdim=True) + EPS)
        out["n"] = n.detach()
        outs, grads = outs + [n], grads + [s["dn"]]
    if s["pass"] == "train":
        have = [k for k in names if f[k] is not None]
        out.update(zip((names[k] for k in have), torch.autograd.grad(outs, [f[k] for k in have], [t.double() for t in grads])))
    return out


def _exact_embedding(s):
    table, ids = s["table"].detach().double(), s["ids"]
    out = {"e": table.index_select(0, ids) * s["factor"]}
    if s["pass"] == "train":
        # sums of runs of the sorted tokens, as differences of running sums
        order = torch.argsort(ids, stable=True)
        running = torch.cumsum(s["dy"].double()[order], 0)
        vocab = torch.arange(s["vocab"], device=ids.device)
        hi = torch.searchsorted(ids[order], vocab, right=True)
        running = torch.cat([torch.zeros_like(running[:1]), running])
        d = running[hi] - running[torch.cat([torch.zeros_like(hi[:1]), hi[:-1]])]
        if s["pad"] is not None:
            d[s["pad"]] = 0
        out["dtable"] = d * s["factor"]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"recurrence": _exact_recurrence, "norm": _exact_norm, "embedding": _exact_embedding}[case["op"]](s)
