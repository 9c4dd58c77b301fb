"""Operators over batches of sequences on the device, with their gradients: what a model does first with the ragged batches
that a pipeline delivers (mel frames, audio samples, token ids).

  linear_recurrence   h_t = a_t h_{t-1} + x_t, or a gated mean of the past, per channel along each sequence
  block_norm          norm after a block, gate, scaled residual and the norm before the next block, in one pass
  embedding_lookup    scaled rows of a table, with a gradient summed over sorted tokens

torch is plumbing here, as in dali_amd.backend: tensors, the current stream, autograd's bookkeeping.  All arithmetic happens
in libdali_amd_kernels.so (include/dali_amd_kernels.h); there is no CPU fallback.  Work is enqueued on the current stream of
the tensors' device and nothing waits; every call can be captured into a HIP graph.  A tensor that another stream is still
writing, or that another stream goes on using, is the caller's to order, as with any torch operator.

Results do not depend on the order in which the device runs things: the same inputs give the same bits."""
import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _capi as capi

_DTYPE = {torch.float32: capi.FLOAT, torch.float16: capi.FLOAT16, torch.bfloat16: capi.BFLOAT16}
_INDEX = {torch.int32: capi.INT32, torch.int64: capi.INT64}
_FORMS = {"decay": capi.RECURRENCE_DECAY, "gate": capi.RECURRENCE_GATE}
_MAX = 1 << 31
_MAX_ROWS, _MAX_CHANNELS = 0x7fff0000, 1 << 20


# ------------------------------------------------------------------ checks and plumbing
def _on_device(t):
    return t.is_cuda


def _tensor(name, t, device=None, dtypes=None, shape=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if not _on_device(t):
        raise ValueError(f"{name} must be on the GPU: the sequence operators have no CPU fallback")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")
    if dtypes is not None and t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d).replace('torch.', '') for d in dtypes)}, got {t.dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have the shape {tuple(shape)}, got {tuple(t.shape)}")
    return t


def _ptr(t):
    return None if t is None else t.data_ptr()


def _rows(t):
    """t with adjacent channels: itself if its last dimension is dense, else a copy."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _flat(t):
    """(t as [rows, channels], distance between rows): in place where all leading dimensions are one, else a copy."""
    t = _rows(t)
    try:
        m = t.view(-1, t.shape[-1])
    except RuntimeError:
        m = t.reshape(-1, t.shape[-1])
    return m, m.stride(0)


def _call(name, device, *args):
    """A Run entry on the current stream of `device`."""
    fn = getattr(capi.kernels(), name)
    if device.index is None or device.index == torch.cuda.current_device():
        capi.check(fn(C.c_void_p(torch.cuda.current_stream(device).cuda_stream), *args))
    else:
        with torch.cuda.device(device):
            capi.check(fn(C.c_void_p(torch.cuda.current_stream(device).cuda_stream), *args))


def _workspace(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _needs_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ------------------------------------------------------------------ linear recurrence
def _recurrence_args(x, decay, initial, offsets, lengths, form):
    a = capi.RecurrenceArgs()
    a.channels = x.shape[-1]
    a.dtype, a.decay_dtype, a.form, a.per_channel = _DTYPE[x.dtype], _DTYPE[decay.dtype], _FORMS[form], int(decay.dim() == 1)
    if offsets is not None:
        a.seq.offsets, a.seq.index_dtype = offsets.data_ptr(), _INDEX[offsets.dtype]
        a.seq.rows, a.seq.sequences = x.shape[0], offsets.shape[0] - 1
        a.x_row = x.stride(0)
        if decay.dim() != 1:
            a.decay_row = decay.stride(0)
    else:
        a.seq.sequences, a.seq.steps = x.shape[0], x.shape[1]
        a.seq.rows = x.shape[0] * x.shape[1]
        a.x_seq, a.x_row = x.stride(0), x.stride(1)
        if decay.dim() != 1:
            a.decay_seq, a.decay_row = decay.stride(0), decay.stride(1)
        if lengths is not None:
            a.seq.lengths, a.seq.index_dtype = lengths.data_ptr(), _INDEX[lengths.dtype]
    a.x, a.decay, a.initial = x.data_ptr(), decay.data_ptr(), _ptr(initial)
    return a


def _recurrence_forward(x, decay, initial, offsets, lengths, form, final, save):
    a = _recurrence_args(x, decay, initial, offsets, lengths, form)
    if final is None:
        final = torch.empty((a.seq.sequences, a.channels), dtype=torch.float32, device=x.device)
    a.final_state = final.data_ptr()
    plan = capi.RecurrencePlan()
    capi.check(capi.kernels().daliamdRecurrenceSetup(C.byref(a), C.byref(plan)))
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    saved = torch.empty(plan.saved_bytes // 4, dtype=torch.float32, device=x.device) if save else None
    ws = _workspace(plan.forward_workspace_bytes, x.device)
    a.y, a.saved = y.data_ptr(), _ptr(saved)
    _call("daliamdRecurrenceRun", x.device, C.byref(a), C.c_void_p(_ptr(ws)), C.c_size_t(plan.forward_workspace_bytes))
    return y, final, saved


class _LinearRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, decay, initial, offsets, lengths, form):
        y, final, saved = _recurrence_forward(x, decay, initial, offsets, lengths, form, None, True)
        ctx.save_for_backward(x, decay, initial, offsets, lengths, saved)
        ctx.form = form
        ctx.set_materialize_grads(False)
        return y, final

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dfinal):
        x, decay, initial, offsets, lengths, saved = ctx.saved_tensors
        a = _recurrence_args(x, decay, initial, offsets, lengths, ctx.form)
        plan = capi.RecurrencePlan()
        capi.check(capi.kernels().daliamdRecurrenceSetup(C.byref(a), C.byref(plan)))
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        ddecay = torch.empty(decay.shape, dtype=decay.dtype, device=x.device)
        dinitial = torch.empty_like(initial) if initial is not None and ctx.needs_input_grad[2] else None
        if dy is not None:
            dy = _rows(dy)
            a.dy = dy.data_ptr()
            if offsets is not None:
                a.dy_row = dy.stride(0)
            else:
                a.dy_seq, a.dy_row = dy.stride(0), dy.stride(1)
        if dfinal is not None:
            dfinal = dfinal.contiguous()
            a.dfinal = dfinal.data_ptr()
        ws = _workspace(plan.backward_workspace_bytes, x.device)
        a.saved, a.dx, a.ddecay, a.dinitial = saved.data_ptr(), dx.data_ptr(), ddecay.data_ptr(), _ptr(dinitial)
        _call("daliamdRecurrenceBackwardRun", x.device, C.byref(a), C.c_void_p(_ptr(ws)), C.c_size_t(plan.backward_workspace_bytes))
        return dx, ddecay, dinitial, None, None, None


def linear_recurrence(x, decay, *, form="decay", initial_state=None, offsets=None, lengths=None, final_state=None):
    """Linear recurrence along each sequence, every channel for itself; returns (y, state).

      form "decay"   h_t = a_t h_{t-1} + x_t                       a = decay
      form "gate"    h_t = f_t h_{t-1} + (1 - f_t) x_t             f = 1 / (1 + exp(-decay))

    y_t = h_t in x's type; state is h of each sequence's last step, in 32 bits, [sequences, channels].

    x              [batch, steps, channels], or [rows, channels] with `offsets`: float32, float16 or bfloat16.  Adjacent
                   channels have to be adjacent in memory (a copy is made otherwise), rows may be any distance apart, as in
                   a slice of a wider projection.
    decay          of x's shape, or [channels]: the same at every step (exponential smoothing); x's type or float32.
    initial_state  h_0, float32 [sequences, channels]; zeros if None.  To go on with a sequence pass the state of the call
                   before: one step at a time gives what one call over all steps gives, up to rounding.
    offsets        int32 or int64 [sequences + 1], ascending, on the device: sequence s has the rows offsets[s] up to
                   offsets[s + 1].  Sequences may be empty: their state is h_0.
    lengths        int32 or int64 [batch], on the device: only the first lengths[b] steps of x[b] are its sequence.
                   Rows of no sequence (padding, rows in front of the first offset and behind the last) give zeros in y and
                   in the gradients, whatever they hold.  The device reads offsets and lengths: values out of range are
                   clamped, not reported.
    final_state    a float32 tensor [sequences, channels] that receives the state and is returned as such; it may be
                   `initial_state` itself, which is then updated in place.  Not while gradients are recorded.

    Gradients with respect to x, decay and initial_state; the state may be differentiated as well."""
    if form not in _FORMS:
        raise ValueError(f'form must be "decay" or "gate", got {form!r}')
    _tensor("x", x, dtypes=tuple(_DTYPE))
    dev = x.device
    if offsets is not None:
        if lengths is not None:
            raise ValueError("offsets and lengths exclude each other")
        _tensor("offsets", offsets, dev, tuple(_INDEX))
        if offsets.dim() != 1 or offsets.shape[0] < 1:
            raise ValueError(f"offsets must be [sequences + 1], got the shape {tuple(offsets.shape)}")
        if x.dim() != 2:
            raise ValueError(f"x must be [rows, channels] with offsets, got the shape {tuple(x.shape)}")
        sequences = offsets.shape[0] - 1
        if sequences == 0 and x.shape[0]:
            raise ValueError("offsets name no sequence but x has rows")
        offsets = offsets.contiguous()
    else:
        if x.dim() != 3:
            raise ValueError(f"x must be [batch, steps, channels] (or [rows, channels] with offsets), got the shape {tuple(x.shape)}")
        sequences = x.shape[0]
        if lengths is not None:
            _tensor("lengths", lengths, dev, tuple(_INDEX), (sequences,))
            lengths = lengths.contiguous()
    channels = x.shape[-1]
    if not 1 <= channels <= _MAX_CHANNELS or x.numel() // channels > _MAX_ROWS:
        raise ValueError(f"x must have between 1 and {_MAX_CHANNELS} channels and at most {_MAX_ROWS} rows, got the shape {tuple(x.shape)}")
    _tensor("decay", decay, dev, (x.dtype,) if x.dtype == torch.float32 else (x.dtype, torch.float32))
    if tuple(decay.shape) != (channels,) and decay.shape != x.shape:
        raise ValueError(f"decay must have x's shape {tuple(x.shape)} or [{channels}], got {tuple(decay.shape)}")
    if initial_state is not None:
        _tensor("initial_state", initial_state, dev, (torch.float32,), (sequences, channels))
    if final_state is not None:
        _tensor("final_state", final_state, dev, (torch.float32,), (sequences, channels))
        if not final_state.is_contiguous():
            raise ValueError("final_state must be contiguous")
    x, decay = _rows(x), _rows(decay)
    initial = None if initial_state is None else initial_state.contiguous()
    if _needs_grad(x, decay, initial):
        if final_state is not None:
            raise ValueError("final_state cannot be given while gradients are recorded")
        return _LinearRecurrence.apply(x, decay, initial, offsets, lengths, form)
    return _recurrence_forward(x, decay, initial, offsets, lengths, form, final_state, False)[:2]


# ------------------------------------------------------------------ norms around a block
def _block_norm_args(x, gate, residual, post_weight, scale, pre_weight, eps):
    a = capi.BlockNormArgs()
    a.rows, a.channels, a.eps = x.shape[0], x.shape[1], eps
    a.dtype = _DTYPE[x.dtype]
    a.residual_dtype = a.dtype if residual is None else _DTYPE[residual.dtype]
    weight = next((w for w in (post_weight, scale, pre_weight) if w is not None), None)
    a.weight_dtype = a.dtype if weight is None else _DTYPE[weight.dtype]
    a.x, a.x_row = x.data_ptr(), x.stride(0)
    if gate is not None:
        a.gate, a.gate_row = gate.data_ptr(), gate.stride(0)
    if residual is not None:
        a.residual, a.residual_row = residual.data_ptr(), residual.stride(0)
    a.post_weight, a.scale, a.pre_weight = _ptr(post_weight), _ptr(scale), _ptr(pre_weight)
    return a


def _block_norm_forward(x, gate, residual, post_weight, scale, pre_weight, eps, save):
    a = _block_norm_args(x, gate, residual, post_weight, scale, pre_weight, eps)
    hidden = torch.empty(x.shape, dtype=x.dtype if residual is None else residual.dtype, device=x.device)
    normed = torch.empty(x.shape, dtype=x.dtype, device=x.device) if pre_weight is not None else None
    rstd = torch.empty((2, a.rows), dtype=torch.float32, device=x.device) if save else None
    a.hidden, a.normed = hidden.data_ptr(), _ptr(normed)
    if save:
        a.rstd_post, a.rstd_pre = rstd.data_ptr(), rstd.data_ptr() + 4 * a.rows
    _call("daliamdBlockNormRun", x.device, C.byref(a))
    return hidden, normed, rstd


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, residual, post_weight, scale, pre_weight, eps):
        hidden, normed, rstd = _block_norm_forward(x, gate, residual, post_weight, scale, pre_weight, eps, True)
        ctx.save_for_backward(x, gate, residual, post_weight, scale, pre_weight, rstd)
        ctx.eps = eps
        ctx.set_materialize_grads(False)
        return hidden, normed

    @staticmethod
    @once_differentiable
    def backward(ctx, dhidden, dnormed):
        x, gate, residual, post_weight, scale, pre_weight, rstd = ctx.saved_tensors
        a = _block_norm_args(x, gate, residual, post_weight, scale, pre_weight, ctx.eps)
        plan = capi.BlockNormPlan()
        capi.check(capi.kernels().daliamdBlockNormSetup(C.byref(a), C.byref(plan)))
        a.rstd_post, a.rstd_pre = rstd.data_ptr(), rstd.data_ptr() + 4 * a.rows
        if dhidden is not None:
            dhidden = _rows(dhidden)
            a.dhidden, a.dhidden_row = dhidden.data_ptr(), dhidden.stride(0)
        if dnormed is not None:
            dnormed = _rows(dnormed)
            a.dnormed, a.dnormed_row = dnormed.data_ptr(), dnormed.stride(0)
        like = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
        grads = [like(t) for t in (x, gate, residual, post_weight, scale, pre_weight)]
        a.dx, a.dgate, a.dresidual, a.dpost_weight, a.dscale, a.dpre_weight = (_ptr(t) for t in grads)
        ws = _workspace(plan.backward_workspace_bytes, x.device)
        _call("daliamdBlockNormBackwardRun", x.device, C.byref(a), C.c_void_p(_ptr(ws)), C.c_size_t(plan.backward_workspace_bytes))
        return (*grads, None)


def block_norm(x, *, gate=None, residual=None, post_weight=None, scale=None, pre_weight=None, eps=1e-6):
    """What stands between two blocks of a layer, in one pass over the rows; returns (hidden, normed).

      u = x rstd(x) post_weight                 norm after the block       (without post_weight: u = x)
      v = u silu(gate)                          gate                       (without gate: v = u)
      hidden = residual + scale v               scaled residual            (without either: 1 and 0 in its place)
      normed = hidden rstd(hidden) pre_weight   norm before the next block (without pre_weight: None)

    rstd(z) = 1 / sqrt(mean(z^2) + eps) over the channels, silu(g) = g / (1 + exp(-g)).  block_norm(x, pre_weight=w)[1] is
    the plain root mean square norm.

    x, gate, residual  [..., channels] of one shape, up to 16384 channels: float32, float16 or bfloat16; gate has x's type, the
                       residual x's or float32.  Adjacent channels have to be adjacent in memory, rows may be any distance
                       apart.
    weights            [channels], all of one type: x's or float32.

    hidden has the residual's type (x's without one), normed x's; the second norm sees hidden before its rounding.
    Gradients with respect to everything; those of the weights are sums over the rows, in 32 bits and a fixed order."""
    _tensor("x", x, dtypes=tuple(_DTYPE))
    if x.dim() < 1:
        raise ValueError("x must be [..., channels]")
    dev, channels = x.device, x.shape[-1]
    if not 1 <= channels <= capi.BLOCK_NORM_MAX_CHANNELS:
        raise ValueError(f"x must have between 1 and {capi.BLOCK_NORM_MAX_CHANNELS} channels, got {channels}")
    if x.numel() // channels >= _MAX:
        raise ValueError("x must have fewer than 2^31 rows")
    wide = (x.dtype,) if x.dtype == torch.float32 else (x.dtype, torch.float32)
    if gate is not None:
        _tensor("gate", gate, dev, (x.dtype,), x.shape)
    if residual is not None:
        _tensor("residual", residual, dev, wide, x.shape)
    weights = [(n, w) for n, w in (("post_weight", post_weight), ("scale", scale), ("pre_weight", pre_weight)) if w is not None]
    for name, w in weights:
        _tensor(name, w, dev, wide, (channels,))
        if w.dtype != weights[0][1].dtype:
            raise TypeError(f"the weights must have one type: {weights[0][0]} is {weights[0][1].dtype}, {name} is {w.dtype}")
    if not (eps >= 0):
        raise ValueError(f"eps must not be negative, got {eps}")
    shape = x.shape
    x2, g2, r2 = (None if t is None else _flat(t)[0] for t in (x, gate, residual))
    w2 = [None if w is None else w.contiguous() for w in (post_weight, scale, pre_weight)]
    if _needs_grad(x2, g2, r2, *w2):
        hidden, normed = _BlockNorm.apply(x2, g2, r2, *w2, float(eps))
    else:
        hidden, normed, _ = _block_norm_forward(x2, g2, r2, *w2, float(eps), False)
    if len(shape) == 2:
        return hidden, normed
    return hidden.view(shape), None if normed is None else normed.view(shape)


# ------------------------------------------------------------------ embedding lookup
def _embedding_args(ids, table, scale, padding, out_dtype):
    a = capi.EmbeddingArgs()
    a.ids, a.index_dtype, a.tokens = ids.data_ptr(), _INDEX[ids.dtype], ids.numel()
    a.table, a.table_row = table.data_ptr(), table.stride(0)
    a.vocab, a.channels = table.shape
    a.dtype, a.out_dtype = _DTYPE[table.dtype], _DTYPE[out_dtype]
    a.padding, a.scale = padding, scale
    return a


def _embedding_forward(ids, table, scale, padding, out_dtype):
    a = _embedding_args(ids, table, scale, padding, out_dtype)
    out = torch.empty((*ids.shape, table.shape[1]), dtype=out_dtype, device=table.device)
    a.out = out.data_ptr()
    _call("daliamdEmbeddingRun", table.device, C.byref(a))
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale, padding, out_dtype):
        ctx.save_for_backward(table, ids)
        ctx.rest = scale, padding, out_dtype
        return _embedding_forward(ids, table, scale, padding, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        table, ids = ctx.saved_tensors
        a = _embedding_args(ids, table, *ctx.rest)
        plan = capi.EmbeddingPlan()
        capi.check(capi.kernels().daliamdEmbeddingSetup(C.byref(a), C.byref(plan)))
        d, row = _flat(dout)
        dtable = torch.empty(table.shape, dtype=table.dtype, device=table.device)
        ws = _workspace(plan.backward_workspace_bytes, table.device)
        a.dout, a.dout_row, a.dtable = d.data_ptr(), row, dtable.data_ptr()
        _call("daliamdEmbeddingBackwardRun", table.device, C.byref(a), C.c_void_p(_ptr(ws)), C.c_size_t(plan.backward_workspace_bytes))
        return dtable, None, None, None, None


def embedding_lookup(ids, table, *, scale=1.0, padding_idx=None, dtype=None):
    """scale * table[ids], rounded once: [*ids.shape, channels].

    ids          int32 or int64, any shape.  The device reads them: an id outside the table gives a row of zeros and takes no
                 part in the gradient; it is not reported.
    table        [vocab, channels]: float32, float16 or bfloat16; adjacent channels adjacent in memory.
    padding_idx  a row of the table whose gradient stays zero (0 <= padding_idx < vocab, or negative: from the end).
    dtype        type of the result (default: the table's).

    The gradient of the table is dense: for each row, scale times the sum of its tokens' gradients, in 32 bits and in the
    order of the tokens, rounded once."""
    _tensor("table", table, dtypes=tuple(_DTYPE))
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1 or table.shape[0] >= _MAX:
        raise ValueError(f"table must be [vocab, channels], got the shape {tuple(table.shape)}")
    _tensor("ids", ids, table.device, tuple(_INDEX))
    if ids.numel() >= _MAX:
        raise ValueError("ids must be fewer than 2^31")
    dtype = table.dtype if dtype is None else dtype
    if dtype not in _DTYPE:
        raise TypeError(f"dtype must be float32, float16 or bfloat16, got {dtype}")
    padding = -1
    if padding_idx is not None:
        vocab = table.shape[0]
        if not -vocab <= padding_idx < vocab:
            raise ValueError(f"padding_idx must be a row of the table, got {padding_idx} of {vocab}")
        padding = int(padding_idx) % vocab
    ids, table = ids.contiguous(), _rows(table)
    if _needs_grad(table):
        return _Embedding.apply(table, ids, float(scale), padding, dtype)
    return _embedding_forward(ids, table, float(scale), padding, dtype)
