"""Operators over batches of sequences on the device, with their gradients: what a model does first with the ragged batches
that a pipeline delivers (mel frames, audio samples, token ids).

  linear_recurrence   h_t = a_t h_{t-1} + x_t, or a gated mean of the past, per channel along each sequence
  block_norm          norm after a block, gate, scaled residual and the norm before the next block, in one pass
  embedding_lookup    scaled rows of a table, with a gradient summed over sorted tokens

torch is plumbing here, as in dali_amd.backend: tensors, the current stream, autograd's bookkeeping (plugin/csrc/sequence.cpp).
All arithmetic happens in libdali_amd_kernels.so (include/dali_amd_kernels.h); there is no CPU fallback.  Work is enqueued on the current stream of
the tensors' device and nothing waits; every call can be captured into a HIP graph.  A tensor that another stream is still
writing, or that another stream goes on using, is the caller's to order, as with any torch operator.

Gradients are backward ones, of first order.  Forward-mode derivatives, a second differentiation and tracing (torch.jit.trace, make_fx)
are refused: they would not see the kernels.

Results do not depend on the order in which the device runs things: the same inputs give the same bits."""
import importlib.util
import os

import torch  # noqa: F401  (the module below is linked against torch's libraries)

from . import _capi as capi

_MODULE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "_sequence.so")
_HOST_MEMORY = False    # the kernel library is a model of the kernels on the CPU (tests)
_module = None


def _ops():
    """The compiled module, bound to the kernel library.  Raises if either has not been built."""
    global _module
    if _module is None:
        if not os.path.exists(_MODULE):
            raise capi.DaliAmdError(f"{_MODULE} is missing: the PyTorch module of the sequence operators has not been built "
                                    "(run `python -c 'import __graft_entry__ as g; g.build()'`).")
        capi.kernels()
        spec = importlib.util.spec_from_file_location("_sequence", _MODULE)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.bind(capi.KERNELS_LIB, capi.DaliAmdError, _HOST_MEMORY)
        _module = module
    return _module


def linear_recurrence(x, decay, *, form="decay", initial_state=None, offsets=None, lengths=None, final_state=None):
    """Linear recurrence along each sequence, every channel for itself; returns (y, state).

      form "decay"   h_t = a_t h_{t-1} + x_t                       a = decay
      form "gate"    h_t = f_t h_{t-1} + (1 - f_t) x_t             f = 1 / (1 + exp(-decay))

    y_t = h_t in x's type; state is h of each sequence's last step, in 32 bits, [sequences, channels].

    x              [batch, steps, channels], or [rows, channels] with `offsets`: float32, float16 or bfloat16.  Adjacent
                   channels have to be adjacent in memory (a copy is made otherwise), rows may be any distance apart, as in
                   a slice of a wider projection.
    decay          of x's shape, or [channels]: the same at every step (exponential smoothing); x's type or float32.  Decays of
                   more than 1 in size are computed as well, but pieces of a sequence are composed: a state that stays small
                   only because what such decays make of its past is taken away again by x loses its digits.
    initial_state  h_0, float32 [sequences, channels]; zeros if None.  To go on with a sequence pass the state of the call
                   before: one step at a time gives what one call over all steps gives, up to rounding.
    offsets        int32 or int64 [sequences + 1], on the device: sequence s has the rows offsets[s] up to offsets[s + 1].
                   Sequences may be empty: their state is h_0.  They have to ascend, or the results are undefined.
    lengths        int32 or int64 [batch], on the device: only the first lengths[b] steps of x[b] are its sequence.
                   Rows of no sequence (padding, rows in front of the first offset and behind the last) give zeros in y and
                   in the gradients, whatever they hold.  The device reads offsets and lengths: values out of range are
                   clamped, not reported.
    final_state    a float32 tensor [sequences, channels] that receives the state and is returned as such; it may be
                   `initial_state` itself, which is then updated in place, or overlap it, but no other input.  Not while
                   gradients are recorded.

    Gradients with respect to x, decay and initial_state; the state may be differentiated as well.

    States and gradients are held in 32 bits, products of decays in 64; the gradient of a decay per channel is a sum in 32 bits over
    256 rows and in 64 bits over these sums.  A gate is taken to the last bits of 32 if `decay` is float32.  Of 16-bit types the
    logistic function leaves out the rounding of its argument, |decay| 2^-24 relative, far below what such a decay is rounded to
    itself; this holds for the state in 32 bits as well.  An infinite x or state makes its channel infinite or NaN up to the end of its
    sequence, and no other."""
    return (_module or _ops()).linear_recurrence(x, decay, form, initial_state, offsets, lengths, final_state)


def block_norm(x, *, gate=None, residual=None, post_weight=None, scale=None, pre_weight=None, eps=1e-6):
    """What stands between two blocks of a layer, in one pass over the rows; returns (hidden, normed).

      u = x rstd(x) post_weight                 norm after the block       (without post_weight: u = x)
      v = u silu(gate)                          gate                       (without gate: v = u)
      hidden = residual + scale v               scaled residual            (without either: 1 and 0 in its place)
      normed = hidden rstd(hidden) pre_weight   norm before the next block (without pre_weight: None)

    rstd(z) = 1 / sqrt(mean(z^2) + eps) over the channels, silu(g) = g / (1 + exp(-g)).  block_norm(x, pre_weight=w)[1] is
    the plain root mean square norm.  Sums of squares are held in 32 bits: a row whose sum passes 3.4e38 is normalised to zeros.

    x, gate, residual  [..., channels] of one shape, up to 16384 channels: float32, float16 or bfloat16; gate has x's type, the
                       residual x's or float32.  Adjacent channels have to be adjacent in memory, rows may be any distance
                       apart.
    weights            [channels], all of one type: x's or float32.

    hidden has the residual's type (x's without one), normed x's; the second norm sees hidden before its rounding.
    Gradients with respect to everything; those of the weights are sums over the rows, in 32 bits and a fixed order."""
    return (_module or _ops()).block_norm(x, gate, residual, post_weight, scale, pre_weight, eps)


def embedding_lookup(ids, table, *, scale=1.0, padding_idx=None, dtype=None):
    """scale * table[ids], in 32 bits (so is scale) and rounded once: [*ids.shape, channels].

    ids          int32 or int64, any shape.  The device reads them: an id outside the table gives a row of zeros and takes no
                 part in the gradient; it is not reported.
    table        [vocab, channels]: float32, float16 or bfloat16; adjacent channels adjacent in memory.
    padding_idx  a row of the table whose gradient stays zero (0 <= padding_idx < vocab, or negative: from the end).
    dtype        type of the result (default: the table's).

    The gradient of the table is dense: for each row, scale times the sum of its tokens' gradients, in 32 bits, in an order that
    the ids alone decide (pieces of up to 32 tokens in their order, then the pieces), rounded once.  It does not depend on the table's values,
    which may change before the backward pass."""
    return (_module or _ops()).embedding_lookup(ids, table, scale, padding_idx, dtype)
