"""Refusals of the sequence operators, in the Python calls and at the C entries: nothing is launched for any of them.  (The calls
look at devices last, so that tensors of this machine get as far as the refusal in question.)"""
import ctypes as C

import numpy as np
import pytest
import torch

from dali_amd import _capi as capi
from dali_amd import sequence

F, BF, HF = torch.float32, torch.bfloat16, torch.float16


def z(*shape, dtype=F):
    return torch.zeros(*shape, dtype=dtype)


def test_host_tensors_are_refused():
    for call in (lambda: sequence.linear_recurrence(z(1, 2, 3), z(3)), lambda: sequence.block_norm(z(2, 3)),
                 lambda: sequence.embedding_lookup(z(2, dtype=torch.int64), z(4, 3))):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(TypeError):
        sequence.block_norm([1.0])


@pytest.mark.parametrize("args,kw,error,match", [
    ((z(1, 2, 3), z(3)), dict(form="sum"), ValueError, "form"),
    ((z(1, 2, 3, dtype=torch.float64), z(3)), {}, TypeError, "x must be"),
    ((z(2, 3), z(3)), {}, ValueError, "batch, steps"),
    ((z(3), z(3)), {}, ValueError, "batch, steps"),
    ((z(1, 2, 0), z(0)), {}, ValueError, "channels"),
    ((z(1, 2, 3), z(4)), {}, ValueError, "decay must have"),
    ((z(1, 2, 3), z(2, 3)), {}, ValueError, "decay must have"),
    ((z(1, 2, 3), z(3, dtype=BF)), {}, TypeError, "decay must be"),
    ((z(1, 2, 3, dtype=BF), z(3, dtype=HF)), {}, TypeError, "decay must be"),
    ((z(1, 2, 3), z(3)), dict(initial_state=z(1, 4)), ValueError, "initial_state"),
    ((z(1, 2, 3), z(3)), dict(initial_state=z(2, 3)), ValueError, "initial_state"),
    ((z(1, 2, 3, dtype=BF), z(3)), dict(initial_state=z(1, 3, dtype=BF)), TypeError, "initial_state"),
    ((z(4, 2, 3), z(3)), dict(final_state=z(3, 4).t()), ValueError, "contiguous"),
    ((z(1, 2, 3), z(3)), dict(offsets=z(2, dtype=torch.int64)), ValueError, "rows, channels"),
    ((z(2, 3), z(3)), dict(offsets=z(2)), TypeError, "offsets"),
    ((z(2, 3), z(3)), dict(offsets=z(1, 2, dtype=torch.int64)), ValueError, "offsets"),
    ((z(2, 3), z(3)), dict(offsets=z(0, dtype=torch.int64)), ValueError, "offsets"),
    ((z(2, 3), z(3)), dict(offsets=z(1, dtype=torch.int64)), ValueError, "no sequence"),
    ((z(2, 3), z(3)), dict(offsets=z(3, dtype=torch.int64), lengths=z(2, dtype=torch.int64)), ValueError, "exclude"),
    ((z(1, 2, 3), z(3)), dict(lengths=z(2, dtype=torch.int64)), ValueError, "lengths"),
    ((z(1, 2, 3), z(3)), dict(lengths=z(1)), TypeError, "lengths"),
])
def test_recurrence_refusals(args, kw, error, match):
    with pytest.raises(error, match=match):
        sequence.linear_recurrence(*args, **kw)


def test_recurrence_state_buffer_and_gradients_exclude_each_other():
    with pytest.raises(ValueError, match="gradients"):
        sequence.linear_recurrence(z(1, 2, 3).requires_grad_(), z(3), final_state=z(1, 3))


@pytest.mark.parametrize("args,kw,error,match", [
    ((z(2, 3, dtype=torch.float64),), {}, TypeError, "x must be"),
    ((torch.tensor(1.0),), {}, ValueError, "channels"),
    ((z(2, 0),), {}, ValueError, "channels"),
    ((z(1, 16385),), {}, ValueError, "16384"),
    ((z(2, 3),), dict(gate=z(2, 4)), ValueError, "gate"),
    ((z(2, 3),), dict(gate=z(3)), ValueError, "gate"),
    ((z(2, 3, dtype=BF),), dict(gate=z(2, 3)), TypeError, "gate"),
    ((z(2, 3),), dict(residual=z(2, 3, dtype=BF)), TypeError, "residual"),
    ((z(2, 3, dtype=BF),), dict(residual=z(2, 3, dtype=HF)), TypeError, "residual"),
    ((z(2, 3),), dict(residual=z(1, 3)), ValueError, "residual"),
    ((z(2, 3),), dict(post_weight=z(2)), ValueError, "post_weight"),
    ((z(2, 3),), dict(scale=z(1)), ValueError, "scale"),
    ((z(2, 3, dtype=BF),), dict(pre_weight=z(3, dtype=HF)), TypeError, "pre_weight"),
    ((z(2, 3, dtype=BF),), dict(post_weight=z(3, dtype=BF), pre_weight=z(3)), TypeError, "one type"),
    ((z(2, 3),), dict(eps=-1e-6), ValueError, "eps"),
    ((z(2, 3),), dict(eps=float("nan")), ValueError, "eps"),
])
def test_block_norm_refusals(args, kw, error, match):
    with pytest.raises(error, match=match):
        sequence.block_norm(*args, **kw)


@pytest.mark.parametrize("ids,table,kw,error,match", [
    (z(2), z(4, 3), {}, TypeError, "ids"),
    (z(2, dtype=torch.int16), z(4, 3), {}, TypeError, "ids"),
    (z(2, dtype=torch.int64), z(4, 3, dtype=torch.float64), {}, TypeError, "table"),
    (z(2, dtype=torch.int64), z(4), {}, ValueError, "table"),
    (z(2, dtype=torch.int64), z(0, 3), {}, ValueError, "table"),
    (z(2, dtype=torch.int64), z(4, 0), {}, ValueError, "table"),
    (z(2, dtype=torch.int64), z(4, 3), dict(padding_idx=4), ValueError, "padding_idx"),
    (z(2, dtype=torch.int64), z(4, 3), dict(padding_idx=-5), ValueError, "padding_idx"),
    (z(2, dtype=torch.int64), z(4, 3), dict(dtype=torch.int32), TypeError, "dtype"),
])
def test_embedding_refusals(ids, table, kw, error, match):
    with pytest.raises(error, match=match):
        sequence.embedding_lookup(ids, table, **kw)


# ------------------------------------------------------------------ the C entries
def recurrence_args(**kw):
    a = capi.RecurrenceArgs()
    a.seq.rows, a.seq.steps, a.seq.sequences = 6, 3, 2
    a.channels, a.dtype, a.decay_dtype = 8, capi.FLOAT, capi.FLOAT
    for k, v in kw.items():
        setattr(a.seq if k in ("rows", "steps", "sequences", "offsets", "lengths", "index_dtype") else a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    ({}, 0), (dict(rows=7), 1), (dict(rows=-1), 3), (dict(rows=1 << 31), 3), (dict(sequences=-2), 3), (dict(channels=0), 3), (dict(channels=(1 << 20) + 1), 3),
    (dict(dtype=capi.INT8), 2), (dict(decay_dtype=capi.FLOAT16), 2), (dict(form=2), 1), (dict(offsets=8, lengths=8, index_dtype=capi.INT32), 1),
    (dict(offsets=8, index_dtype=capi.FLOAT), 2), (dict(offsets=8, index_dtype=capi.INT64, sequences=0, steps=0), 1),
    (dict(offsets=8, index_dtype=capi.INT64, rows=100, steps=0), 0)])
def test_recurrence_setup_checks(kw, code):
    a, plan = recurrence_args(**kw), capi.RecurrencePlan()
    assert capi.kernels().daliamdRecurrenceSetup(C.byref(a), C.byref(plan)) == code
    for run in ("daliamdRecurrenceRun", "daliamdRecurrenceBackwardRun"):    # and no run without its tensors
        assert getattr(capi.kernels(), run)(None, C.byref(a), None, C.c_size_t(0)) == (code or 1)
        assert capi.kernels().daliamdGetLastErrorMessage()


@pytest.mark.parametrize("kw,code", [
    ({}, 0), (dict(rows=-1), 3), (dict(channels=0), 3), (dict(channels=16385), 3), (dict(dtype=capi.UINT8), 2), (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1),
    (dict(residual=8, residual_dtype=capi.FLOAT16), 2), (dict(scale=8, weight_dtype=capi.INT8), 2)])
def test_block_norm_setup_checks(kw, code):
    a, plan = capi.BlockNormArgs(), capi.BlockNormPlan()
    a.rows, a.channels, a.dtype, a.residual_dtype, a.weight_dtype = 4, 16, capi.BFLOAT16, capi.BFLOAT16, capi.BFLOAT16
    for k, v in kw.items():
        setattr(a, k, v)
    lib = capi.kernels()
    assert lib.daliamdBlockNormSetup(C.byref(a), C.byref(plan)) == code
    assert lib.daliamdBlockNormRun(None, C.byref(a)) == (code or 1)
    assert lib.daliamdBlockNormBackwardRun(None, C.byref(a), None, C.c_size_t(0)) == (code or 1)


@pytest.mark.parametrize("kw,code", [
    ({}, 0), (dict(tokens=-1), 3), (dict(tokens=1 << 31), 3), (dict(vocab=0), 3), (dict(vocab=1 << 31), 3), (dict(channels=0), 3),
    (dict(dtype=capi.INT8), 2), (dict(out_dtype=capi.INT8), 2), (dict(index_dtype=capi.FLOAT), 2)])
def test_embedding_setup_checks(kw, code):
    a, plan = capi.EmbeddingArgs(), capi.EmbeddingPlan()
    a.tokens, a.vocab, a.channels, a.dtype, a.out_dtype, a.index_dtype = 4, 9, 16, capi.FLOAT, capi.FLOAT, capi.INT64
    for k, v in kw.items():
        setattr(a, k, v)
    lib = capi.kernels()
    assert lib.daliamdEmbeddingSetup(C.byref(a), C.byref(plan)) == code
    assert lib.daliamdEmbeddingRun(None, C.byref(a)) == (code or 1)
    assert lib.daliamdEmbeddingBackwardRun(None, C.byref(a), None, C.c_size_t(0)) == (code or 1)


def test_workspaces_that_are_too_small_or_not_aligned_are_refused():
    lib = capi.kernels()
    one = 16            # (no address is looked at)
    a = recurrence_args(rows=1000, steps=1000, sequences=1, x=one, decay=one, y=one, dx=one, ddecay=one, saved=one)
    plan = capi.RecurrencePlan()
    assert lib.daliamdRecurrenceSetup(C.byref(a), C.byref(plan)) == 0
    b = capi.EmbeddingArgs(tokens=4, vocab=9, channels=16, dtype=capi.FLOAT, out_dtype=capi.FLOAT, index_dtype=capi.INT64, ids=one, dout=one, dtable=one)
    plan_b = capi.EmbeddingPlan()
    assert lib.daliamdEmbeddingSetup(C.byref(b), C.byref(plan_b)) == 0
    n = capi.BlockNormArgs(rows=4, channels=16, dtype=capi.FLOAT, residual_dtype=capi.FLOAT, weight_dtype=capi.FLOAT, x=one, dx=one, post_weight=one,
                           dpost_weight=one, rstd_post=one)
    plan_n = capi.BlockNormPlan()
    assert lib.daliamdBlockNormSetup(C.byref(n), C.byref(plan_n)) == 0
    for run, args, size in (("daliamdRecurrenceRun", a, plan.forward_workspace_bytes), ("daliamdRecurrenceBackwardRun", a, plan.backward_workspace_bytes),
                            ("daliamdEmbeddingBackwardRun", b, plan_b.backward_workspace_bytes),
                            ("daliamdBlockNormBackwardRun", n, plan_n.backward_workspace_bytes)):
        assert size > 0
        for workspace, given, message in ((4096, size - 1, b"too small"), (None, size, b"too small"), (4096 + 8, size, b"multiple of 16")):
            assert getattr(lib, run)(None, C.byref(args), workspace and C.c_void_p(workspace), C.c_size_t(given)) == 1
            lib.daliamdGetLastErrorMessage.restype = C.c_char_p
            assert message in lib.daliamdGetLastErrorMessage(), run


def test_struct_sizes_match_the_c_header(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"daliamdSequenceRows": capi.SequenceRows, "daliamdRecurrenceArgs": capi.RecurrenceArgs, "daliamdRecurrencePlan": capi.RecurrencePlan,
             "daliamdBlockNormArgs": capi.BlockNormArgs, "daliamdBlockNormPlan": capi.BlockNormPlan, "daliamdEmbeddingArgs": capi.EmbeddingArgs,
             "daliamdEmbeddingPlan": capi.EmbeddingPlan}
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "dali_amd_kernels.h"\nint main() {\n' +
                   "".join(f'  printf("%zu\\n", sizeof({n}));\n' for n in names) + "  return 0;\n}\n")
    subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "s")])
    sizes = [int(v) for v in subprocess.check_output([str(tmp_path / "s")]).split()]
    assert sizes == [C.sizeof(m) for m in names.values()]


def test_packed_rows_refuses_a_batch_in_host_memory():
    from dali_amd import fn
    from dali_amd.pipeline import Pipeline
    from dali_amd.plugin.pytorch import packed_rows
    pipe = Pipeline(batch_size=2, num_threads=1, device_id=None)
    with pipe:
        pipe.set_outputs(fn.external_source(source=lambda: [np.zeros((3, 2), np.float32), np.zeros((1, 2), np.float32)]))
    pipe.build()
    with pytest.raises(TypeError, match="no CPU fallback"):
        packed_rows(pipe.run()[0])
