"""The sequence operators where their inputs are at an end of their range or their work at the end of a piece: excluded tokens behind
the last real one, gates that are wide open or shut, states that share memory.  Bounds are derived beside each test from half a
step of each type and 2^-24 per operation in 32 bits."""
import ctypes as C
import os

import numpy as np
import pytest
import torch

from dali_amd import _capi as capi
from tests import sequence_reference as R
from tests.test_gpu_sequence import BF, F, HF

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
