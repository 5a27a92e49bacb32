"""Trainer.token_logprobs and Trainer.distill_step where a call goes wrong: what
is refused, and that a refusal comes before any work."""
import ctypes as C

import numpy as np
import pytest

import test_gpu_logits as base

pytestmark = pytest.mark.gpu


def test_refused_device_arguments_queue_nothing():
    """Device pointers that the kernel refuses (ids off their alignment, outputs
    that overlap) are refused before the forward pass is queued."""
    import torch
    from tmnn_b200 import _abi
    n = 64
    pos = torch.rand(n, 3, device="cuda")
    ids = torch.zeros(4 * n + 1, dtype=torch.int32, device="cuda")
    y = torch.zeros(n, 2, device="cuda")
    out = torch.zeros(6 * n, device="cuda")
    loss = C.c_float(5.0)
    torch.cuda.synchronize()
    with base._field(16) as tr:
        h, lib, dev = tr._handle(), _abi.lib, _abi.PTR_DEVICE

        def at(t, byte=0):
            return C.c_void_p(t.data_ptr() + byte)

        def read(tokens, kind, lp, ent, k=0, top=None, lps=None):
            return lib.tmnn_cuda_ctx_token_logprobs(
                h, at(pos), tokens, kind, n, k, 1.0, dev, lp, ent, top, lps)

        def step(tokens, kind, logits):
            return lib.tmnn_cuda_distill_step(h, at(pos), tokens, kind, logits, n,
                                              2, 1.0, dev, C.byref(loss))

        assert read(at(ids), _abi.INDEX_I64, at(out), at(out, 4 * n)) == 0
        before, weights = tr.launch_count(), tr.weights()
        bad = [
            lambda: read(at(ids, 4), _abi.INDEX_I64, at(out), at(out, 4 * n)),
            lambda: read(at(ids, 2), _abi.INDEX_I32, at(out), at(out, 4 * n)),
            lambda: read(at(ids), _abi.INDEX_I64, at(out), at(out, 4)),
            lambda: read(at(ids), _abi.INDEX_I64, at(out), at(ids, 8)),
            lambda: read(at(ids), _abi.INDEX_I32, at(out, 1), None),
            lambda: read(None, _abi.INDEX_I32, None, at(out), 2, at(out, 4 * n),
                         at(out, 8 * n)),
            lambda: step(at(ids, 4), _abi.INDEX_I64, at(y)),
            lambda: step(at(ids), _abi.INDEX_I64, at(y, 2)),
        ]
        for i, call in enumerate(bad):
            assert call() == _abi.ERR_INVALID_ARGUMENT, i
            assert tr.launch_count() == before, i
        assert tr.step() == 0
        assert all(np.array_equal(a, b) for a, b in zip(weights, tr.weights()))
        assert step(at(ids), _abi.INDEX_I64, at(y)) == 0 and tr.step() == 1
