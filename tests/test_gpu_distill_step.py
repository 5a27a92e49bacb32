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


# ------------------------------------------------------------ the numerics guard
FAMILIES = [(16, "FullyFused"), (16, "Tiled"), (19, "SafeDebug")]


def _guarded_field(n_out, family, recovery, **kw):
    import tmnn_b200 as t
    cfg = dict(base.CFG, b200=dict(family=family, bad_step_recovery=recovery, **kw))
    return t.Trainer.from_config(cfg, n_input=3, n_output=n_out)


def _state(tr):
    from tmnn_b200 import _abi
    return [tr.read_buffer(r) for r in (_abi.BUF_FUSED_WEIGHTS, _abi.BUF_FUSED_M,
                                        _abi.BUF_FUSED_V)]


def _same(a, b):
    return all(np.array_equal(x, y) for x, y in zip(a, b))


def _bad_batches(ids, y, n_out):
    """The batch with one entry that makes its point's row NaN."""
    i = ids.copy()
    i[7, 1] = n_out
    yield i, y
    for value in (np.nan, np.inf):
        i, z = ids.copy(), y.copy()
        i[7, 1], z[7, 1] = 0, value
        yield i, z


@pytest.mark.parametrize("n_out,family", FAMILIES)
@pytest.mark.parametrize("recovery,action", [("Skip", "Skipped"),
                                             ("Rollback", "RolledBack"),
                                             ("Throw", None)])
def test_a_bad_row_does_not_reach_the_weights(n_out, family, recovery, action):
    """One point whose teacher's entry names no class, or is NaN or infinite:
    the recovery mode keeps weights and optimizer state as they were, and the
    next step is a good one."""
    import torch
    import tmnn_b200 as t
    pos, ids, y = base._teacher(300, n_out, 4, 8)
    with _guarded_field(n_out, family, recovery) as tr, \
            _guarded_field(n_out, family, recovery) as twin:
        tr.distill_step(pos, ids, y)
        twin.distill_step(pos, ids, y)
        before, hash_before, steps = _state(tr), tr.weights()[0], tr.step()
        count = 0
        for bad_ids, bad_y in _bad_batches(ids, y, n_out):
            for args in ((pos, bad_ids, bad_y),
                         [torch.from_numpy(a).cuda() for a in (pos, bad_ids, bad_y)]):
                count += 1
                if recovery == "Throw":
                    with pytest.raises(t.TmnnError, match="numerics anomaly"):
                        tr.distill_step(*args)
                    assert tr.step() == steps
                else:
                    assert np.isnan(tr.distill_step(*args))
                    n = tr.last_numerics()
                    assert n["anomaly"] and not n["finite_forward"]
                    assert n["recovery_action"] == action
                    assert tr.step() == steps + count
                assert _same(_state(tr), before)
                assert np.array_equal(tr.weights()[0], hash_before)
        stats = tr.numerics_stats()
        assert stats["anomalies"] == count
        assert stats["skipped"] == (count if recovery == "Skip" else 0)
        assert stats["rolled_back"] == (count if recovery == "Rollback" else 0)
        # no gradient of the bad batches is left
        loss, want = tr.distill_step(pos, ids, y), twin.distill_step(pos, ids, y)
        assert np.isfinite(loss) and not tr.last_numerics()["anomaly"]
        # (the twin's MLP differs by the order of float additions in one step)
        assert abs(loss - want) <= 1e-4 * abs(want)
        if recovery == "Throw":  # the same step number, so the same update
            a, b = tr.weights()[0], twin.weights()[0]
            assert np.mean(np.abs(a - b) > 1e-5) < 0.01
        assert np.isfinite(tr.weights()[1]).all()


@pytest.mark.parametrize("n_out,family", FAMILIES)
def test_signal_only_reports_the_anomaly(n_out, family):
    """SignalOnly reports and applies, like training_step; a good step reports
    what the probe saw."""
    pos, ids, y = base._teacher(300, n_out, 4, 9)
    with _guarded_field(n_out, family, "SignalOnly") as tr:
        loss = tr.distill_step(pos, ids, y)
        n = tr.last_numerics()
        assert n["probed"] and not n["anomaly"] and n["max_abs_gradient"] > 0
        assert tr.last_result.loss == loss and tr.last_result.batch_size == 300
        assert tr.last_result.step == 0 and tr.step() == 1
        # an empty batch is no step and changes no report
        assert tr.distill_step(pos[:0], ids[:0], y[:0]) == 0.0
        assert tr.last_result.loss == loss
        bad_ids, bad_y = next(_bad_batches(ids, y, n_out))
        assert np.isnan(tr.distill_step(pos, bad_ids, bad_y))
        n = tr.last_numerics()
        assert n["anomaly"] and n["recovery_action"] == "None"
        assert not n["finite_forward"] and not n["finite_backward"]
        assert tr.numerics_stats()["anomalies"] == 1


def test_fallback_retries_with_the_safe_family():
    """An anomaly of the fp16 tensor cores alone (hidden values above fp16's
    range) is redone by the fp32 family; one that stays is an error."""
    import tmnn_b200 as t
    pos, ids, y = base._teacher(300, 16, 4, 10)
    bad_ids, bad_y = next(_bad_batches(ids, y, 16))
    mode = "FallbackAndRetryWithSafeFamily"
    with _guarded_field(16, "FullyFused", mode) as tr:
        hw, mw = tr.weights()
        tr.set_initial_weights(np.full_like(hw, 6.0e4), np.abs(mw) + 0.05)
        before = tr.weights()
        loss = tr.distill_step(pos, ids, y)
        n = tr.last_numerics()
        assert np.isfinite(loss) and not n["anomaly"]
        assert n["recovery_action"] == "RetriedWithSafeFamily"
        assert tr.last_result.family == 2 and tr.step() == 1
        after = tr.weights()
        assert all(np.isfinite(w).all() for w in after)
        assert not np.array_equal(after[1], before[1])
        with pytest.raises(t.TmnnError, match="already active"):
            tr.distill_step(pos, bad_ids, bad_y)
        assert tr.step() == 1
    with _guarded_field(16, "Tiled", mode) as tr:
        before = tr.weights()
        with pytest.raises(t.TmnnError, match="retry still produced"):
            tr.distill_step(pos, bad_ids, bad_y)
        assert tr.step() == 0 and _same(tr.weights(), before)
        assert np.isfinite(tr.distill_step(pos, ids, y))


def test_guard_between_training_steps():
    """Steps of both kinds under one guard: each reports its own loss."""
    pos, ids, y = base._teacher(300, 16, 4, 11)
    tgt = np.zeros((300, 16), np.float32)
    with _guarded_field(16, "FullyFused", "Skip") as tr:
        first = tr.training_step(pos, tgt)
        assert first == tr.last_result.loss
        tr.distill_step(pos, ids, y)
        assert tr.last_result.step == 1
        bad_ids, bad_y = next(_bad_batches(ids, y, 16))
        assert np.isnan(tr.distill_step(pos, bad_ids, bad_y))
        loss = tr.training_step(pos, tgt)
        assert np.isfinite(loss) and tr.last_result.loss == loss
        assert not tr.last_numerics()["anomaly"] and tr.step() == 4


@pytest.mark.parametrize("n", [2, 777, 4096])
def test_the_tiled_family_takes_the_split_step(n):
    """The family of large tables: distill_step is the split step there too."""
    base.test_distill_step_is_the_split_step(16, "Tiled", n)


def test_result_before_any_step():
    from tmnn_b200 import _abi
    res = _abi.StepResult()
    with base._field(16) as tr:
        assert _abi.lib.tmnn_cuda_distill_result(tr._handle(), C.byref(res)) == 0
        assert res.batch_size == 0 and res.loss == 0.0
        assert _abi.lib.tmnn_cuda_distill_result(tr._handle(), None) \
            == _abi.ERR_INVALID_ARGUMENT
    assert _abi.lib.tmnn_cuda_distill_result(None, C.byref(res)) == 2
