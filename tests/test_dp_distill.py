"""Trainer.distill_step under data parallelism (2 or more GPUs): every rank's
points, averaged over all ranks' points, against one process on the whole
batch; and a bad row of one rank, which every rank's guard sees."""
import os

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from test_dp import KW_FUSED, ROOT, _free_port

KW = dict(KW_FUSED, O=16)
POINTS = 512  # of a rank


def _batches(world, steps=3):
    rng = np.random.default_rng(33)
    for _ in range(steps):
        n = POINTS * world
        pos = rng.uniform(-1, 1, (n, 3)).astype(np.float32)
        ids = np.argsort(rng.random((n, 16)), axis=1)[:, :4].astype(np.int64)
        ids[rng.random((n, 4)) < 0.1] = -1
        yield pos, ids, rng.normal(size=(n, 4)).astype(np.float32)


def _trainer(family, grad, extra, device=0):
    from _util import cuda_trainer
    return cuda_trainer(**KW, family=family, grad=grad, device=device,
                        cfg_extra=extra)


def _rank(rank, world, port, q, family, grad, extra):
    import sys
    for p in (ROOT, os.path.join(ROOT, "tests"), os.path.join(ROOT, "tiny-metal-nn_b200"),
              os.path.join(ROOT, "oracle")):
        sys.path.insert(0, p)
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    os.environ.setdefault("NCCL_NVLS_ENABLE", "0")
    os.environ["TMNN_DP_BUCKETS"] = "4"
    torch.cuda.set_device(rank)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    import tmnn_b200 as t
    tr = _trainer(family, grad, extra, rank)
    uid = [t.dp_unique_id() if rank == 0 else None]
    dist.broadcast_object_list(uid, src=0)
    tr.dp_init(uid[0], rank, world)
    init = tr.weights()
    mine = slice(rank * POINTS, (rank + 1) * POINTS)
    losses = []
    for batch in _batches(world):
        part = [np.ascontiguousarray(a[mine]) for a in batch]
        losses.append(tr.distill_step(*part, temperature=2.0))
    tr.dp_sync_state()
    good = tr.weights()
    # one bad id on the last rank: no rank's weights move
    if rank == world - 1:
        part[1][5, 2] = 16
    bad = tr.distill_step(*part, temperature=2.0)
    action = tr.last_numerics()["recovery_action"]
    tr.dp_sync_state()
    kept = all(np.array_equal(a, b) for a, b in zip(good, tr.weights()))
    q.put((rank, good, losses, init, np.isnan(bad), action, kept))
    tr.close()
    dist.destroy_process_group()


def _run(world, family, grad, sharded):
    from tmnn_b200 import _abi
    extra = {"bad_step_recovery": _abi.BAD_STEP["Skip"]}
    if sharded:
        extra["dp_replicated_optimizer"] = -1
    port = _free_port()
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, world, port, q, family, grad, extra))
             for r in range(world)]
    for p in procs:
        p.start()
    res = {}
    for _ in procs:
        got = q.get(timeout=120)
        res[got[0]] = got[1:]
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    (h0, m0), l0, (hi, mi), *_ = res[0]
    for (h, m), losses, _, bad, action, kept in res.values():
        assert np.array_equal(h, h0) and np.array_equal(m, m0) and losses == l0
        assert bad and action == "Skipped" and kept
    with _trainer(family, grad, extra) as one:
        want = [one.distill_step(*b, temperature=2.0) for b in _batches(world)]
        hr, mr = one.weights()
    assert np.allclose(l0, want, rtol=1e-3)

    def cos(a, b):
        a, b = a.astype(np.float64), b.astype(np.float64)
        return a @ b / max(np.linalg.norm(a) * np.linalg.norm(b), 1e-300)
    # Adam moves a weight by about lr whatever its gradient's size, and sums
    # are taken in another order: changes are compared by their direction
    assert cos(h0 - hi, hr - hi) >= 0.99
    assert cos(m0 - mi, mr - mi) >= 0.99


@pytest.mark.gpu
@pytest.mark.parametrize("family,grad,sharded", [
    ("SafeDebug", "Fixed16", False), ("FullyFused", "F32", False),
    ("Tiled", "F32", False), ("Tiled", "F32", True),
    ("FullyFused", "Fixed16", True)])
def test_ranks_match_one_process(family, grad, sharded):
    if torch.cuda.device_count() < 2:
        pytest.skip("needs 2 GPUs")
    _run(min(4, torch.cuda.device_count()), family, grad, sharded)


@pytest.mark.gpu
@pytest.mark.parametrize("family,grad", [("SafeDebug", "Fixed16"),
                                         ("Tiled", "F32")])
def test_one_rank(family, grad):
    """The same with a communicator of one rank."""
    _run(1, family, grad, False)
