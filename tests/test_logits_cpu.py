"""Class-logit operators without a GPU: refusals of the C ABI and the Python
functions (arguments are checked before any device work), and the 64-bit
reference of the GPU tests against central differences."""
import ctypes as C

import numpy as np
import pytest

import _logits_ref as ref

P = 1 << 20  # an aligned address that is never read: every call is refused


def _logits(**kw):
    from tmnn_b200 import _abi
    a = dict(data=P, row_stride=100, rows=4, classes=100, dtype=0,
             temperature=1.0)
    a.update(kw)
    return _abi.Logits(*[a[f] for f, _ in _abi.Logits._fields_])


def _refused(st, frag):
    from tmnn_b200 import _abi
    msg = _abi.lib.tmnn_cuda_logits_last_error().decode()
    assert st == _abi.ERR_INVALID_ARGUMENT, (st, msg)
    assert frag in msg, msg


@pytest.mark.parametrize("kw,frag", [
    (dict(classes=0), "classes must be in [1, 524288]"),
    (dict(classes=524289), "classes must be in [1, 524288]"),
    (dict(dtype=3), "logits must be F32, F16 or BF16"),
    (dict(temperature=0.0), "temperature must be in"),
    (dict(temperature=-1.0), "temperature must be in"),
    (dict(temperature=float("nan")), "temperature must be in"),
    (dict(temperature=float("inf")), "temperature must be in"),
    (dict(row_stride=-1), "row_stride must be in"),
    (dict(row_stride=(1 << 40) + 1), "row_stride must be in"),
    (dict(row_stride=1 << 40, rows=1 << 17), "span more than memory"),
    (dict(data=0), "logits is null"),
    (dict(data=P + 2), "logits is not aligned"),
])
def test_bad_logits_refused(kw, frag):
    from tmnn_b200 import lib
    x = _logits(**kw)
    _refused(lib.tmnn_cuda_token_logprobs(0, None, x, P, 0, 0, P, P, None, None,
                                          None), frag)
    _refused(lib.tmnn_cuda_token_logprobs_backward(
        0, None, x, P, 0, P, P, None, 2 * P, 100), frag)
    _refused(lib.tmnn_cuda_distill(0, None, x, P, 0, P, 0, 5, None, P, None, 0),
             frag)


def test_null_logits():
    from tmnn_b200 import lib
    assert lib.tmnn_cuda_token_logprobs(0, None, None, P, 0, 0, P, P, None,
                                        None, None) == 2


@pytest.mark.parametrize("args,frag", [
    ((P, 0, 101, P, P, P, P, None), "top_k must be at most"),
    ((P, 0, 3, P, P, None, P, None), "top_ids is null"),
    ((P, 0, 3, P, P, P, None, None), "top_logprobs is null"),
    ((None, 0, 0, P, P, None, None, None), "logprob needs tokens"),
    ((P, 2, 0, P, P, None, None, None), "index_type"),
    ((P + 4, 1, 0, P, P, None, None, None), "tokens is not aligned"),
    ((P, 0, 0, P + 1, P, None, None, None), "logprob is not aligned"),
    ((P, 0, 0, P, P, None, None, P + 2), "stats is not aligned"),
    ((2 * P, 0, 0, P + 1596, 3 * P, None, None, None), "an output overlaps"),
    ((2 * P, 0, 0, 3 * P, 2 * P + 12, None, None, None), "an output overlaps"),
    ((2 * P, 0, 0, 3 * P, 3 * P + 12, None, None, None), "an output overlaps"),
    ((2 * P, 0, 3, 3 * P, 4 * P, 5 * P, 5 * P + 44, None), "an output overlaps"),
])
def test_token_logprobs_refusals(args, frag):
    from tmnn_b200 import lib
    _refused(lib.tmnn_cuda_token_logprobs(0, None, _logits(), *args), frag)


def test_top_k_limit():
    from tmnn_b200 import lib
    x = _logits(classes=1000, row_stride=1000)
    _refused(lib.tmnn_cuda_token_logprobs(0, None, x, P, 0, 129, P, P, P, P,
                                          None), "top_k must be at most")


@pytest.mark.parametrize("args,frag", [
    ((P, 0, None, P, None, 2 * P, 100), "stats is null"),
    ((None, 0, P, P, None, 2 * P, 100), "d_logprob needs tokens"),
    ((P, 0, P, P, None, None, 100), "d_logits is null"),
    ((P, 0, P, P, None, 2 * P, 99), "d_row_stride must be in"),
    ((P, 0, P, P, None, P + 4, 100), "overlaps the logits in part"),
    ((P, 0, P, P, None, P, 101), "overlaps the logits in part"),
    ((P, 0, P, P, None, P + 4 * 399, 100), "overlaps the logits in part"),
    ((P, 0, P, P, None, P - 4 * 399, 100), "overlaps the logits in part"),
    ((P, 3, P, P, None, 2 * P, 100), "index_type"),
    ((2 * P + 8, 0, P, P, None, 2 * P, 100), "d_logits overlaps another"),
    ((3 * P, 0, 2 * P + 1596, P, None, 2 * P, 100), "d_logits overlaps another"),
    ((3 * P, 0, 4 * P, P, 2 * P, 2 * P, 100), "d_logits overlaps another"),
    ((3 * P, 0, 4 * P, P, None, 2 * P, 1 << 41), "d_row_stride must be in"),
])
def test_backward_refusals(args, frag):
    from tmnn_b200 import lib
    _refused(lib.tmnn_cuda_token_logprobs_backward(0, None, _logits(), *args),
             frag)


@pytest.mark.parametrize("args,frag", [
    ((P, 0, P, 0, 0, None, P, None, 0), "k must be in [1, 128]"),
    ((P, 0, P, 0, 129, None, P, None, 0), "k must be in [1, 128]"),
    ((P, 0, P, 5, 4, None, P, None, 0), "teacher_logits must be F32"),
    ((P, 7, P, 0, 4, None, P, None, 0), "index_type"),
    ((None, 0, P, 0, 4, None, P, None, 0), "teacher_ids is null"),
    ((P, 0, None, 0, 4, None, P, None, 0), "teacher_logits is null"),
    ((P, 0, P, 0, 4, None, None, None, 0), "loss is null"),
    ((2 * P, 0, 3 * P, 0, 4, None, 4 * P, 5 * P, 50), "d_row_stride must be in"),
    ((P, 0, P, 0, 4, P + 2, P, 2 * P, 100), "row_weight is not aligned"),
    ((2 * P, 0, 3 * P, 0, 4, None, 4 * P, P + 40, 100),
     "overlaps the logits in part"),
    ((2 * P, 0, 3 * P, 0, 4, None, P, None, 0), "loss overlaps another"),
    ((2 * P, 0, 3 * P, 0, 4, None, 3 * P + 60, None, 0), "loss overlaps another"),
    ((2 * P, 0, 3 * P, 0, 4, None, 4 * P, 2 * P, 100), "d_logits overlaps another"),
    ((2 * P, 0, 3 * P, 0, 4, 5 * P, 4 * P, 5 * P - 1596, 100),
     "d_logits overlaps another"),
])
def test_distill_refusals(args, frag):
    from tmnn_b200 import lib
    _refused(lib.tmnn_cuda_distill(0, None, _logits(), *args), frag)


def test_null_context():
    from tmnn_b200 import lib
    assert lib.tmnn_cuda_distill_step(None, P, P, 0, P, 1, 1, 1.0, 0, None) == 2
    assert lib.tmnn_cuda_ctx_token_logprobs(None, P, P, 0, 1, 0, 1.0, 0, P, P,
                                            None, None) == 2


def test_host_tensors_refused():
    import torch
    import tmnn_b200 as t
    x = torch.zeros(2, 5)
    with pytest.raises(ValueError, match="CUDA tensor"):
        t.token_logprobs(x)
    with pytest.raises(ValueError, match="CUDA tensor"):
        t.distill_loss(x, torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1))
    with pytest.raises(ValueError, match="CUDA tensor"):
        t.token_logprobs_backward(x, None, torch.zeros(2, 3))


def test_reference_import_name_has_them():
    import tiny_metal_nn
    import tmnn_b200
    for name in ("token_logprobs", "token_logprobs_backward", "distill_loss",
                 "distill_forward_backward", "TokenLogprobs"):
        assert getattr(tiny_metal_nn, name) is getattr(tmnn_b200, name)
    for name in ("token_logprobs", "distill_step"):
        assert hasattr(tiny_metal_nn.Trainer, name)


# ---- the reference against central differences (64 bits: with a step of
# 1e-5 the truncation is ~1e-10 and the round-off ~1e-11 of the value)
@pytest.mark.parametrize("T", [1.0, 0.7, 2.0])
def test_reference_gradients_by_differences(T):
    rng = np.random.default_rng(5)
    n, V, K, eps = 3, 7, 4, 1e-5
    x = rng.normal(size=(n, V)) * 2
    x[1, 3] = -np.inf
    tok = np.array([2, 0, 6])
    g, h = rng.normal(size=n), rng.normal(size=n)
    ids = np.array([[0, 3, 5, 3], [1, 2, -1, 4], [6, 0, 1, 2]])
    y = rng.normal(size=(n, K))
    w = rng.uniform(0.5, 1.5, n)

    def values(x):
        lp, H, *_ = ref.token_logprobs(x, T, tok, 0)
        loss = ref.distill(x, T, ids, y, w)[0]
        return (g * lp + h * H).sum(), (w * loss).sum()

    stats = ref.token_logprobs(x, T, tok, 0)[4]
    da, _ = ref.token_logprobs_backward(x, T, tok, stats, g, h)
    db = ref.distill(x, T, ids, y, w)[2]
    for i in range(n):
        for v in range(V):
            if x[i, v] == -np.inf:
                assert da[i, v] == 0 and db[i, v] == 0
                continue
            up, dn = x.copy(), x.copy()
            up[i, v] += eps
            dn[i, v] -= eps
            a, b = values(up), values(dn)
            assert abs((a[0] - b[0]) / (2 * eps) - da[i, v]) < 1e-7
            assert abs((a[1] - b[1]) / (2 * eps) - db[i, v]) < 1e-7
