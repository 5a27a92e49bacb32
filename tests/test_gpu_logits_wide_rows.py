"""Class-logit operators on fp32 rows of more than 1 MB (262145 to 524288
classes), which take clusters of 16 CTAs where a row is not streamed by one:
the checks of test_gpu_logits.py at those sizes, and the same rows in numbers."""
import numpy as np
import pytest

import _logits_ref as ref
import test_gpu_logits as base

pytestmark = pytest.mark.gpu

# the first width above 1 MB, odd ones, the last but one and the widest
SIZES = [(2, 262145), (13, 300007), (3, 400003), (10, 524287), (1, 524288)]


@pytest.mark.parametrize("n,V", SIZES)
@pytest.mark.parametrize("T,k,pad,offset", [(1.0, 5, 0, 0), (0.7, 40, 3, 1),
                                            (2.0, 128, 0, 2)])
def test_token_logprobs(n, V, T, k, pad, offset):
    base.test_token_logprobs(n, V, "f32", T, k, pad, offset)


@pytest.mark.parametrize("n,V", SIZES)
@pytest.mark.parametrize("T,pad,offset,which", [(1.0, 0, 0, "both"),
                                                (0.7, 3, 1, "logprob")])
def test_token_logprobs_backward(n, V, T, pad, offset, which):
    base.test_token_logprobs_backward(n, V, "f32", T, pad, offset, which)


@pytest.mark.parametrize("n,V", SIZES)
@pytest.mark.parametrize("T,K,pad,offset", [(1.0, 4, 0, 0), (2.0, 37, 3, 1),
                                            (0.7, 128, 0, 0)])
def test_distill(n, V, T, K, pad, offset):
    base.test_distill(n, V, "f32", T, K, pad, offset)


def test_rows_in_numbers():
    """The rows of a few again and again until they fill the SMs: the same
    alternatives, and values within the bounds of either order of summation."""
    import torch
    import tmnn_b200 as t
    n, V, k, times = 13, 300007, 20, 12
    x, xd = base.make(n, V, "f32", seed=3)
    tk, tok = base.make_tokens(n, V, V)
    r = t.token_logprobs(x.repeat(times, 1), tk.repeat(times), top_k=k, stats=True)
    lp, H, ids, _, stats, rows = ref.token_logprobs(xd, 1.0, tok, k)
    d = rows.d[np.arange(n), np.clip(tok, 0, V - 1)]
    tol = np.nan_to_num(rows.tol_lp(d, np.where(np.isfinite(lp), lp, 0)))
    tol_s = np.nan_to_num(np.stack([np.zeros(n), rows.s * rows.ds * 1.1,
                                    rows.tol_H], 1))
    for i in range(times):
        part = slice(i * n, (i + 1) * n)
        ref.assert_close(r.logprob[part].cpu(), lp, tol, "logprob")
        ref.assert_close(r.entropy[part].cpu(), H, np.nan_to_num(rows.tol_H), "H")
        ref.assert_close(r.stats[part].cpu(), stats, tol_s, "stats")
        assert np.array_equal(r.top_ids[part].cpu().numpy(), ids)


def test_ties_over_a_cluster():
    """Rows of few values, whose ties go over all CTAs of the cluster: the
    lowest classes come first."""
    import torch
    import tmnn_b200 as t
    V, k = 524288, 100
    x = np.zeros((5, V), np.float32)
    x[0] = np.arange(V) % 3
    x[1, ::32768] = 1  # one class of every CTA's part
    x[2] = -np.inf
    x[2, -7:] = -3
    x[3, 1::2] = base.LOWEST["f32"]
    r = t.token_logprobs(torch.from_numpy(x).cuda(), top_k=k)
    assert np.array_equal(r.top_ids.cpu().numpy(),
                          ref.token_logprobs(x.astype(np.float64), 1.0, None, k)[2])
