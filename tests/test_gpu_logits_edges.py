"""Class-logit operators on the GPU at the edges of their number range and of
what may be asked of them, in a size of every kernel (test_gpu_logits.py has
the ordinary range and the tolerances' reference)."""
import numpy as np
import pytest

import _logits_ref as ref
import test_gpu_logits as base

pytestmark = pytest.mark.gpu

# rows of a thread, of some lanes, of a CTA, of a CTA for the loss and a cluster
# for the gradient, of a cluster, of a cluster of 16
KERNELS = [(40, 19), (33, 127), (30, 1000), (20, 9001), (170, 33000), (5, 131072),
           (2, 300007)]


@pytest.mark.parametrize("T", [0.5, 0.7, 1.0, 2.0])
@pytest.mark.parametrize("n,V", KERNELS)
def test_entries_of_classes_at_the_lowest_value(n, V, T):
    """A teacher's entries that name classes masked with fp32's lowest value:
    the loss is in range although the log probability, divided by T, is not."""
    import torch
    import tmnn_b200 as t
    rng = np.random.default_rng(V)
    K = 5
    x = rng.normal(size=(n, V)).astype(np.float32) * 2
    x[:, 3:9] = base.LOWEST["f32"]
    ids = np.tile([0, 4, 1, 8, 5], (n, 1))
    ids[0] = [0, 1, 2, 10, 11]  # none of them
    y = rng.normal(size=(n, K)).astype(np.float32)
    w = rng.uniform(0.5, 1.5, n).astype(np.float32)
    loss, tl, d, td = ref.distill(x.astype(np.float64), T, ids, y, w)
    # a share is at least e^(-13 / 0.5) / 5 > 1e-12
    assert np.isfinite(loss).all() and (loss[1:] > 1e25).all()
    # T times a difference of 3.4e38 may be out of fp32's range, which is
    # infinity then; no loss is as near to its border as its bound
    most = -base.LOWEST["f32"]
    assert (np.abs(loss - most) > 2 * tl + 1e32).all() and (T > 1 or loss.max() < most)
    loss[loss > most] = np.inf
    args = [torch.from_numpy(a).cuda() for a in (x, ids, y)]
    ref.assert_close(t.distill_loss(*args, temperature=T).cpu(), loss, tl, "loss")
    l, g = t.distill_forward_backward(*args, temperature=T,
                                      row_weight=torch.from_numpy(w).cuda())
    ref.assert_close(l.cpu(), loss, tl, "loss with gradient")
    ref.assert_close(g.double().cpu(), d, base._round(d, td, "f32"), "gradient")


@pytest.mark.parametrize("T", [1.0, 2.0])
@pytest.mark.parametrize("n,V", KERNELS)
def test_small_shares_of_masked_classes(n, V, T):
    """A masked class (-inf) under an entry whose e^y is above fp32's zero makes
    the loss infinite, also where the share of all entries rounds to zero;
    one whose e^y is zero counts nothing.  Gradients are finite."""
    import torch
    import tmnn_b200 as t
    torch.manual_seed(V)
    x = torch.randn(n, V, device="cuda")
    x[:, 5] = float("-inf")
    ids = torch.tensor([[0, 1, 2, 5]], device="cuda").repeat(n, 1)
    # the smallest number above zero is 2^-149: e^-103 is 1.3 of it, and a third
    # of that rounds to none; e^-110 is none of it
    for far, inf in ((-95.0, True), (-103.0, True), (-110.0, False)):
        y = torch.tensor([[0.0, 0.0, 0.0, far * T]], device="cuda").repeat(n, 1)
        loss = t.distill_loss(x, ids, y, temperature=T)
        both, g = t.distill_forward_backward(x, ids, y, temperature=T)
        assert not loss.isnan().any() and not both.isnan().any(), far
        assert bool(loss.isinf().all()) == inf and bool(both.isinf().all()) == inf
        assert g.isfinite().all()
        if not inf:
            want = t.distill_loss(x, ids[:, :3].contiguous(),
                                  y[:, :3].contiguous(), temperature=T)
            # the same shares and sums: three roundings of terms below 20 T
            assert (loss - want).abs().max() <= 3 * 2 ** -24 * 20 * T * T
            assert loss.isfinite().all()


def test_leaves_that_require_a_gradient_are_not_written():
    """out= a leaf that requires a gradient, or a view of one, is refused where
    torch's own in-place calls refuse it, and written where they write."""
    import torch
    import tmnn_b200 as t
    tok = torch.zeros(4, dtype=torch.int64, device="cuda")
    one = torch.ones(4, device="cuda")
    ids = torch.ones(4, 2, dtype=torch.int64, device="cuda")
    y = torch.zeros(4, 2, device="cuda")

    def distil(x, out):
        return t.distill_forward_backward(x, ids, y, out=out)[1]

    def policy(x, out):
        st = t.token_logprobs(x, tok, stats=True).stats
        return t.token_logprobs_backward(x, tok, st, one, out=out)

    for write in (distil, policy):
        values = torch.randn(4, 9, device="cuda")
        want = write(values, None)
        leaf = values.clone().requires_grad_()
        wide = torch.zeros(4, 12, device="cuda", requires_grad=True)
        for out in (leaf, wide[:, :9]):
            before, version = out.detach().clone(), out._version
            with pytest.raises(ValueError, match="leaf"):
                write(values, out)
            with pytest.raises(RuntimeError):
                out.zero_()  # as torch does
            assert torch.equal(out.detach(), before) and out._version == version
        assert torch.equal(write(values, leaf.detach()), want)
        leaf = values.clone().requires_grad_()
        with torch.no_grad():
            assert torch.equal(write(leaf, leaf), want)
        leaf = values.clone().requires_grad_()
        made = leaf * 1  # no leaf: in place as before
        assert torch.equal(write(made, made).detach(), want)


def _device_us(call):
    """Device time of a call, the best of several replays of a graph of them."""
    import torch
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(5):
            call()
    best = np.inf
    for _ in range(8):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        graph.replay()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) * 1e3 / 5)
    return best


@pytest.mark.parametrize("n,V,k", [(1024, 65536, 64), (64, 131072, 20),
                                   (2000, 5000, 20), (4096, 600, 64)])
def test_a_constant_added_to_the_logits(n, V, k):
    """softmax does not see a constant added to fp32 logits: the alternatives are
    those of the shifted values, and are found in about the same time (a bound
    with 8 bits of a logit's fraction took 4 to 7 times as long)."""
    import torch
    import tmnn_b200 as t
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(n, V, device="cuda", generator=g) * 2.5
    far = x + 30000.0  # a step of 2^-9
    near = far - 30000.0  # exact: the same order and the same ties
    a, b = (t.token_logprobs(v, top_k=k) for v in (near, far))
    assert torch.equal(a.top_ids, b.top_ids)
    # each is off by the reference's bound of a log probability: V / 256 + 80
    # additions, differences d of at most 30, ln s of at most 20
    tol = 2 * 1.1 * ref.U * (3 * 30 + ref.chain(V) + 4 + 3 * 30 + 4 * 20)
    assert (a.top_logprobs - b.top_logprobs).abs().max() <= tol
    plain = _device_us(lambda: t.token_logprobs(near, top_k=k))
    shifted = _device_us(lambda: t.token_logprobs(far, top_k=k))
    assert shifted <= 2.5 * plain + 2, (shifted, plain)


@pytest.mark.parametrize("T", [1e-4, 1e4])
@pytest.mark.parametrize("n,V", KERNELS)
def test_first_and_last_temperature(n, V, T):
    """The ends of the range of temperatures, where a row is one class or all
    alike."""
    import torch
    import tmnn_b200 as t
    x, xd = base.make(n, V, "f32", seed=V + 1)
    tk, tok = base.make_tokens(n, V, V)
    Tf = float(np.float32(T))
    r = t.token_logprobs(x, tk, top_k=5, temperature=T, stats=True)
    lp, H, ids, _, stats, rows = ref.token_logprobs(xd, Tf, tok, 5)
    d = rows.d[np.arange(n), np.clip(tok, 0, V - 1)]
    # (d is 0 in the reference where e^-d is: there the logit's own distance)
    with np.errstate(all="ignore"):
        far = (rows.m - xd[np.arange(n), np.clip(tok, 0, V - 1)]) / Tf
    d = np.where(np.isfinite(far), np.maximum(d, far), d)
    ref.assert_close(r.logprob.cpu(), lp, np.nan_to_num(
        rows.tol_lp(d, np.where(np.isfinite(lp), lp, 0))), "logprob")
    ref.assert_close(r.entropy.cpu(), H, np.nan_to_num(rows.tol_H), "entropy")
    assert np.array_equal(r.top_ids.cpu().numpy(), ids)
    one = np.ones(n, np.float32)
    want, tol = ref.token_logprobs_backward(xd, Tf, tok, r.stats.cpu().numpy(),
                                            one, one)
    c = torch.ones(n, device="cuda")
    g = t.token_logprobs_backward(x, tk, r.stats, c, c, temperature=T)
    # an e^-d below 2^-126 may be flushed; the gradient has it times
    # (g + h (d + ln s + H)) / T with g = h = 1, d of at most 88 there, and ln s
    # and H of at most ln 524288 < 14
    flushed = 2.0 ** -126 * (1 + 88 + 2 * 14) / Tf
    ref.assert_close(g.double().cpu(), want,
                     base._round(want, np.nan_to_num(tol) + flushed, "f32"),
                     "backward")
    ti, ty = base.make_teacher(n, V, min(4, V), V)
    loss, tl, dx, td = ref.distill(xd, Tf, ti, ty.astype(np.float64), one)
    at = np.clip(ti, 0, V - 1)
    with np.errstate(all="ignore"):
        # the same for an entry's class: its distance counts 3 u, times T^2 q
        far = np.where(ti < 0, 0, rows.m[:, None] - np.take_along_axis(xd, at, 1)) / Tf
        far = np.where(np.isfinite(far), far, 0)
    tl = np.nan_to_num(tl) + 1.1 * Tf * Tf * 3 * ref.U * far.max(1)
    args = (x, torch.from_numpy(ti).cuda(), torch.from_numpy(ty).cuda())
    got, gx = t.distill_forward_backward(*args, temperature=T, row_weight=c)
    ref.assert_close(got.cpu(), loss, tl, "loss with gradient")
    ref.assert_close(t.distill_loss(*args, temperature=T).cpu(), loss, tl, "loss")
    ref.assert_close(gx.double().cpu(), dx,
                     base._round(dx, np.nan_to_num(td) + 2.0 ** -126 * Tf, "f32"),
                     "gradient")


def test_more_rows_than_a_launch_takes():
    """Rows beyond 2^26 go to a second launch: each row's results are its
    own."""
    import torch
    import tmnn_b200 as t
    n, V, period = (1 << 26) + 1027, 3, 1024
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(period, V, device="cuda", generator=g).bfloat16()
    tok = torch.randint(-1, V, (period,), device="cuda", generator=g).int()
    y = torch.randn(period, 1, device="cuda", generator=g)
    w = torch.rand(period, device="cuda", generator=g)

    def many(a):
        return a.repeat(n // period + 1, *[1] * (a.dim() - 1))[:n]

    def run(x, tok, y, w):
        r = t.token_logprobs(x, tok, top_k=2, stats=True)
        d = t.token_logprobs_backward(x, tok, r.stats, w, w)
        loss, e = t.distill_forward_backward(x, tok.view(-1, 1), y, row_weight=w)
        return [*r, d, loss, e]

    want = run(x, tok, y, w)
    for got, few in zip(run(many(x), many(tok), many(y), many(w)), want):
        whole = n // period * period
        assert (got[:whole].view(-1, period, *few.shape[1:]) == few).all()
        assert (got[whole:] == few[:n - whole]).all()
