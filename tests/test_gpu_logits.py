"""Class-logit operators on the GPU against their definitions in 64 bits
(tests/_logits_ref.py, which derives the error bounds): log probabilities,
entropy and alternatives, their backward pass, and distillation, over types,
sizes, strides, masks, padding and rows that are no distributions; then
streams, graphs, in-place gradients and the Trainer paths that call them."""
import ctypes as C

import numpy as np
import pytest

import _logits_ref as ref

pytestmark = pytest.mark.gpu

TORCH = {"f32": "float32", "bf16": "bfloat16", "fp16": "float16"}
LOWEST = {"f32": -3.4028234663852886e38, "bf16": -3.3895313892515355e38,
          "fp16": -65504.0}


def _t(name):
    import torch
    return getattr(torch, TORCH[name])


def make(n, V, dtype, seed, pad=0, offset=0):
    """(CUDA tensor [n, V] whose rows lie V + pad apart and start `offset`
    elements into their memory, float64 values).  With 10 rows or more, rows
    1..8 are the ones that go wrong: nothing left, all equal, lowest value,
    lowest value but one, NaN, +inf, a mask with one class left, and -0 / +0."""
    import torch
    rng = np.random.default_rng(seed)
    x = rng.normal(size=(n, V)) * 3
    hot = rng.integers(0, V, n)
    x[np.arange(n), hot] += 6
    x[rng.random((n, V)) < 0.1] = -np.inf
    if n >= 10:
        x[1] = -np.inf
        x[2] = 1.25
        x[3] = LOWEST[dtype]
        x[4] = LOWEST[dtype]
        x[4, V // 2] = 3.0
        x[5, V // 3] = np.nan
        x[6, V - 1] = np.inf
        x[7] = -np.inf
        x[7, V - 1] = -7.0
        x[8] = 0.0
        x[8, ::2] = -0.0
    mem = torch.full((offset + n * (V + pad),), 77.0, dtype=_t(dtype),
                     device="cuda")
    t = mem[offset:].view(n, V + pad)[:, :V]
    t.copy_(torch.from_numpy(x).to("cuda").to(_t(dtype)))
    return t, t.double().cpu().numpy()


def make_tokens(n, V, seed, dtype="int64"):
    import torch
    rng = np.random.default_rng(seed + 1000)
    tok = rng.integers(0, V, n)
    if n >= 10:
        tok[0] = V - 1
        tok[9] = -1
        tok[n - 1] = V  # no such class
    if n >= 12:
        tok[10] = -100
    return torch.from_numpy(tok).to("cuda").to(getattr(torch, dtype)), tok


# 150 rows and more: wide rows in numbers that fill the SMs
SIZES = [(1, 1), (3, 2), (40, 3), (13, 19), (70000, 5), (33, 31), (300, 64),
         (12, 65), (50, 127), (11, 257), (64, 1000), (5, 1023), (17, 1024),
         (17, 1025), (10, 2047), (12, 2311), (10, 4097), (21, 8192), (2, 32768),
         (11, 32003), (300, 5000), (1, 131072), (10, 50021), (3, 262143),
         (12, 131071), (1, 524288), (320, 9001), (160, 33000), (600, 2500),
         (155, 24999), (152, 66001), (150, 40000)]
DTYPES = ["f32", "bf16", "fp16"]


def _sizes(dtypes=DTYPES):
    # every size in one type, the types taken in turn, and a few in all
    for i, (n, V) in enumerate(SIZES):
        for j, d in enumerate(dtypes):
            if i % 3 == j or V in (19, 1025, 32003, 131071):
                yield n, V, d


@pytest.mark.parametrize("n,V,dtype", list(_sizes()))
@pytest.mark.parametrize("T,k,pad,offset", [(1.0, 5, 0, 0), (0.7, 40, 3, 1)])
def test_token_logprobs(n, V, dtype, T, k, pad, offset):
    import tmnn_b200 as t
    k = min(k, V)
    x, xd = make(n, V, dtype, seed=n + V, pad=pad, offset=offset)
    tk, tok = make_tokens(n, V, V, "int32" if pad else "int64")
    r = t.token_logprobs(x, tk, top_k=k, temperature=T, stats=True)
    lp, H, ids, top, stats, rows = ref.token_logprobs(xd, float(np.float32(T)),
                                                      tok, k)
    at = np.clip(tok, 0, V - 1)
    d = rows.d[np.arange(n), at]
    ref.assert_close(r.entropy.cpu(), H, np.nan_to_num(rows.tol_H), "entropy")
    ref.assert_close(r.logprob.cpu(), lp, np.nan_to_num(
        rows.tol_lp(d, np.where(np.isfinite(lp), lp, 0))), "logprob")
    assert np.array_equal(r.top_ids.cpu().numpy(), ids)
    fin = np.where(np.isfinite(top), top, 0)
    dk = np.take_along_axis(rows.d, np.clip(ids, 0, V - 1), 1)
    tol = 1.1 * (ref.U * 3 * dk + np.nan_to_num(rows.tol_ln)[:, None]
                 + 2 * ref.U * np.abs(fin)) + 1e-37
    ref.assert_close(r.top_logprobs.cpu(), top, np.nan_to_num(tol), "top")
    tol = np.stack([np.zeros(n), rows.s * rows.ds * 1.1, rows.tol_H], 1)
    ref.assert_close(r.stats.cpu(), stats, np.nan_to_num(tol), "stats")
    # fewer outputs are the same outputs
    q = t.token_logprobs(x, tk, temperature=T)
    assert q.top_ids is None and q.stats is None
    # (sums may be taken in another order)
    ref.assert_close(q.logprob.cpu(), lp, np.nan_to_num(
        rows.tol_lp(d, np.where(np.isfinite(lp), lp, 0))), "logprob alone")
    # without tokens no row is padding
    q = t.token_logprobs(x, top_k=k, temperature=T)
    assert q.logprob is None
    full = ref.token_logprobs(xd, float(np.float32(T)), None, k)
    assert np.array_equal(q.top_ids.cpu().numpy(), full[2])
    ref.assert_close(q.entropy.cpu(), full[1], np.nan_to_num(rows.tol_H), "entropy")


@pytest.mark.parametrize("k", [1, 2, 31, 32, 33, 64, 100, 128])
@pytest.mark.parametrize("V", [128, 700, 4100, 70000])
def test_many_alternatives(V, k):
    """Every count of alternatives; values with many ties (few distinct
    values), ascending rows, and rows whose largest values lie a fixed distance
    apart (one thread's or one granule's share of the row)."""
    import torch
    import tmnn_b200 as t
    rng = np.random.default_rng(V + k)
    x = np.zeros((11, V))
    x[0] = rng.integers(0, 4, V)
    x[1] = np.arange(V) % 2048
    x[2] = rng.normal(size=V)
    x[2, ::256] += 50
    x[3] = rng.normal(size=V)
    x[3, 5::2048] += 50
    x[4] = -np.arange(V) / 64.0
    x[5, rng.permutation(V)[:k // 2]] = 1  # the rest ties at 0
    x[6] = -np.inf
    x[6, rng.permutation(V)[:max(1, k // 2)]] = 2.5
    x[7] = np.arange(V) / 64.0
    x[8, : V // 2] = rng.normal(size=V // 2) + 9
    x[9] = -np.inf
    x[9, V // 2:] = LOWEST["f32"]
    x[10] = 0.5
    for dtype in DTYPES:
        x[9, V // 2:] = LOWEST[dtype]
        c = torch.from_numpy(x).to("cuda").to(_t(dtype))
        xd = c.double().cpu().numpy()
        r = t.token_logprobs(c, top_k=k)
        _, _, ids, top, _, rows = ref.token_logprobs(xd, 1.0, None, k)
        # the same rows in numbers that fill the SMs
        many = t.token_logprobs(c.repeat(60, 1), top_k=k)
        assert torch.equal(many.top_ids, r.top_ids.repeat(60, 1))
        assert np.array_equal(r.top_ids.cpu().numpy(), ids), dtype
        dk = np.take_along_axis(rows.d, np.clip(ids, 0, V - 1), 1)
        tol = 1.1 * (ref.U * 3 * dk + rows.tol_ln[:, None] + 2 * ref.U *
                     np.abs(np.where(np.isfinite(top), top, 0))) + 1e-37
        ref.assert_close(r.top_logprobs.cpu(), top, tol, dtype)
        ref.assert_close(many.top_logprobs.cpu(), np.tile(top, (60, 1)),
                         np.tile(tol, (60, 1)), dtype)


def _round(d, tol, dtype):
    return tol + np.abs(np.nan_to_num(d)) * ref.HALF_STEP[dtype] * 1.01 + ref.TINY[dtype]


@pytest.mark.parametrize("n,V,dtype", list(_sizes()))
@pytest.mark.parametrize("T,pad,offset,which", [(1.0, 0, 0, "both"),
                                                (0.7, 3, 1, "logprob"),
                                                (2.0, 8, 0, "entropy")])
def test_token_logprobs_backward(n, V, dtype, T, pad, offset, which):
    import torch
    import tmnn_b200 as t
    x, xd = make(n, V, dtype, seed=n * 3 + V, pad=pad, offset=offset)
    tk, tok = make_tokens(n, V, V)
    st = t.token_logprobs(x, tk, temperature=T, stats=True).stats
    rng = np.random.default_rng(n + V)
    g = rng.normal(size=n).astype(np.float32)
    h = rng.normal(size=n).astype(np.float32)
    gc, hc = torch.from_numpy(g).cuda(), torch.from_numpy(h).cuda()
    kw = dict(d_logprob=None if which == "entropy" else gc,
              d_entropy=None if which == "logprob" else hc)
    want, tol = ref.token_logprobs_backward(
        xd, float(np.float32(T)), tok, st.cpu().numpy(),
        None if which == "entropy" else g, None if which == "logprob" else h)
    tol = _round(want, np.nan_to_num(tol), dtype)
    d = t.token_logprobs_backward(x, tk, st, temperature=T, **kw)
    assert d.dtype == x.dtype and d.is_contiguous()
    ref.assert_close(d.double().cpu(), want, tol, "gradient")
    # rows of another layout; what lies between them is left alone
    mem = torch.full((n * (V + 5) + 3,), 9.0, dtype=x.dtype, device="cuda")
    out = mem[3:].view(n, V + 5)[:, :V]
    got = t.token_logprobs_backward(x, tk, st, temperature=T, out=out, **kw)
    assert got is out and _same(out, d)
    assert (mem[3:].view(n, V + 5)[:, V:] == 9.0).all() and (mem[:3] == 9.0).all()
    # in place
    got = t.token_logprobs_backward(x, tk, st, temperature=T, out=x, **kw)
    assert got is x and _same(x, d)


def _same(a, b):
    """Equal bit for bit, NaN beside NaN."""
    import torch
    return torch.equal(torch.nan_to_num(a, nan=123.0), torch.nan_to_num(b, nan=123.0)) \
        and torch.equal(a.isnan(), b.isnan())


def make_teacher(n, V, K, seed):
    """ids and logits [n, K]; with 10 rows or more: row 2 has no entries, row 3
    one class named twice, row 4 one entry, row 0 an entry at -inf, row n - 1
    an id that names no class, row n - 2 a NaN."""
    rng = np.random.default_rng(seed)
    ids = np.argsort(rng.random((n, V)), axis=1)[:, :K] if n * V < 4e6 else \
        rng.integers(0, V, (n, K))
    y = rng.normal(size=(n, K)).astype(np.float32) * 2
    if n >= 10:
        ids[2] = -1
        ids[3, K - 1] = ids[3, 0]
        ids[4, 1:] = -5
        if K > 1:
            y[0, K // 2] = -np.inf
        ids[n - 1, K // 2] = V
        y[n - 1, K // 2] = 1.0
        y[n - 2, 0] = np.nan
    if n >= 14:
        y[11] = -np.inf
    return ids, y


@pytest.mark.parametrize("n,V,dtype", list(_sizes()))
@pytest.mark.parametrize("T,K,pad,offset", [(1.0, 4, 0, 0), (2.0, 37, 3, 1)])
def test_distill(n, V, dtype, T, K, pad, offset):
    import torch
    import tmnn_b200 as t
    K = min(K, max(V, 2))
    x, xd = make(n, V, dtype, seed=n * 7 + V, pad=pad, offset=offset)
    ids, y = make_teacher(n, V, K if K <= V else V, n + V)
    K = ids.shape[1]
    rng = np.random.default_rng(V)
    w = rng.uniform(0.5, 1.5, n).astype(np.float32)
    yt = {0: "f32", 3: "bf16"}[pad]
    yc = torch.from_numpy(y).cuda().to(_t(yt))
    ic = torch.from_numpy(ids).cuda().to(torch.int32 if pad else torch.int64)
    wc = torch.from_numpy(w).cuda()
    Tf = float(np.float32(T))
    loss, tol_l, d, tol_d = ref.distill(xd, Tf, ids, yc.double().cpu().numpy(), w)
    got = t.distill_loss(x, ic, yc, temperature=T)
    ref.assert_close(got.cpu(), loss, np.nan_to_num(tol_l), "loss")
    l2, g = t.distill_forward_backward(x, ic, yc, temperature=T, row_weight=wc)
    ref.assert_close(l2.cpu(), loss, np.nan_to_num(tol_l), "loss with gradient")
    tol = _round(d, np.nan_to_num(tol_d), dtype)
    ref.assert_close(g.double().cpu(), d, tol, "gradient")
    # the default weight is the mean's
    lm, gm = t.distill_forward_backward(x, ic, yc, temperature=T)
    one = ref.distill(xd, Tf, ids, yc.double().cpu().numpy(),
                      np.full(n, np.float32(1.0 / n)))
    ref.assert_close(gm.double().cpu(), one[2],
                     _round(one[2], np.nan_to_num(one[3]), dtype), "mean")
    # another layout, then in place
    mem = torch.full((n * (V + 5) + 3,), 9.0, dtype=x.dtype, device="cuda")
    out = mem[3:].view(n, V + 5)[:, :V]
    t.distill_forward_backward(x, ic, yc, temperature=T, row_weight=wc, out=out)
    assert _same(out, g)
    assert (mem[3:].view(n, V + 5)[:, V:] == 9.0).all() and (mem[:3] == 9.0).all()
    l3, gi = t.distill_forward_backward(x, ic, yc, temperature=T, row_weight=wc,
                                        out=x)
    assert gi is x and _same(x, g) and _same(l3, l2)


@pytest.mark.parametrize("K", [1, 2, 31, 32, 33, 64, 127, 128])
@pytest.mark.parametrize("V", [2, 130, 5000, 40000])
def test_distill_entry_counts(V, K):
    """Every count of entries, more entries than classes among them (classes
    named again and again)."""
    import torch
    import tmnn_b200 as t
    rng = np.random.default_rng(V * K)
    n = 6
    x = rng.normal(size=(n, V)) * 2
    ids = rng.integers(0, V, (n, K))
    ids[rng.random((n, K)) < 0.1] = -1
    y = rng.normal(size=(n, K)).astype(np.float32)
    w = np.ones(n, np.float32)
    for dtype in DTYPES:
        c = torch.from_numpy(x).cuda().to(_t(dtype))
        loss, tl, d, td = ref.distill(c.double().cpu().numpy(), 1.0, ids, y, w)
        l, g = t.distill_forward_backward(
            c, torch.from_numpy(ids).cuda(), torch.from_numpy(y).cuda(),
            row_weight=torch.from_numpy(w).cuda())
        ref.assert_close(l.cpu(), loss, tl, dtype)
        ref.assert_close(g.double().cpu(), d, _round(d, td, dtype), dtype)


# a size of every kernel: rows of a thread, of some lanes, of a CTA, of a cluster
EVERY = [(40, 19), (30, 1000), (20, 9001), (170, 33000), (5, 131072)]


@pytest.mark.parametrize("n,V", EVERY)
def test_ids_beyond_32_bits(n, V):
    """Ids keep their 64 bits: one whose low half names a class is still none,
    one below -2^31 is still padding."""
    import torch
    import tmnn_b200 as t
    x, _ = make(n, V, "bf16", seed=V)
    x[:5] = torch.linspace(-2, 2, V, device="cuda").bfloat16()
    far = torch.tensor([(1 << 32) + 1, 1 << 31, (1 << 63) - 1, -(1 << 63),
                        -(1 << 32) + 1], device="cuda")
    tok = torch.ones(n, dtype=torch.int64, device="cuda")
    tok[:5] = far
    r = t.token_logprobs(x, tok, top_k=2, stats=True)
    assert r.logprob[:3].isnan().all() and not r.entropy[:5].isnan().any()
    assert (r.logprob[3:5] == 0).all() and (r.entropy[3:5] == 0).all()
    first = (x[0] == x[0].max()).nonzero()[0]  # several classes round to 2
    assert (r.top_ids[:3, 0] == first).all() and (r.top_ids[3:5] == -1).all()
    one = torch.ones(n, device="cuda")
    g = t.token_logprobs_backward(x, tok, r.stats, one, one)
    assert g[:3].isnan().all() and (g[3:5] == 0).all()
    ids = torch.stack([tok, torch.full_like(tok, 2)], 1)
    y = torch.zeros(n, 2, device="cuda")
    loss, g = t.distill_forward_backward(x, ids, y)
    assert loss[:3].isnan().all() and g[:3].isnan().all()
    ids[3:5, 0] = -1  # left out like the entries far below 0
    l2, g2 = t.distill_forward_backward(x, ids, y)
    assert torch.equal(loss[3:5], l2[3:5]) and torch.equal(g[3:5], g2[3:5])
    assert not l2[3:5].isnan().any()
    assert torch.equal(t.distill_loss(x, ids, y)[:3].isnan(), loss[:3].isnan())


@pytest.mark.parametrize("n,V", EVERY)
def test_gradient_factors_of_padding(n, V):
    """Whatever the row weights and incoming gradients of padded rows and of
    rows without a distribution hold, their gradient is 0; a weight of 0 gives
    0 elsewhere."""
    import torch
    import tmnn_b200 as t
    torch.manual_seed(V)
    x = torch.randn(n, V, device="cuda")
    x[2] = float("nan")
    x[3] = float("-inf")
    tok = torch.ones(n, dtype=torch.int64, device="cuda")
    tok[1:3] = -1
    ids = torch.ones(n, 3, dtype=torch.int64, device="cuda")
    ids[1:3] = -1
    w = torch.ones(n, device="cuda")
    w[0], w[1], w[2], w[3] = 0.0, float("nan"), float("inf"), float("nan")
    y = torch.zeros(n, 3, device="cuda")
    _, g = t.distill_forward_backward(x, ids, y, row_weight=w)
    assert (g[:4] == 0).all() and not g.isnan().any()
    assert (g[4:].abs().amax(1) > 0).all()
    r = t.token_logprobs(x, tok, stats=True)
    g = t.token_logprobs_backward(x, tok, r.stats, w, w)
    assert (g[:4] == 0).all() and not g.isnan().any()
    assert (g[4:].abs().amax(1) > 0).all()


def test_gradients_by_differences():
    """Central differences of the kernels' own values.  f32 values are off by
    about 16 u |value| < 4e-5 (derived bounds are below that at V = 9), so a
    step of 0.05 gives 4e-5 / 0.05 = 8e-4 of round-off and its third-order
    term is below 0.05^2 / 6 * 4 = 2e-3 (third derivatives of these functions
    of a softmax stay below 4 for unit weights); both are inside 5e-3."""
    import torch
    import tmnn_b200 as t
    torch.manual_seed(3)
    x = torch.randn(4, 9, device="cuda")
    tok = torch.tensor([0, 8, 3, 3], device="cuda")
    ids = torch.tensor([[1, 2], [0, 8], [3, 3], [5, -1]], device="cuda")
    y = torch.randn(4, 2, device="cuda")
    one = torch.ones(4, device="cuda")
    st = t.token_logprobs(x, tok, stats=True).stats
    ga = t.token_logprobs_backward(x, tok, st, one, one)
    _, gb = t.distill_forward_backward(x, ids, y, row_weight=one)
    for v in range(9):
        up, dn = x.clone(), x.clone()
        up[:, v] += 0.05
        dn[:, v] -= 0.05
        a, b = t.token_logprobs(up, tok), t.token_logprobs(dn, tok)
        da = (a.logprob + a.entropy - b.logprob - b.entropy) / 0.1
        db = (t.distill_loss(up, ids, y) - t.distill_loss(dn, ids, y)) / 0.1
        assert (da - ga[:, v]).abs().max() < 5e-3
        assert (db - gb[:, v]).abs().max() < 5e-3


def test_far_rows_and_repeated_rows():
    """Rows 2^31 elements apart (offsets pass 32 bits), and rows that share
    their memory (stride 0)."""
    import torch
    import tmnn_b200 as t
    V, far = 5003, 1 << 31
    mem = torch.empty(far + V, dtype=torch.bfloat16, device="cuda")
    x = mem.as_strided((2, V), (far, 1))
    torch.manual_seed(1)
    x.copy_(torch.randn(2, V, device="cuda"))
    # near rows that start on the same boundaries: rows that start elsewhere are
    # summed in another order, which is within the bounds but not bit for bit
    near = torch.empty(2, V + 5, dtype=torch.bfloat16, device="cuda")[:, :V]
    near.copy_(x)
    tok = torch.tensor([7, V - 1], device="cuda")
    a = t.token_logprobs(x, tok, top_k=9, stats=True)
    b = t.token_logprobs(near, tok, top_k=9, stats=True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    one = torch.ones(2, device="cuda")
    want = t.token_logprobs_backward(near, tok, b.stats, one, one)
    ids = torch.tensor([[1, 2], [0, V - 1]], device="cuda")
    y = torch.randn(2, 2, device="cuda")
    wl, wg = t.distill_forward_backward(near, ids, y)
    save = near.clone()
    l, _ = t.distill_forward_backward(x, ids, y, out=x)
    assert torch.equal(l, wl) and torch.equal(x, wg)
    x.copy_(save)
    t.token_logprobs_backward(x, tok, b.stats, one, one, out=x)
    assert torch.equal(x, want)
    del mem, x
    same = near[:1].expand(5, V)
    c = t.token_logprobs(same, torch.full((5,), 7, device="cuda"), top_k=9)
    assert torch.equal(c.logprob, a.logprob[:1].expand(5))
    assert torch.equal(c.top_ids, a.top_ids[:1].expand(5, 9))


def test_one_row_in_place():
    """A single row's stride does not matter, in place either."""
    import torch
    import tmnn_b200 as t
    for V in (7, 900, 70001):
        x = torch.randn(V, device="cuda").expand(1, V)
        tok = torch.tensor([V - 1], device="cuda")
        one = torch.ones(1, device="cuda")
        st = t.token_logprobs(x, tok, stats=True).stats
        want = t.token_logprobs_backward(x, tok, st, one, one)
        _, dist = t.distill_forward_backward(x, tok.view(1, 1), one.view(1, 1))
        y = x.clone().as_strided((1, V), (0, 1))
        assert torch.equal(t.token_logprobs_backward(y, tok, st, one, one, out=y),
                           want)
        y = x.clone().as_strided((1, V), (0, 1))
        t.distill_forward_backward(y, tok.view(1, 1), one.view(1, 1), out=y)
        assert torch.equal(y, dist)


def test_in_place_gradients_are_seen_by_autograd():
    """A gradient written over a tensor that an autograd graph has saved makes
    that graph's backward pass an error, as torch's own in-place calls do;
    tensors without a version are written as well."""
    import torch
    import tmnn_b200 as t
    w = torch.ones(4, 9, device="cuda", requires_grad=True)
    ids = torch.ones(4, 2, dtype=torch.int64, device="cuda")
    y = torch.zeros(4, 2, device="cuda")
    tok = torch.zeros(4, dtype=torch.int64, device="cuda")
    one = torch.ones(4, device="cuda")

    def distil(x):
        t.distill_forward_backward(x, ids, y, out=x)

    def policy(x):
        r = t.token_logprobs(x, tok, stats=True)
        t.token_logprobs_backward(x, tok, r.stats, one, out=x)

    for write in (distil, policy):
        x = w * 2
        z = (x * x).sum()  # saves x
        write(x.detach())
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            z.backward()
        with torch.inference_mode():
            x = w * 2
            write(x)
            assert not torch.equal(x, w * 2)


def test_empty_batches():
    import torch
    import tmnn_b200 as t
    x = torch.empty(0, 17, device="cuda")
    i = torch.empty(0, dtype=torch.int64, device="cuda")
    r = t.token_logprobs(x, i, top_k=3, stats=True)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 3)
    g = t.token_logprobs_backward(x, i, r.stats, r.logprob, r.entropy)
    assert g.shape == (0, 17)
    l, g = t.distill_forward_backward(x, i.view(0, 1).expand(0, 2).contiguous(),
                                      torch.empty(0, 2, device="cuda"))
    assert l.shape == (0,) and g.shape == (0, 17)


def test_refusals():
    import torch
    import tmnn_b200 as t
    x = torch.zeros(4, 10, device="cuda")
    tok = torch.zeros(4, dtype=torch.int64, device="cuda")
    y = torch.zeros(4, 2, device="cuda")
    ids = torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    st = t.token_logprobs(x, tok, stats=True).stats
    for bad in (lambda: t.token_logprobs(x.double(), tok),
                lambda: t.token_logprobs(x, tok.float()),
                lambda: t.token_logprobs(x, tok.short()),
                lambda: t.distill_loss(x, ids, y.double()),
                lambda: t.distill_forward_backward(x, ids, y, out=x.half()),
                lambda: t.token_logprobs_backward(x, tok, st.half())):
        with pytest.raises(t.DTypeError):
            bad()
    for bad in (lambda: t.token_logprobs(x.view(2, 2, 10), tok),
                lambda: t.token_logprobs(x.t(), tok),
                lambda: t.token_logprobs(x, tok[:3]),
                lambda: t.token_logprobs(x, tok.cpu()),
                lambda: t.token_logprobs(x, tok, top_k=11),
                lambda: t.token_logprobs(x, tok, top_k=-1),
                lambda: t.token_logprobs(x, tok, temperature=0.0),
                lambda: t.token_logprobs(x[:, :0], tok),
                lambda: t.distill_loss(x, ids[:, :0], y[:, :0]),
                lambda: t.distill_loss(x, ids, y.t().contiguous().t()),
                lambda: t.distill_loss(x, ids[:, :1], y),
                lambda: t.distill_forward_backward(x, ids, y, row_weight=y),
                lambda: t.distill_forward_backward(x, ids, y, out=x[:3]),
                lambda: t.distill_forward_backward(
                    x, ids, y, out=torch.zeros(10, device="cuda").expand(4, 10)),
                lambda: t.distill_forward_backward(
                    x[:, :9], ids, y, out=x[:, 1:]),
                lambda: t.distill_forward_backward(
                    x, ids, y, out=torch.zeros(8, 10, device="cuda")[::2, :8]),
                lambda: t.token_logprobs_backward(x, tok, st[:, :2], y[:, 0]),
                lambda: t.token_logprobs_backward(x, None, st, y[:, 0].contiguous())):
        with pytest.raises(ValueError):
            bad()


def test_streams_graphs_and_repeats():
    """The current stream is used; captured calls replay on new values; two
    calls give the same bits."""
    import torch
    import tmnn_b200 as t
    for n, V in ((64, 64), (3, 100000), (40, 9001)):
        torch.manual_seed(n)
        data = [torch.randn(n, V, device="cuda").bfloat16() * 3 for _ in range(2)]
        tok = torch.randint(0, V, (n,), device="cuda")
        ids = torch.randint(0, V, (n, 8), device="cuda")
        y = torch.randn(n, 8, device="cuda")
        one = torch.ones(n, device="cuda")

        def run(x):
            r = t.token_logprobs(x, tok, top_k=8, stats=True)
            g = t.token_logprobs_backward(x, tok, r.stats, one, one)
            return [*r, g, *t.distill_forward_backward(x, ids, y),
                    t.distill_loss(x, ids, y)]

        want = [run(x) for x in data]
        for x, w in zip(data, want):
            assert all(torch.equal(a, b) for a, b in zip(run(x), w))
        x = data[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            late = torch.empty_like(x)
            torch.cuda._sleep(20_000_000)  # only stream order makes it right
            late.copy_(data[1])
            got = run(late)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(x)
        for data_x, w in zip(data[::-1], want[::-1]):
            x.copy_(data_x)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, w))


def test_two_threads_on_two_streams():
    """Calls of several threads, each on a stream of its own, at once."""
    import threading
    import torch
    import tmnn_b200 as t
    out, errors = {}, []

    def work(seed, V):
        try:
            g = torch.Generator(device="cuda").manual_seed(seed)
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                x = torch.randn(150, V, device="cuda", generator=g)
                tok = torch.randint(0, V, (150,), device="cuda", generator=g)
                y = torch.randn(150, 3, device="cuda", generator=g)
                ids = torch.randint(0, V, (150, 3), device="cuda", generator=g)
                one = torch.ones(150, device="cuda")
                for _ in range(20):
                    r = t.token_logprobs(x, tok, top_k=5, stats=True)
                    d = t.token_logprobs_backward(x, tok, r.stats, one, one)
                    e = t.distill_forward_backward(x, ids, y)
            stream.synchronize()
            out.setdefault((seed, V), []).append([*r, d, *e])
        except Exception as ex:  # reported by the test's thread
            errors.append(ex)

    for _ in range(2):  # the second round's results are the first's
        threads = [threading.Thread(target=work, args=(i, V))
                   for i, V in enumerate((40, 700, 5000, 30000))]
        for th in threads:
            th.start()
        for th in threads:
            th.join()
    assert not errors, errors
    for first, second in out.values():
        assert all(torch.equal(a, b) for a, b in zip(first, second))
    for (seed, V), (first, _) in out.items():
        torch.manual_seed(0)
        g = torch.Generator(device="cuda").manual_seed(seed)
        x = torch.randn(150, V, device="cuda", generator=g)
        tok = torch.randint(0, V, (150,), device="cuda", generator=g)
        lone = t.token_logprobs(x, tok, top_k=5, stats=True)
        assert all(torch.equal(a, b) for a, b in zip(first, lone))


# ------------------------------------------------------ as they are used
def test_teacher_to_student_run():
    """A teacher's logits -> its top classes -> the student's distillation
    gradient, against the definitions; a teacher equal to the student over all
    classes gives no loss."""
    import torch
    import tmnn_b200 as t
    n, V, K, T = 50, 1500, 20, 2.0
    torch.manual_seed(11)
    teacher = (torch.randn(n, V, device="cuda") * 3).bfloat16()
    student = (torch.randn(n, V, device="cuda") * 3).bfloat16()
    tk = torch.randint(0, V, (n,), device="cuda")
    top = t.token_logprobs(teacher, tk, top_k=K)
    loss, g = t.distill_forward_backward(student, top.top_ids, top.top_logprobs,
                                         temperature=T)
    ids = top.top_ids.cpu().numpy().astype(np.int64)
    y = np.take_along_axis(teacher.double().cpu().numpy(), ids, 1)
    want, tl, d, td = ref.distill(student.double().cpu().numpy(), T, ids, y,
                                  np.full(n, np.float32(1.0 / n)))
    # the entries are log probabilities of the teacher: each is off by at most
    # 1e-5 (the bound of logprob above), and moves its row's loss by T^2 2e-5
    # |log ratio| <= T^2 2e-5 30 / T, its gradient by w T 2e-5 / T
    ref.assert_close(loss.cpu(), want, tl + T * 6e-4)
    ref.assert_close(g.double().cpu(), d, _round(d, td + 2e-5 / n, "bf16"))
    small = student[:, :128].float()
    full = t.token_logprobs(small, top_k=128)
    zero = t.distill_loss(small, full.top_ids, full.top_logprobs)
    # ln s of both sides: (64 + 17 + 4 + 3 * 10) u each (the reference's ds at
    # 128 classes), and a few u of values below 20: under 3e-5
    assert zero.abs().max() < 3e-5


CFG = {"encoding": {"n_levels": 8, "n_features_per_level": 2,
                    "log2_hashmap_size": 14, "base_resolution": 16,
                    "per_level_scale": 1.447},
       "network": {"n_neurons": 64, "n_hidden_layers": 1},
       "optimizer": {"learning_rate": 1e-2}}


def _field(n_out, family="Auto"):
    import tmnn_b200 as t
    cfg = dict(CFG, b200={"family": family})
    return t.Trainer.from_config(cfg, n_input=3, n_output=n_out)


@pytest.mark.parametrize("n_out,family", [(16, "Auto"), (19, "SafeDebug"),
                                          (64, "SafeDebug")])
def test_trainer_token_logprobs(n_out, family):
    """Trainer.token_logprobs is inference() read by token_logprobs, for host
    arrays and CUDA tensors."""
    import torch
    import tmnn_b200 as t
    rng = np.random.default_rng(2)
    pos = rng.uniform(-1, 1, (700, 3)).astype(np.float32)
    tok = rng.integers(-1, n_out, 700)
    with _field(n_out, family) as tr:
        want = t.token_logprobs(torch.from_numpy(tr.inference(pos)).cuda(),
                                torch.from_numpy(tok).cuda(), top_k=5,
                                temperature=0.7)
        host = tr.token_logprobs(pos, tok, top_k=5, temperature=0.7)
        dev = tr.token_logprobs(torch.from_numpy(pos).cuda(),
                                torch.from_numpy(tok).cuda().int(), top_k=5,
                                temperature=0.7)
        for h, d, w in zip(host[:4], dev[:4], want[:4]):
            assert np.array_equal(h, w.cpu().numpy())
            assert torch.equal(d, w)
        r = tr.token_logprobs(pos[:9])
        assert r.logprob is None and r.top_ids is None and r.entropy.shape == (9,)
        assert tr.token_logprobs(pos[:0], tok[:0], top_k=2).top_ids.shape == (0, 2)
        for bad in (lambda: tr.token_logprobs(pos, tok[:5]),
                    lambda: tr.token_logprobs(pos, tok, top_k=n_out + 1),
                    lambda: tr.token_logprobs(pos, tok, temperature=-1.0),
                    lambda: tr.token_logprobs(pos, torch.from_numpy(tok).cuda())):
            with pytest.raises(ValueError):
                bad()
        with pytest.raises(t.DTypeError):
            tr.token_logprobs(pos, tok.astype(np.float32))
    with pytest.raises(t.ClosedError):
        tr.token_logprobs(pos, tok)


def test_trainer_empty_cuda_batch():
    """An empty CUDA batch, whose tensors have no address, is a no-op."""
    import torch
    with _field(16) as tr:
        pos = torch.empty(0, 3, device="cuda")
        r = tr.token_logprobs(pos, torch.empty(0, dtype=torch.int64,
                                               device="cuda"), top_k=3)
        assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 3)
        assert tr.token_logprobs(pos, top_k=2).entropy.shape == (0,)
        ids = torch.empty(0, 2, dtype=torch.int32, device="cuda")
        assert tr.distill_step(pos, ids, torch.empty(0, 2, device="cuda")) == 0.0
        assert tr.step() == 0


def test_trainer_refuses_host_memory_as_device_memory():
    """Pointers flagged as device pointers that are the host's are refused
    before anything is queued (another device's go the same way)."""
    import ctypes as C
    import torch
    from tmnn_b200 import _abi
    pos = torch.zeros(8, 3, device="cuda")
    ids = torch.zeros(8, 2, dtype=torch.int32, device="cuda")
    y = torch.zeros(8, 2, device="cuda")
    ent = torch.zeros(8, device="cuda")
    host = np.zeros((8, 3), np.float32)
    at, far = (lambda t: C.c_void_p(t.data_ptr())), C.c_void_p(host.ctypes.data)
    with _field(16) as tr:
        h, lib, dev = tr._handle(), _abi.lib, _abi.PTR_DEVICE
        for a in ((far, None, at(ent)), (at(pos), far, at(ent)),
                  (at(pos), None, far)):
            assert lib.tmnn_cuda_ctx_token_logprobs(
                h, a[0], a[1], _abi.INDEX_I32, 8, 0, 1.0, dev, None, a[2], None,
                None) == _abi.ERR_INVALID_ARGUMENT
        loss = C.c_float(1.0)
        for a in ((far, at(ids), at(y)), (at(pos), far, at(y)),
                  (at(pos), at(ids), far)):
            assert lib.tmnn_cuda_distill_step(
                h, a[0], a[1], _abi.INDEX_I32, a[2], 8, 2, 1.0, dev,
                C.byref(loss)) == _abi.ERR_INVALID_ARGUMENT
        assert tr.step() == 0
        assert tr.distill_step(pos, ids, y) >= 0.0


def _teacher(n, n_out, K, seed):
    rng = np.random.default_rng(seed)
    pos = rng.uniform(-1, 1, (n, 3)).astype(np.float32)
    ids = np.argsort(rng.random((n, n_out)), axis=1)[:, :K].astype(np.int64)
    y = rng.normal(size=(n, K)).astype(np.float32)
    ids[rng.random((n, K)) < 0.1] = -1
    ids[n // 2] = -1
    return pos, np.ascontiguousarray(ids), y


@pytest.mark.parametrize("n_out,family,n", [(16, "FullyFused", 1000),
                                            (19, "SafeDebug", 300)])
def test_distill_step_is_the_split_step(n_out, family, n):
    """distill_step does what forward_for_training, distill_forward_backward,
    backward_accumulate and adam_step do by hand, from host arrays and from
    CUDA tensors: the same loss and, with the integer hash gradients, the same
    hash weights; the MLP's gradients are float atomics, whose order moves an
    Adam step only where a gradient is next to zero."""
    import torch
    import tmnn_b200 as t
    pos, ids, y = _teacher(n, n_out, 4, 5)
    cu = [torch.from_numpy(a).cuda() for a in (pos, ids, y)]
    a, b, c = (_field(n_out, family) for _ in range(3))
    la = a.distill_step(pos, ids, y, temperature=2.0)
    lc = c.distill_step(*cu, temperature=2.0)
    out = b.forward_for_training(cu[0])
    loss, g = t.distill_forward_backward(out, cu[1], cu[2], temperature=2.0)
    torch.cuda.synchronize()
    b.backward_accumulate(cu[0], g)
    b.adam_step()
    assert abs(la - loss.double().mean().item()) <= 2 ** -23 * abs(la)
    assert la == lc
    (ha, ma), (hb, mb), (hc, mc) = a.weights(), b.weights(), c.weights()
    assert np.array_equal(ha, hb) and np.array_equal(ha, hc)
    assert np.mean(np.abs(ma - mb) > 1e-5) < 0.01
    assert a.step() == b.step() == c.step() == 1
    # the batch's gradient reached the weights
    with _field(n_out, family) as fresh:
        assert not np.array_equal(fresh.weights()[0], ha)
        assert fresh.distill_step(pos[:0], ids[:0], y[:0]) == 0.0
    for tr in (a, b, c):
        tr.close()


def test_distill_step_refusals():
    import torch
    import tmnn_b200 as t
    pos, ids, y = _teacher(64, 16, 4, 6)
    with _field(16) as tr:
        for bad in (lambda: tr.distill_step(pos, ids[:5], y),
                    lambda: tr.distill_step(pos, ids, y[:, :3]),
                    lambda: tr.distill_step(pos, ids[:, 0], y),
                    lambda: tr.distill_step(pos, ids, y, temperature=0.0),
                    lambda: tr.distill_step(pos, torch.from_numpy(ids).cuda(), y),
                    lambda: tr.distill_step(pos, np.zeros((64, 0), np.int64),
                                            np.zeros((64, 0), np.float32))):
            with pytest.raises(ValueError):
                bad()
        with pytest.raises(t.DTypeError):
            tr.distill_step(pos, ids.astype(np.int16), y)
        with pytest.raises(t.DTypeError):
            tr.distill_step(pos, ids, y.astype(np.float64))
        tgt = np.zeros((64, 16), np.float32)
        tr.training_step_enqueue(pos, tgt)
        with pytest.raises(ValueError, match="pending"):
            tr.distill_step(pos, ids, y)
        tr.training_step_finalize()
        before = tr.launch_count()
        tr.distill_step(pos, ids, y)
        assert tr.launch_count() > before


def test_distill_step_after_a_cuda_producer():
    """CUDA inputs that are still being written on the current stream are
    waited for."""
    import torch
    pos, ids, y = _teacher(500, 16, 4, 7)
    want = _field(16).distill_step(pos, ids, y)
    cu = [torch.from_numpy(a).cuda() for a in (pos, ids, y)]
    late = [torch.zeros_like(a) for a in cu]
    tr = _field(16)
    torch.cuda.synchronize()
    torch.cuda._sleep(50_000_000)
    for a, b in zip(late, cu):
        a.copy_(b)
    assert tr.distill_step(*late) == want
