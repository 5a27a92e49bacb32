"""The class-logit operators from their definitions in 64 bits (numpy), with
the error bounds that fp32 arithmetic allows.

Bounds: u = 2^-24 is half a step of fp32.  With d = (max - x) / T >= 0,
  t = (x - max) * (1 / T) rounds three times (difference, 1 / T, product):
      |error| <= 3 u d
  e = 2^(t log2 e) by ex2.approx, 2 ulp: relative error <= 3 u d + 4 u
  s = sum e: no term of the sum goes through more than `chain` additions, so
      its relative error is <= ds = u (chain + 4 + 3 sum p d)
  ln s: |error| <= ds + 2 u |ln s| (the logarithm is within an ulp)
Bounds of results follow by adding the errors of their terms; second-order
terms are covered by a factor of 1.1.  Results in bf16 / fp16 are rounded once
more, by half a step."""
import numpy as np

U = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
# what a value below the type's normal range is off by after rounding (fp32
# results and intermediates below 2^-126 may be flushed)
TINY = {"f32": 2.0 ** -125, "fp16": 2.0 ** -25, "bf16": 2.0 ** -125}


def chain(V):
    """Additions any term goes through: a lane of a narrow row sums up to 64
    elements, a thread of a wide one V / 256, and a reduction over lanes, warps
    and blocks follows."""
    return min(V, 64) + V / 256 + 16


class Rows:
    """Statistics of logits x [n, V] (float64 of the values the kernel reads)."""

    def __init__(self, x, T):
        self.x, self.T = x, T
        n, V = x.shape
        with np.errstate(all="ignore"):
            self.m = x.max(1)  # NaN propagates
            self.bad = ~(self.m < np.inf)
            self.empty = self.m == -np.inf
            m = np.where(self.bad | self.empty, 0.0, self.m)
            self.t = np.where(x == -np.inf, -np.inf, (x - m[:, None]) / T)
            self.t[self.bad] = np.nan
            e = np.exp(self.t)
            self.s = e.sum(1)
            self.p = e / self.s[:, None]
            d = np.where(e > 0, -self.t, 0.0)
            self.d = d
            self.Ed = (self.p * d).sum(1)
            self.ds = U * (chain(V) + 4 + 3 * self.Ed)
            self.ln_s = np.log(self.s)
            self.H = np.where(self.empty, 0.0, self.ln_s + self.Ed)
            self.lp = self.t - self.ln_s[:, None]
            self.lp[self.empty] = -np.inf
            self.tol_ln = self.ds + 2 * U * np.abs(self.ln_s)
            # H = ln s + sum e d / s: a term e d is off by (3 u d + 6 u) of
            # itself, the sum by chain u, the quotient by ds + 2 u
            pd = self.p * d
            self.tol_H = 1.1 * (self.tol_ln + U * (pd * (3 * d + 6)).sum(1)
                                + self.Ed * (U * (chain(V) + 4) + self.ds)
                                + 2 * U * np.abs(self.H)) + 1e-37
            self.tol_p = 1.1 * self.p * (U * (3 * d + 10) + self.ds[:, None])

    def tol_lp(self, d, lp):
        """Bound of t - ln s where t = -d."""
        return 1.1 * (U * 3 * d + self.tol_ln + 2 * U * np.abs(lp)) + 1e-37


def token_logprobs(x, T, tokens, k):
    """(logprob, entropy, ids, top, stats) and the Rows; padded rows as the
    calls define them."""
    r = Rows(x, T)
    n, V = x.shape
    rows = np.arange(n)
    if tokens is None:
        lp, pad = None, np.zeros(n, bool)
    else:
        pad = tokens < 0
        out = tokens >= V
        lp = r.lp[rows, np.clip(tokens, 0, V - 1)]
        lp = np.where(out, np.nan, lp)
        lp = np.where(pad, 0.0, lp)
    H = np.where(pad, 0.0, np.where(r.bad, np.nan, r.H))
    ids = np.argsort(-np.where(np.isnan(x), -np.inf, x), axis=1, kind="stable")[:, :k]
    none = (np.take_along_axis(x, ids, 1) == -np.inf) | r.bad[:, None] | pad[:, None]
    top = np.take_along_axis(r.lp, ids, 1)
    top = np.where(none, -np.inf, top)
    top[r.bad & ~pad] = np.nan
    ids = np.where(none, -1, ids)
    stats = np.stack([np.where(r.bad, np.nan, r.m),
                      np.where(r.empty, 0.0, r.s), H], 1)
    stats[r.bad] = np.nan
    stats[pad] = 0.0
    return lp, H, ids, top, stats, r


def token_logprobs_backward(x, T, tokens, stats, g, h):
    """(d_x, bound) from given float32 stats."""
    n, V = x.shape
    m, s, H = (stats[:, i].astype(np.float64)[:, None] for i in range(3))
    idle = (stats[:, 1] == 0) | (tokens < 0 if tokens is not None else False)
    with np.errstate(all="ignore"):
        t = np.where(x == -np.inf, -np.inf, (x - m) / T)
        p = np.exp(t) / s
        lp = t - np.log(s)
        g = np.zeros((n, 1)) if g is None else g.astype(np.float64)[:, None] / T
        h = np.zeros((n, 1)) if h is None else h.astype(np.float64)[:, None] / T
        if tokens is not None:
            g = np.where((tokens >= V)[:, None], np.nan, g)
        plp = np.where(p > 0, p * (lp + H), 0.0)
        d = -g * p - h * plp
        # p off by (3 d + 10) u; lp + H by 3 u d + 2 u of each of its terms;
        # the products and their sum by 4 u
        dd = np.where(p > 0, -t, 0.0)
        rel = U * (3 * dd + 14)
        lnH = np.abs(np.log(s)) + np.abs(H)
        tol = 1.1 * (np.abs(g) * p * rel + np.abs(plp) * np.abs(h) * rel
                     + np.abs(h) * p * U * (5 * dd + 4 * lnH))
        if tokens is not None:
            rows = np.arange(n)
            at = np.clip(tokens, 0, V - 1)
            d[rows, at] += g[:, 0]
            tol[rows, at] += 4 * U * np.abs(g[:, 0])
    d[idle] = 0.0
    tol[idle] = 0.0
    return d, tol


def distill(x, T, ids, y, w):
    """(loss, bound, d_x, bound) of each row."""
    n, V = x.shape
    r = Rows(x, T)
    with np.errstate(all="ignore"):
        left = (ids < 0) | (y == -np.inf)
        y = np.where(left, -np.inf, np.where(ids >= V, np.nan, y))
        pad = left.all(1)
        ym = np.where(pad, 0.0, y.max(1))
        bad = (r.bad | ~(ym < np.inf)) & ~pad
        ty = (y - ym[:, None]) / T
        ey = np.exp(ty)
        ys = ey.sum(1, keepdims=True)
        q = np.where(left, 0.0, ey / ys)
        lq = ty - np.log(ys)
        at = np.where(left, 0, np.clip(ids, 0, V - 1))
        lpk = np.take_along_axis(r.lp, at, 1)
        terms = np.where(q > 0, q * (lq - lpk), 0.0)
        loss = T * T * terms.sum(1)
        loss = np.where(pad, 0.0, np.where(bad, np.nan, loss))
        loss = np.where(r.empty & ~pad & ~bad, np.inf, loss)
        # a term: q off by (3 dy + 6 + K) u of itself, the difference by the
        # errors of its three parts; their sum by K u; T^2 by 2 u
        K = ids.shape[1]
        dy = np.where(q > 0, -ty, 0.0)
        dk = np.take_along_axis(r.d, at, 1)
        sub = (U * (3 * dy + 3 * dk + 2 * np.abs(np.log(ys)) + K + 8
                    + 2 * np.abs(np.where(q > 0, lq, 0.0))
                    + 2 * np.abs(np.where(q > 0, lpk, 0.0)))
               + r.tol_ln[:, None])
        tol_loss = 1.1 * T * T * np.where(
            q > 0, q * sub + np.abs(terms) * U * (3 * dy + 2 * K + 10), 0.0
        ).sum(1) + 1e-37
        d = np.where(r.empty[:, None], 0.0, r.p)
        tol = np.where(r.empty[:, None], 0.0, r.tol_p + 4 * U * r.p)
        for k in range(K):
            # a row with nothing left has no gradient
            on = ~left[:, k] & ~r.empty & ~bad
            rows = np.nonzero(on)[0]
            d[rows, at[rows, k]] -= q[rows, k]
            tol[rows, at[rows, k]] += (q[rows, k] * U
                                       * (3 * dy[rows, k] + 2 * K + 12))
        f = (w.astype(np.float64) * T)[:, None]
        d, tol = d * f, tol * np.abs(f)
        d[bad], d[pad], tol[pad] = np.nan, 0.0, 0.0
    return loss, tol_loss, d, tol


def assert_close(got, want, tol, what=""):
    """|got - want| <= tol, NaN and infinities in the same places."""
    got = np.asarray(got, np.float64)
    want = np.asarray(want, np.float64)
    # a value beyond the fp32 range (the lowest fp32 number over T = 0.7 is
    # -4.9e38) rounds to infinity
    want = np.where(want > 3.5e38, np.inf, np.where(want < -3.5e38, -np.inf, want))
    tol = np.broadcast_to(tol, want.shape)
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), (what, "NaN places")
    inf = ~fin & ~np.isnan(want)
    assert np.array_equal(got[inf], want[inf]), (what, "infinities")
    err = np.abs(got[fin] - want[fin])
    over = err > tol[fin]
    assert not over.any(), (what, int(over.sum()), float(err[over].max()),
                            float((err[over] / tol[fin][over]).max()))
