"""Measured calls of the class-logit operators: log probabilities of given
tokens (with the entropy and the top alternatives of each row), their backward
pass, and distillation from a teacher's top logits.

A case is a dict of plain values.  `own` false computes the plain form with
elementary torch operations; `own` true makes the framework's calls.

Definitions, for a row x[0..V) of logits, temperature T, z = x / T:
  lse = log sum_v exp(z_v),  p_v = exp(z_v - lse)
  logprob = z_token - lse,   entropy = -sum_v p_v (z_v - lse)
  top: the K largest logits, ties to the lowest class; a class at -inf is no
       alternative (id -1, log probability -inf)
  d_x = (d_logprob (delta_token - p) - d_entropy p (z - lse + entropy)) / T
  distillation: q = softmax of the teacher's top logits / T,
       loss = T^2 sum_k q_k (log q_k - (z_id_k - lse)),
       d_x = weight T (p - q)
A token below zero, or a row whose teacher ids are all below zero, is padding:
its outputs are 0 (no alternatives) and its gradient is zero.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "fp16": 2}
_INF = float("inf")
_lib = None


def _framework():
    global _lib
    if _lib is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "tiny-metal-nn_b200"))
        import tmnn_b200
        _lib = tmnn_b200
    return _lib


def _case(name, op, rows, classes, dtype, top=0, pad=0, padded=0.0,
          masked=0.0, temperature=1.0, index="i64", teacher="f32",
          ragged=False):
    """top: alternatives (logprobs) or teacher entries (distill); pad: columns
    between two rows; padded: share of padded rows at the end; masked: share of
    classes at -inf; ragged: rows with fewer teacher entries."""
    return {"name": name, "op": op, "rows": rows, "classes": classes,
            "dtype": dtype, "top": top, "pad": pad, "padded": padded,
            "masked": masked, "temperature": temperature, "index": index,
            "teacher": teacher, "ragged": ragged}


def listed():
    return [
        # one decoded token answered with its log probability and 5
        # alternatives: latency
        _case("decode-1x32768-bf16-top5", "logprobs", 1, 32768, "bf16", 5),
        # a decode batch over a large vocabulary
        _case("decode-64x131072-bf16-top20", "logprobs", 64, 131072, "bf16", 20,
              temperature=0.7),
        # scoring the tokens of a padded batch for a policy update
        _case("score-4096x131072-bf16", "logprobs", 4096, 131072, "bf16",
              padded=0.1),
        # constrained scoring: odd vocabulary, padded rows of memory, masks
        _case("score-1531x50003-fp16-top8", "logprobs", 1531, 50003, "fp16", 8,
              pad=61, masked=0.3, index="i32"),
        # class probabilities of a field's batch (2^18 points, 64 outputs)
        _case("field-262144x64-f32-top4", "logprobs", 262144, 64, "f32", 4),
        # a teacher's top logits, taken to distil from them
        _case("teacher-2048x131072-bf16-top64", "logprobs", 2048, 131072,
              "bf16", 64),
        # policy-gradient step: backward of log probability and entropy
        _case("policy-4096x131072-bf16", "logprobs_backward", 4096, 131072,
              "bf16", padded=0.1),
        _case("policy-1021x32003-f32", "logprobs_backward", 1021, 32003, "f32",
              temperature=0.7, index="i32"),
        # distillation step of a large-vocabulary student
        _case("distill-4096x131072-bf16-k64", "distill", 4096, 131072, "bf16",
              64, temperature=2.0, teacher="bf16", padded=0.1),
        # a field (2^18 points, 19 classes) distilled from a labelling teacher
        _case("distill-262144x19-f32-k4", "distill", 262144, 19, "f32", 4,
              index="i32", ragged=True),
        # odd sizes and rows with fewer teacher entries
        _case("distill-777x50021-fp16-k20", "distill", 777, 50021, "fp16", 20,
              pad=27, ragged=True),
        # held-out loss of a small batch
        _case("heldout-8x32768-f32-k16", "distill_loss", 8, 32768, "f32", 16,
              temperature=2.0),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "logprobs_backward", "distill",
                     "distill_loss"])
    classes = _log_uniform(rng, 2, 262144)
    if rng.random() < 0.5:
        classes |= 1
    rows = _log_uniform(rng, 1, min(524288, max(2, (1 << 28) // classes)))
    most = min(classes, 128)
    if op == "distill" or op == "distill_loss":
        top = _log_uniform(rng, 1, most)
    elif op == "logprobs" and rng.random() < 0.7:
        top = _log_uniform(rng, 1, min(most, 64))
    else:
        top = 0
    return {"op": op, "rows": rows, "classes": classes,
            "dtype": rng.choice(["f32", "bf16", "fp16"]), "top": top,
            "pad": rng.choice([0, 0, rng.randrange(1, 64)]),
            "padded": rng.choice([0.0, 0.0, 0.2]),
            "masked": rng.choice([0.0, 0.3]) if op.startswith("logprobs") else 0.0,
            "temperature": rng.choice([1.0, 1.0, 0.7, 2.0]),
            "index": rng.choice(["i32", "i64"]),
            "teacher": rng.choice(["f32", "bf16", "fp16"]),
            "ragged": rng.random() < 0.5}


def _live(case):
    """Rows that are not padding."""
    return case["rows"] - int(case["rows"] * case["padded"])


def work(case):
    n, v, k = _live(case), case["classes"], case["top"]
    rows, size = case["rows"], _SIZE[case["dtype"]]
    index = 8 if case["index"] == "i64" else 4
    if case["op"] == "logprobs":  # read the logits, write the row results
        return {"bytes": n * v * size + rows * (index + 8 + 8 * k),
                "flops": 5 * n * v}
    if case["op"] == "logprobs_backward":  # and write a gradient of their size
        return {"bytes": (n + rows) * v * size + rows * (index + 12 + 8),
                "flops": 8 * n * v}
    entries = rows * k * (index + _SIZE[case["teacher"]])
    if case["op"] == "distill":
        return {"bytes": (n + rows) * v * size + entries + rows * 8,
                "flops": 7 * n * v}
    return {"bytes": n * v * size + entries + rows * 4, "flops": 4 * n * v}


def prepare(case, seed):
    n, v, k = case["rows"], case["classes"], case["top"]
    live, dtype = _live(case), _DTYPES[case["dtype"]]
    index = torch.int64 if case["index"] == "i64" else torch.int32
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    # a mean over the rows; gradients in fp16 are kept in its range by a loss
    # scale, as training in fp16 has it
    scale = 1024.0 if case["dtype"] == "fp16" else 1.0 / max(1, live)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    # logits: a broad bulk with a few raised classes a row
    x = normal(n, v).mul_(2.5)
    peaks = torch.randint(0, v, (n, min(4, v)), device="cuda", generator=g)
    x.scatter_add_(1, peaks, 4.0 + 2.0 * normal(n, min(4, v)))
    if case["masked"]:
        x.masked_fill_(torch.rand((n, v), device="cuda", generator=g)
                       < case["masked"], -_INF)
        if live > 4:
            x[1] = -_INF  # a mask that leaves nothing
    # rows lie `pad` columns apart; what stands there is no logit
    hold = torch.full((n, v + case["pad"]), 100.0, device="cuda", dtype=dtype)
    logits = hold[:, :v]
    logits.copy_(x)
    state = {"case": case, "logits": logits}
    if case["op"].startswith("logprobs"):
        tokens = torch.randint(0, v, (n,), device="cuda", generator=g)
        pick = torch.rand((n,), device="cuda", generator=g) < 0.7
        tokens = torch.where(pick, peaks[:, 0], tokens)
        tokens[live:] = -1
        state["tokens"] = tokens.to(index)
        if case["op"] == "logprobs_backward":
            state["stats"] = _stats(logits, state["tokens"], case["temperature"])
            state["d_logprob"] = normal(n) * scale
            state["d_entropy"] = torch.full((n,), -0.01 * scale, device="cuda")
    else:
        x.add_(normal(n, v))  # the teacher: the student with noise
        values, ids = torch.topk(x, k, dim=1)
        if case["ragged"]:
            fewer = torch.randint(1, k + 1, (n, 1), device="cuda", generator=g)
            ids[torch.arange(k, device="cuda") >= fewer] = -1
        ids[live:] = -1
        state["ids"] = ids.to(index)
        state["teacher"] = values.to(_DTYPES[case["teacher"]])
        weight = torch.rand((n,), device="cuda", generator=g).add_(0.5)
        state["weight"] = weight * scale
    return state


def _stats(logits, tokens, t):
    """[row maximum, sum of exp((x - maximum) / T), entropy], what the forward
    call keeps for its backward pass."""
    x = logits.float()
    m = x.amax(1, keepdim=True)
    d = torch.where(x == -_INF, -_INF, x - m) / t
    e = d.exp()
    s = e.sum(1, keepdim=True)
    ed = torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True)
    h = torch.where(s > 0, s.log() - ed / s, 0.0)
    out = torch.cat([m, s, h], 1)
    return torch.where((tokens < 0)[:, None], 0.0, out)


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------ the framework
def _own(state):
    lib, case = _framework(), state["case"]
    t, op = case["temperature"], case["op"]
    if op == "logprobs":
        if case["top"]:
            r = lib.token_logprobs(state["logits"], state["tokens"],
                                   top_k=case["top"], temperature=t)
            return [r.logprob, r.entropy, r.top_ids, r.top_logprobs]
        r = lib.token_logprobs(state["logits"], state["tokens"], temperature=t,
                               stats=True)
        return [r.logprob, r.entropy, r.stats]
    if op == "logprobs_backward":
        return lib.token_logprobs_backward(
            state["logits"], state["tokens"], state["stats"],
            state["d_logprob"], state["d_entropy"], temperature=t)
    if op == "distill":
        return lib.distill_forward_backward(
            state["logits"], state["ids"], state["teacher"], temperature=t,
            row_weight=state["weight"])
    return lib.distill_loss(state["logits"], state["ids"], state["teacher"],
                            temperature=t)


# ------------------------------------------------------------ the plain form
def _top(x, k):
    """The k largest of each row, ties to the lowest class."""
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
    v = x.shape[1]
    key = order * (1 << 32) + (v - 1 - torch.arange(v, device=x.device))
    best = torch.topk(key, k, dim=1, sorted=True).values
    return v - 1 - (best & 0xFFFFFFFF)


def _plain(state):
    case, logits = state["case"], state["logits"]
    t, op = case["temperature"], case["op"]
    x = logits.float()
    n = x.shape[0]
    if op == "logprobs_backward":
        stats = state["stats"]
        tok = state["tokens"].to(torch.int64)
        m, s, h = stats[:, 0:1], stats[:, 1:2], stats[:, 2:3]
        logp = torch.where(x == -_INF, -_INF, x - m) / t - s.log()
        p = logp.exp()
        a, b = state["d_logprob"][:, None], state["d_entropy"][:, None]
        g = -a * p - b * torch.where(p > 0, p * (logp + h), 0.0)
        g.scatter_add_(1, tok.clamp(min=0)[:, None], a)
        g = torch.where((tok < 0)[:, None] | (m == -_INF), 0.0, g / t)
        return g.to(logits.dtype)
    m = x.amax(1, keepdim=True)
    empty = m[:, 0] == -_INF
    z = torch.where(x == -_INF, -_INF, x - m) / t
    e = z.exp()
    s = e.sum(1, keepdim=True)
    logp = z - s.log()
    if op == "logprobs":
        tok = state["tokens"].to(torch.int64)
        padded = tok < 0
        logprob = logp.gather(1, tok.clamp(min=0)[:, None])[:, 0]
        logprob = torch.where(empty, -_INF, logprob)
        ed = torch.where(e > 0, e * z, 0.0).sum(1)
        entropy = torch.where(empty, 0.0, s[:, 0].log() - ed / s[:, 0])
        logprob = torch.where(padded, 0.0, logprob)
        entropy = torch.where(padded, 0.0, entropy)
        k = case["top"]
        if not k:
            stats = torch.stack([m[:, 0], s[:, 0], entropy], 1)
            return [logprob, entropy,
                    torch.where(padded[:, None], 0.0, stats)]
        ids = _top(x, k)
        none = (x.gather(1, ids) == -_INF) | padded[:, None]
        top = torch.where(none, -_INF, logp.gather(1, ids))
        return [logprob, entropy, torch.where(none, -1, ids).to(torch.int32), top]
    # distillation
    ids = state["ids"].to(torch.int64)
    y = torch.where(ids < 0, -_INF, state["teacher"].float() / t)
    idle = (ids < 0).all(1)
    y = y - torch.where(idle, 0.0, y.amax(1))[:, None]
    q = y.exp()
    total = q.sum(1, keepdim=True)
    logq = y - total.log()
    q = torch.where(idle[:, None], 0.0, q / total)
    at = ids.clamp(min=0)
    loss = (t * t) * torch.where(q > 0, q * (logq - logp.gather(1, at)), 0.0).sum(1)
    if op == "distill_loss":
        return loss
    g = (e / s).scatter_add_(1, at, -q)
    g = g * (state["weight"] * t)[:, None]
    return [loss, torch.where(idle[:, None], 0.0, g).to(logits.dtype)]


# --------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    n, v, k, t = case["rows"], case["classes"], case["top"], case["temperature"]
    step = max(1, (1 << 25) // v)
    parts = [_exact_rows(state, case["op"], slice(i, min(n, i + step)), k, t)
             for i in range(0, n, step)]
    out = [torch.cat(p) for p in zip(*parts)]
    return out if case["op"] in ("logprobs", "distill") else out[0]


def _exact_rows(state, op, rows, k, t):
    x = state["logits"][rows].double()
    z = x / t
    lse = torch.logsumexp(z, 1)
    p = torch.exp(z - lse[:, None])
    if op.startswith("logprobs"):
        tok = state["tokens"][rows].long()
        skip, row = tok < 0, torch.arange(x.shape[0], device=x.device)
        dead = torch.isinf(lse)
        entropy = -torch.nan_to_num(p * (z - lse[:, None]), nan=0.0).sum(1)
        if op == "logprobs_backward":
            m, s, h = state["stats"][rows].double().unbind(1)
            lse = m / t + s.log()  # the saved statistics are inputs
            logp = z - lse[:, None]
            p = torch.exp(logp)
            a = state["d_logprob"][rows].double()
            b = state["d_entropy"][rows].double()
            g = -(a[:, None] * p)
            g[row, tok.clamp(min=0)] += a
            g -= b[:, None] * torch.nan_to_num(p * (logp + h[:, None]), nan=0.0)
            g[skip | torch.isinf(m)] = 0.0
            return [g / t]
        lp = z[row, tok.clamp(min=0)] - lse
        lp[dead] = -_INF
        lp[skip] = 0.0
        entropy[skip | dead] = 0.0
        if not k:
            m = x.max(1).values
            stats = torch.stack([m, torch.exp(lse - m / t), entropy], 1)
            stats[dead, 1] = 0.0
            stats[skip] = 0.0
            return [lp, entropy, stats]
        value, ids = torch.sort(x, dim=1, descending=True, stable=True)
        value, ids = value[:, :k], ids[:, :k].to(torch.int32)
        top = value / t - lse[:, None]
        none = torch.isinf(value) | skip[:, None]
        ids[none] = -1
        top[none] = -_INF
        return [lp, entropy, ids, top]
    ids = state["ids"][rows].long()
    valid = ids >= 0
    y = torch.where(valid, state["teacher"][rows].double() / t, -_INF)
    some = valid.any(1)
    logq = torch.where(some[:, None], torch.log_softmax(y, 1), -_INF)
    q = torch.exp(logq)
    logp = z.gather(1, ids.clamp(min=0)) - lse[:, None]
    loss = t * t * torch.where(valid, q * (logq - logp), 0.0).sum(1)
    if op == "distill_loss":
        return [loss]
    p.scatter_add_(1, ids.clamp(min=0), -q)
    g = p * (state["weight"][rows].double() * t)[:, None]
    g[~some] = 0.0
    return [loss, g]
