"""Operators over class logits (include/tmnn_cuda.h, tmnn_cuda_token_logprobs*
and tmnn_cuda_distill): log probabilities of given tokens with entropy and top
alternatives, their backward pass, and distillation from a teacher's top
logits.

The functions take CUDA torch tensors and queue their kernel on the current
stream of the tensors' device (whichever device is current); they do not wait
and can be captured into CUDA graphs.  They are plain functions of their
arguments: results are new tensors unless `out` is given, and no autograd graph
is recorded (the backward passes are calls of their own, as in the Trainer's
split API)."""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

from . import _abi
from ._abi import lib

_DTYPE = {"torch.float32": _abi.DTYPE_F32, "torch.float16": _abi.DTYPE_F16,
          "torch.bfloat16": _abi.DTYPE_BF16}
_INDEX = {"torch.int32": _abi.INDEX_I32, "torch.int64": _abi.INDEX_I64}


class TokenLogprobs(NamedTuple):
    """Row results of token_logprobs: `logprob` [n] (None without tokens),
    `entropy` [n], `top_ids` int32 and `top_logprobs` [n, top_k] (None without
    alternatives), `stats` [n, 3] (None unless asked for).  All but the ids
    are float32."""
    logprob: Optional[object]
    entropy: object
    top_ids: Optional[object]
    top_logprobs: Optional[object]
    stats: Optional[object]


def _check(status):
    if status != _abi.OK:
        msg = lib.tmnn_cuda_logits_last_error().decode()
        if status == _abi.ERR_INVALID_ARGUMENT:
            raise ValueError(msg)
        from . import TmnnError
        raise TmnnError(status, msg)


def _dtype_error(msg):
    from . import DTypeError
    return DTypeError(msg)


def _logits(x, temperature):
    """The C descriptor of a [n, classes] tensor of logits."""
    if not getattr(x, "is_cuda", False):
        raise ValueError("logits must be a CUDA tensor")
    dtype = _DTYPE.get(str(x.dtype))
    if dtype is None:
        raise _dtype_error(
            f"logits must be float32, float16 or bfloat16, got {x.dtype}")
    if x.dim() != 2:
        raise ValueError("logits must be 2D (rows, classes)")
    n, v = x.shape
    if v > 1 and x.stride(1) != 1:
        raise ValueError("the classes of a row of logits must be contiguous")
    if n >= 1 << 32 or v >= 1 << 32:
        raise ValueError("logits must have fewer than 2^32 rows and classes")
    return _abi.Logits(x.data_ptr(), x.stride(0), n, v, dtype, temperature)


def _vector(t, name, like, shape, kinds):
    """Pointer of a contiguous tensor of the given shape on like's device;
    `kinds` maps the dtypes it may have to their C values."""
    if not getattr(t, "is_cuda", False) or t.device != like.device:
        raise ValueError(f"{name} must be a CUDA tensor on the logits' device")
    kind = kinds.get(str(t.dtype))
    if kind is None:
        raise _dtype_error(f"{name} must be "
                           + " or ".join(k[6:] for k in kinds)
                           + f", got {t.dtype}")
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr(), kind


_F32 = {"torch.float32": _abi.DTYPE_F32}


def _gradient(out, x):
    import torch
    if out is None:
        return torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if (not getattr(out, "is_cuda", False) or out.device != x.device
            or out.shape != x.shape):
        raise ValueError("out must be a CUDA tensor of the logits' shape and device")
    if out.dtype != x.dtype:
        raise _dtype_error(f"out must have the logits' type {x.dtype}")
    if out.dim() == 2 and out.shape[1] > 1 and out.stride(1) != 1:
        raise ValueError("the classes of a row of out must be contiguous")
    return out


def _grad_stride(out):
    """Distance of the gradient's rows; of one row or none it is never used."""
    n, v = out.shape
    return out.stride(0) if n > 1 else max(v, out.stride(0))


def _stream(x):
    import torch
    return x.device.index, torch.cuda.current_stream(x.device).cuda_stream


def token_logprobs(logits, tokens=None, *, top_k=0, temperature=1.0,
                   stats=False) -> TokenLogprobs:
    """Per row of logits [n, classes] (float32, float16 or bfloat16, rows any
    distance apart): the log probability of tokens[i] under
    softmax(logits[i] / temperature), the entropy of that distribution in nats,
    and the top_k most likely classes with their log probabilities (ties to
    the lowest class; id -1 and -inf where fewer classes are above -inf).
    tokens [n]: int32 or int64; below 0 marks a padded row (results 0, no
    alternatives), at or above `classes` gives NaN.  stats=True also returns
    what token_logprobs_backward needs."""
    import torch
    x = _logits(logits, temperature)
    n = logits.shape[0]
    tp, it = (None, 0) if tokens is None else _vector(tokens, "tokens", logits,
                                                      (n,), _INDEX)
    k = int(top_k)
    if not 0 <= k <= min(logits.shape[1], _abi.MAX_TOP):
        raise ValueError("top_k must be in [0, min(classes, 128)]")
    dev = logits.device
    new = torch.empty
    lp = None if tokens is None else new((n,), dtype=torch.float32, device=dev)
    ent = new((n,), dtype=torch.float32, device=dev)
    ids = new((n, k), dtype=torch.int32, device=dev) if k else None
    top = new((n, k), dtype=torch.float32, device=dev) if k else None
    st = new((n, 3), dtype=torch.float32, device=dev) if stats else None
    d, s = _stream(logits)
    _check(lib.tmnn_cuda_token_logprobs(
        d, s, x, tp, it, k, None if lp is None else lp.data_ptr(),
        ent.data_ptr(), ids.data_ptr() if k else None,
        top.data_ptr() if k else None, st.data_ptr() if stats else None))
    return TokenLogprobs(lp, ent, ids, top, st)


def token_logprobs_backward(logits, tokens, stats, d_logprob=None,
                            d_entropy=None, *, temperature=1.0, out=None):
    """d_logits [n, classes], in the logits' type, of
    sum(d_logprob * logprob) + sum(d_entropy * entropy), from the arguments of
    a token_logprobs(..., stats=True) call and its stats.  Either of the
    incoming gradients (float32 [n]) may be None.  out: where to write it; it
    may be `logits` itself, whose values are then lost.  The alternatives'
    log probabilities carry no gradient."""
    x = _logits(logits, temperature)
    n = logits.shape[0]
    tp, it = (None, 0) if tokens is None else _vector(tokens, "tokens", logits,
                                                      (n,), _INDEX)
    sp, _ = _vector(stats, "stats", logits, (n, 3), _F32)
    gp = None if d_logprob is None else _vector(d_logprob, "d_logprob", logits,
                                                (n,), _F32)[0]
    hp = None if d_entropy is None else _vector(d_entropy, "d_entropy", logits,
                                                (n,), _F32)[0]
    out = _gradient(out, logits)
    d, s = _stream(logits)
    _check(lib.tmnn_cuda_token_logprobs_backward(
        d, s, x, tp, it, sp, gp, hp, out.data_ptr(), _grad_stride(out)))
    return out


def _distill(logits, teacher_ids, teacher_logits, temperature, row_weight, out):
    import torch
    x = _logits(logits, temperature)
    n = logits.shape[0]
    if teacher_ids.dim() != 2:
        raise ValueError("teacher_ids must be 2D (rows, k)")
    k = teacher_ids.shape[1]
    ip, it = _vector(teacher_ids, "teacher_ids", logits, (n, k), _INDEX)
    yp, yt = _vector(teacher_logits, "teacher_logits", logits, (n, k), _DTYPE)
    wp = None if row_weight is None else _vector(row_weight, "row_weight",
                                                 logits, (n,), _F32)[0]
    loss = torch.empty((n,), dtype=torch.float32, device=logits.device)
    d, s = _stream(logits)
    _check(lib.tmnn_cuda_distill(
        d, s, x, ip, it, yp, yt, k, wp, loss.data_ptr(),
        None if out is None else out.data_ptr(),
        0 if out is None else _grad_stride(out)))
    return loss


def distill_loss(logits, teacher_ids, teacher_logits, *, temperature=1.0):
    """Distillation loss of each row [n], float32: T^2 KL(q || p) of the
    teacher's distribution q = softmax(teacher_logits / T) over the k classes
    teacher_ids names, and p = softmax(logits / T) over all classes.
    teacher_ids [n, k] int32 or int64 (below 0: no entry; a row without
    entries is padding with loss 0), teacher_logits [n, k] float32, float16 or
    bfloat16 -- the top_ids and top_logprobs of token_logprobs fit both."""
    return _distill(logits, teacher_ids, teacher_logits, temperature, None, None)


def distill_forward_backward(logits, teacher_ids, teacher_logits, *,
                             temperature=1.0, row_weight=None, out=None):
    """(loss [n], d_logits [n, classes]): distill_loss and, from the same read
    of the logits, the gradient of sum(row_weight * loss) in the logits' type.
    row_weight float32 [n]; None is 1 / n, the gradient of the mean loss.  out:
    where to write the gradient; it may be `logits` itself."""
    _logits(logits, temperature)
    out = _gradient(out, logits)
    return _distill(logits, teacher_ids, teacher_logits, temperature,
                    row_weight, out), out
