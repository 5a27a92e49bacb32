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

from typing import NamedTuple, Optional

from . import _abi
from ._abi import lib

# torch, its dtypes' C values and the function that gives a device's current
# stream; filled at the first call (importing this package does not import
# torch, and small calls cost as much in Python as on the GPU)
_torch = None
_DTYPE: dict = {}
_INDEX: dict = {}
_F32: dict = {}
_raw_stream = None


def _load_torch():
    global _torch, _raw_stream
    import torch
    _DTYPE.update({torch.float32: _abi.DTYPE_F32, torch.float16: _abi.DTYPE_F16,
                   torch.bfloat16: _abi.DTYPE_BF16})
    _INDEX.update({torch.int32: _abi.INDEX_I32, torch.int64: _abi.INDEX_I64})
    _F32[torch.float32] = _abi.DTYPE_F32
    _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
        lambda index: torch.cuda.current_stream(index).cuda_stream)
    _torch = torch
    return torch


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
    if _torch is None:
        _load_torch()
    dtype = _DTYPE.get(x.dtype)
    if dtype is None:
        raise _dtype_error(
            f"logits must be float32, float16 or bfloat16, got {x.dtype}")
    if x.dim() != 2:
        raise ValueError("logits must be 2D (rows, classes)")
    n, v = x.shape
    stride, step = x.stride()
    if step != 1 and v > 1:
        raise ValueError("the classes of a row of logits must be contiguous")
    if n >= 1 << 32 or v >= 1 << 32:
        raise ValueError("logits must have fewer than 2^32 rows and classes")
    return _abi.Logits(x.data_ptr(), stride, n, v, dtype, temperature)


def _vector(t, name, device, shape, kinds):
    """(pointer, C type) of a contiguous tensor of the given shape on `device`;
    `kinds` maps the dtypes it may have to their C values."""
    if not getattr(t, "is_cuda", False) or t.device != device:
        raise ValueError(f"{name} must be a CUDA tensor on the logits' device")
    kind = kinds.get(t.dtype)
    if kind is None:
        raise _dtype_error(f"{name} must be "
                           + " or ".join(str(k)[6:] for k in kinds)
                           + f", got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr(), kind


def _gradient(out, x):
    if out is None:
        return _torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if (not getattr(out, "is_cuda", False) or out.device != x.device
            or out.shape != x.shape):
        raise ValueError("out must be a CUDA tensor of the logits' shape and device")
    if out.dtype != x.dtype:
        raise _dtype_error(f"out must have the logits' type {x.dtype}")
    if out.shape[1] > 1 and out.stride(1) != 1:
        raise ValueError("the classes of a row of out must be contiguous")
    if out.requires_grad and _torch.is_grad_enabled() and (
            out.is_leaf or (out._is_view() and out._base.is_leaf)):
        raise ValueError("out is a leaf that requires a gradient, or a view of "
                         "one: pass out.detach(), or call under torch.no_grad()")
    return out


def _written(out):
    """Tells autograd that a tensor of the caller's has new values, so that a
    graph that saved the old ones refuses its backward pass."""
    if not out.is_inference():  # those have no version
        _torch.autograd.graph.increment_version(out)


def _grad_stride(out):
    """Distance of the gradient's rows; of one row or none it is never used."""
    n, v = out.shape
    return out.stride(0) if n > 1 else max(v, out.stride(0))


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
    x = _logits(logits, temperature)
    n, dev = x.rows, logits.device
    k = int(top_k)
    if not 0 <= k <= min(x.classes, _abi.MAX_TOP):
        raise ValueError("top_k must be in [0, min(classes, 128)]")
    empty, f32 = _torch.empty, _torch.float32
    lp = lpp = tp = ids = top = idp = topp = st = stp = None
    it = 0
    if tokens is not None:
        tp, it = _vector(tokens, "tokens", dev, (n,), _INDEX)
        lp = empty(n, dtype=f32, device=dev)
        lpp = lp.data_ptr()
    ent = empty(n, dtype=f32, device=dev) if lp is None else _torch.empty_like(lp)
    if k:
        top = ent.new_empty(n, k)
        ids = _torch.empty_like(top, dtype=_torch.int32)
        idp, topp = ids.data_ptr(), top.data_ptr()
    if stats:
        st = empty(n, 3, dtype=f32, device=dev)
        stp = st.data_ptr()
    index = dev.index
    _check(lib.tmnn_cuda_token_logprobs(
        index, _raw_stream(index), x, tp, it, k, lpp, ent.data_ptr(), idp, topp,
        stp))
    return TokenLogprobs(lp, ent, ids, top, st)


def token_logprobs_backward(logits, tokens, stats, d_logprob=None,
                            d_entropy=None, *, temperature=1.0, out=None):
    """d_logits [n, classes], in the logits' type, of
    sum(d_logprob * logprob) + sum(d_entropy * entropy), from the arguments of
    a token_logprobs(..., stats=True) call and its stats.  Either of the
    incoming gradients (float32 [n]) may be None.  out: where to write it; it
    may be `logits` itself, whose values are then lost, but no leaf that
    requires a gradient.  The alternatives' log probabilities carry no
    gradient."""
    x = _logits(logits, temperature)
    n, dev = x.rows, logits.device
    tp, it = (None, 0) if tokens is None else _vector(tokens, "tokens", dev,
                                                      (n,), _INDEX)
    sp, _ = _vector(stats, "stats", dev, (n, 3), _F32)
    gp = None if d_logprob is None else _vector(d_logprob, "d_logprob", dev,
                                                (n,), _F32)[0]
    hp = None if d_entropy is None else _vector(d_entropy, "d_entropy", dev,
                                                (n,), _F32)[0]
    given, out = out, _gradient(out, logits)
    index = dev.index
    _check(lib.tmnn_cuda_token_logprobs_backward(
        index, _raw_stream(index), x, tp, it, sp, gp, hp, out.data_ptr(),
        _grad_stride(out)))
    if given is not None:
        _written(out)
    return out


def _distill(x, logits, teacher_ids, teacher_logits, row_weight, out):
    n, dev = x.rows, logits.device
    if not getattr(teacher_ids, "is_cuda", False) or teacher_ids.dim() != 2:
        raise ValueError("teacher_ids must be a 2D CUDA tensor (rows, k)")
    k = teacher_ids.shape[1]
    ip, it = _vector(teacher_ids, "teacher_ids", dev, (n, k), _INDEX)
    yp, yt = _vector(teacher_logits, "teacher_logits", dev, (n, k), _DTYPE)
    wp = dp = None
    stride = 0
    if row_weight is not None:
        wp, _ = _vector(row_weight, "row_weight", dev, (n,), _F32)
    if out is not None:
        dp, stride = out.data_ptr(), _grad_stride(out)
    loss = _torch.empty(n, dtype=_torch.float32, device=dev)
    index = dev.index
    _check(lib.tmnn_cuda_distill(index, _raw_stream(index), x, ip, it, yp, yt, k,
                                 wp, loss.data_ptr(), dp, stride))
    return loss


def distill_loss(logits, teacher_ids, teacher_logits, *, temperature=1.0):
    """Distillation loss of each row [n], float32: T^2 KL(q || p) of the
    teacher's distribution q = softmax(teacher_logits / T) over the k classes
    teacher_ids names, and p = softmax(logits / T) over all classes.
    teacher_ids [n, k] int32 or int64 (below 0: no entry; a row without
    entries is padding with loss 0), teacher_logits [n, k] float32, float16 or
    bfloat16 -- the top_ids and top_logprobs of token_logprobs at temperature 1
    fit both (the temperature here divides them, too)."""
    return _distill(_logits(logits, temperature), logits, teacher_ids,
                    teacher_logits, None, None)


def distill_forward_backward(logits, teacher_ids, teacher_logits, *,
                             temperature=1.0, row_weight=None, out=None):
    """(loss [n], d_logits [n, classes]): distill_loss and, from the same read
    of the logits, the gradient of sum(row_weight * loss) in the logits' type.
    row_weight float32 [n]; None is 1 / n, the gradient of the mean loss.  out:
    where to write the gradient; it may be `logits` itself, but no leaf that
    requires a gradient."""
    x = _logits(logits, temperature)
    given, out = out, _gradient(out, logits)
    loss = _distill(x, logits, teacher_ids, teacher_logits, row_weight, out)
    if given is not None:
        _written(out)
    return loss, out
