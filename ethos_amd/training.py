"""Operators of a language model's training step around its blocks, as HIP kernels
(include/ethos_hip.h):

  linear_cross_entropy  softmax cross entropy of hidden rows against a head matrix, and its
                        gradients, without the logits in memory (their exponentials may be)
  embedding             rows of a table, scaled; the table's gradient by sorted tokens
  balance_loss          how often each expert was chosen, the load-balance loss, its gradient
  clip_grads            the global norm of many gradients, and the clipped gradients

The reference trains through torch operations (F.cross_entropy of model.py:396's logits, nn.Embedding,
nn.utils.clip_grad_norm_) and has no balance loss.  Inputs are HIP tensors on the current device, bf16
or float32; there is no CPU path.  All work goes to the current stream.  Results are the same on
every run.  The gradients are those of a single backward (no create_graph); forward-mode derivatives and
torch.jit.trace, which would not see the kernels' results, are refused."""
from __future__ import annotations

import math
import operator

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import hip

__all__ = ["balance_loss", "clip_grads", "embedding", "linear_cross_entropy"]


_FLOATS = set(hip.FLOATS)
_TENSORS = {torch.Tensor, torch.nn.Parameter}
_dtype, _shape = operator.attrgetter("dtype"), operator.attrgetter("shape")


def _contiguous(t):
    return t.contiguous() if isinstance(t, torch.Tensor) and not t.is_contiguous() else t


# (both without gradients: within autograd functions, or on tensors that need none)
def _dense(t: torch.Tensor) -> torch.Tensor:
    """t contiguous at a 16-byte address (a copy where it is not)."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[n, d] rows of t [..., d] that the kernels can read: evenly spaced, 16-byte aligned."""
    ld = hip.row_stride(t)
    if ld >= t.shape[-1] and ld * t.element_size() % 16 == 0 and t.data_ptr() % 16 == 0:
        n = t.numel() // t.shape[-1] if t.numel() else 0
        return t.as_strided((n, t.shape[-1]), (ld, 1))
    return _dense(t).view(-1, t.shape[-1])


def _is_followed() -> bool:
    return torch._C._is_tracing() or forward_ad._current_level >= 0


def _refuse_followed(what: str, *ts) -> None:
    """Raise where something follows the operations on the tensors that the kernels, which take addresses, hide
    from it: forward-mode derivatives would be lost, a trace would record results that nothing writes."""
    if torch.jit.is_tracing():
        raise RuntimeError(f"{what} cannot be traced by torch.jit.trace")
    if any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise RuntimeError(f"{what} has no forward-mode derivative")


def _device_check(name: str, t: torch.Tensor) -> None:
    if isinstance(t, torch.Tensor) and t.is_cuda and t.get_device() == hip._current_device():
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be on a HIP device (got {t.device}); the ETHOS kernels have no CPU path")
    raise RuntimeError(f"{name} is on {t.device}, not on the current device")


# -------------------------------------------------------------------------- cross entropy
class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, weight, labels, ignore_index, reduction, keep_bytes):
        rows, w = _rows(h), _dense(weight)
        # the weight itself is saved, so that a change in place before the backward is noticed
        loss, state, exps = hip.linear_ce(rows, w, labels, ignore_index, reduction, keep_bytes)
        ctx.save_for_backward(weight, state, exps)
        ctx.copy = w if w.data_ptr() != weight.data_ptr() else None
        ctx.shape, ctx.reduction = h.shape, reduction
        ctx.fresh, ctx.capture = True, hip.capture_id()
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        weight, state, exps = ctx.saved_tensors
        # the first backward uses the exponentials up: a second one of a retained graph has none, nor has one that
        # is captured apart from its forward, to be replayed more often than that
        if not ctx.fresh or (exps is not None and hip.capture_id() not in (0, ctx.capture)):
            exps = None
        else:
            ctx.fresh = False
        w = weight if ctx.copy is None else ctx.copy
        n = math.prod(ctx.shape[:-1])
        want_h, want_w = ctx.needs_input_grad[:2]
        dh, dw = hip.linear_ce_grad(state, exps, w, dloss.float().contiguous(), n, ctx.reduction, want_h, want_w)
        return dh.view(ctx.shape) if want_h else None, dw, None, None, None, None


class _NoRows(torch.autograd.Function):
    """The loss of no rows (`value`), with zero gradients."""

    @staticmethod
    def forward(ctx, h, weight, value):
        ctx.like = h.shape, weight.shape, weight.dtype, weight.device
        return value

    @staticmethod
    @once_differentiable
    def backward(ctx, _):
        rows, table, dtype, device = ctx.like
        return torch.zeros(rows, dtype=dtype, device=device), torch.zeros(table, dtype=dtype, device=device), None


def linear_cross_entropy(h: torch.Tensor, weight: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100,
                         reduction: str = "mean", keep_bytes: int = 1 << 30) -> torch.Tensor:
    """Softmax cross entropy of h @ weight.T against labels, without forming the logits.

    h [..., d] and weight [vocab, d] of one dtype (bf16 or float32), d a multiple of 8 up to 32768;
    labels int64 [...].  Positions whose label is `ignore_index` have no part in the loss or its
    gradients; another label outside the vocabulary makes the loss NaN.  `reduction`: "mean" over the
    labelled positions (NaN without one), "sum", or "none" (float32 [...], zero where ignored).  The
    loss is float32.  Gradients go to h and weight, in their dtype.  For them the backward forms the logits
    again, a piece of the vocabulary at a time; in bf16 the forward leaves the exponentials behind instead, in
    16 bits, where these take at most `keep_bytes`.  They take what the backward would take anyway, but from the
    forward on, once for every loss that waits for its backward."""
    if _is_followed():
        _refuse_followed("linear_cross_entropy", h, weight)
    for name, t in (("h", h), ("weight", weight), ("labels", labels)):
        _device_check(name, t)
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', got {reduction!r}")
    if h.dtype not in hip.FLOATS or weight.dtype != h.dtype:
        raise TypeError(f"h and weight must both be bfloat16 or both float32, got {h.dtype} and {weight.dtype}")
    if labels.dtype != torch.int64:
        raise TypeError(f"labels must be int64, got {labels.dtype}")
    if h.dim() < 1 or weight.dim() != 2 or h.shape[-1] != weight.shape[1] or labels.shape != h.shape[:-1]:
        raise RuntimeError(f"linear_cross_entropy: inconsistent shapes {tuple(h.shape)}, {tuple(weight.shape)}, {tuple(labels.shape)}")
    d = h.shape[-1]
    if weight.shape[0] == 0 or d == 0 or d % 8 or d > 32768:
        raise RuntimeError(f"linear_cross_entropy: needs a vocabulary and d a multiple of 8 up to 32768, got weight {tuple(weight.shape)}")
    if labels.numel() == 0:
        shape = labels.shape if reduction == "none" else ()
        value = torch.full(shape, math.nan if reduction == "mean" else 0.0, dtype=torch.float32, device=h.device)
        return _NoRows.apply(h, weight, value)
    flat = labels.contiguous().view(-1)
    if torch.is_grad_enabled() and (h.requires_grad or weight.requires_grad):
        loss = _LinearCrossEntropy.apply(h, weight, flat, int(ignore_index), reduction, int(keep_bytes))
    else:
        loss = hip.linear_ce(_rows(h), _dense(weight), flat, int(ignore_index), reduction)[0]
    return loss.view(labels.shape) if reduction == "none" else loss


# -------------------------------------------------------------------------- embedding
class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, ids, scale, padding):
        out, keys = hip.embedding(ids, weight, scale, padding, True)
        ctx.keys, ctx.vocab, ctx.scale = keys, weight.shape[0], scale  # keys: this node's own tensor
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return hip.embedding_grad(ctx.keys, _dense(dy), ctx.vocab, ctx.scale), None, None, None


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: int | None = None) -> torch.Tensor:
    """scale * weight[ids], [*ids.shape, d], for a table weight [vocab, d] (bf16 or float32) and ids of
    any shape (int32 or int64).  The table's gradient is dense, leaves out positions of `padding_idx`
    (negative ones count from the end) and adds a token's positions in a fixed order, in float32.  An
    id outside the table gives a row of NaN."""
    if _is_followed():
        _refuse_followed("embedding", weight)
    ids, w = _contiguous(ids), _contiguous(weight)  # (types and devices: hip.embedding)
    if isinstance(w, torch.Tensor) and (w.dim() != 2 or w.numel() == 0):
        raise RuntimeError(f"embedding: weight must be [vocab, d], got {tuple(w.shape)}")
    padding = -1
    if padding_idx is not None:
        if not -weight.shape[0] <= padding_idx < weight.shape[0]:
            raise ValueError(f"padding_idx {padding_idx} is outside the table of {weight.shape[0]} rows")
        padding = padding_idx % weight.shape[0]
    if torch.is_grad_enabled() and isinstance(w, torch.Tensor) and w.requires_grad:
        return _Embedding.apply(w, ids, float(scale), padding)  # (a copied weight's gradient goes through the copy)
    return hip.embedding(ids, w, float(scale))[0]


# -------------------------------------------------------------------------- balance
class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gates, ids, n_experts):
        loss, counts = hip.balance(gates, ids, n_experts)
        ctx.save_for_backward(ids, counts)
        ctx.dtype = gates.dtype
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return loss, counts

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        if dloss is None:
            return None, None, None
        ids, counts = ctx.saved_tensors
        return hip.balance_grad(ids, counts, dloss, ctx.dtype), None, None


def balance_loss(gates: torch.Tensor, ids: torch.Tensor, n_experts: int):
    """(loss, counts): the load-balance loss of a routing and how often each expert was chosen.

    gates [..., heads, k] (bf16 or float32) and ids of the same shape (int32 or int64), as
    ProductKeyRouter returns them.  With n tokens (the product of the leading dimensions),
    loss = n_experts * sum_e f_e s_e (float32), f_e = counts[e] / (n heads k) held fixed and s_e the
    sum of expert e's gates over (n heads); it is 1 when both are even over the experts.  counts is int32
    [n_experts].  Ids outside [0, n_experts) count nowhere.  Without tokens both are zero."""
    if _is_followed():
        _refuse_followed("balance_loss", gates)
    gates, ids = _contiguous(gates), _contiguous(ids)  # (types, shapes and devices: hip.balance)
    if n_experts <= 0:
        raise ValueError(f"n_experts must be positive, got {n_experts}")
    if torch.is_grad_enabled() and isinstance(gates, torch.Tensor) and gates.requires_grad:
        return _Balance.apply(gates, ids, int(n_experts))
    return hip.balance(gates, ids, int(n_experts))


# -------------------------------------------------------------------------- clipping
@torch.no_grad()
def clip_grads(grads, max_norm: float, norm_type: float = 2.0, out=None) -> torch.Tensor:
    """The global norm of `grads` (tensors, bf16 or float32, all taken as one vector), a float32 scalar
    on the device, and the gradients times min(1, max_norm / (norm + 1e-6)) in `out` (tensors of the same
    shapes and dtypes, for example parts of a reduction's buffer), or in place without it.
    norm_type: 2 (squares summed in float64) or inf.  A NaN gradient makes norm and outputs NaN.  Tensors
    may not overlap, but an output may be its own input."""
    grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
    out = grads if out is None else [out] if isinstance(out, torch.Tensor) else list(out)
    if norm_type not in (2, math.inf):
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    if not max_norm >= 0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    if len(out) != len(grads):
        raise ValueError(f"{len(grads)} gradients but {len(out)} outputs")
    # (a training step has hundreds of tensors: each check is one pass of a C function over them)
    ts = grads if out is grads else grads + out
    if _is_followed():
        _refuse_followed("clip_grads", *ts)
    if not set(map(type, ts)) <= _TENSORS and not all([isinstance(t, torch.Tensor) for t in ts]):
        raise TypeError("clip_grads takes tensors")
    if not ts:
        return torch.zeros((), dtype=torch.float32, device="cuda")
    devices = set(map(torch.Tensor.get_device, ts))
    if -1 in devices or devices != {hip._current_device()}:
        raise RuntimeError(f"clip_grads: tensors must be on the current HIP device, got some on {sorted({str(t.device) for t in ts})}")
    dtypes = list(map(_dtype, grads))
    kinds = set(dtypes)
    if not kinds <= _FLOATS:
        raise TypeError(f"clip_grads: tensors must be bfloat16 or float32, got {kinds - _FLOATS}")
    if out is not grads and (list(map(_dtype, out)) != dtypes or list(map(_shape, out)) != list(map(_shape, grads))):
        raise RuntimeError("clip_grads: outputs must have the gradients' shapes and dtypes")
    src = grads if all(map(torch.Tensor.is_contiguous, grads)) else [g.contiguous() for g in grads]
    dst = out if all(map(torch.Tensor.is_contiguous, out)) else [o if o.is_contiguous() else torch.empty_like(s) for s, o in zip(src, out)]
    sizes, to = list(map(torch.Tensor.numel, src)), list(map(torch.Tensor.data_ptr, dst))
    if len(set(to)) != len(to) and len({p for p, n in zip(to, sizes) if n}) != sum(n > 0 for n in sizes):
        raise ValueError("clip_grads: an output is given twice")
    codes = [int(dt == torch.bfloat16) for dt in dtypes] if len(kinds) > 1 else [int(torch.bfloat16 in kinds)] * len(dtypes)
    total = hip.clip_grads(to if dst is src else list(map(torch.Tensor.data_ptr, src)), to, sizes, codes, grads[0].device, float(max_norm),
                           norm_type == math.inf)
    for o, t in zip(out, dst) if dst is not out else ():
        if o is not t:
            o.copy_(t)
    try:
        torch.autograd.graph.increment_version(out)  # written by address
    except RuntimeError:  # some are inference tensors, which have none
        torch.autograd.graph.increment_version([o for o in out if not o.is_inference()])
    return total
