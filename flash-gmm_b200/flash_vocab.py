"""Operators over a vocabulary table W (V, D): the two ends of a language model
that read it, and the labelled counterpart of the isotropic E-step.

    loss = linear_cross_entropy(X, W, targets, bias)       # X (..., D), targets (...)
    rows = embedding_lookup(W, ids, scale=D ** 0.5)        # (..., D)
    loss.backward()                                        # dX, dW, dbias

With W = mu / sigma^2 and bias = log pi - |mu|^2 / (2 sigma^2) the cross
entropy is -log p(component | x) of a mixture of one variance; its logZ is the
E-step's up to -|x|^2 / (2 sigma^2) - D/2 log(2 pi sigma^2), and the gradients
of sum(logZ) by W and bias are the E-step's mu_acc and Nk.  The lookup's
gradient is mu_acc with hard labels.

Nothing of size N x V is kept: the logits run through the chip in pieces of the
vocabulary, forward and again backward.  W and X are bfloat16, float16 or
float32 (both alike); sums, exponentials and logZ are float32.  Calls run on
torch's current stream, do not synchronise, keep no state and can be captured
into CUDA graphs.  There is no CPU fallback, and no forward-mode derivative
(arguments with tangents are refused).
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

import _fgmm_lib as L


def _need_gpu(**tensors):
    dev = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{name} must be on GPU")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the other arguments on {dev}")


def _values(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """t with its values in memory: the imaginary part of a conjugate holds their negatives
    and a bit that says so, which a kernel does not see."""
    return t.resolve_neg() if t is not None and t.is_neg() else t


def _has_tangent(*tensors) -> bool:
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _refuse_tangents(name: str, *tensors):
    """The kernels see primal values only: a tangent would be lost without a word."""
    if _has_tangent(*tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative: its arguments may not "
                                  "carry tangents")


def _tracked(*tensors) -> bool:
    """Whether autograd has to see the call."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _need_type(name: str, t: torch.Tensor):
    if t.dtype not in L.FGMM_TYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")


def _labels(name: str, t: torch.Tensor) -> torch.Tensor:
    if t.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"{name} must be int64 or int32, got {t.dtype}")
    if t.dim() != 1:
        t = t.reshape(-1)
    if t.dtype != torch.int64:
        t = t.long()
    return t if t.is_contiguous() else t.contiguous()


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, X, W, bias, targets, ignore_index, reduction):
        loss, logZ, reduced, count = L.xent_fwd(X, W, targets, bias, ignore_index, reduction)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(X, W, bias, targets, logZ, count if reduction == "mean" else None)
        ctx.ignore_index = ignore_index
        return (loss if reduced is None else reduced), logZ

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, dlogZ):
        X, W, bias, targets, logZ, count = ctx.saved_tensors
        if dloss is None and dlogZ is None:
            return (None,) * 6
        dloss = None if dloss is None else _values(dloss).contiguous()
        dlogZ = None if dlogZ is None else _values(dlogZ).contiguous()
        grads = L.xent_bwd(X, W, targets, bias, ctx.ignore_index, logZ, dloss, count, dlogZ,
                           ctx.needs_input_grad[:3])
        return (*grads, None, None, None)


def linear_cross_entropy(X: torch.Tensor, W: torch.Tensor, targets: torch.Tensor,
                         bias: Optional[torch.Tensor] = None, *, ignore_index: int = -100,
                         reduction: str = "mean", return_logZ: bool = False):
    """Cross entropy of softmax(X W^T + bias) against ``targets``.

    X: (..., D); W: (V, D) of the same type, any strides; targets: (...) int64
    or int32; bias: (V,), used in float32, -inf removes an entry.
    reduction: "none" gives float32 losses of the shape of targets; "sum" and
    "mean" a float32 scalar, the mean over the rows that are not ignored (NaN
    when there is none).
    return_logZ: also return logZ = log sum_v exp(S_v), of the shape of targets
    (0 on ignored rows); it is differentiable, e.g. for a penalty on logZ^2.

    A row whose target is ``ignore_index`` has loss 0 and gradient 0, whatever
    its X holds.  Another target outside [0, V) makes its loss and the
    gradients NaN: labels live on the device and are not read back to raise.
    Gradients have the types of X and W (float32 for bias).  float16 ones keep
    their bits down to 2^-26 of the largest weight of a row's loss, with an
    error of 2^-37 of it below; bfloat16 and float32 ones over their range.
    """
    if reduction not in L.FGMM_REDUCE:
        raise ValueError("reduction must be 'none', 'sum' or 'mean'")
    if W.dim() != 2 or X.dim() < 1 or X.shape[-1] != W.shape[1]:
        raise ValueError(f"X must be (..., D) and W (V, D), got {tuple(X.shape)} and "
                         f"{tuple(W.shape)}")
    if W.shape[0] < 1 or W.shape[1] < 1:
        raise ValueError(f"W must not be empty, got {tuple(W.shape)}")
    if targets.shape != X.shape[:-1]:
        raise ValueError(f"targets must be {tuple(X.shape[:-1])}, got {tuple(targets.shape)}")
    _need_type("X", X)
    if W.dtype != X.dtype:
        raise ValueError(f"X and W must have one type, got {X.dtype} and {W.dtype}")
    if bias is not None:
        if bias.shape != W.shape[:1]:
            raise ValueError(f"bias must be ({W.shape[0]},), got {tuple(bias.shape)}")
        if not bias.is_floating_point():
            raise ValueError(f"bias must be floating point, got {bias.dtype}")
    _refuse_tangents("linear_cross_entropy", X, W, bias)
    labels = _labels("targets", targets)
    _need_gpu(X=X, W=W, targets=targets, bias=bias)
    X, W, bias = _values(X), _values(W), _values(bias)
    if bias is not None:
        bias = bias.float().contiguous()
    shape = targets.shape
    if X.dim() != 2:
        X = X.reshape(-1, X.shape[-1])
    if _tracked(X, W, bias):
        loss, logZ = _LinearCrossEntropy.apply(X, W, bias, labels, int(ignore_index), reduction)
    else:
        loss, logZ, reduced, _ = L.xent_fwd(X, W, labels, bias, int(ignore_index), reduction)
        loss = loss if reduced is None else reduced
    if len(shape) != 1:
        logZ = logZ.reshape(shape)
        if reduction == "none":
            loss = loss.reshape(shape)
    return (loss, logZ) if return_logZ else loss


class _EmbeddingLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale, ignore_index):
        ctx.save_for_backward(ids)
        ctx.table_shape = tuple(table.shape)
        ctx.scale, ctx.ignore_index = scale, ignore_index
        return L.embed_fwd(table, ids, scale, ignore_index)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        ids, = ctx.saved_tensors
        dout = _values(dout)
        out = torch.empty(ctx.table_shape, device=dout.device, dtype=dout.dtype)
        return L.embed_bwd(dout, ids, ctx.scale, ctx.ignore_index, out, False), None, None, None


def embedding_lookup(table: torch.Tensor, ids: torch.Tensor, *, scale: float = 1.0,
                     ignore_index: int = -100) -> torch.Tensor:
    """out[..., :] = scale * table[ids] (scaled in float32, rounded once).

    table: (V, D), any strides; ids: int64 or int32 of any shape.  An id equal
    to ``ignore_index`` gives a row of zeros and no gradient; another id
    outside [0, V) a row of NaN and no gradient.  The gradient by the table is
    summed in float32 over sorted ids (`embedding_grad`).
    """
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError(f"table must be (V, D) and not empty, got {tuple(table.shape)}")
    _need_type("table", table)
    _refuse_tangents("embedding_lookup", table)
    flat = _labels("ids", ids)
    _need_gpu(table=table, ids=ids)
    fn = _EmbeddingLookup.apply if _tracked(table) else L.embed_fwd
    out = fn(_values(table), flat, float(scale), int(ignore_index))
    return out if ids.dim() == 1 else out.reshape(*ids.shape, table.shape[1])


def lookup_takes(table: torch.Tensor) -> bool:
    """Whether `embedding_lookup` can stand for indexing the rows of ``table`` in every
    respect: its type and size, and no derivative (indexing has those of any order)."""
    return (table.dim() == 2 and table.dtype in L.FGMM_TYPES
            and 0 < table.shape[0] < L.FGMM_VOCAB_MAX_ROWS
            and 0 < table.shape[1] <= L.FGMM_VOCAB_MAX_D
            and not _tracked(table) and not _has_tangent(table))


def embedding_grad(dout: torch.Tensor, ids: torch.Tensor, V: int, *, scale: float = 1.0,
                   ignore_index: int = -100, out: Optional[torch.Tensor] = None,
                   accumulate: bool = False) -> torch.Tensor:
    """dtable[v] = scale * sum of dout over the positions whose id is v: the
    gradient of `embedding_lookup`, for programs that keep their own gradients.

    dout: (..., D); ids: (...).  ``out`` may supply the (V, D) result buffer
    (contiguous, of dout's type); with ``accumulate`` the sums are added to it,
    e.g. to the other gradient of a tied table, and its other rows are left as
    they are.  ``out`` may not share memory with dout or ids (refused).
    Bitwise the same on every run.  The result is not tracked by autograd.
    """
    if ids.shape != dout.shape[:-1] or dout.dim() < 1:
        raise ValueError(f"ids must be {tuple(dout.shape[:-1])}, got {tuple(ids.shape)}")
    _need_type("dout", dout)
    D = dout.shape[-1]
    if V < 1 or D < 1:
        raise ValueError(f"V and D must be positive, got {V} and {D}")
    if out is None and accumulate:
        raise ValueError("accumulate=True needs the out= buffer to add into")
    _refuse_tangents("embedding_grad", dout, out)
    flat = _labels("ids", ids)
    _need_gpu(dout=dout, ids=ids, out=out)
    if out is None:
        out = torch.empty(V, D, device=dout.device, dtype=dout.dtype)
    elif (out.shape != (V, D) or out.dtype != dout.dtype or not out.is_contiguous()
          or out.is_neg()):
        raise ValueError(f"out must be a contiguous ({V}, {D}) tensor of {dout.dtype}")
    got = L.embed_bwd(_values(dout.detach()).reshape(-1, D), flat, float(scale), int(ignore_index),
                      out.detach(), bool(accumulate))
    if not out.is_inference():   # the kernel wrote to it: autograd has to see that
        torch.autograd.graph.increment_version(out)
    return got
