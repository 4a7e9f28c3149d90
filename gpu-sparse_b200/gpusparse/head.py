"""The vocabulary head: the projection that term weights come from, and its training losses.

A learned-sparse encoder ends in a projection of its hidden states onto the vocabulary,
s[t, v] = hidden[t] . weight[v] + bias[v].  The operators here run that projection on the
tensor cores and reduce the logits where they are made, so none of them ever holds logits
(backward passes write their gradient, in the inputs' type and for a piece of the vocabulary of
512 MiB at a time; kept for them are the packed rows, 16 bytes per teacher entry, and the sparse
head's weights and winners):

* ``sparse_head``: term weights log1p(relu(max over a text's tokens of s)), [B, V];
  ``encode_documents`` / ``encode_queries`` turn them into what the index builders and the
  scorer take, ``build_index_from_hidden`` into an index;
* ``vocab_cross_entropy``: softmax cross entropy over the vocabulary (masked tokens, or
  with documents as the rows of ``weight`` a contrastive loss);
* ``topk_distillation``: KL divergence from a teacher's top scores, in the (scores, ids)
  form ``score_topk`` and ``compacted_topk`` return.

Types: hidden and weight both bf16 or both fp16, bias in any floating type (used as fp32);
logits and sums are fp32, and so are the results.  All three differentiate in hidden,
weight and bias; gradients come in the inputs' types, and equal inputs give equal bits.
Tokens that take no part (ignored targets, masked tokens, rows without teacher entries)
are packed away on the GPU first: they cost nothing, and what they hold is never used.
No call synchronises except ``encode_documents`` and ``build_index_from_hidden``, whose
results' sizes depend on the data; the others can be captured in a CUDA graph.  (As with any
torch operator, a backward pass is captured only while no uncaptured graph of the same leaves is
alive: that graph's accumulation nodes belong to another stream.)  Forward-mode derivatives and
gradients of gradients raise.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
from typing import Iterable, Optional, Tuple

import torch
import torch.autograd.forward_ad as forward_ad

from . import _lib as L
from .index import GPUInvertedIndex, build_from_csr_tensors
from .scoring import compacted_topk

_DTYPES = {torch.bfloat16: L.W_BF16, torch.float16: L.W_F16}


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x as rows of unit element stride that do not overlap, copied only if it has others."""
    if x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < x.shape[1]):
        x = x.contiguous()
    return x


def _as(x: torch.Tensor, dtype) -> torch.Tensor:
    """x contiguous and of that type (x itself where it is)."""
    if x.dtype != dtype:
        x = x.to(dtype)
    return x if x.is_contiguous() else x.contiguous()


def _is_integer(x: torch.Tensor) -> bool:
    return not (x.dtype.is_floating_point or x.dtype.is_complex or x.dtype == torch.bool)


def _differentiated(hidden, weight, bias) -> bool:
    """Whether the call belongs in an autograd function: for a gradient, or for a forward-mode
    tangent, which the function has no rule for and raises."""
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad or
                                    (bias is not None and bias.requires_grad)):
        return True
    return forward_ad._current_level >= 0 and any(
        x is not None and forward_ad.unpack_dual(x).tangent is not None for x in (hidden, weight, bias))


def _check(what: str, hidden, weight, bias):
    L.require_cuda(hidden, "hidden")
    L.require_cuda(weight, "weight")
    if hidden.dtype not in _DTYPES or weight.dtype != hidden.dtype:
        raise ValueError(f"{what}: hidden and weight must both be bfloat16 or both float16, got "
                         f"{hidden.dtype} and {weight.dtype}")
    if weight.dim() != 2 or hidden.dim() < 2 or hidden.shape[-1] != weight.shape[1]:
        raise ValueError(f"{what}: hidden must be [..., D] and weight [V, D], got "
                         f"{tuple(hidden.shape)} and {tuple(weight.shape)}")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"{what}: weight must not be empty")
    if weight.device != hidden.device:
        raise ValueError(f"{what}: weight must live on {hidden.device}")
    if bias is not None:
        if bias.shape != (weight.shape[0],) or not bias.dtype.is_floating_point:
            raise ValueError(f"{what}: bias must be a floating tensor of {weight.shape[0]} entries")
        if bias.device != hidden.device:
            raise ValueError(f"{what}: bias must live on {hidden.device}")


def _view(hidden, weight, bias) -> L.VocabView:
    """View of row tensors (see _rows); hidden may be (T, D) of a backward call without data."""
    V, D = weight.shape
    if isinstance(hidden, torch.Tensor):
        T = hidden.shape[0]
        ldh, ptr = hidden.stride(0) if T > 1 else D, hidden.data_ptr()
    else:
        T, ldh, ptr = hidden[0], D, None
    return L.VocabView(T, V, D, ldh, weight.stride(0) if V > 1 else D, ptr, weight.data_ptr(),
                       bias.data_ptr() if bias is not None else None, _DTYPES[weight.dtype], 0)


@functools.lru_cache(maxsize=1024)
def _sizes(T, V, D, ld_weight, aligned, K, kind, backward, device_index):
    """(state, workspace) bytes of a call: a function of its sizes alone (and of the device's
    number of SMs)."""
    lib = L.lib()
    v = L.VocabView(T, V, D, D, ld_weight, None, None if aligned else 2, None, L.W_BF16, 0)
    sb = lib.gsp_vocab_state_bytes(ctypes.byref(v), K, kind)
    wb = lib.gsp_vocab_ws_bytes(ctypes.byref(v), K, kind, int(backward))
    if sb < 0 or wb < 0:
        L.check(int(-min(sb, wb)), "vocabulary head")
    return sb, wb


def _bytes(v: L.VocabView, K: int, kind: int, backward: bool, dev):
    return _sizes(v.T, v.V, v.D, v.ld_weight, v.weight % 16 == 0, K, kind, backward, dev.index)


def _buffer(nbytes: int, dev) -> torch.Tensor:
    return torch.empty(nbytes, dtype=torch.uint8, device=dev)


def _state_and_ws(sb: int, wb: int, train: bool, dev):
    """(buffers, address of the state, address of the workspace): the first buffer is the state
    to keep for the backward pass, or both in one when there is none to keep it for.  The caller
    holds the buffers until the call has been issued."""
    if train:
        state, ws = _buffer(sb, dev), _buffer(wb, dev)
        return (state, ws), state.data_ptr(), ws.data_ptr()
    sb = (sb + 255) // 256 * 256
    both = _buffer(sb + wb, dev)
    return (both,), both.data_ptr(), both.data_ptr() + sb


_HERE = contextlib.nullcontext()


def _on(dev):
    """The device's context, or nothing to do where it is current already."""
    return _HERE if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _stream(dev) -> int:
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _read_in_place(weight: torch.Tensor) -> bool:
    """Whether tensor maps describe these rows; the state of a forward call holds a copy of
    others."""
    ld = weight.stride(0) if weight.shape[0] > 1 else weight.shape[1]
    return ld % 8 == 0 and weight.data_ptr() % 16 == 0


# Hooks on saved tensors may have given them another layout; the backward calls read them as the
# forward calls left them: contiguous, the state on a 256-byte boundary.
def _saved(x: torch.Tensor) -> torch.Tensor:
    return x if x.is_contiguous() else x.contiguous()


def _saved_state(state: torch.Tensor) -> torch.Tensor:
    state = _saved(state)
    return state if state.data_ptr() % 256 == 0 else state.clone()


def _saved_weight(weight: torch.Tensor, in_place: bool) -> torch.Tensor:
    """The forward call's weight as its state expects it (which holds a copy of rows that are not
    read in place)."""
    weight = _rows(weight)
    if not in_place or _read_in_place(weight):
        return weight
    V, D = weight.shape
    rows = weight.new_empty((V, (D + 7) // 8 * 8))[:, :D]
    return rows.copy_(weight)


# ---------------------------------------------------------------------------- losses
def _loss_forward(hidden, weight, bias, args, train):
    kind, targets, ignore_index, scores, ids, tau, reduction = args
    dev = hidden.device
    with _on(dev):
        v = _view(hidden, weight, bias)
        K = ids.shape[1] if kind == L.VOCAB_DISTILL else 0
        sb, wb = _bytes(v, K, kind, False, dev)
        held, sp, wp = _state_and_ws(sb, wb, train, dev)
        loss = torch.empty((v.T,) if reduction == 0 else (), dtype=torch.float32, device=dev)
        if kind == L.VOCAB_CE:
            rc = L.lib().gsp_vocab_ce(ctypes.byref(v), targets.data_ptr(), ignore_index, reduction,
                                      loss.data_ptr(), sp, sb, wp, wb, _stream(dev))
        else:
            rc = L.lib().gsp_vocab_distill(ctypes.byref(v), scores.data_ptr(), ids.data_ptr(), K, tau,
                                           reduction, loss.data_ptr(), sp, sb, wp, wb, _stream(dev))
        if rc:
            L.check(rc, "vocab_cross_entropy" if kind == L.VOCAB_CE else "topk_distillation")
    return loss, held[0], K


def _grad_buffers(ctx, T, weight):
    """d_hidden, d_weight and d_bias as the backward pass needs them, else None."""
    V, D = weight.shape
    need_h, need_w, need_b = ctx.needs_input_grad[:3]
    dev = weight.device
    return (torch.empty((T, D), dtype=weight.dtype, device=dev) if need_h else None,
            torch.empty((V, D), dtype=weight.dtype, device=dev) if need_w else None,
            torch.empty(V, dtype=torch.float32, device=dev) if need_b else None)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _loss_backward(ctx, grad):
    weight, state = ctx.saved_tensors
    kind, K, tau, reduction, T, in_place = ctx.args
    dev = weight.device
    with _on(dev):
        weight, state = _saved_weight(weight, in_place), _saved_state(state)
        v = _view((T, None), weight, None)
        grad = _as(grad, torch.float32)
        _, wb = _bytes(v, K, kind, True, dev)
        ws = _buffer(wb, dev)
        dh, dw, db = _grad_buffers(ctx, T, weight)
        rc = L.lib().gsp_vocab_loss_backward(
            ctypes.byref(v), kind, K, tau, reduction, grad.data_ptr(), _ptr(dh), _ptr(dw), _ptr(db),
            state.data_ptr(), state.numel(), ws.data_ptr(), wb, _stream(dev))
        if rc:
            L.check(rc, "vocab loss backward")
    return dh, dw, db, None


# The same for a caller that builds a graph of the gradients: differentiating them again raises.
_loss_backward_once = torch.autograd.function.once_differentiable(_loss_backward)


class _VocabLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, args):
        kind, tau, reduction = args[0], args[-2], args[-1]
        loss, state, K = _loss_forward(hidden, weight, bias, args, True)
        ctx.save_for_backward(weight, state)
        ctx.args = (kind, K, tau, reduction, hidden.shape[0], _read_in_place(weight))
        return loss

    @staticmethod
    def backward(ctx, grad):
        return (_loss_backward_once if torch.is_grad_enabled() else _loss_backward)(ctx, grad)


def _loss(kind, hidden, weight, bias, targets, ignore_index, scores, ids, tau, reduction):
    lead = hidden.shape[:-1]
    hidden = _rows(hidden if len(lead) == 1 else hidden.reshape(-1, hidden.shape[-1]))
    weight = _rows(weight)
    if bias is not None:
        bias = _as(bias, torch.float32)
    red = L.REDUCE[reduction]
    args = (kind, targets, ignore_index, scores, ids, tau, red)
    if _differentiated(hidden, weight, bias):
        loss = _VocabLoss.apply(hidden, weight, bias, args)
    else:
        loss = _loss_forward(hidden, weight, bias, args, False)[0]
    return loss.reshape(lead) if red == 0 and len(lead) > 1 else loss


def _check_reduction(what: str, reduction: str) -> None:
    if reduction not in L.REDUCE:
        raise ValueError(f"{what}: reduction must be 'mean', 'sum' or 'none', got {reduction!r}")


def vocab_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
                        bias: Optional[torch.Tensor] = None, ignore_index: int = -100,
                        reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of hidden @ weight.T + bias against ``targets``, in fp32.

    hidden [..., D], weight [V, D], targets integer [...].  Tokens whose target is
    ``ignore_index`` or lies outside [0, V) take no part: they add no loss, get zero
    gradients, and their hidden states are never used.  ``reduction`` "mean" divides by the
    tokens that take part (0 when there are none), "none" gives the losses in targets' shape.
    """
    _check("vocab_cross_entropy", hidden, weight, bias)
    _check_reduction("vocab_cross_entropy", reduction)
    if targets.shape != hidden.shape[:-1] or not _is_integer(targets):
        raise ValueError(f"vocab_cross_entropy: targets must be an integer tensor of shape "
                         f"{tuple(hidden.shape[:-1])}, got {targets.dtype} {tuple(targets.shape)}")
    if targets.device != hidden.device:
        raise ValueError(f"vocab_cross_entropy: targets must live on {hidden.device}")
    targets = _as(targets if targets.dim() == 1 else targets.reshape(-1), torch.int64)
    return _loss(L.VOCAB_CE, hidden, weight, bias, targets, int(ignore_index), None, None, 1.0,
                 reduction)


def topk_distillation(hidden: torch.Tensor, weight: torch.Tensor, teacher_scores: torch.Tensor,
                      teacher_ids: torch.Tensor, bias: Optional[torch.Tensor] = None,
                      temperature: float = 1.0, reduction: str = "mean") -> torch.Tensor:
    """Distillation from a teacher's top scores: with p = softmax(teacher_scores /
    temperature) over a token's K entries, temperature^2 KL(p || softmax(s / temperature)),
    s = hidden @ weight.T + bias, in fp32.

    hidden [..., D], weight [V, D], teacher_scores and teacher_ids [..., K] with K <= 1024,
    in any order (``score_topk`` and ``compacted_topk`` return this pair).  Entries with an
    id outside [0, V) or a score of -inf are left out, an id listed twice adds its
    probabilities, and a token without entries takes no part (as an ignored target in
    ``vocab_cross_entropy``).  No gradient flows to the teacher's scores.  The temperature's
    square has to be a normal fp32 number (1.1e-19 to 1.8e19).
    """
    _check("topk_distillation", hidden, weight, bias)
    _check_reduction("topk_distillation", reduction)
    if teacher_scores.shape != teacher_ids.shape or \
            teacher_scores.shape[:-1] != hidden.shape[:-1] or teacher_scores.dim() != hidden.dim():
        raise ValueError(f"topk_distillation: teacher scores and ids must be "
                         f"{tuple(hidden.shape[:-1])} + [K], got {tuple(teacher_scores.shape)} and "
                         f"{tuple(teacher_ids.shape)}")
    if not _is_integer(teacher_ids) or not teacher_scores.dtype.is_floating_point:
        raise ValueError("topk_distillation: teacher ids must be an integer tensor and teacher scores "
                         f"a floating one, got {teacher_ids.dtype} and {teacher_scores.dtype}")
    if teacher_scores.device != hidden.device or teacher_ids.device != hidden.device:
        raise ValueError(f"topk_distillation: teacher scores and ids must live on {hidden.device}")
    K = teacher_ids.shape[-1]
    if not 1 <= K <= L.DISTILL_MAX_K:
        raise ValueError(f"topk_distillation: {K} teacher entries, 1 to {L.DISTILL_MAX_K} are supported")
    if not 0.0 < temperature < float("inf"):
        raise ValueError("topk_distillation: temperature must be positive")
    scores = _as(teacher_scores.detach().reshape(-1, K), torch.float32)
    ids = _as(teacher_ids.reshape(-1, K), torch.int64)
    return _loss(L.VOCAB_DISTILL, hidden, weight, bias, None, 0, scores, ids, float(temperature),
                 reduction)


# ---------------------------------------------------------------------------- sparse head
def _head_forward(hidden, weight, bias, mask, Lt: int, train: bool):
    dev = hidden.device
    with _on(dev):
        v = _view(hidden, weight, bias)
        B = v.T // Lt
        sb, wb = _bytes(v, 0, L.VOCAB_HEAD, False, dev)
        held, sp, wp = _state_and_ws(sb, wb, train, dev)
        y = torch.empty((B, v.V), dtype=torch.float32, device=dev)
        win = torch.empty((B, v.V), dtype=torch.int32, device=dev) if train else None
        rc = L.lib().gsp_sparse_head(ctypes.byref(v), Lt, _ptr(mask), y.data_ptr(), _ptr(win), sp, sb, wp,
                                     wb, _stream(dev))
        if rc:
            L.check(rc, "sparse_head")
    return y, win, held[0]


def _head_backward(ctx, dy):
    weight, y, win, state = ctx.saved_tensors
    T, Lt, in_place = ctx.args
    dev = weight.device
    with _on(dev):
        weight, state = _saved_weight(weight, in_place), _saved_state(state)
        y, win = _saved(y), _saved(win)
        v = _view((T, None), weight, None)
        dy = _as(dy, torch.float32)
        _, wb = _bytes(v, 0, L.VOCAB_HEAD, True, dev)
        ws = _buffer(wb, dev)
        dh, dw, db = _grad_buffers(ctx, T, weight)
        rc = L.lib().gsp_sparse_head_backward(
            ctypes.byref(v), Lt, y.data_ptr(), win.data_ptr(), dy.data_ptr(), _ptr(dh), _ptr(dw), _ptr(db),
            state.data_ptr(), state.numel(), ws.data_ptr(), wb, _stream(dev))
        if rc:
            L.check(rc, "sparse_head backward")
    return dh, dw, db, None, None


_head_backward_once = torch.autograd.function.once_differentiable(_head_backward)


class _SparseHead(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, mask, Lt):
        y, win, state = _head_forward(hidden, weight, bias, mask, Lt, True)
        ctx.save_for_backward(weight, y, win, state)
        ctx.args = (hidden.shape[0], Lt, _read_in_place(weight))
        return y

    @staticmethod
    def backward(ctx, dy):
        return (_head_backward_once if torch.is_grad_enabled() else _head_backward)(ctx, dy)


def sparse_head(hidden: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Term weights fp32 [B, V] of B texts: log1p(relu(max over the text's tokens of
    hidden @ weight.T + bias)).

    hidden [B, L, D], weight [V, D], mask [B, L] (nonzero or True = the token takes part, in
    any pattern; None = all do).  A text without tokens has zero weights.  The gradient goes
    to the token that won the maximum, the first one on ties; a NaN wins, and both the weight
    and its gradients are NaN.
    """
    _check("sparse_head", hidden, weight, bias)
    if hidden.dim() != 3:
        raise ValueError(f"sparse_head: hidden must be [B, L, D], got {tuple(hidden.shape)}")
    B, Lt, D = hidden.shape
    if mask is not None:
        if mask.shape != (B, Lt):
            raise ValueError(f"sparse_head: mask must be {(B, Lt)}, got {tuple(mask.shape)}")
        if mask.device != hidden.device:
            raise ValueError(f"sparse_head: mask must live on {hidden.device}")
        mask = _as(mask if mask.dtype == torch.bool else mask != 0, torch.bool)
    if B > 65534:
        raise ValueError(f"sparse_head: {B} texts in one call, at most 65534 are supported")
    if Lt == 0:          # texts of one token that takes no part
        hidden, Lt = torch.nn.functional.pad(hidden, (0, 0, 0, 1)), 1
        mask = torch.zeros((B, 1), dtype=torch.bool, device=hidden.device)
    rows = _rows(hidden.reshape(B * Lt, D))
    weight = _rows(weight)
    if bias is not None:
        bias = _as(bias, torch.float32)
    if _differentiated(rows, weight, bias):
        return _SparseHead.apply(rows, weight, bias, mask, Lt)
    return _head_forward(rows, weight, bias, mask, Lt, False)[0]


# ---------------------------------------------------------------------------- index and queries
def encode_documents(hidden: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                     mask: Optional[torch.Tensor] = None, min_weight: float = 0.0):
    """Documents as CSR rows for the index builders: ``(indptr int64 [B + 1], indices int32,
    data fp32)`` on the GPU, the terms of ``sparse_head`` with a weight above ``min_weight``
    (>= 0) in ascending order.  Synchronises once for the number of terms.  Raises RuntimeError
    where weights are NaN (hidden states that are, or a wait that ran out)."""
    if not min_weight >= 0.0:
        raise ValueError("encode_documents: min_weight must be >= 0")
    with torch.no_grad():
        y = sparse_head(hidden, weight, bias, mask)
    B, V = y.shape
    dev = y.device
    lib = L.lib()
    with torch.cuda.device(dev):
        st = L.stream_of(dev)
        nnz = torch.empty(B, dtype=torch.int32, device=dev)
        indptr = torch.empty(B + 1, dtype=torch.int64, device=dev)
        ws = L.workspace(lib.gsp_scan_ws_bytes(B), dev)
        L.check(lib.gsp_dense_rows_count(L.ptr(y), B, V, min_weight, L.ptr(nnz), st), "encode_documents")
        L.check(lib.gsp_scan_i32(L.ptr(nnz), B, L.ptr(indptr), L.ptr(ws), ws.numel(), st),
                "encode_documents")
        # weights are >= 0: a sum is NaN where one of them is
        total, bad = torch.stack((indptr[B], y.sum().isnan().to(torch.int64))).tolist()
        if bad:
            rows = torch.isnan(y.sum(dim=1)).nonzero().flatten()
            raise RuntimeError(f"encode_documents: the weights of {rows.numel()} of {B} documents are NaN, "
                               f"the first is document {int(rows[0])}")
        indices = torch.empty(total, dtype=torch.int32, device=dev)
        data = torch.empty(total, dtype=torch.float32, device=dev)
        L.check(lib.gsp_dense_rows_fill(L.ptr(y), B, V, min_weight, L.ptr(indptr), L.ptr(indices),
                                        L.ptr(data), st), "encode_documents")
    return indptr, indices, data


def encode_queries(hidden: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                   mask: Optional[torch.Tensor] = None, max_terms: int = 128
                   ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Queries as the scorer takes them: term ids int32 and weights fp32, both [B, max_terms]
    (-1 / 0 padded), the ``max_terms`` strongest terms of ``sparse_head``, ties by ascending
    term id.  A query with a NaN weight (hidden states that are NaN, or a wait that ran out) has
    NaN in all of its weights, and one term at least."""
    if max_terms < 1:
        raise ValueError("encode_queries: max_terms must be positive")
    with torch.no_grad():
        y = sparse_head(hidden, weight, bias, mask)
        B, V = y.shape
        tau = torch.full((B,), torch.finfo(torch.float32).tiny, device=y.device)
        w, t = compacted_topk(y, tau, max_terms)
        pad = w == float("-inf")
        qi = torch.where(pad, torch.full_like(t, -1), t).to(torch.int32)
        qs = torch.where(pad, torch.zeros_like(w), w)
        if qi.shape[1] < max_terms:
            qi = torch.nn.functional.pad(qi, (0, max_terms - qi.shape[1]), value=-1)
            qs = torch.nn.functional.pad(qs, (0, max_terms - qs.shape[1]))
        bad = y.sum(dim=1).isnan()
        qs.masked_fill_(bad[:, None], float("nan"))
        qi[:, 0] = torch.where(bad, qi[:, 0].clamp(min=0), qi[:, 0])
    return qi, qs


def build_index_from_hidden(batches: Iterable, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                            min_weight: float = 0.0, weight_dtype: str = "fp32",
                            doc_base: int = 0) -> GPUInvertedIndex:
    """Index of the documents whose hidden states ``batches`` yields, in order: each batch
    hidden [B, L, D], or a pair (hidden, mask).  The vocabulary is weight's rows; the other
    arguments are ``encode_documents``' and ``build_from_csr_tensors``'."""
    ptrs, indices, data = [], [], []
    base = 0
    for batch in batches:
        hidden, mask = batch if isinstance(batch, (tuple, list)) else (batch, None)
        ip, ix, dt = encode_documents(hidden, weight, bias, mask, min_weight)
        ptrs.append(ip[:-1] + base)
        indices.append(ix)
        data.append(dt)
        base += ix.numel()
    dev = weight.device
    ptrs.append(torch.full((1,), base, dtype=torch.int64, device=dev))
    empty_i = torch.empty(0, dtype=torch.int32, device=dev)
    empty_f = torch.empty(0, dtype=torch.float32, device=dev)
    return build_from_csr_tensors(torch.cat(ptrs), torch.cat(indices or [empty_i]),
                                  torch.cat(data or [empty_f]), weight.shape[0], dev,
                                  weight_dtype=weight_dtype, doc_base=doc_base)
