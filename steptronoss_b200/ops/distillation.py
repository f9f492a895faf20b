"""Distillation from a teacher's top logits, on logits and fused with the LM-head projection.

Per token, with the student's logits ``s [V]`` and ``K`` teacher entries ``(id_j, t_j)`` (logits or log-probabilities:
a constant per token drops out), at temperature ``tau``::

    q = softmax_j(t / tau)      p = softmax_v(s / tau)      loss = sum_j q_j (log q_j - log p[id_j])
    d loss / d s_v = (p_v - sum_{j: id_j = v} q_j) / tau

An entry of ``-inf`` is no entry (rows of different length are padded with it, whatever their id), nor is one whose id
lies outside the vocabulary; ids may repeat.  A token without entries has loss 0 and gradient 0, whatever its logits
hold, and a token of weight 0 has gradient 0.  The factor ``tau ** 2`` that some recipes put in front is left to the
caller's weights.

The CUDA path is ``csrc/distill.cu``: a thread-block cluster takes a row, so that one read of the logits from DRAM gives
the loss and the gradient.  Rows longer than the cluster holds, and vocabularies that are sharded over a
group, take the same sums in three kernels (statistics, loss, gradient) with the statistics all-reduced in between.
The reference has no distillation loss; the layout follows its vocab-parallel cross-entropy
(``steptronoss/core/tensor_parallel/cross_entropy.py:28-166``).
"""
from __future__ import annotations

import math

import torch
import torch.distributed as dist

from . import native
from .cross_entropy import _all_reduce
from .gemm import _tma_compatible, count_launch, gemm

MAX_ENTRIES = 1024
MAX_TOKENS, MAX_VOCAB = 0x0FFFFFFF, 1 << 30      # of a call; what the C entry points take, as 32-bit numbers
P, I, L, F = native.P, native.I, native.L, native.F
native.register_signature("stb_distill_row_limit", [I])
native.register_signature("stb_distill_row", [P, L, P, L, P, I, L, P, L, P, P, P, I, I, I, F, I, I, P, P])
native.register_signature("stb_distill_stats", [P, L, P, I, L, P, L, P, P, I, I, I, L, L, F, I, P])
native.register_signature("stb_distill_loss", [P, I, L, P, L, P, P, P, I, I, L, F, P])
native.register_signature("stb_distill_live", [P, L, P, I, L, P, L, P, P, I, I, I, L, P])
native.register_signature("stb_distill_total", [P, P, I, P, P])
native.register_signature("stb_distill_scale", [P, P, P, L, P])
native.register_signature("stb_distill_grad", [P, L, P, L, P, I, L, P, L, P, P, I, I, I, L, L, F, I, I, P, P])


# --------------------------------------------------------------------------------------------------- arguments
def _group_size(group) -> int:
    return dist.get_world_size(group) if group is not None else 1


def _checked(rows: int, vocab: int, index: int, teacher_ids, teacher_logits, temperature, what: str):
    """Teacher entries as ``[rows, K]`` with a contiguous last dimension (ids int32 / int64, logits fp32); ``index`` is
    the student's device."""
    if rows > MAX_TOKENS or vocab > MAX_VOCAB:
        raise ValueError(f"{what}: {rows} tokens of {vocab} logits, at most {MAX_TOKENS} of {MAX_VOCAB} are taken")
    shape = teacher_ids.shape
    if shape != teacher_logits.shape or len(shape) < 1:
        raise ValueError(f"{what}: teacher_ids {tuple(shape)} and teacher_logits {tuple(teacher_logits.shape)} differ")
    K = shape[-1]
    if K > MAX_ENTRIES:
        raise ValueError(f"{what}: {K} teacher entries per token, at most {MAX_ENTRIES} are taken")
    if math.prod(shape[:-1]) != rows:
        raise ValueError(f"{what}: teacher entries for {math.prod(shape[:-1])} tokens, logits for {rows}")
    if teacher_ids.dtype != torch.int64 and teacher_ids.dtype != torch.int32:
        raise TypeError(f"{what}: teacher_ids are int64 or int32, got {teacher_ids.dtype}")
    if not teacher_logits.is_floating_point():
        raise TypeError(f"{what}: teacher_logits are floating point, got {teacher_logits.dtype}")
    if teacher_logits.requires_grad:
        raise ValueError(f"{what}: no gradient flows to the teacher, detach teacher_logits")
    if teacher_ids.get_device() != index or teacher_logits.get_device() != index:
        raise ValueError(f"{what}: teacher entries on {teacher_ids.device} / {teacher_logits.device}, not on the student's "
                         "device")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"{what}: temperature must lie between 1e-6 and 1e6, got {temperature}")
    if len(shape) != 2:
        teacher_ids, teacher_logits = teacher_ids.reshape(rows, K), teacher_logits.reshape(rows, K)
    if teacher_logits.dtype != torch.float32:
        teacher_logits = teacher_logits.float()
    return (teacher_ids if teacher_ids.stride(1) == 1 else teacher_ids.contiguous(),
            teacher_logits if teacher_logits.stride(1) == 1 else teacher_logits.contiguous())


def _check_shard(V: int, vocab_start: int, group, what: str) -> None:
    if not 0 <= vocab_start <= V * (_group_size(group) - 1):
        raise ValueError(f"{what}: a shard of {V} from {vocab_start} on does not lie in a vocabulary of {_group_size(group)} "
                         "such shards")


def _rows_of(logits: torch.Tensor, what: str) -> torch.Tensor:
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: logits need a vocabulary dimension, got {tuple(logits.shape)}")
    if logits.is_cuda and logits.dtype != torch.bfloat16 and logits.dtype != torch.float32:
        raise TypeError(f"{what}: logits are bf16 or fp32 on the GPU, got {logits.dtype}")
    x = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    return x if x.stride(1) == 1 else x.contiguous()


def _token_weights(weights, rows: int, index: int, what: str) -> torch.Tensor:
    if weights.numel() != rows or weights.get_device() != index:
        raise ValueError(f"{what}: one weight per token on the student's device, got {tuple(weights.shape)} on {weights.device}")
    if weights.dtype == torch.float32 and weights.dim() == 1 and not weights.requires_grad and weights.is_contiguous():
        return weights
    return weights.detach().reshape(rows).float().contiguous()


# --------------------------------------------------------------------------------------------------- PyTorch statement
def _teacher_q(ids, t, temperature: float, vocab: int):
    """``(q, log q, has)``; entries that do not count have q = 0."""
    entry = (ids >= 0) & (ids < vocab) & (t != -math.inf)
    if t.shape[-1] == 0:
        return t, t, torch.zeros(t.shape[0], dtype=torch.bool, device=t.device)
    has = entry.any(-1)
    t = torch.where(entry, t, -math.inf)
    t = torch.where(has.unsqueeze(-1), (t - t.amax(-1, keepdim=True)) / temperature, 0.0)
    logq = torch.log_softmax(t, dim=-1)
    return torch.where(entry, logq.exp(), 0.0), logq, has


def _statement(logits, ids, t, temperature: float, vocab_start: int, group):
    """``(loss [T], gradient [T, V] for a unit weight)`` in fp32 (fp64 for fp64 logits) from (a vocab shard of) the logits.

    The maximum is subtracted before the division: logits of the type's lowest value are finite and stay so.  The few
    numbers of an entry's loss are taken in fp64, where differences of such logits are finite, too."""
    s = logits if logits.dtype == torch.float64 else logits.float()
    V = s.shape[-1]
    q, logq, has = _teacher_q(ids, t.to(s.dtype), temperature, V * _group_size(group))
    top = _all_reduce(s.amax(-1), dist.ReduceOp.MAX, group)
    e = ((s - top.unsqueeze(-1)) / temperature).exp()
    total = _all_reduce(e.sum(-1), dist.ReduceOp.SUM, group)
    local = ids - vocab_start
    here = (local >= 0) & (local < V) & (q != 0)
    safe = local.masked_fill(~here, 0).long()
    picked = _all_reduce(torch.where(here, s.gather(-1, safe), 0.0), dist.ReduceOp.SUM, group)
    logp = (picked.double() - top.double().unsqueeze(-1)) / temperature - total.double().log().unsqueeze(-1)
    loss = torch.where(q != 0, q.double() * (logq.double() - logp), 0.0).sum(-1).to(s.dtype)
    grad = (e / total.unsqueeze(-1)).scatter_add(-1, safe, -torch.where(here, q, 0.0)) / temperature
    return loss, torch.where(has.unsqueeze(-1), grad, 0.0)


def _weighted(grad, weights):
    w = weights.unsqueeze(-1)
    return torch.where(w == 0, 0.0, grad * w)


# --------------------------------------------------------------------------------------------------- kernels
_ROW_LIMIT: dict[int, int] = {}


def _fits_row(V: int, elem: int) -> bool:
    limit = _ROW_LIMIT.get(elem)
    if limit is None:
        limit = _ROW_LIMIT[elem] = native.load().stb_distill_row_limit(elem)
    return V <= limit


def _row_kernel(x, ids, t, temperature, weights=None, grad=None, stats=None, loss=None):
    """One pass over whole rows: the loss, and on request the gradient and the statistics."""
    T, V = x.shape
    if loss is None:
        loss = x.new_empty(T, dtype=torch.float32)
    size = x.element_size()
    gp, gld, gsize = (None, 0, size) if grad is None else (grad.data_ptr(), grad.stride(0), grad.element_size())
    rc = native.launch(
        native.load().stb_distill_row, x.get_device(), x.data_ptr(), x.stride(0), gp, gld, ids.data_ptr(),
        int(ids.dtype == torch.int64), ids.stride(0), t.data_ptr(), t.stride(0),
        None if weights is None else weights.data_ptr(), loss.data_ptr(), None if stats is None else stats.data_ptr(), T, V,
        ids.shape[1], 1.0 / temperature, size, gsize, native.status_ptr(x.get_device()))
    if rc:
        native.check(rc, f"distill_row T={T} V={V} K={ids.shape[1]}")
    count_launch()
    return loss


def _stats_kernels(x, ids, t, temperature, vocab_start=0, group=None, loss=None):
    """``(loss, statistics)`` of rows of any length, or of the shards of a group."""
    T, V = x.shape
    K, vocab, index = ids.shape[1], V * _group_size(group), x.get_device()
    lib = native.load()
    stats = x.new_empty((T, 4), dtype=torch.float32)
    picked = x.new_empty((T, K), dtype=torch.float32)
    native.check(native.launch(
        lib.stb_distill_stats, index, x.data_ptr(), x.stride(0), ids.data_ptr(), int(ids.dtype == torch.int64),
        ids.stride(0), t.data_ptr(), t.stride(0), stats.data_ptr(), picked.data_ptr(), T, V, K, vocab_start, vocab,
        1.0 / temperature, x.element_size()), f"distill_stats T={T} V={V} K={K}")
    count_launch()
    if _group_size(group) > 1:
        _join_shards(stats, picked, group)
    if loss is None:
        loss = x.new_empty(T, dtype=torch.float32)
    native.check(native.launch(
        lib.stb_distill_loss, index, ids.data_ptr(), int(ids.dtype == torch.int64), ids.stride(0), t.data_ptr(), t.stride(0),
        stats.data_ptr(), picked.data_ptr(), loss.data_ptr(), T, K, vocab, 1.0 / temperature), "distill_loss")
    count_launch()
    return loss, stats


def _shard_keys(stats):
    """``[2, T]``, whose maxima over the shards are the whole rows': ``c * max`` (infinite for large rows, which have a
    negative sum) and the maximum of large rows itself."""
    top, large = stats[:, 0], stats[:, 1] < 0
    return torch.stack([torch.where(large, torch.copysign(torch.full_like(top, math.inf), top), top),
                        torch.where(large, top, -math.inf)])


def _shard_sums(stats, keys):
    """A shard's sums relative to the maxima of the whole rows, and which of these are large."""
    (top, total), large = (stats[:, 0], stats[:, 1]), stats[:, 1] < 0
    rows = keys[0].isinf() & (keys[1] != -math.inf)
    # a shard that holds nothing but -inf has top = -inf and sum 0; beside a large one only equal maxima count
    usual = torch.where(top == -math.inf, total, total * torch.exp2(top - keys[0]))
    sums = torch.where(rows, torch.where(large & (top == keys[1]), -total, 0.0), torch.where(large, 0.0, usual))
    return torch.where(total.isnan(), total, sums), rows


def _join_shards(stats, picked, group) -> None:
    """Statistics of whole rows from those of the group's vocabulary shards, in place.  The first two columns are ``(top,
    sum of 2^(c s - top))``, or for large rows ``(max, -number of elements that equal it)``; the teacher's columns are
    equal on all ranks."""
    keys = _all_reduce(_shard_keys(stats), dist.ReduceOp.MAX, group)
    sums, rows = _shard_sums(stats, keys)
    sums = _all_reduce(sums, dist.ReduceOp.SUM, group)
    stats[:, 0] = torch.where(rows, keys[1], keys[0])
    stats[:, 1] = torch.where(rows, -sums, sums)
    _all_reduce(picked, dist.ReduceOp.SUM, group)


def _grad_kernel(x, ids, t, temperature, weights, stats, grad, vocab_start=0, vocab=None):
    T, V = x.shape
    index = x.get_device()
    rc = native.launch(
        native.load().stb_distill_grad, index, x.data_ptr(), x.stride(0), grad.data_ptr(), grad.stride(0),
        ids.data_ptr(), int(ids.dtype == torch.int64), ids.stride(0), t.data_ptr(), t.stride(0), weights.data_ptr(),
        stats.data_ptr(), T, V, ids.shape[1], vocab_start, V if vocab is None else vocab, 1.0 / temperature,
        x.element_size(), grad.element_size(), native.status_ptr(index))
    if rc:
        native.check(rc, f"distill_grad T={T} V={V} K={ids.shape[1]}")
    count_launch()


def _whole_rows(x, vocab_start: int, group) -> bool:
    """Whether the one-pass kernel takes these rows: the whole vocabulary, of a length that a cluster takes."""
    return vocab_start == 0 and (group is None or _group_size(group) == 1) and _fits_row(x.shape[1], x.element_size())


def _loss_and_grad(x, ids, t, temperature, weights, grad, vocab_start=0, group=None, loss=None):
    """Loss of the rows of ``x``, their weighted gradient into ``grad`` (which may be ``x``)."""
    if x.shape[0] == 0:
        return torch.empty(0, dtype=torch.float32, device=x.device)
    if _whole_rows(x, vocab_start, group):
        return _row_kernel(x, ids, t, temperature, weights, grad, loss=loss)
    loss, stats = _stats_kernels(x, ids, t, temperature, vocab_start, group, loss)
    _grad_kernel(x, ids, t, temperature, weights, stats, grad, vocab_start, x.shape[1] * _group_size(group))
    return loss


def _first_order(what: str) -> None:
    if torch.is_grad_enabled():              # create_graph=True
        raise RuntimeError(f"{what} has no second derivative")


# --------------------------------------------------------------------------------------------------- logits
class _TopkDistillationFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, t, temperature, vocab_start, group):
        x = _rows_of(logits, "topk_distillation")
        ctx.args = (temperature, vocab_start, group)
        if not x.is_cuda:
            loss, grad = _statement(x, ids, t, temperature, vocab_start, group)
            ctx.save_for_backward(grad)
        elif x.shape[0] == 0:
            loss = torch.empty(0, dtype=torch.float32, device=x.device)
            ctx.save_for_backward(x, ids, t, loss)
        else:
            if _whole_rows(x, vocab_start, group):
                stats = x.new_empty((x.shape[0], 4), dtype=torch.float32)
                loss = _row_kernel(x, ids, t, temperature, stats=stats)
            else:
                loss, stats = _stats_kernels(x, ids, t, temperature, vocab_start, group)
            ctx.save_for_backward(x, ids, t, stats)
        ctx.shape, ctx.dtype = logits.shape, logits.dtype
        return loss if logits.dim() == 2 else loss.view(logits.shape[:-1])

    @staticmethod
    def backward(ctx, gloss):
        _first_order("topk_distillation")
        temperature, vocab_start, group = ctx.args
        w = gloss if gloss.dim() == 1 else gloss.reshape(-1)
        if w.dtype != torch.float32 or not w.is_contiguous():
            w = w.float().contiguous()
        if len(ctx.saved_tensors) == 1:
            (unit,) = ctx.saved_tensors
            return _weighted(unit, w).to(ctx.dtype).view(ctx.shape), None, None, None, None, None
        x, ids, t, stats = ctx.saved_tensors
        grad = x.new_empty(x.shape)
        if x.shape[0]:
            _grad_kernel(x, ids, t, temperature, w, stats, grad, vocab_start, x.shape[1] * _group_size(group))
        return grad if len(ctx.shape) == 2 else grad.view(ctx.shape), None, None, None, None, None


def topk_distillation(logits, teacher_ids, teacher_logits, temperature: float = 1.0, vocab_start: int = 0, group=None):
    """Per-token loss ``[...]`` (fp32) of ``logits [..., V]`` against teacher entries ``[..., K]``.

    ``logits`` may be a vocabulary shard of equal size on every rank of ``group``, starting at ``vocab_start``;
    ``teacher_ids`` are always ids of the whole vocabulary.  Differentiable with respect to ``logits``."""
    temperature, vocab_start = float(temperature), int(vocab_start)
    rows = math.prod(logits.shape[:-1])
    V = logits.shape[-1] if logits.dim() else 0
    _check_shard(V, vocab_start, group, "topk_distillation")
    ids, t = _checked(rows, V, logits.get_device(), teacher_ids, teacher_logits, temperature, "topk_distillation")
    return _TopkDistillationFn.apply(logits, ids, t, temperature, vocab_start, group)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    def span(x):
        last = sum((n - 1) * s for n, s in zip(x.shape, x.stride()))
        return x.data_ptr(), x.data_ptr() + (last + 1) * x.element_size()

    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def topk_distillation_loss_and_grad(logits, teacher_ids, teacher_logits, weights, temperature: float = 1.0, out=None):
    """``(loss [T] fp32, gradient of sum_t weights[t] * loss[t])`` of ``logits [T, V]`` in one pass over them.

    For loops that feed the gradient straight into the next product instead of going through autograd; no graph is
    recorded.  ``out`` receives the gradient: ``[T, V]`` of the logits' type, or bf16 for fp32 logits, with any row
    stride; it may be ``logits`` itself (they are overwritten).  The loss is returned without its weight."""
    what = "topk_distillation_loss_and_grad"
    temperature = float(temperature)
    if logits.dim() != 2:
        raise ValueError(f"{what}: logits are [T, V], got {tuple(logits.shape)}")
    x, index = _rows_of(logits.detach() if logits.requires_grad else logits, what), logits.get_device()
    ids, t = _checked(x.shape[0], x.shape[1], index, teacher_ids, teacher_logits, temperature, what)
    w = _token_weights(weights, x.shape[0], index, what)
    if out is None:
        out = x.new_empty(x.shape)
        if index >= 0:
            return _loss_and_grad(x, ids, t, temperature, w, out), out
    else:
        if out.shape != x.shape or out.device != x.device:
            raise ValueError(f"{what}: out is {tuple(out.shape)} on {out.device}, logits {tuple(x.shape)} on {x.device}")
        if out.dtype != x.dtype and not (out.dtype == torch.bfloat16 and x.dtype == torch.float32):
            raise TypeError(f"{what}: out is {out.dtype} for logits of {x.dtype}")
        if out.stride(-1) != 1 and out.shape[-1] > 1:
            raise ValueError(f"{what}: the last dimension of out must be contiguous")
        if out.shape[0] > 1 and out.stride(0) < out.shape[1]:
            raise ValueError(f"{what}: the rows of out overlap")
        same = out.data_ptr() == logits.data_ptr() and out.dtype == logits.dtype and out.stride() == logits.stride()
        if x.numel() and not same and _overlap(out, logits):
            raise ValueError(f"{what}: out overlaps logits without being the same tensor")
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{what}: out is part of an autograd graph")
    if not x.is_cuda:
        loss, grad = _statement(x, ids, t, temperature, 0, None)
        with torch.no_grad():
            out.copy_(_weighted(grad, w).to(out.dtype))
        return loss, out
    loss = _loss_and_grad(x, ids, t, temperature, w, out)
    torch.autograd.graph.increment_version(out)
    return loss, out


# --------------------------------------------------------------------------------------------------- LM head
class _FusedLinearTopkDistillationFn(torch.autograd.Function):
    """Per block of tokens: fp32 logits from the tcgen05 GEMM, loss and bf16 gradient in one pass over them, dgrad and
    wgrad GEMMs.  The logits stay fp32 because the loss is a difference of log-probabilities: rounded to bf16, logits
    of size 20 would carry an error of 0.04 into a divergence that is itself of that size late in training.

    Their gradient is rounded to bf16 (2^-8 of itself at most), because the two products behind it take bf16 operands: dh
    and dW are sums of such terms and then rounded to bf16 themselves, and come out 2.4e-3 off instead of the 1.7e-3 of
    that last rounding alone.  A second product with the remainders would take it back for twice the time.  The
    cross-entropy next to this one makes the same choice.  The tensor cores truncate where they add, which leaves 2e-6 of
    the loss."""

    @staticmethod
    def forward(ctx, h, w, ids, t, weights, temperature, vocab_start, group, chunk):
        T, H = h.shape
        V = w.shape[0]
        need_dh, need_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        main_grad = getattr(w, "main_grad", None) if need_dw else None
        # elsewhere than on 16-byte boundaries the product would be the library's, rounded to bf16 once per block
        into_main_grad = main_grad is not None and _tma_compatible(main_grad)
        f32 = torch.float32
        loss, total = h.new_empty(T, dtype=f32), h.new_empty((), dtype=f32)
        dh = h.new_empty((T, H), dtype=f32) if need_dh else None
        dw = main_grad if into_main_grad else None
        if need_dw and dw is None:
            dw = h.new_empty((V, H), dtype=f32) if T else h.new_zeros((V, H), dtype=f32)
        rows = min(chunk, T)
        logits = h.new_empty((rows, V), dtype=f32)
        grad = h.new_empty((rows, V)) if need_dh or need_dw else None
        live = h.new_empty((rows, H)) if need_dw else None
        for t0 in range(0, T, chunk):
            n = min(T - t0, chunk)
            whole = n == T
            s, hc = (logits, h) if whole else (logits[:n], h[t0:t0 + n])
            gemm(hc, w, out=s)
            args = (s, ids, t, temperature) if whole else (s, ids[t0:t0 + n], t[t0:t0 + n], temperature)
            lc = loss if whole else loss[t0:t0 + n]
            if grad is None:
                if _whole_rows(s, vocab_start, group):
                    _row_kernel(*args, loss=lc)
                else:
                    _stats_kernels(*args, vocab_start, group, loss=lc)
                continue
            g = grad if n == rows else grad[:n]
            _loss_and_grad(*args, weights if whole else weights[t0:t0 + n], g, vocab_start, group, loss=lc)
            if need_dh:
                gemm(g, w, b_mn_major=True, out=dh if whole else dh[t0:t0 + n])
            if need_dw:
                hl = _live_states(hc, *args[1:3], weights if whole else weights[t0:t0 + n], V * _group_size(group), live[:n])
                gemm(g, hl, a_mn_major=True, b_mn_major=True, out=dw, accumulate=into_main_grad or t0 > 0)
        if main_grad is not None and not into_main_grad:
            main_grad.add_(dw)
        native.check(native.launch(native.load().stb_distill_total, h.get_device(), loss.data_ptr(), weights.data_ptr(), T,
                                   total.data_ptr()), "distill_total")
        count_launch()
        ctx.save_for_backward(dh)
        ctx.dw = None if main_grad is not None else dw
        ctx.w_ref = w
        ctx.used_main_grad = main_grad is not None
        ctx.mark_non_differentiable(loss)
        return total, loss

    @staticmethod
    def backward(ctx, gloss, _):
        _first_order("fused_linear_topk_distillation")
        (dh,) = ctx.saved_tensors
        gh = gw = None
        if gloss.dtype != torch.float32:
            gloss = gloss.float()
        if ctx.needs_input_grad[0]:
            gh = _scaled(dh, gloss)
        if ctx.needs_input_grad[1]:
            if ctx.used_main_grad:
                # dW already sits in main_grad with unit upstream gradient: the loss returned by this function has to
                # be the quantity that backward() is called on.
                ctx.w_ref.grad_added_to_main_grad = True
            else:
                gw = _scaled(ctx.dw, gloss)
        return gh, gw, None, None, None, None, None, None, None


def _live_states(h, ids, t, weights, vocab, out):
    """``h`` into ``out``, with zeros for tokens that do not count: of weight 0, or without an entry."""
    T, H = h.shape
    native.check(native.launch(
        native.load().stb_distill_live, h.get_device(), h.data_ptr(), h.stride(0), ids.data_ptr(),
        int(ids.dtype == torch.int64), ids.stride(0), t.data_ptr(), t.stride(0), weights.data_ptr(), out.data_ptr(), T, H,
        ids.shape[1], vocab), "distill_live")
    count_launch()
    return out


def _rows_for_gemm(x: torch.Tensor) -> bool:
    """Whether the tcgen05 GEMM takes these bf16 rows; it leaves others to a library product that rounds to bf16."""
    return _tma_compatible(x) and (x.shape[0] < 2 or x.stride(0) >= x.shape[1])


def _scaled(x: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """bf16 ``x * scale`` for a contiguous fp32 matrix and a scalar on the device."""
    y = x.new_empty(x.shape, dtype=torch.bfloat16)
    native.check(native.launch(native.load().stb_distill_scale, x.get_device(), x.data_ptr(), scale.data_ptr(), y.data_ptr(),
                               x.numel()), "distill_scale")
    count_launch()
    return y


def fused_linear_topk_distillation(h, w, teacher_ids, teacher_logits, weights, temperature: float = 1.0,
                                   vocab_start: int = 0, group=None, chunk_tokens: int = 2048):
    """``sum_t weights[t] * loss[t]`` of the logits ``h @ w.T`` with vocab-parallel ``w``, and the per-token loss.

    The counterpart of ``fused_linear_cross_entropy`` for a teacher: ``weights`` holds the loss mask already divided by
    its normaliser (and times ``temperature ** 2`` where the recipe wants that), so the returned scalar is what
    ``backward()`` is called on; with ``w.main_grad`` the weight gradient is added there during the forward pass, unless
    gradients are switched off (``torch.no_grad()``): then only the losses are computed.  The per-token loss carries no gradient."""
    what = "fused_linear_topk_distillation"
    temperature = float(temperature)
    if h.dim() != 2 or w.dim() != 2 or h.shape[1] != w.shape[1]:
        raise ValueError(f"{what}: h is [T, H] and w [V, H], got {tuple(h.shape)} and {tuple(w.shape)}")
    if not w.numel():
        raise ValueError(f"{what}: w needs a vocabulary and a hidden size, got {tuple(w.shape)}")
    main_grad = getattr(w, "main_grad", None)
    if main_grad is not None and (main_grad.shape != w.shape or main_grad.device != w.device
                                  or main_grad.dtype not in (torch.float32, torch.bfloat16)):
        raise ValueError(f"{what}: main_grad is fp32 or bf16 and lies beside w {tuple(w.shape)}, got {main_grad.dtype} "
                         f"{tuple(main_grad.shape)} on {main_grad.device}")
    if chunk_tokens < 1:
        raise ValueError(f"{what}: chunk_tokens must be positive, got {chunk_tokens}")
    _check_shard(w.shape[0], int(vocab_start), group, what)
    if w.device != h.device:
        raise ValueError(f"{what}: h on {h.device}, w on {w.device}")
    ids, t = _checked(h.shape[0], w.shape[0], h.get_device(), teacher_ids, teacher_logits, temperature, what)
    wt = _token_weights(weights, h.shape[0], h.get_device(), what)
    if torch.is_grad_enabled():
        if weights.requires_grad:
            raise ValueError(f"{what}: no gradient flows to the weights, detach them")
    else:
        h, w = h.detach(), w.detach()        # a Function is told that they need gradients in any mode: main_grad stays as it is
    if not h.is_cuda:
        linear = torch.nn.functional.linear
        entries = (ids >= 0) & (ids < w.shape[0] * _group_size(group)) & (t != -math.inf)
        live = ((wt != 0) & entries.any(-1)).unsqueeze(-1)
        logits = torch.where(live, linear(torch.where(live, h, 0.0), w), linear(h, w).detach())
        loss = topk_distillation(logits, ids, t, temperature, vocab_start, group)
        return torch.where(wt == 0, 0.0, loss * wt).sum(), loss.detach()
    if h.dtype != torch.bfloat16 or w.dtype != torch.bfloat16:
        raise TypeError(f"{what}: h and w are bf16, got {h.dtype} and {w.dtype}")
    if h.get_device() != torch.cuda.current_device():
        raise ValueError(f"{what}: h is on {h.device}, which is not the current device (the GEMMs go to the current one)")
    if w.shape[0] % 8 or w.shape[1] % 8 or not _rows_for_gemm(w):
        raise ValueError(f"{what}: w needs a vocabulary and a hidden size that are multiples of 8 and separate 16-byte aligned "
                         f"rows, got {tuple(w.shape)} with strides {w.stride()}")
    if not _rows_for_gemm(h):
        h = h.clone(memory_format=torch.contiguous_format)     # contiguous() would return a shifted or single row as it is
    return _FusedLinearTopkDistillationFn.apply(h, w, ids, t, wt, temperature, int(vocab_start), group, int(chunk_tokens))
