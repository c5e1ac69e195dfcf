"""Vocab-parallel cross entropy and the masked mean loss: dhellam/operators/loss.py:15-164.

Same calling convention as the reference (dict in, dict out, ``bwd(context, dout)``).  The
reference materialises the softmax in the forward and turns it into the gradient in the
backward; with ``keep_softmax=False`` the forward keeps only two numbers per row (maximum and
exponential sum) and the backward recomputes the softmax from the logits, which removes one
[rows, vocab] write and one read from the pair and leaves nothing of that size alive in
between.  ``output_dict["softmax"]`` is then None.

The all-reduces over the tensor-parallel group (loss.py:22-24,52-56,61-66) are the caller's:
with a world size above one the outputs are this rank's share.  The ranks join their row
statistics as

    M = max_r row_max_r,   S = sum_r sum_exp_r * exp(row_max_r - M),
    P = sum over the rank that holds the target of (predicted_r + row_max_r - M),
    loss = log S - P,

(two all-reduces of [rows] floats instead of the reference's three) and each rank's share of
the gradient comes from ``cross_entropy_bwd`` with ``row_max`` / ``sum_exp`` in its context
replaced by M / S (``keep_softmax=False``; a kept softmax is normalised by the rank's own sum).
"""
from __future__ import annotations

import torch

from .. import _host, _lib
from ..common.parallel_state import get_tensor_model_parallel_rank, get_tensor_model_parallel_world_size
from .embedding import vocab_range_from_per_partition_vocab_size


def cross_entropy_fwd(inputs, label_smoothing=0.0, keep_softmax=True):
    logits, target = inputs["vocab_parallel_logits"], inputs["target"]
    cols = logits.shape[-1]
    start, _ = vocab_range_from_per_partition_vocab_size(cols, get_tensor_model_parallel_rank(),
                                                        get_tensor_model_parallel_world_size())
    stats, softmax, mask, masked_target = _host.cross_entropy_fwd(logits, target, start, label_smoothing, keep_softmax)
    rows = mask.shape[0]
    if stats.shape[1] != rows:                         # no rows at all
        stats = stats[:, :rows]
    loss, row_max, sum_exp, predicted = stats.unbind(0)
    return {
        "loss": loss.view(target.shape),
        "label_smoothing": label_smoothing,
        "vocab_size": cols,
        "softmax": softmax.view(logits.shape) if keep_softmax else None,
        "target_mask": mask.view(target.shape),
        "masked_target_1d": masked_target,
        "row_max": row_max, "sum_exp": sum_exp, "predicted": predicted.view(target.shape),
    }


def cross_entropy_bwd(context, dout, grad_out=None):
    """Returns d loss / d logits scaled by ``dout`` per row.  With the softmax kept it is written
    over the softmax, as in the reference (loss.py:105-126); otherwise into ``grad_out`` (default:
    a new tensor; pass the logits themselves to overwrite them)."""
    inputs, out = context[0], context[1]
    logits, target = inputs["vocab_parallel_logits"], inputs["target"]
    cols = out["vocab_size"]
    start, _ = vocab_range_from_per_partition_vocab_size(cols, get_tensor_model_parallel_rank(),
                                                        get_tensor_model_parallel_world_size())
    if out["softmax"] is None:
        return _host.cross_entropy_bwd(logits, out["row_max"], out["sum_exp"], target, dout, start, out["label_smoothing"], grad_out)
    d = dout.to(torch.float32).contiguous()
    tgt = target.contiguous()
    rows = tgt.numel()
    assert d.numel() == rows
    sm = out["softmax"]
    s2 = sm.view(-1, cols)
    _lib.check(_lib.load().dh_cross_entropy_bwd(s2.data_ptr(), s2.stride(0), 0, None, None, tgt.data_ptr(), d.data_ptr(),
                                                rows, cols, start, float(out["label_smoothing"]), _lib.dt(sm),
                                                s2.data_ptr(), s2.stride(0), _host.stream_ptr(None)))
    return sm


def _vocabulary(cols):
    """(first id of this rank's slice, ids of all ranks)"""
    world = get_tensor_model_parallel_world_size()
    start, _ = vocab_range_from_per_partition_vocab_size(cols, get_tensor_model_parallel_rank(), world)
    return start, cols * world


def distill_fwd(inputs, temperature=1.0, alpha=1.0):
    """Distillation from a teacher's top logits, mixed with the labels' cross entropy.  inputs:

    * ``vocab_parallel_logits`` [..., cols]: the student's, x
    * ``teacher_ids`` int32 or int64 [..., K], ``teacher_logits`` [..., K] (any of the float types): the teacher's largest logits t and
      the ids of the WHOLE vocabulary that they belong to, K <= 1024.  An id outside it (-1) is no entry; an entry listed twice counts twice
    * ``teacher_lse`` fp32 [...] or None: log-sum-exp of the teacher's t / temperature over its whole vocabulary.  With it the teacher's
      probabilities are what it gave them and what lies behind its list is left out; without it the list is normalised to one
    * ``target`` int64 [...], needed for alpha < 1

    p = exp(t / temperature - lse), q = softmax(x / temperature):

        loss = alpha temperature^2 sum_k p_k (log p_k - log q_k) + (1 - alpha) cross entropy(x, target)

    A row without entries has no first term.  Returns {"loss" [...], "stats" (what the backward needs and ``distill_statistics`` names),
    "temperature", "alpha", "vocab_size"}."""
    logits, target = inputs["vocab_parallel_logits"], inputs.get("target")
    start, total = _vocabulary(logits.shape[-1])
    loss, stats = _host.distill_fwd(logits, inputs["teacher_ids"], inputs["teacher_logits"], inputs.get("teacher_lse"), target, start, total,
                                    temperature, alpha)
    return {"loss": loss, "stats": stats, "temperature": temperature, "alpha": alpha,
            "vocab_size": logits.shape[-1]}


def distill_statistics(out):
    """The rows of ``out["stats"]`` by name, views of [rows].  With a tensor-parallel world above one the outputs of ``distill_fwd`` are
    this rank's share and the caller joins them: with M = max_r row_max_r,

        S  = sum_r sum_exp_t_r exp((row_max_r - M) / temperature),   S1 = sum_r sum_exp_r exp(row_max_r - M)      (alpha < 1)
        D  = sum_r dot_r + (mass_local_r (row_max_r - M)) / temperature
        P  = sum over the rank that holds the target of (predicted_r + row_max_r - M)
        loss = alpha temperature^2 (entropy - D + mass log S) + (1 - alpha) (log S1 - P)

    and each rank's share of the gradient comes from ``distill_bwd`` after M, S and S1 are written over ``row_max``, ``sum_exp_t`` and
    ``sum_exp``.  A slice of a row that holds nothing but -inf has the lowest float as its ``row_max`` and sums of 0, so it adds nothing
    to any of these (the product before the quotient: (row_max_r - M) / temperature may be past the floats)."""
    names = ("loss", "row_max", "sum_exp_t", "sum_exp", "teacher_norm", "mass", "dot", "mass_local", "entropy", "predicted")
    return dict(zip(names, out["stats"].unbind(0)))


def distill_bwd(context, dout, grad_out=None):
    """d loss / d logits of ``distill_fwd`` scaled by ``dout`` per row, into ``grad_out`` (default: a new tensor; pass the logits themselves
    to overwrite them).  A row whose dout is 0 gets zeros, whatever it holds."""
    inputs, out = context[0], context[1]
    logits = inputs["vocab_parallel_logits"]
    start, total = _vocabulary(out["vocab_size"])
    return _host.distill_bwd(logits, inputs["teacher_ids"], inputs["teacher_logits"], inputs.get("target"), out["stats"], dout, start, total,
                             out["temperature"], out["alpha"], grad_out)


def mask_scale_loss_fwd(inputs):
    """loss = sum(losses * mask) / sum(mask) / num_microbatch * loss_scale (loss.py:131-153).  The NaN
    assertion of the reference needs a host sync and is left to the caller."""
    scale = float(inputs["loss_scale"]) / float(inputs["num_microbatch"])
    out, m = _host.masked_mean_fwd(inputs["output_tensor"], inputs["loss_mask"], scale)
    return {"loss": out[0], "mask_sum": out[1:2], "mask_f32": m}


def mask_scale_loss_bwd(context, dout=None):
    """d loss / d output_tensor; like the reference (loss.py:155-164) the incoming gradient is one."""
    inputs, out = context[0], context[1]
    losses, m = inputs["output_tensor"], out["mask_f32"]
    scale = float(inputs["loss_scale"]) / float(inputs["num_microbatch"])
    return _host.masked_mean_bwd(m, out["mask_sum"], scale).view(losses.shape).to(losses.dtype)
