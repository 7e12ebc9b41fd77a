"""Operators of the `ocl` device that torch has no function for."""
from __future__ import annotations

import torch

from . import _C  # noqa: F401  (registers torch.ops.ocl)

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def linear_cross_entropy(input, weight, target, bias=None, *, ignore_index=-100, reduction="mean", label_smoothing=0.0):
    """``F.cross_entropy(F.linear(input, weight, bias), target, ...)`` in one operator.

    ``input`` is ``[..., features]``, ``weight`` ``[classes, features]`` (a
    linear layer's), both fp32, bf16 or fp16, ``target`` int64 ``[...]``; any
    number of classes, from a classifier's to a language model's vocabulary.
    The loss is fp32 whatever the operands' type: one number, or one per row
    with ``reduction="none"``.  A call without gradients keeps no logits.  A
    backward pass needs their softmax: of as many classes as fit into
    ``B200_CE_KEEP_MB`` (2048 MB by default, for each loss that is alive; 0 keeps
    nothing) the forward pass keeps it, as 16-bit exponentials (12 bits each,
    those below 2^-27 of the largest of 64 neighbours as 0) or, for fp32
    operands, as the fp32 logits, until the graph is freed; of the others, or
    where there is no memory for it, the backward pass forms the logits again,
    piece by piece.  The same call with as much kept gives the same bits.

    Gradients of ``input``, ``weight`` and ``bias`` have the operands' type.
    They are fp32 sums of products with the logits' gradient, which is rounded to
    the operands' type before (to 22 bits for fp32, and in fp32 and fp16 to steps
    of 2^-39 of a row's).  With ``reduction="none"`` a row's gradient of
    ``input`` depends on no other row's upstream gradient; those of ``weight``
    and ``bias`` are formed relative to the largest of them.

    Rows whose target is ``ignore_index`` or out of range have no loss and no
    gradient, whatever they hold.  fp32 operands are multiplied to 22
    bits, in either math mode (of an element below 2^-17 of its tensor's
    largest magnitude fewer take part: those above 2^-39 of that).  Forward mode
    and second derivatives are refused.
    """
    if reduction not in _REDUCTIONS:
        raise ValueError(f"{reduction} is not a valid value for reduction")
    return torch.ops.ocl.linear_cross_entropy(input, weight, target, bias, ignore_index, _REDUCTIONS[reduction],
                                              float(label_smoothing))


def relative_position_bias(table, q_len, k_len, *, bidirectional=True, max_distance=128, q_offset=0):
    """Learned relative position bias of attention scores: ``[1, heads, q_len, k_len]``.

    ``out[0, h, i, j] = table[bucket(j - i - q_offset), h]`` with ``table``
    ``[num_buckets, heads]`` (fp32, bf16 or fp16; 2 to 512 buckets).  With
    ``n = num_buckets`` (``num_buckets // 2`` for each sign if
    ``bidirectional``), distances below ``n // 2`` have a bucket each and those
    from there to ``max_distance`` (at most 2**20) share the others, evenly in
    the distance's logarithm; what is further takes the last one.  If not
    ``bidirectional``, keys behind the query take bucket 0.  ``q_offset`` is
    the position of the first query among the keys (``k_len - 1`` for one new
    token against a cache).  The gradient of ``table`` is summed in a fixed
    order.  In fp32 the result goes to ``scaled_dot_product_attention`` as
    ``attn_mask`` (whose products are fp32, as all of this device's layers; with
    a mask it takes its unfused path); in 16 bits, to scores of a program's own.
    """
    return torch.ops.ocl.relative_position_bias(table, q_len, k_len, bidirectional, max_distance, q_offset)


def rms_norm(input, weight=None, residual=None, *, eps=1e-6):
    """Root-mean-square norm over the last dimension, with the residual's addition before it.

    ``y = h / sqrt(mean(h**2) + eps) * weight`` with ``h = input``, or with
    ``h = input + residual`` rounded to their type; then the result is ``(y, h)``,
    ``h`` being the residual stream as it goes on.  fp32, bf16 or fp16, all of
    one type; ``weight`` ``[features]`` or None.  The mean of squares is summed in
    64 bits, the rest is fp32, rounded once; with an ``eps`` of next to nothing rows
    may be as small as fp32's normal numbers, but rows whose mean of squares is
    beyond fp32 (1.8e19 and more) are 0.  Gradients of ``input``, ``residual`` and
    ``weight`` (the last in a fixed order); forward mode and second derivatives are
    refused.
    """
    if residual is None:
        return torch.ops.ocl.rms_norm(input, weight, eps)
    return torch.ops.ocl.rms_norm_add(input, residual, weight, eps)


def rms_norm_8bit(input, weight=None, residual=None, *, eps=1e-6):
    """``rms_norm`` whose output is ``quantize_8bit``'s: ``(codes, scales)``, or ``(codes, scales, h)`` with a residual.

    The codes are those of ``y`` before it is rounded to the input's type.  They
    have no gradient: tensors that require one are refused outside
    ``torch.no_grad()``.
    """
    return tuple(torch.ops.ocl.rms_norm_8bit(input, weight, residual, eps))


def quantize_8bit(input, *, block_rows=1):
    """``(codes, scales)`` of fp32, bf16 or fp16 numbers in 8-bit floating point.

    ``codes`` are uint8 and hold e4m3 numbers (``codes.cpu().view(torch.float8_e4m3fn)``
    shows them), rows beginning on 16-byte boundaries.  One fp32 scale belongs to
    128 consecutive elements of a row (``block_rows=1``: activations, scales
    ``[..., ceil(features / 128)]``) or to 128 x 128 elements of a matrix
    (``block_rows=128``: weights, scales ``[ceil(rows / 128), ceil(features / 128)]``).
    The scale is the largest magnitude over 448, the largest code; a block whose
    magnitudes are 2**-100 or less becomes 0, one that holds an infinity or a NaN
    is NaN throughout.
    """
    if block_rows not in (1, 128):
        raise ValueError(f"block_rows is 1 or 128, got {block_rows!r}")
    return torch.ops.ocl.quantize_8bit(input, block_rows == 128)


def dequantize_8bit(codes, scales, *, dtype=torch.float32):
    """The numbers that ``quantize_8bit``'s or ``rms_norm_8bit``'s codes stand for."""
    return torch.ops.ocl.dequantize_8bit(codes, scales, dtype)


def linear_8bit(codes, scales, weight_codes, weight_scales, bias=None, *, dtype=torch.bfloat16):
    """``F.linear`` of operands in 8 bits: ``x w^T + bias`` as fp32, bf16 or fp16.

    ``codes`` ``[..., features]`` with a scale for every 128 of a row
    (``rms_norm_8bit``, ``quantize_8bit(x)``), ``weight_codes`` ``[outputs, features]``
    with one for every 128 x 128 (``quantize_8bit(w, block_rows=128)``, once);
    ``bias`` ``[outputs]`` of the output's type.  Any sizes, one row as well as
    many.  Codes whose rows do not begin on 16-byte boundaries are copied first.
    Products are exact and summed in fp32: by the tensor cores over 128 features,
    then block by block with the scales, whose product may lie outside fp32 where
    the result does not (of many rows, those with such products take much longer).
    No gradients (they are refused).
    """
    return torch.ops.ocl.linear_8bit(codes, scales, weight_codes, weight_scales, bias, dtype)


def token_log_probs(logits, tokens, *, top=0):
    """Log probabilities of given tokens and the entropy of their distributions, ``(log_probs, entropy)``, in fp32.

    ``logits`` ``[..., vocabulary]`` in fp32, bf16 or fp16, ``tokens`` int64
    ``[...]``: ``log_probs = log_softmax(logits)[tokens]``, ``entropy = -sum(p log p)``
    in nats.  With ``top`` (at most 32 and the vocabulary) also the best
    alternatives, ``(log_probs, entropy, top_log_probs, top_tokens)`` with
    ``[..., top]``, by falling logit and of equal ones the lower token first.

    ``log_probs`` and ``entropy`` have gradients (the alternatives have none);
    forward mode and second derivatives are refused.  Logits of -inf have no
    probability and no gradient, but for a given token's own: its log probability is
    -inf, and it gets that one's gradient.  Tokens outside the vocabulary (-100 for a
    prompt's, say) have the log probability 0 and no gradient through it, whatever
    their entropy's.  A row whose logits are all -inf has -inf, the entropy 0 and no
    gradient; one that holds a NaN or +inf is NaN.
    """
    out = torch.ops.ocl.token_log_probs(logits, tokens, top)
    return out if top else out[:2]
