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
