"""Operators of the `ocl` device that torch has no function for."""
from __future__ import annotations

import torch

from . import _C  # noqa: F401  (registers torch.ops.ocl)


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
    order.  The result goes to ``scaled_dot_product_attention`` as
    ``attn_mask``.
    """
    return torch.ops.ocl.relative_position_bias(table, q_len, k_len, bidirectional, max_distance, q_offset)
