"""Attention over whole prompts of different lengths, packed one behind the other.

A model attends to a prompt before its keys and values go into a cache.  ``prompt_attention`` is that step for batches whose prompts
differ in length: tensors ``[tokens, heads, 128]`` without padding, ``cu_seqlens`` saying where each sequence starts and ends.
``ResKVLlama(cache="int4")`` calls it; the models with a compressed or dense cache have one length per batch and use the library's
attention for the prompt.  The kernel is ``csrc/prompt_attention.cu``.
"""

from __future__ import annotations

import torch

from ._extension import host, require_device


def prompt_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    cu_seqlens: torch.Tensor,
    *,
    scaling: float | None = None,
    causal: bool = True,
    out: torch.Tensor | None = None,
    return_lse: bool = False,
    status: torch.Tensor | None = None,
):
    """Attention of every token to the tokens of its own sequence (``causal``: up to itself).

    ``query`` is FP16 or BF16 ``[T,H,128]``, ``key`` and ``value`` ``[T,KH,128]`` of the same type, ``H`` a multiple of
    ``KH`` (query head ``h`` reads KV head ``h // (H / KH)``; at most 128 per KV head); views of a fused projection are read
    where they lie.  ``cu_seqlens`` is int32 ``[n+1]`` on the same device, non-decreasing: sequence ``i`` holds
    the tokens ``[cu_seqlens[i], cu_seqlens[i+1])``; lengths may be 0, bounds are clamped to ``[0, T]``.  ``scaling`` (positive) defaults
    to ``128**-0.5``.

    Returns ``[T,H,128]`` of the query's type, written to ``out`` if that is given (contiguous, not overlapping the inputs);
    with ``return_lse`` also FP32 ``[T,H]``, the natural logarithm of each row's sum of exponentials.  Rows that belong to no
    sequence are not written.  Scores, sums and products are FP32, the weights are rounded once to the type of ``value`` for
    the product with it.  A row whose scores are all minus infinity has no weights: NaN, with a logarithm of minus infinity.  Infinities and NaN count only where they are attended to.  Inference only: tensors that ask for
    a gradient, carry a tangent, are no plain tensors (subclasses, vmap) or are being traced are refused.

    ``status``, an int32 tensor on the device (``PagedInt4Cache.status``, whose ``check()`` then speaks for this call too), gets a
    bit if a bounded wait on the device ran out and rows were left unwritten.
    """
    if isinstance(query, torch.Tensor) and query.is_cuda:
        require_device(query.get_device())
    return host().prompt_attention(query, key, value, cu_seqlens, scaling, bool(causal), out, bool(return_lse), status)
