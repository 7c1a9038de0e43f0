"""A key / value cache in pages: places for new tokens, the tokens' way into them, attention over them.

A cache is two tensors ``[pages, kv heads, page_size, D]`` (any strides with a contiguous last dimension: a transposed view of
``[pages, page_size, kv heads, D]`` will do).  A request's tokens lie in the pages that its row of the block table lists; token
``j`` is token ``j % page_size`` of page ``block_table[b, j // page_size]``, and its slot is ``page * page_size + j % page_size``.

The pages may be in 8 bits: int8, with a float32 scale for each token and kv head (``key_scales`` and ``value_scales``, ``[pages, kv heads, page_size]``,
any strides).  ``rotary_append`` then stores a row ``y`` as ``round(y / scale)`` with ``scale = max|y| / 127``, which keeps it to 1 / 254 of its largest
value, in half of the memory and of the time that reading takes.

A decoding step is ``page_step`` once, and then, for every layer, ``rotary_append`` and ``paged_attention``.  None of
them waits for the GPU or depends on a length that only the GPU knows, so that a step can be captured in a CUDA graph.
What would look on (a tracer, a dispatch mode, a functorch transform, a tensor class with a ``__torch_function__`` of its own) is
refused with ``NotImplementedError``.
(No counterpart in the reference, whose keys and values are contiguous.)
"""
from __future__ import annotations

from typing import Callable, NamedTuple, Optional, Tuple, Union

import torch

from .blockmask import device_buffers, identity_score, module_for, noop_mask
from .modtrace import lower_mods
from .rotary import native


class PageStep(NamedTuple):
    """What ``page_step`` returns.  All int32 but ``slots`` (int64)."""

    lengths: torch.Tensor    # [B] tokens of each request with the new ones
    positions: torch.Tensor  # [num_tokens] place of each new token in its request
    slots: torch.Tensor      # [num_tokens] its place in the pages, -1: it has none
    requests: torch.Tensor   # [num_tokens] its request
    starts: torch.Tensor     # [B + 1] where the new tokens of a request begin
    taken: torch.Tensor      # [1] pages of the free list that are in use now


def page_step(lengths, new_tokens, block_table, free_pages, page_size: int, num_tokens: int, taken=None) -> PageStep:
    """Finds places for the new tokens of a batch of requests, in one launch.

    ``lengths`` and ``new_tokens`` (int32 ``[B]``): tokens that the requests have and get (below 0 counts as 0).  The entries of
    ``block_table`` (int32 ``[B, width]``) for the pages they need in addition are filled in **in place**, from ``free_pages`` (int32)
    in the order of the requests, beginning behind the first ``taken`` (int32, one value, default 0).  ``num_tokens`` is the sum of
    ``new_tokens``, which the host has to know to have made the tokens; the new tokens are numbered through, request after request.

    Where the free list or the row of a table is too short, tokens get the slot -1 (``rotary_append`` leaves them out) and table
    entries -1; ``taken`` then is beyond the list's length.  If ``num_tokens`` is larger than the sum, the rest is padding: position 0,
    slot and request -1.  Nothing else is changed, so that a call may be repeated, with the same results.  The list is only gone through
    forwards: pages that are given back go into a new one, with ``taken`` beginning at 0 again.
    """
    return PageStep._make(native().page_step(lengths, new_tokens, block_table, free_pages, page_size, num_tokens, taken))


def rotary_append(query, key, value, key_pages, value_pages, slots, table=None, positions=None, *, query_weight=None,
                  key_weight=None, eps: float = 1e-6, interleaved: bool = False, bhln: bool = True, key_scales=None,
                  value_scales=None) -> Optional[torch.Tensor]:
    """``rotary_embedding`` for new tokens, whose keys and values go straight into the cache: ``key`` (normed and rotated)
    and ``value`` (as it is) are written to ``slots`` of ``key_pages`` and ``value_pages`` **in place**; the normed and rotated
    ``query`` is returned.  One launch.

    ``query`` ``[B, Hq, S, D]`` (or ``None``), ``key`` ``[B, Hkv, S, D]`` and ``value`` ``[B, Hkv, S, Dv]``; ``bhln=False``: ``[B, S, H, D]``,
    for instance ``[1, tokens, H, D]`` for the prompts of a batch laid end to end.  ``slots`` (int64 ``[B, S]`` or ``[B * S]``) as ``page_step`` gives
    them; a slot below 0 is left out, one beyond the pages too, and the next call raises ``FlaxAttnError``.  No two
    tokens may have the same slot.  ``table``, ``positions`` and the weights are those of ``rotary_embedding``.

    With ``key_scales`` and ``value_scales`` the pages are int8 and the scales are written too (float16 and bfloat16 tensors).  What is stored is
    rounded once, from the fp32 value behind the rotation.  A row of zeros has the scale 0; one with an infinity or no number in it has no number
    for a scale, and is read as that throughout.
    """
    return native().rotary_append(query, key, value, key_pages, value_pages, slots, table, positions, query_weight, key_weight, eps,
                                  interleaved, not bhln, key_scales, value_scales)


def read_pages(key_pages, value_pages, block_table, starts, num_tokens: int, *, key_scales=None, value_scales=None, dtype: Optional[torch.dtype] = None,
               bhln: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cached tokens of a batch laid end to end, ``(key, value)`` of ``[1, kv heads, num_tokens, D]`` (``bhln=False``: ``[1, num_tokens, kv heads, D]``).

    Row ``t`` is token ``t - starts[b]`` of the request ``b`` with ``starts[b] <= t < starts[b + 1]`` (``starts``: int32 ``[B + 1]``, never decreasing; of whole requests
    the sums of their lengths).  ``num_tokens`` is ``starts[B]``, which the host has to know; rows beyond it, or in front of ``starts[0]``, are 0.
    Pages in 8 bits (with their scales) are multiplied out and rounded to ``dtype``, others are copied.  A table entry that is no page, or a token that the table has no
    room for, leaves the row 0, and the next call raises ``FlaxAttnError`` (``check_status``); so do starts that decrease, with which rows are some tokens or other.

    It is what attention over more than a few new tokens takes: the next piece of a prompt (``prompt_attention`` with ``key_starts``), or the
    tokens that requests have in common (``prefix`` of ``paged_attention``).  One launch, no gradient.
    """
    return native().read_pages(key_pages, value_pages, block_table, starts, num_tokens, key_scales, value_scales, dtype, not bhln)


def known_mods(score_mod, mask_mod, device):
    """(handle, buffers) of mods that the native path does not know yet, or that capture tensors elsewhere than on `device`."""
    module = module_for(score_mod, mask_mod)
    lowered = lower_mods(None if score_mod is identity_score else score_mod, None if mask_mod is noop_mask else mask_mod)
    return module.handle.value, tuple(device_buffers(lowered, device))


def paged_attention(query, key_pages, value_pages, block_table, lengths, score_mod: Optional[Callable] = None,
                    mask_mod: Optional[Callable] = None, *, window: Optional[int] = None, sm_scale: Optional[float] = None,
                    bhln: bool = True, return_lse: bool = False, b_offset: int = 0, h_offset: int = 0,
                    kernel_options: Optional[dict] = None, key_scales=None, value_scales=None,
                    prefix: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of the newest tokens of each request over its pages.

    ``query`` ``[B, Hq, Sq, D]`` (``bhln=False``: ``[B, Sq, Hq, D]``) holds the last ``Sq`` tokens of each request, ``lengths`` (int32 ``[B]``) counts
    its tokens with them, and ``block_table`` (int32 ``[B, width]``) lists its pages; entries behind its length are not looked at.
    ``Hq`` is a multiple of the pages' heads.  Query ``i`` is token ``p = lengths[b] - Sq + i``.  It sees the keys up to itself, with
    ``window`` those at most ``window`` tokens behind it (as ``masks.generate_sliding_window``), of these the ones that ``mask_mod`` keeps,
    and ``score_mod`` changes their scores; both see ``p`` as ``q_idx``.  A query that sees nothing (a request of length 0, a query in front of the
    first token) is 0, with a logsumexp of ``-inf``.  Returns the output in the shape of ``query`` and, with ``return_lse``, the natural-log
    logsumexp ``[B, Hq, Sq]`` in float32.

    Scores, softmax and sums are in fp32; 16-bit probabilities are rounded to the dtype for the product with the values (up to 16 query rows per
    kv head in two parts, which leaves nothing of it), and a ``score_mod`` over 16-bit inputs divides scores and takes their ``tanh`` to some 2^-22; where a
    quotient decides something (a mask, a comparison, a rounding, an index) it is exact, as in ``flax_attention``.  As there, a ``score_mod`` takes a key out with
    any score below -2.3e38 (the lowest of float32, ``-inf``), and a row with no other is 0.  Cached values of keys that ``mask_mod`` takes out must be
    finite; what lies behind a request's length or out of the window is not looked at, so that pages which the window has left may be given back.  A
    table entry that is no page, or a length beyond the table, leaves the keys out, and the next call raises ``FlaxAttnError``
    (``check_status``).  Meant for a few tokens per request; there is no gradient.  ``kernel_options``: ``{"kernels": "general"}`` takes keys and values in
    16-byte pieces where TMA would do.

    With ``key_scales`` and ``value_scales`` (float32 ``[pages, kv heads, page_size]``) the pages are in 8 bits, as ``rotary_append`` writes them, and queries float16 or
    bfloat16.  A scale that is no number or infinite makes the rows that see its token no numbers, and no others.
    What else is rounded then: up to 8 query rows per kv head, queries are whole numbers of 23 bits of their row's largest value, and probabilities times the values' scales
    whole numbers of 16 bits of the largest among 32 keys; with more rows, these products are two bfloat16 parts.  Pages in 8 bits save time for up to 8 rows per kv head (head
    dims above 128: 16); with more the way from 8 to 16 bits takes longer than the smaller pages save.

    ``prefix``: keys and values ``[1, kv heads, tokens, D]`` (``bhln=False``: ``[1, tokens, kv heads, D]``) that all requests begin with, in front of those in
    their pages, of the queries' dtype also where the pages are in 8 bits (``read_pages`` takes them out of pages).  They are read once for all requests, not
    once for each.  ``lengths`` still counts what lies in the pages; a query's token is ``p = tokens + lengths[b] - Sq + i``, for the mods and the window too, and a
    query in front of the request's first token in the pages sees nothing, the prefix neither.  Probabilities over the prefix are rounded to the dtype once (over 16-bit pages up to 16 rows per
    kv head lose nothing): tokens moved from the pages into the prefix are as exact as in ``prompt_attention``.  Over a prefix and over 8-bit pages a ``score_mod`` takes ``tanh`` of scores to
    4e-7 in proportion.  A score over the prefix that is no number or ``+inf`` makes the rows that see its key no numbers.
    """
    general = kernel_options is not None and kernel_options.get("kernels") == "general"
    call = native().paged_attention
    res = call(query, key_pages, value_pages, block_table, lengths, score_mod, mask_mod, window, sm_scale, not bhln, return_lse, b_offset,
               h_offset, general, key_scales, value_scales, prefix, None)
    if res is None:
        res = call(query, key_pages, value_pages, block_table, lengths, score_mod, mask_mod, window, sm_scale, not bhln, return_lse, b_offset,
                   h_offset, general, key_scales, value_scales, prefix, known_mods(score_mod, mask_mod, query.device))
    return res
