"""Attention of whole prompts, or of pieces of them, that lie end to end.

A batch of prompts of different lengths is one sequence, ``[1, heads, tokens, D]``, in which request after request has its
tokens; ``starts`` says where each begins.  It is what ``page_step`` numbers new tokens by and what ``rotary_append`` takes.
(No counterpart in the reference, whose sequences have one length; there, and in ``flax_attention`` here, requests that share a
sequence are told apart by a mask over their ids.)
"""
from __future__ import annotations

from typing import Callable, Optional, Tuple, Union

import torch

from .paged import known_mods
from .rotary import native


def prompt_attention(query, key, value, starts, score_mod: Optional[Callable] = None, mask_mod: Optional[Callable] = None, *,
                     key_starts=None, window: Optional[int] = None, sm_scale: Optional[float] = None, bhln: bool = True,
                     return_lse: bool = False, b_offset: int = 0, h_offset: int = 0,
                     kernel_options: Optional[dict] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Causal attention of each request's queries over its own keys.

    ``query`` ``[1, Hq, T, D]``, ``key`` ``[1, Hkv, T, D]`` and ``value`` ``[1, Hkv, T, Dv]`` (``bhln=False``: ``[1, T, H, D]``), float16, bfloat16 or float32, with any
    strides of whole 16 bytes and a contiguous head dimension, a multiple of 16 up to 256; ``Hq`` is a multiple of ``Hkv``.  The tokens of request ``b`` are rows ``starts[b]`` to
    ``starts[b + 1] - 1`` (int32 ``[B + 1]``, never decreasing, on the device; a request may have none).  With ``key_starts`` keys and values are of another number of
    rows, those of request ``b`` from ``key_starts[b]`` on: a piece of a prompt over all that came before it (``read_pages``), its last query the last key's token.

    Query ``i`` of ``n`` is token ``p = m - n + i`` of a request with ``m`` keys.  It sees the keys up to itself, with ``window`` those at most ``window`` tokens behind it, of
    these the ones that ``mask_mod`` keeps, and ``score_mod`` changes their scores; both see the request as ``b``, ``p`` as ``q_idx`` and the key's place in the request as
    ``kv_idx``.  A query that sees nothing is 0, with a logsumexp of ``-inf``, and so are rows of no request.  Returns the output in the layout of ``query`` and, with
    ``return_lse``, the natural-log logsumexp ``[1, Hq, T]`` in float32.

    Scores, softmax and sums are in fp32 (to 2.7e-6 in proportion: some exponentials are a polynomial's); 16-bit probabilities are rounded to the dtype for the product with the values,
    and a ``score_mod`` over 16-bit inputs divides scores to some 2^-22 and takes their ``tanh`` to 4e-7 in proportion; where a quotient decides something it is exact, as in ``paged_attention``.
    A score that is no number or ``+inf`` makes the rows that see its key no numbers.  The values of a request must be finite also where a query does not see them (behind it, or taken out by
    ``mask_mod``: they are multiplied with 0); other requests' may hold anything.  Starts in front of the rows or beyond them are cut to what is there, and the next call raises ``FlaxAttnError``
    (``check_status``); so it does for starts that decrease, with which the call has no results (there may be rows that nothing is written to).  Nothing waits for the GPU or depends on a
    length on the host.  There is no gradient: training over sequences of several documents is ``flax_attention`` with a mask over their ids.  ``kernel_options``:
    ``{"kernels": "general"}`` takes the general kernel where the tcgen05 one would do.
    """
    general = kernel_options is not None and kernel_options.get("kernels") == "general"
    call = native().prompt_attention
    res = call(query, key, value, starts, key_starts, score_mod, mask_mod, window, sm_scale, not bhln, return_lse, b_offset, h_offset, general, None)
    if res is None:
        res = call(query, key, value, starts, key_starts, score_mod, mask_mod, window, sm_scale, not bhln, return_lse, b_offset, h_offset, general,
                   known_mods(score_mod, mask_mod, query.device))
    return res
