"""``sb_attn_decode``: stick-breaking attention of new tokens over a paged key-value cache.

The serving form of ``sb_attn``: the same function of the same keys, evaluated for the newest tokens of each sequence only.  The
reference has no counterpart (its operators attend over whole sequences, ``sb_varlen/__init__.py:24-82``).
"""
from __future__ import annotations

import math

import torch

from . import _sb_torch, ops


def sb_attn_decode(q, k_pages, v_pages, page_table, seq_lens, inv_temp=None, attend_current=False):
    """q: ``(batch, heads, new_tokens, head_dim)``, the newest tokens of each sequence, whose keys and values the cache already
    holds (``kv_append``).  k_pages, v_pages: ``(pages, kv_heads, page_size, head_dim)``, any strides with the last one 1;
    ``heads`` is a multiple of ``kv_heads``, query head h reads key head ``h // (heads // kv_heads)``.  page_table: int32
    ``(batch, pages per sequence)``, the pages of a sequence in order; seq_lens: int32 ``(batch,)``, new tokens included; both on
    the device.  Returns ``o`` like q and ``rem (batch, heads, new_tokens)``, as ``sb_attn`` does for these rows.

    Query t of sequence b has position ``seq_lens[b] - new_tokens + t`` and attends to the keys before it (``attend_current``:
    and its own).  A row without keys, or in front of its sequence (a padded batch), gets o = 0 and rem = 1.  A length that
    cannot be, and what a page that is none would have gone into, gives NaN and an error at ``check_status()``.

    Serving only: no derivative, so call it under ``torch.no_grad()``.  It does not synchronise, and can be captured into a graph.
    """
    if inv_temp is None:
        inv_temp = 1 / math.sqrt(q.size(-1))
    if torch.compiler.is_compiling():
        return ops.decode_op(q, k_pages, v_pages, page_table, seq_lens, float(inv_temp), bool(attend_current))
    return _sb_torch.decode(q, k_pages, v_pages, page_table, seq_lens, inv_temp, attend_current, ops.switch_flags())
