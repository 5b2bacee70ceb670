"""The paged key-value cache that ``sb_attn_decode`` reads: the write of new keys and values, and the keeping of its pages.

Everything a step needs stays on the device: page tables, lengths and the count of sequences that hold each page are int32
tensors which the operators read and write in place.  No call synchronises, all can be captured into a graph, and which page a
sequence gets is a rule (the lowest free ones, in the order of sequences and positions), so that runs repeat.  A call that
cannot do all it is asked to (too few pages, an index that is no sequence, a length that cannot be) changes nothing;
``check_status()`` raises.

``PagedKVCache`` holds the tensors of a cache; the functions work on any tensors laid out like them.  The reference has no cache.
"""
from __future__ import annotations

import torch

from . import _sb_torch, ops
from .sb_decode import sb_attn_decode


def kv_append(k, v, k_pages, v_pages, page_table, seq_lens, cu_seqlens=None, zero_start=True):
    """Writes the keys and values of the newest tokens into their pages (``k_pages``, ``v_pages``: one layer, as in
    ``sb_attn_decode``).  ``seq_lens`` counts the new tokens already: the last n positions of a sequence are written.

    k, v: ``(batch, kv_heads, n, head_dim)``, or, with ``cu_seqlens`` (as in ``sb_attn_varlen``: a leading 0 iff ``zero_start``),
    packed ``(kv_heads, tokens, head_dim)`` with a number of tokens per sequence.  Tokens in front of position 0 (a padded batch)
    and packed tokens behind the last sequence are left out.  No other sequence may share a page that is written to."""
    if torch.compiler.is_compiling():
        ops.append_op(k, v, k_pages, v_pages, page_table, seq_lens, cu_seqlens, bool(zero_start))
    else:
        _sb_torch.append(k, v, k_pages, v_pages, page_table, seq_lens, cu_seqlens, bool(zero_start) and cu_seqlens is not None)


def kv_extend(page_table, seq_lens, page_refs, counts, page_size):
    """Makes room for new tokens: ``seq_lens`` grows by ``counts`` (an int32 tensor with an entry per sequence, or one number for
    every sequence that is not empty), and the sequences get the pages they lack."""
    tensor = counts if torch.is_tensor(counts) else None
    _sb_torch.kv_extend(page_table, seq_lens, page_refs, tensor, 0 if tensor is not None else int(counts), page_size)


def kv_fork(k_cache, v_cache, page_table, seq_lens, page_refs, src, dst):
    """Sequence ``dst[i]``, which must be empty, becomes a copy of ``src[i]`` (int32 tensors): full pages are shared, the tokens of
    a last page that is not full are copied to a page of its own.  Caches ``([layers,] pages, kv_heads, page_size, head_dim)``.
    A sequence may be forked several times in a call, but not be forked and become a fork in the same one."""
    _sb_torch.kv_fork(k_cache, v_cache, page_table, seq_lens, page_refs, src, dst)


def kv_free(page_table, seq_lens, page_refs, seqs, page_size):
    """The listed sequences (int32 tensor) give their pages back and are empty.  A page goes free when no sequence holds it.
    Empty sequences, and the same one twice, are allowed.  An entry that names no page, or a free one, goes out of its row, counts
    nothing down, and is an error at ``check_status()``."""
    _sb_torch.kv_free(page_table, seq_lens, page_refs, seqs, page_size)


def kv_compact(k_cache, v_cache, page_table, seq_lens, page_refs):
    """Moves the pages in use to the front of the cache: with N in use, the r-th of those at or behind N goes to the r-th free
    one before N, in all layers, and the tables follow.  With a negative count nothing is changed; an entry that names no page, or a
    free one behind N, is left as it is, an error at ``check_status()``."""
    _sb_torch.kv_compact(k_cache, v_cache, page_table, seq_lens, page_refs)


class PagedKVCache:
    """A cache of ``layers`` x ``num_pages`` pages for up to ``max_seqs`` sequences of up to ``max_len`` tokens.

    ::

        cache = PagedKVCache(layers, num_pages, kv_heads, page_size, head_dim, max_seqs, max_len)
        cache.extend(counts)                      # per step: room for the new tokens (their number, per sequence)
        cache.append(layer, k, v)                 # per layer: write them, then attend
        o, rem = cache.attend(layer, q)

    A sequence is a row of ``page_table`` and of ``seq_lens``; length 0 is an empty one.  ``append`` and ``attend`` take a batch of
    all ``max_seqs`` rows, or of the rows ``rows`` (a slice)."""

    def __init__(self, layers, num_pages, kv_heads, page_size, head_dim, max_seqs, max_len, dtype=torch.bfloat16, device="cuda"):
        shape = (layers, num_pages, kv_heads, page_size, head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        self.page_size = page_size
        self.page_table = torch.full((max_seqs, -(-max_len // page_size)), -1, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(max_seqs, dtype=torch.int32, device=device)
        self.page_refs = torch.zeros(num_pages, dtype=torch.int32, device=device)

    def extend(self, counts):
        kv_extend(self.page_table, self.seq_lens, self.page_refs, counts, self.page_size)

    def append(self, layer, k, v, cu_seqlens=None, zero_start=True, rows=slice(None)):
        kv_append(k, v, self.k[layer], self.v[layer], self.page_table[rows], self.seq_lens[rows], cu_seqlens, zero_start)

    def attend(self, layer, q, inv_temp=None, attend_current=False, rows=slice(None)):
        return sb_attn_decode(q, self.k[layer], self.v[layer], self.page_table[rows], self.seq_lens[rows], inv_temp, attend_current)

    def fork(self, src, dst):
        kv_fork(self.k, self.v, self.page_table, self.seq_lens, self.page_refs, src, dst)

    def free(self, seqs):
        kv_free(self.page_table, self.seq_lens, self.page_refs, seqs, self.page_size)

    def compact(self):
        kv_compact(self.k, self.v, self.page_table, self.seq_lens, self.page_refs)
