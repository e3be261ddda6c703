"""An exact K/V cache in pages for a batch of sequences that may share prefixes.

Beside ``EvictingKVCache`` (exact rows of a fixed budget) and ``LogStructuredKVCache`` (compressed rows): memory follows
the rows in use, and what many sequences have in common - an instruction, a document, also one that a LogKV cache has
compressed - is stored and read once. No counterpart in the reference, whose dense cache has a full row per sequence.
"""

from __future__ import annotations

import math

import torch

from ._lib import check_activation_dtype, refuse_tangents
from .log_kv_cache import LogStructuredKVCache
from .log_kv_pack import _check_backend, log_kv_prefix_attention
from .paged_attention import MIN_PAGE, SharedPrefix, log_kv_paged_append, log_kv_paged_attention
from .rotary import log_kv_rotary
from .row_attention import _ROW_DTYPES
from .streaming import LogKVStreamingAttention


class PagedKVCache:
    """Up to ``max_rows`` rows of ``batch_size`` sequences in a pool of ``pages`` pages of ``page_size`` rows.

    ``cache(q, k, v, counts=None)`` stores T new tokens of every sequence and returns their causal attention ``[batch,
    n_heads, T, v_dim]`` over the sequence's prefix, its rows and each other; ``cache.draft(q, k, v, visible)`` attends a
    tree of drafted tokens without a change. Queries and keys come as they leave the projections: with ``frequencies``
    (``rotary_frequencies``) both are rotated here, a token's position being its prefix's tokens and its row.

    A prefix belongs to each of N equal runs of consecutive sequences: ``cache.prefix(q, k, v)`` writes the next tokens of
    N prefixes into the pool, returning their own causal attention (a prompt may come in blocks), or ``cache.share(x)``
    takes a compressed document: a ``LogKVStreamingAttention`` or its ``LogStructuredKVCache`` of batch N. Prefixes come
    before the sequences' first rows.

    Pages are handed out as rows come and taken back by ``free``, ``trim`` and ``reset``; a call that finds too few raises
    ``RuntimeError``, and a call that raises changes nothing. ``lengths`` (int32 ``[batch]``) and the page table are on the
    device; the host keeps an upper bound of the lengths and never waits. Calls cannot be captured into a HIP graph, since
    the host hands out pages in them: capture ``log_kv_paged_append`` and ``log_kv_paged_attention`` on a cache's tensors
    instead."""

    def __init__(self, batch_size: int, n_groups: int, k_dim: int, v_dim: int, pages: int, *, scale: float, max_rows: int,
                 page_size: int = 64, frequencies=None, interleaved: bool = False, amplitude: float = 1.0,
                 dtype=torch.bfloat16, device="cuda") -> None:
        if min(batch_size, n_groups, pages, max_rows) < 1:
            raise ValueError("sizes and pages must be positive")
        if k_dim % 8 or v_dim % 8 or not 8 <= k_dim <= 256 or not 8 <= v_dim <= 256:
            raise ValueError("key and value widths must be multiples of 8 up to 256")
        if page_size < MIN_PAGE or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from {MIN_PAGE} on")
        if max_rows > 2 ** 30 or batch_size * n_groups > 65535:
            raise ValueError("at most 2^30 rows a sequence and 65535 lanes")
        if dtype not in _ROW_DTYPES:
            raise ValueError("the cache must be bfloat16 or float16")
        if not 0.0 < scale < math.inf or not math.isfinite(amplitude):
            raise ValueError("attention scale must be positive, amplitude finite")
        if frequencies is not None and (frequencies.ndim != 1 or 2 * frequencies.numel() > k_dim
                                        or frequencies.dtype not in (torch.float64, torch.float32)):
            raise ValueError("frequencies must be float64 or float32 [rotated features / 2] for at most the keys' features")
        if frequencies is not None and frequencies.requires_grad:
            raise NotImplementedError("frequencies have no gradient")
        self.batch_size, self.n_groups, self.page_size, self.max_rows = batch_size, n_groups, page_size, max_rows
        self.scale, self.interleaved, self.amplitude = float(scale), bool(interleaved), float(amplitude)
        self.frequencies = None if frequencies is None else frequencies.to(device)
        self.k_pages = torch.empty(pages, n_groups, page_size, k_dim, dtype=dtype, device=device)
        self.v_pages = torch.empty(pages, n_groups, page_size, v_dim, dtype=dtype, device=device)
        self.lengths = torch.zeros(batch_size, dtype=torch.int32, device=device)
        self.table = torch.full((batch_size, -(-max_rows // page_size)), -1, dtype=torch.int32, device=device)
        self._free = list(range(pages - 1, -1, -1))
        self._pages = [[] for _ in range(batch_size)]
        self._bound = [0] * batch_size          # no sequence has more rows than this
        self._forget_prefix()

    def _forget_prefix(self):
        self._prefix_pages, self._prefix_rows, self._prefix_table = [], 0, None      # of prefixes in the pool
        self._compressed = None                                                      # or a compressed document
        self._first = 0                                                              # position of a sequence's row 0

    @property
    def prefix_rows(self) -> int:
        """Rows of all prefixes in the pool."""
        return self._prefix_rows * len(self._prefix_pages)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def reset(self) -> None:
        """Empty the cache: sequences and prefixes."""
        self.free()
        for line in self._prefix_pages:
            self._free += line
        self._forget_prefix()

    def free(self, sequences=None) -> None:
        """Drop the rows of ``sequences`` (indices; all without them), whose pages others may take. Prefixes stay."""
        self._refuse_capture()
        rows = range(self.batch_size)
        if sequences is not None:
            given = sequences.tolist() if hasattr(sequences, "tolist") else list(sequences)
            rows = [b.item() if hasattr(b, "item") else b for b in (given if isinstance(given, list) else [given])]
            if any(not isinstance(b, int) or isinstance(b, bool) or not 0 <= b < self.batch_size for b in rows):
                raise ValueError("sequences must be indices of the batch")
        if sequences is None:
            self.lengths.zero_()
            self.table.fill_(-1)
        elif len(rows):
            index = self._upload(torch.tensor(rows, dtype=torch.int64))
            self.lengths.index_fill_(0, index, 0)
            self.table.index_fill_(0, index, -1)
        for b in rows:
            self._free += self._pages[b]
            self._pages[b], self._bound[b] = [], 0

    def trim(self) -> None:
        """Take back the pages that padded batches reserved and did not fill. Waits for the device, which knows how many."""
        self._refuse_capture()
        for b, n in enumerate(self.lengths.tolist()):
            keep = -(-n // self.page_size)
            if keep < len(self._pages[b]):
                self.table[b, keep:].fill_(-1)
                self._free += self._pages[b][keep:]
                del self._pages[b][keep:]
            self._bound[b] = n

    def _upload(self, host):
        return host.pin_memory().to(self.lengths.device, non_blocking=True) if self.lengths.is_cuda else host

    def _reserve(self, lines, table, rows):
        """Pages for ``rows[i]`` rows of every line, returned as (line, place, page); too few of them change nothing."""
        need = [max(0, -(-n // self.page_size) - len(line)) for line, n in zip(lines, rows)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"the pool has {len(self._free)} pages left, {sum(need)} are needed"
                               " (trim() takes back what padded batches left unused)")
        places = [(i, len(line) + j) for i, (line, n) in enumerate(zip(lines, need)) for j in range(n)]
        new = [(*x, page) for x, page in zip(places, reversed(self._free))]
        if new:
            at = self._upload(torch.tensor(list(zip(*new)), dtype=torch.int64))
            table.index_put_((at[0], at[1]), at[2].to(torch.int32))
            del self._free[-len(new):]
        for i, _, page in new:
            lines[i].append(page)
        return new

    def _give_back(self, lines, table, new):
        """Undoes a ``_reserve`` whose call failed. What is on its way to the pages comes before what others write there."""
        for i, _, page in reversed(new):
            lines[i].pop()
            self._free.append(page)
        if new:
            at = self._upload(torch.tensor(list(zip(*new)), dtype=torch.int64))
            table.index_put_((at[0], at[1]), torch.full_like(at[2], -1, dtype=torch.int32))

    def _check(self, q, k, v, batch, sharing):
        """A call's tokens; refuses what an append or an attention would, before a page is handed out. ``sharing``: the
        sequences whose queries read the same rows."""
        refuse_tangents(q, k, v)
        shape = q.shape
        if len(shape) != 4 or shape[0] != batch or shape[2] < 1 or shape[1] < 1 or shape[1] % self.n_groups:
            raise ValueError("queries must be [batch, n_heads, T, k_dim] with n_groups dividing the heads")
        tokens, dk, dv = shape[2], self.k_pages.size(3), self.v_pages.size(3)
        if shape[3] != dk or k.shape != (batch, self.n_groups, tokens, dk) or v.shape != (batch, self.n_groups, tokens, dv):
            raise ValueError("new rows must be k [batch, n_groups, T, k_dim] and v [batch, n_groups, T, v_dim]")
        if not q.dtype == k.dtype == v.dtype:
            raise ValueError("queries, keys and values must be of one dtype")
        check_activation_dtype(q.dtype)
        if not q.device == k.device == v.device == self.k_pages.device:
            raise ValueError("queries and new rows must be on the cache's device")
        if shape[1] // self.n_groups * tokens * sharing > 2 ** 19:
            raise ValueError("too many queries a KV group at once: split the call")
        self._refuse_capture()
        return tokens

    def _refuse_capture(self):
        if self.k_pages.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a PagedKVCache's calls cannot be captured: capture log_kv_paged_append and "
                               "log_kv_paged_attention on its tensors instead")

    def _sharing(self):
        """Sequences behind one prefix, 1 without one."""
        prefixes = len(self._prefix_pages) if self._compressed is None else self._compressed[0].batch_size
        return self.batch_size // prefixes if prefixes else 1

    def _append(self, q, k, v, table, lengths, **position):
        return log_kv_paged_append(k, v, self.k_pages, self.v_pages, table, lengths, q=q, frequencies=self.frequencies,
                                   interleaved=self.interleaved, amplitude=self.amplitude, **position)

    def _attend(self, q, k, v, **kw):
        if self._compressed is not None:
            cache, engine = self._compressed
            pending = None if engine is None else engine._log_kv_pending
            return log_kv_prefix_attention(cache, q, k, v, self.k_pages, self.v_pages, self.table, self.lengths, self.scale,
                                           pending=None if pending is None else pending[:2], **kw)
        prefix = SharedPrefix(self._prefix_rows, table=self._prefix_table) if self._prefix_pages else None
        return log_kv_paged_attention(q, k, v, self.k_pages, self.v_pages, self.table, self.lengths, self.scale,
                                      prefix=prefix, **kw)

    @torch.no_grad()
    def prefix(self, q, k, v):
        """Attention ``[N, n_heads, T, v_dim]`` of the next T tokens of N prefixes (all of one length), which join them."""
        runs = len(self._prefix_pages) or (q.size(0) if q.ndim == 4 else 0)
        if self._compressed is not None or any(self._bound):
            raise RuntimeError("a prefix comes before the sequences' rows and beside no other one: reset() the cache first")
        if runs < 1 or self.batch_size % runs:
            raise ValueError(f"{runs} prefixes do not divide a batch of {self.batch_size}")
        tokens = self._check(q, k, v, runs, 1)
        if self._prefix_rows + tokens > 2 ** 30:
            raise ValueError("at most 2^30 rows a prefix")
        lines = [list(line) for line in self._prefix_pages] or [[] for _ in range(runs)]
        width = -(-(self._prefix_rows + tokens) // self.page_size)
        table = torch.full((runs, width), -1, dtype=torch.int32, device=self.k_pages.device)
        if self._prefix_table is not None:
            table[:, :self._prefix_table.size(1)] = self._prefix_table
        new = self._reserve(lines, table, [self._prefix_rows + tokens] * runs)
        try:
            q, stored = self._append(q, k, v, table, self._prefix_rows)
            out = log_kv_paged_attention(q, stored, v, self.k_pages, self.v_pages, table, self._prefix_rows, self.scale)
        except Exception:
            self._give_back(lines, table, new)
            raise
        self._prefix_pages, self._prefix_table = lines, table
        self._prefix_rows += tokens
        self._first = self._prefix_rows
        return out

    def share(self, source) -> None:
        """Take a compressed document of batch N (a ``LogKVStreamingAttention``, whose pending token is part of it, or a
        ``LogStructuredKVCache``) as the sequences' prefix. It is read at every call, not copied: leave it as it is."""
        engine = source if isinstance(source, LogKVStreamingAttention) else None
        cache = source.cache if engine is not None else source
        if not isinstance(cache, LogStructuredKVCache):
            raise ValueError("a shared document is a LogKVStreamingAttention or a LogStructuredKVCache")
        if self._prefix_pages or self._compressed is not None or any(self._bound):
            raise RuntimeError("a prefix comes before the sequences' rows and beside no other one: reset() the cache first")
        _check_backend(cache.semantic_pack_backend)
        if (self.batch_size % cache.batch_size or cache.n_groups != self.n_groups or cache.k_dim != self.k_pages.size(3)
                or cache.v_dim != self.v_pages.size(3) or self.k_pages.dtype != torch.bfloat16
                or cache.recent_k.device != self.k_pages.device):
            raise ValueError("a shared document has this cache's groups, widths and device, a batch that divides it, and "
                             "bfloat16 rows")
        pending = 0 if engine is None or engine._log_kv_pending is None else engine._log_kv_pending[0].size(2)
        self._compressed, self._first = (cache, engine), cache.token_count + pending

    @torch.no_grad()
    def draft(self, q, k, v, visible, positions=None):
        """Attention of T drafted tokens of every sequence over its prefix, its rows and the drafted rows that ``visible``
        (bool, ``[T, T]`` or ``[B, T, T]``) shows each; nothing is stored. With ``frequencies``, ``positions`` (``[T]`` or
        ``[B, T]``) are the tokens' own, those of their depths in the tree."""
        self._check(q, k, v, self.batch_size, self._sharing())
        if self.frequencies is not None:
            if positions is None:
                raise ValueError("drafted tokens that are rotated need their positions")
            q, k = log_kv_rotary(q, k, self.frequencies, positions, interleaved=self.interleaved, amplitude=self.amplitude)
        return self._attend(q, k, v, visible=visible)

    @torch.no_grad()
    def __call__(self, q, k, v, counts=None):
        """Attention ``[batch, n_heads, T, v_dim]`` of T new tokens, which join the cache. ``counts`` (int32 ``[batch]`` on
        the device) gives the tokens that exist per sequence of a padded batch; the host, which does not wait for them, counts
        all T against ``max_rows`` and the pool until ``trim``."""
        tokens = self._check(q, k, v, self.batch_size, self._sharing())
        if counts is not None:
            if (counts.shape != (self.batch_size,) or counts.dtype not in (torch.int32, torch.int64)
                    or counts.device != self.k_pages.device):
                raise ValueError("counts must be an int32 tensor [batch] on the cache's device")
            counts = counts.clamp(0, tokens).to(torch.int32)
        if max(self._bound) + tokens > self.max_rows:
            raise RuntimeError(f"a sequence has at most {self.max_rows} rows: {max(self._bound)} may be in use, {tokens} are "
                               "new (trim() counts anew what padded batches left unused)")
        new = self._reserve(self._pages, self.table, [n + tokens for n in self._bound])
        try:
            q, stored = self._append(q, k, v, self.table, self.lengths, first=self._first, counts=counts)
            out = self._attend(q, stored, v, counts=counts)
        except Exception:
            self._give_back(self._pages, self.table, new)
            raise
        self.lengths.add_(tokens if counts is None else counts)
        self._bound = [n + tokens for n in self._bound]
        return out
