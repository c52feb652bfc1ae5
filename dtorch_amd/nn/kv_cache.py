"""KV caches for the decode loop: a padded per-sequence cache and a paged one.

The reference's Llama port keeps no cache and recomputes causal attention over the whole sequence at
every step (python/dtorch/test/modules/llama.py:126-156, with repeat_kv for GQA at :80-85).  These
classes hold the keys and values of the tokens seen so far, so that a step appends its new tokens and
attends with the split-KV decode kernels:

    cache = KVCache(batch, kv_heads, max_len, head_dim)
    out = cache.prefill(q, k, v)          # prompt: causal attention, then its K/V into the cache
    out = cache.decode(q1, k1, v1)        # one token per sequence: append, then decode attention

Prompts in one prefill call share their length; per-sequence lengths then diverge only through the
caller's own use of `lengths`.

With ``dtype=torch.float8_e4m3fn`` a cache holds codes and a scale for each block of tokens and kv head
(half the bytes of a 16-bit one): the prompt's own attention still runs on the tensors as they come, and
decode reads the codes.  ``KVCache(track_weights=True)`` also sums the attention weight that each cached
token has received, and ``evict(keep, recent)`` shrinks every sequence to the tokens that received the most
(and the newest ones), so that a bounded cache serves an unbounded sequence.

Sequences may share what they have in common.  ``PagedKVCache.fork(parents)`` lets sequences continue others (beams, samples of
one prompt) on the same pages, which are copied only where they are written; ``share(groups)`` then reads the common
pages once for a group; ``KVCache.decode(..., prefix=cache)`` does so for a prefix in a cache of its own:

    cache = PagedKVCache(8, ...)
    cache.prefill(q, k, v)                # two prompts, in the first two rows
    cache.fork([0, 0, 0, 0, 1, 1, 1, 1])  # four sequences of each
    cache.share(2)
    out = cache.decode(q1, k1, v1)        # the prompts' pages are read once per group

With ``bounds_block`` a cache keeps the smallest and largest key of each block of tokens, and ``decode(..., keep=)`` attends
to the blocks with the largest bounds of their scores only.
"""
from __future__ import annotations

from typing import Optional

import numpy as np
import torch

from . import functional as F


_CODES = torch.float8_e4m3fn


def _scales(cache: torch.Tensor, block: int):
    """K and V scales of a cache of codes, one per block of tokens and kv head (None, None for other caches)."""
    if cache.dtype != _CODES:
        return None, None
    if block not in (16, 32, 64, 128, 256) or cache.shape[2] % block:
        raise ValueError(f"the tokens of a scale must be a power of two from 16 to 256 that divides a page; got {block}")
    if cache.shape[3] % 16 or cache.shape[3] > 128:
        raise ValueError(f"a cache of codes takes a head_dim that is a multiple of 16 up to 128; got {cache.shape[3]}")
    scale = torch.ones(cache.shape[0], cache.shape[1], cache.shape[2] // block, device=cache.device)
    return scale, torch.ones_like(scale)


def _bounds(cache: torch.Tensor, block: int):
    """Key bounds of a cache, one row per block of tokens and kv head (None, None without a block)."""
    if not block:
        return None, None
    if block not in (16, 32, 64, 128, 256) or cache.shape[2] % block:
        raise ValueError(f"the tokens of key bounds must be a power of two from 16 to 256 that divides a page; got {block}")
    if cache.dtype == _CODES or cache.shape[3] > 128 or cache.shape[3] * cache.element_size() % 16:
        raise ValueError("key bounds take a bf16, fp16 or fp32 cache with a head_dim up to 128 whose rows are multiples of 16 bytes")
    low = torch.zeros(cache.shape[0], cache.shape[1], cache.shape[2] // block, cache.shape[3], dtype=cache.dtype, device=cache.device)
    return low, torch.zeros_like(low)


def _check_selection(keep: int, recent: int, block: int) -> None:
    """The sizes that select_key_blocks takes, before anything is appended."""
    if keep % block or recent % block or not block <= recent <= keep:
        raise ValueError(f"decode: keep {keep} and recent {recent} must be multiples of the block of {block} tokens with block <= recent <= keep")


class KVCache:
    """Padded cache [B, Hkv, max_len, D] plus device lengths [B] (int32).

    dtype float8_e4m3fn: codes with fp32 scales [B, Hkv, max_len / block], max_len rounded up to whole blocks of
    ``block`` tokens (a power of two from 16 to 256).  track_weights: fp32 ``weights`` [B, Hkv, max_len], for evict().
    bounds_block: tokens of a block of key bounds (a power of two from 16 to 256; 0: none), for decode(keep=).
    """

    def __init__(self, batch: int, kv_heads: int, max_len: int, head_dim: int, dtype=torch.bfloat16,
                 device="cuda", scale: Optional[float] = None, block: int = 32, track_weights: bool = False,
                 bounds_block: int = 0):
        self.block = max(block, 1) if dtype == _CODES else 1  # tokens that share a scale, and that evict() keeps or drops together
        self.bounds_block = bounds_block
        max_len = -(-max_len // max(self.block, bounds_block)) * max(self.block, bounds_block)
        self.k = torch.zeros(batch, kv_heads, max_len, head_dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.k_scale, self.v_scale = _scales(self.k, self.block)
        if track_weights and (head_dim > 128 or head_dim * self.k.element_size() % 16):
            raise ValueError(f"track_weights takes a head_dim up to 128 whose rows are multiples of 16 bytes; got {head_dim}")
        self.weights = torch.zeros(batch, kv_heads, max_len, device=device) if track_weights else None
        self.k_min, self.k_max = _bounds(self.k, bounds_block)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.scale = scale
        self._host_len = np.zeros(batch, dtype=np.int64)  # mirrors `lengths` for capacity checks
        self._host_stale = False  # a step was recorded under graph capture: replays outrun _host_len

    @property
    def capacity(self) -> int:
        return self.k.shape[2]

    def _span(self) -> int:
        """Cache positions the decode kernel covers.  Its split grid is sized by S_max, so in eager use the
        cache is passed as a view up to the longest sequence rather than the whole capacity (one split per
        384 tokens of S_max, empty ones included: a 32K-token cache holding 2K-token sequences would launch
        16x the workgroups).  Under graph capture, and after it until sync_lengths(), the host does not
        know the lengths the replays reach, so the whole capacity is covered."""
        if torch.cuda.is_current_stream_capturing():
            self._host_stale = True
        if self._host_stale:
            return self.capacity
        unit = max(self.block, self.bounds_block)
        return -(-max(int(self._host_len.max(initial=0)), 1) // unit) * unit

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor) -> None:
        """Append [B, Hkv, n, D] keys and values after each sequence's current length."""
        n = k_new.shape[2]
        if int(self._host_len.max(initial=0)) + n > self.capacity:
            raise ValueError(f"KV cache full: {int(self._host_len.max())} + {n} tokens > capacity {self.capacity}")
        if self.k_scale is not None:
            F.kv_cache_append_fp8(self.k, self.v, self.k_scale, self.v_scale, self.lengths, k_new, v_new)
        else:
            F.kv_cache_append(self.k, self.v, self.lengths, k_new, v_new)
        self._host_len += n  # only once the append was accepted
        if self.k_min is not None:
            F.kv_key_bounds(self.k, self.k_min, self.k_max, self.lengths, n)

    def prefill(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        """Causal attention over a prompt of equal length per sequence (the cache must be empty for the
        causal alignment to hold), then the prompt's K/V into the cache."""
        if int(self._host_len.max(initial=0)) != 0:
            raise ValueError("prefill expects an empty cache; use decode() for later tokens")
        if self.weights is None:
            out = F.scaled_dot_product_attention(q, k, v, is_causal=True, scale=self.scale, enable_gqa=True)
            self.append(k, v)
            return out
        out, lse = F.scaled_dot_product_attention_with_lse(q, k, v, is_causal=True, scale=self.scale, enable_gqa=True)
        self.append(k, v)
        F.attention_weight_accumulate(self.weights[:, :, :k.shape[2]], q, k, lse, is_causal=True, scale=self.scale)
        return out

    def decode(self, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, prefix: Optional["KVCache"] = None,
               keep: int = 0, recent: int = 0) -> torch.Tensor:
        """One new token per sequence: append its K/V, then attend over everything cached.

        prefix: a cache of G sequences, each the prefix of B / G consecutive sequences of this one, which attend to it first
        (F.decode_attention_shared).  keep: attend to ``keep`` tokens only, the last ``recent`` (a block of bounds by default) and the
        blocks with the largest score bounds (F.select_key_blocks; multiples of ``bounds_block``)."""
        if keep and (self.k_min is None or self.weights is not None or prefix is not None):
            raise ValueError("decode(keep=) needs a cache with bounds_block, without track_weights and prefix")
        if prefix is not None and (self.weights is not None or self.k_scale is not None or prefix.k_scale is not None):
            raise ValueError("decode(prefix=) takes caches without codes and track_weights")
        if keep:
            _check_selection(keep, recent or self.bounds_block, self.bounds_block)
        if prefix is not None:
            p, own = prefix.k, self.k
            if own.shape[0] % p.shape[0] or (p.shape[1], p.shape[3], p.dtype, p.device) != (own.shape[1], own.shape[3], own.dtype, own.device):
                raise ValueError("decode(prefix=) takes a cache of the same kv heads, head_dim, dtype and device whose sequences divide this one's")
            if own.shape[3] > 128 or own.shape[3] * own.element_size() % 16:
                raise ValueError("decode(prefix=) takes a head_dim up to 128 whose rows are multiples of 16 bytes")
            if p.shape[0] > 1024:
                raise ValueError(f"decode(prefix=) takes up to 1024 prefixes; got {p.shape[0]}")
        self.append(k_new, v_new)
        n = self._span()
        k, v, ks = self.k[:, :, :n], self.v[:, :, :n], None
        if prefix is not None:
            m = prefix._span()
            return F.decode_attention_shared(q, prefix.k[:, :, :m], prefix.v[:, :, :m], prefix.lengths, k, v, self.lengths, scale=self.scale)[0]
        if keep:
            block = self.bounds_block
            blocks = F.select_key_blocks(q, self.k_min[:, :, :n // block], self.k_max[:, :, :n // block], self.lengths, keep,
                                         recent or block, block, scale=self.scale)
            return F.decode_attention_blocks(q, k, v, self.lengths, blocks, block, scale=self.scale)[0]
        if self.k_scale is not None:
            ks = self.k_scale[:, :, :n // self.block]
            out, lse = F.decode_attention_fp8(q, k, v, ks, self.v_scale[:, :, :n // self.block], self.lengths, scale=self.scale)
        else:
            out, lse = F.decode_attention(q, k, v, self.lengths, scale=self.scale)
        if self.weights is not None:
            F.attention_weight_accumulate(self.weights[:, :, :n], q, k, lse, lengths=self.lengths, scale=self.scale, key_scale=ks)
        return out

    def evict(self, keep: int, recent: int) -> torch.Tensor:
        """Shrink each sequence to ``keep`` tokens: its last ``recent`` and, kv head by kv head, those of the others
        that received the most attention (F.kv_cache_evict; both are multiples of ``block``).  The order of the
        tokens stays, and keys keep the positions they were rotated with.  Returns the kept block indices."""
        if self.weights is None:
            raise ValueError("evict needs a cache with track_weights=True")
        kept = F.kv_cache_evict(self.k, self.v, self.lengths, self.weights, keep, recent, block=self.block,
                                k_scale=self.k_scale, v_scale=self.v_scale)
        if torch.cuda.is_current_stream_capturing():
            self._host_stale = True
        blocks = -(-self._host_len // self.block)  # as the kernel shortens them
        self._host_len = np.where(blocks > keep // self.block, keep + self._host_len - blocks * self.block, self._host_len)
        if self.k_min is not None:  # tokens have moved
            F.kv_key_bounds(self.k, self.k_min, self.k_max, self.lengths, keep)  # what any sequence has at most
        return kept

    def sync_lengths(self) -> np.ndarray:
        """Refresh the host copy of the lengths from the device (one synchronising copy).

        A decode step captured in a HIP graph advances the host copy once, at capture; every replay
        advances only the device lengths.  Call this after replays and before eager use, so that the
        capacity check sees the true lengths.  The caller bounds the number of replays by
        capacity - current length: the append kernel drops tokens past the capacity (and the lengths
        saturate there), so later replays would attend over a truncated cache.  A caller that has shortened
        `lengths` itself calls it as well; it then clears the weights of the tokens that are gone.
        """
        self._host_len = self.lengths.to("cpu", torch.int64).numpy().copy()
        self._host_stale = False
        if self.weights is not None:
            gone = torch.arange(self.capacity, device=self.weights.device) >= self.lengths[:, None]
            self.weights.masked_fill_(gone[:, None], 0.0)
        return self._host_len.copy()


class PagedKVCache:
    """Paged cache: pools [num_pages, Hkv, page_size, D], a block table [B, max_pages] and lengths [B].

    Pages come from a host-side free list when a sequence's next tokens cross into a new page; the block
    table rows that change are copied to the device before the append that writes them.  dtype float8_e4m3fn:
    codes with fp32 scales [num_pages, Hkv, page_size / block], ``block`` tokens (at most a page) to a scale.
    bounds_block: tokens (at most a page) of a block of key bounds (0: none), for decode(keep=).

    From the first fork(), free() or compact() on, ``page_refs`` (int32 [num_pages], how many slots of the table name
    each page) is kept on the device, and pages are given out there by the same rule as here: the lowest free one first.  Call one
    of them before a step is captured, if sequences are to share pages later.
    """

    def __init__(self, batch: int, kv_heads: int, num_pages: int, page_size: int, max_pages: int, head_dim: int,
                 dtype=torch.bfloat16, device="cuda", scale: Optional[float] = None, block: int = 32, bounds_block: int = 0):
        self.k = torch.zeros(num_pages, kv_heads, page_size, head_dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.k_scale, self.v_scale = _scales(self.k, min(block, page_size))
        self.bounds_block = bounds_block
        self.k_min, self.k_max = _bounds(self.k, bounds_block)
        self.page_size = page_size
        self.scale = scale
        self._free = list(range(num_pages - 1, -1, -1))
        # unassigned slots hold -1, which names no page: the append kernel drops a token written through one
        # (a graph replay past a sequence's pages), and decode reads never reach past the length
        self._table = np.full((batch, max_pages), -1, dtype=np.int32)
        self._pages = np.zeros(batch, dtype=np.int64)  # pages assigned per sequence
        self._host_len = np.zeros(batch, dtype=np.int64)
        self.block_table = torch.from_numpy(self._table.copy()).to(device)
        self.lengths = torch.zeros(batch, dtype=torch.int32, device=device)
        self.page_refs: Optional[torch.Tensor] = None
        self._lacking: Optional[torch.Tensor] = None  # pages that steps lacked on the device since the last sync_lengths()
        self.prefix_lengths: Optional[torch.Tensor] = None  # of each group, where sequences share pages that are read once
        self._shares = {}  # the same for every number of groups so far: a captured step reads its own as long as it lives
        self._append_captured = False  # before page_refs were there: its replays write the pages that the table names
        self._fork_captured = False  # a captured fork updates the _shares that were there, and may be replayed at any time
        self._host_stale = False  # a step was recorded under graph capture, or its parents were on the device: _host_len is behind

    def _span_pages(self) -> int:
        """Block-table columns the decode kernel covers: the most pages any sequence holds in eager use
        (the split grid is sized by max_pages * page_size), the whole table under graph capture and after
        it until sync_lengths()."""
        if torch.cuda.is_current_stream_capturing():
            self._host_stale = True
        if self._host_stale:
            return self._table.shape[1]
        return max(int(self._pages.max(initial=0)), 1)

    def _pools(self):
        return [x for x in (self.k, self.v, self.k_scale, self.v_scale, self.k_min, self.k_max) if x is not None]

    def _refs(self) -> np.ndarray:
        """References of each page, by the host's table."""
        return np.bincount(self._table[self._table >= 0], minlength=self.k.shape[0]).astype(np.int32)

    def _set_free(self) -> None:
        self._free = np.flatnonzero(self._refs() == 0)[::-1].tolist()

    def _track_pages(self) -> None:
        if self.page_refs is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("PagedKVCache: call fork() or compact() once before they are captured")
            self.page_refs = torch.from_numpy(self._refs()).to(self.lengths.device)
            self._lacking = torch.zeros(1, dtype=torch.int32, device=self.lengths.device)

    def _reserve_shared(self, rows: int, n: int) -> None:
        """Pages for the next n tokens of the first sequences, on the device; the host's table follows by the same rule."""
        if torch.cuda.is_current_stream_capturing():
            self._host_stale = True
        table = None if self._host_stale else self._table.copy()
        if table is not None:
            refs, free, writers = self._refs(), list(self._free), {}
            for b, s in self._written(rows, n):
                page = int(self._table[b, s])
                if page >= 0:
                    writers[page] = writers.get(page, -1) + 1
                    if writers[page] >= refs[page] - 1:  # the last one keeps the page
                        continue
                if not free:
                    raise ValueError("PagedKVCache: out of pages")
                table[b, s] = free.pop()
        lacking = F.kv_pages_reserve(self._pools(), self.block_table[:rows], self.lengths[:rows], self.page_refs, n)
        if table is None:
            self._lacking += lacking
        else:
            self._table = table
            self._pages = (table >= 0).sum(1)
            self._set_free()

    def _written(self, rows: int, n: int):
        """(sequence, slot) pairs that the next n tokens of the first sequences lie in."""
        for b in range(rows):
            t = int(self._host_len[b])
            for s in range(t // self.page_size, (t + n - 1) // self.page_size + 1):
                yield b, s

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor) -> None:
        """Append [B, Hkv, n, D] keys and values after each sequence's current length; fewer than B: to the first sequences, and
        nothing to the others."""
        rows, n = k_new.shape[0], k_new.shape[2]
        if rows > len(self._host_len):
            raise ValueError(f"PagedKVCache: {rows} sequences in a cache of {len(self._host_len)}")
        stale = self._host_stale and self.page_refs is not None  # the device gives out the pages
        if stale and not torch.cuda.is_current_stream_capturing() and int(self._host_len[:rows].max(initial=0)) + n > self._table.shape[1] * self.page_size:
            self.sync_lengths()  # by what the host knows the tokens might not fit
            stale = False
        if not stale:
            need = (self._host_len[:rows] + n + self.page_size - 1) // self.page_size
            if int(need.max(initial=0)) > self._table.shape[1]:
                raise ValueError("PagedKVCache: a sequence exceeds max_pages * page_size tokens")
        if self.page_refs is not None:
            if n > 0:
                self._reserve_shared(rows, n)
        else:
            if int((need - self._pages[:rows]).sum()) > len(self._free):
                raise ValueError("PagedKVCache: out of pages")
            changed = False
            for b in range(rows):
                while self._pages[b] < need[b]:
                    self._table[b, self._pages[b]] = self._free.pop()
                    self._pages[b] += 1
                    changed = True
            if changed:
                self.block_table.copy_(torch.from_numpy(self._table), non_blocking=False)
            self._append_captured |= torch.cuda.is_current_stream_capturing()
        table, lengths = self.block_table[:rows], self.lengths[:rows]
        if self.k_scale is not None:
            F.kv_cache_append_fp8_paged(self.k, self.v, self.k_scale, self.v_scale, table, lengths, k_new, v_new)
        else:
            F.kv_cache_append_paged(self.k, self.v, table, lengths, k_new, v_new)
        self._host_len[:rows] += n  # only once the append was accepted
        if self.k_min is not None:
            F.kv_key_bounds_paged(self.k, self.k_min, self.k_max, table, lengths, n)

    def prefill(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        """Causal attention over a prompt of equal length per sequence, then its K/V into the (empty) cache; fewer prompts
        than sequences go to the first ones."""
        if int(self._host_len[:k.shape[0]].max(initial=0)) != 0:
            raise ValueError("prefill expects an empty cache; use decode() for later tokens")
        out = F.scaled_dot_product_attention(q, k, v, is_causal=True, scale=self.scale, enable_gqa=True)
        self.append(k, v)
        return out

    def decode(self, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, keep: int = 0, recent: int = 0) -> torch.Tensor:
        """One new token per sequence: append its K/V, then attend over everything cached, or, with ``keep``, to ``keep`` tokens
        only: the last ``recent`` (a block of bounds by default) and the blocks with the largest score bounds
        (F.select_key_blocks_paged; multiples of ``bounds_block``)."""
        if keep and self.k_min is None:
            raise ValueError("decode(keep=) needs a cache with bounds_block")
        if keep:
            _check_selection(keep, recent or self.bounds_block, self.bounds_block)
        if k_new.shape[0] != len(self._host_len):
            raise ValueError(f"PagedKVCache: decode takes a token for each of the {len(self._host_len)} sequences; got {k_new.shape[0]}")
        self.append(k_new, v_new)
        table = self.block_table[:, :self._span_pages()]
        if self.k_scale is not None:
            return F.decode_attention_fp8_paged(q, self.k, self.v, self.k_scale, self.v_scale, table, self.lengths, scale=self.scale)[0]
        if keep:
            block = self.bounds_block
            blocks = F.select_key_blocks_paged(q, self.k_min, self.k_max, table, self.lengths, keep, recent or block, block, scale=self.scale)
            return F.decode_attention_blocks_paged(q, self.k, self.v, table, self.lengths, blocks, block, scale=self.scale)[0]
        if self.prefix_lengths is not None:
            return F.decode_attention_shared_paged(q, self.k, self.v, table, self.lengths, self.prefix_lengths, scale=self.scale)[0]
        return F.decode_attention_paged(q, self.k, self.v, table, self.lengths, scale=self.scale)[0]

    def fork(self, parents) -> None:
        """Sequence b continues what sequence parents[b] is, on the same pages (F.kv_pages_fork); a parent outside the batch, such
        as -1, frees the sequence.  parents: B whole numbers on the host, or an int32 tensor [B] on the device.  The latter does not
        wait for the device (and may be captured): the host's lengths are then behind until sync_lengths() (which an eager step calls
        by itself where its token might not fit), and a group that has a parent from another one, or a sequence without parent,
        shares nothing until the next share().  A captured fork does so for the
        numbers of groups that share() has had before the capture; others are refused from then on.  A step captured before the first
        fork() or compact() does not copy what it writes, so that sequences cannot share pages behind it.  A cache that runs out of pages
        meanwhile drops tokens, which sync_lengths() reports; until then what the sequences without pages attend to says nothing."""
        batch = len(self._host_len)
        on_device = isinstance(parents, torch.Tensor) and parents.is_cuda
        if not on_device:
            parents = np.asarray(parents, dtype=np.int64).reshape(-1)
        if len(parents) != batch:
            raise ValueError(f"fork takes a parent for each of the {batch} sequences; got {len(parents)}")
        if not on_device and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("PagedKVCache: a captured fork takes its parents on the device")
        if self._append_captured:
            living = None if on_device else parents[(parents >= 0) & (parents < batch)]
            if living is None or len(np.unique(living)) < len(living):
                raise RuntimeError("PagedKVCache: a step was captured before the first fork() or compact(), and its replays would write pages that "
                                   "sequences share; call compact() once before the capture")
        if not on_device and self._host_stale:
            parents = torch.from_numpy(parents.clip(-1, batch).astype(np.int32)).to(self.lengths.device)
            on_device = True
        self._track_pages()
        if on_device:
            F.kv_pages_fork(self.block_table, self.lengths, self.page_refs, parents)
            self._host_stale = True
            self._host_len[:] = self._host_len.max(initial=0)  # no sequence is longer, until sync_lengths()
            self._fork_captured |= torch.cuda.is_current_stream_capturing()
            for groups, shared in self._shares.items():  # a group with a parent from elsewhere, or none, has nothing in common
                per = batch // groups
                home = torch.arange(batch, dtype=torch.int64, device=parents.device) // per
                stays = torch.where(parents.div(per, rounding_mode="floor") == home, 0x7fffffff, 0).to(torch.int32)
                shared.scatter_reduce_(0, home, stays, "amin")
            return
        lives = (parents >= 0) & (parents < batch)
        source = np.where(lives, parents, 0)
        F.kv_pages_fork(self.block_table, self.lengths, self.page_refs,
                        torch.from_numpy(np.where(lives, parents, -1).astype(np.int32)).to(self.lengths.device))
        self._table = np.where(lives[:, None], self._table[source], -1).astype(np.int32)
        self._pages = np.where(lives, self._pages[source], 0)
        self._host_len = np.where(lives, self._host_len[source], 0)
        self._set_free()
        for groups in self._shares:
            self._set_shared(groups)

    def free(self, sequences) -> None:
        """Free sequences (their indices): length 0, and pages that no other one names are free again.  decode() appends to every row, so a
        freed one takes a page again at the next step, and ends what its group shares; the row of a sequence that has ended can
        follow a living one instead (fork() with a sibling as its parent).  prefill() fills the first rows: a prompt for a
        freed row elsewhere needs a fork() that brings that row to the front."""
        parents = np.arange(len(self._host_len))
        sequences = np.asarray(sequences, dtype=np.int64).reshape(-1)
        if np.any((sequences < 0) | (sequences >= len(parents))):
            raise ValueError(f"free takes sequences from 0 to {len(parents) - 1}; got {sequences.tolist()}")
        parents[sequences] = -1
        self.fork(parents)

    def share(self, groups: int) -> None:
        """Read the pages that the sequences of a group have in common once per step: ``groups`` equal groups of consecutive
        sequences (0: no longer).  Takes effect for the pages they share now, and stays right as sequences grow; a group with
        an empty sequence shares nothing, nor once that sequence grows again.  Call it once with each number of groups that will
        be wanted before a fork is captured: the fork's replays keep those right and know no others, which are refused."""
        if groups == 0:
            self.prefix_lengths = None
            return
        if groups < 0 or len(self._host_len) % groups:
            raise ValueError(f"{len(self._host_len)} sequences are not {groups} equal groups")
        if groups > 1024:
            raise ValueError(f"share takes up to 1024 groups; got {groups}")
        if self.k_scale is not None or self.k.shape[3] > 128 or self.k.shape[3] * self.k.element_size() % 16:
            raise ValueError("share takes a bf16, fp16 or fp32 cache with a head_dim up to 128 whose rows are multiples of 16 bytes")
        if self._host_stale:
            raise RuntimeError("PagedKVCache: call sync_lengths() before share()")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("PagedKVCache: share() cannot be captured")
        if groups not in self._shares:
            if self._fork_captured:
                raise RuntimeError(f"PagedKVCache: a fork was captured before the first share({groups}), and its replays would not keep the "
                                   f"prefixes right; call share({groups}) once before the capture")
            self._shares[groups] = torch.zeros(groups, dtype=torch.int32, device=self.lengths.device)
        self._set_shared(groups)
        self.prefix_lengths = self._shares[groups]

    def _set_shared(self, groups: int, most=None) -> None:
        """The tokens on pages that all of a group have; no more than ``most``, where that is given for each group."""
        common = []
        for table, lengths in zip(np.split(self._table, groups), np.split(self._host_len, groups)):
            whole = int(lengths.min()) // self.page_size
            same = (table[:, :whole] == table[:1, :whole]).all(0)
            common.append((int(same.argmin()) if not same.all() else whole) * self.page_size)
        if most is not None:
            common = np.minimum(common, most).tolist()
        self._shares[groups].copy_(torch.tensor(common, dtype=torch.int32))

    def compact(self) -> torch.Tensor:
        """Move the pages in use to the front of the pools (F.kv_pages_compact).  Returns their number, int32 [1] on the device."""
        self._track_pages()
        if torch.cuda.is_current_stream_capturing():
            self._host_stale = True
        used = F.kv_pages_compact(self._pools(), self.block_table, self.page_refs)
        if not self._host_stale:
            live = self._refs() > 0
            n = int(live.sum())
            to = np.arange(len(live), dtype=np.int32)
            to[n:][live[n:]] = np.flatnonzero(~live[:n])
            self._table = np.where(self._table >= 0, to[np.maximum(self._table, 0)], self._table)
            self._set_free()
        return used

    def sync_lengths(self) -> np.ndarray:
        """Refresh the host copy of the lengths from the device after HIP-graph replays (and, once pages are shared, the table
        too; what share() reads once comes down to what the groups still have in common).

        Without shared pages replays assign none: the block-table slots past a sequence's assigned pages hold -1, so the
        caller bounds the replays by the tokens left on the pages already assigned.  Raises if a replay
        went past them, or found no free page: those tokens were dropped (no page was written) and the sequence's cache is
        incomplete.  Raises until such sequences are freed, and once if they have ended meanwhile.
        """
        self._host_stale = True  # unless all is found well
        dev = self.lengths.to("cpu", torch.int64).numpy().copy()
        if self.page_refs is not None:
            self._table = self.block_table.to("cpu").numpy().copy()
            self._pages = np.where((self._table < 0).any(1), (self._table < 0).argmax(1), self._table.shape[1])
            self._set_free()
            lacking = self._lacking.item()
            self._lacking.zero_()
            if lacking:
                raise RuntimeError(f"PagedKVCache: steps appended past the assigned pages: {lacking} times a sequence found no page, and dropped tokens")
        if np.any(dev > self._pages * self.page_size):
            raise RuntimeError("PagedKVCache: graph replays appended past the assigned pages")
        self._host_len = dev
        self._host_stale = False
        for groups, shared in self._shares.items():
            self._set_shared(groups, most=shared.tolist())
        return dev.copy()
