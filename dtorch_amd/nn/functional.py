"""Python front end of the MI355X attention path.

Mirrors ``dtorch.nn.functional.scaled_dot_product_attention`` and ``SdpaOption``
(python/dtorch/nn/functional.py:169-238) on local torch device tensors: same signature, same
defaults, same validation; the call lands in the C++ ``SdpaOp`` host operator, whose ``Compute``
launches the gfx950 kernels through the dtattn C ABI on the current HIP stream.

New entry points (no reference counterpart, see the host operators):
``scaled_dot_product_attention_with_lse``, ``decode_attention``, ``lse_merge``,
``ring_attention_step`` and ``quantize_fp8_per_head``; over an 8-bit KV cache ``kv_cache_append_fp8`` and
``decode_attention_fp8`` (and their paged forms); to bound a cache ``attention_weight_accumulate`` and
``kv_cache_evict``; over pages that sequences share ``kv_pages_fork``, ``kv_pages_reserve`` and ``kv_pages_compact``;
over a prefix that sequences share ``decode_attention_shared`` (and ``_paged``); to read a long cache in part
``kv_key_bounds``, ``select_key_blocks`` and ``decode_attention_blocks`` (and their paged forms).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple, Union

import torch

from .._lib import load

_h = load()

_SAGE_TYPES = ("auto", "qk_int8_pv_fp8", "qk_int8_pv_fp16")


@dataclass
class SdpaOption:
    """Per-call attention options (python/dtorch/nn/functional.py:169-188).

    ``sage_attn_type`` keeps the reference's candidates ("", "auto", "qk_int8_pv_fp8",
    "qk_int8_pv_fp16") and adds ``"native_fp8"``: per-head absmax e4m3fn quantization of q/k/v and
    fp8 MFMA for both products, bf16 output.
    """

    # cp
    ulysess_cp_dim: Optional[Union[int, str]] = "ulysess_cp"
    ring_cp_dim: Optional[Union[int, str]] = "ring_cp"

    # candidate: "", "auto", "qk_int8_pv_fp8", "qk_int8_pv_fp16", "native_fp8"
    sage_attn_type: Optional[str] = None

    def check_valid(self):
        return self.sage_attn_type in (None, "", "native_fp8") + _SAGE_TYPES


def _param(is_causal: bool, scale: Optional[float], enable_gqa: bool, sdpa_option: SdpaOption):
    return _h.SdpaParam(bool(is_causal), None if scale is None else float(scale), bool(enable_gqa),
                        _h.SdpaOption(sdpa_option.sage_attn_type or ""))


def _check_option(query, sdpa_option: SdpaOption):
    assert sdpa_option.check_valid(), f"sdpa_option invalid: {sdpa_option}"
    if sdpa_option.sage_attn_type in _SAGE_TYPES:
        # python/dtorch/nn/functional.py:216-220
        try:
            import sageattention  # noqa: F401
        except ImportError:
            raise RuntimeError("Require sageattention, please install sageattention.")
    mesh = getattr(query, "device_mesh", None)
    if (isinstance(sdpa_option.ulysess_cp_dim, int) or isinstance(sdpa_option.ring_cp_dim, int) or
            (mesh is not None and (mesh.has_dim_name(sdpa_option.ulysess_cp_dim or "") or
                                   mesh.has_dim_name(sdpa_option.ring_cp_dim or "")))):
        raise NotImplementedError(
            "context parallelism across devices is not part of this single-GPU build; "
            "ring_attention_step() computes one device's share")


def scaled_dot_product_attention(
    query: torch.Tensor,  # N, Hq, L, E
    key: torch.Tensor,  # N, H, S, E
    value: torch.Tensor,  # N, H, S, E
    attn_mask=None,
    dropout_p: float = 0.0,
    is_causal: bool = False,
    scale: Optional[float] = None,
    enable_gqa=False,
    sdpa_option: SdpaOption = SdpaOption(),
) -> torch.Tensor:
    """O = softmax(scale Q K^T [causal, top-left]) V on the gfx950 kernels.

    ``dropout_p`` is accepted and ignored, as in the reference (neural_network.cc:147-154 drops it and
    SdpaOp::Compute passes 0.0).  ``attn_mask`` follows torch: broadcastable to [..., Hq, L, S], boolean
    (True keeps a key) or floating point (added to the scaled logits), applied together with ``is_causal``;
    not supported with ``native_fp8``.
    """
    _check_option(query, sdpa_option)
    op = _h.SdpaOp(_param(is_causal, scale, enable_gqa, sdpa_option))
    return op.compute([query, key, value, attn_mask])[0]


def scaled_dot_product_attention_with_lse(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    is_causal: bool = False,
    scale: Optional[float] = None,
    enable_gqa: bool = False,
    q_offset: int = 0,
    k_offset: int = 0,
    sdpa_option: SdpaOption = SdpaOption(),
    attn_mask: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """(O, LSE[..., Hq, L] fp32).  Causal rule: key j visible to query i iff j + k_offset <= i + q_offset.
    ``attn_mask`` as in scaled_dot_product_attention, applied together with the causal rule."""
    _check_option(query, sdpa_option)
    op = _h.SdpaWithLseOp(_param(is_causal, scale, enable_gqa, sdpa_option), int(q_offset), int(k_offset))
    o, lse = op.compute([query, key, value, attn_mask])
    return o, lse


def decode_attention(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor,
                     scale: Optional[float] = None, chunk: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """Single-token attention per sequence over k_cache[b, :, :lengths[b]] (split-KV + LSE merge).

    query [B, Hq, 1, D]; caches [B, Hkv, S_max, D]; lengths int32 [B] on the device.
    Returns (O [B, Hq, 1, D], LSE [B, Hq] fp32).
    """
    op = _h.SdpaDecodeOp(None if scale is None else float(scale), int(chunk))
    o, lse = op.compute([query, k_cache, v_cache, lengths])
    return o, lse


def decode_attention_paged(query: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                           block_table: torch.Tensor, lengths: torch.Tensor, scale: Optional[float] = None,
                           chunk: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """decode_attention over a paged KV cache.

    query [B, Hq, 1, D]; k_pages / v_pages are page pools viewed as [num_pages, Hkv, page_size, D]
    (any strides with unit stride on D, so a [num_pages, page_size, Hkv, D] pool passed through
    .permute(0, 2, 1, 3) works without a copy); block_table int32 [B, max_pages] holds the page of
    each sequence's p-th block; lengths int32 [B].  page_size is a power of two >= 16.
    Returns (O [B, Hq, 1, D], LSE [B, Hq] fp32).
    """
    op = _h.SdpaDecodePagedOp(None if scale is None else float(scale), int(chunk))
    o, lse = op.compute([query, k_pages, v_pages, block_table, lengths])
    return o, lse


def kv_cache_append(k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor, k_new: torch.Tensor,
                    v_new: torch.Tensor) -> None:
    """Write n_new tokens per sequence into a [B, Hkv, S_max, D] cache, in place.

    k_new / v_new are [B, Hkv, n_new, D] (any strides with unit stride on D, e.g. a transposed projection
    output).  Token j of sequence b lands at position lengths[b] + j; positions at or past S_max are not
    written.  lengths (contiguous int32 [B]) then advances by n_new, saturating at S_max.
    """
    _h.KvCacheAppendOp().compute([k_cache, v_cache, lengths, k_new, v_new])


def kv_cache_append_paged(k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                          lengths: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor) -> None:
    """kv_cache_append for the paged cache of decode_attention_paged; the block table must already name
    the pages of the positions being written."""
    _h.KvCacheAppendPagedOp().compute([k_pages, v_pages, block_table, lengths, k_new, v_new])


def kv_cache_append_fp8(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                        lengths: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor) -> None:
    """kv_cache_append into an 8-bit cache, in place: e4m3fn codes with one scale per block of tokens and kv head.

    k_cache / v_cache float8_e4m3fn [B, Hkv, S_max, D]; k_scale / v_scale fp32 [B, Hkv, S_max / block] (the block,
    a power of two from 16 to 256, follows from the shapes); k_new / v_new bf16, fp16 or fp32 [B, Hkv, n_new, D].
    A value is code * scale.  A block's scale is the smallest power of two that holds its largest value within
    +-448 (and at least 2^-126, which is that of a block of zeros); a block that outgrows its scale re-encodes its older
    tokens (exact, subnormal codes apart).  NaN and infinite inputs become NaN codes; they and zeros leave the scale to
    the others, whichever come first.
    """
    _h.KvCacheAppendFp8Op().compute([k_cache, v_cache, k_scale, v_scale, lengths, k_new, v_new])


def kv_cache_append_fp8_paged(k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                              block_table: torch.Tensor, lengths: torch.Tensor, k_new: torch.Tensor,
                              v_new: torch.Tensor) -> None:
    """kv_cache_append_fp8 into a paged cache: pools float8_e4m3fn [num_pages, Hkv, page_size, D], scales fp32
    [num_pages, Hkv, page_size / block]; block table and dropped tokens as for kv_cache_append_paged."""
    _h.KvCacheAppendFp8PagedOp().compute([k_pages, v_pages, k_scale, v_scale, block_table, lengths, k_new, v_new])


def decode_attention_fp8(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                         v_scale: torch.Tensor, lengths: torch.Tensor,
                         scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """decode_attention over an 8-bit cache (kv_cache_append_fp8), any positive scales.

    query bf16, fp16 or fp32 [B, Hq, 1, D], D a multiple of 16 up to 128.  Returns (O [B, Hq, 1, D] in the query's
    type, LSE [B, Hq] fp32).
    """
    o, lse = _h.SdpaDecodeFp8Op(None if scale is None else float(scale)).compute(
        [query, k_cache, v_cache, k_scale, v_scale, lengths])
    return o, lse


def decode_attention_fp8_paged(query: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                               k_scale: torch.Tensor, v_scale: torch.Tensor, block_table: torch.Tensor,
                               lengths: torch.Tensor,
                               scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """decode_attention_fp8 over a paged 8-bit cache (kv_cache_append_fp8_paged)."""
    o, lse = _h.SdpaDecodeFp8PagedOp(None if scale is None else float(scale)).compute(
        [query, k_pages, v_pages, k_scale, v_scale, block_table, lengths])
    return o, lse


def attention_weight_accumulate(weights: torch.Tensor, query: torch.Tensor, key: torch.Tensor, lse: torch.Tensor,
                                lengths: Optional[torch.Tensor] = None, is_causal: bool = False, q_offset: int = 0,
                                scale: Optional[float] = None,
                                key_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Add the attention weight that each key has received to ``weights`` (fp32 [B, Hkv, S]), in place.

    weights[b, hk, j] += sum over the query heads of hk and the queries i that see key j of
    exp(scale q_i . k_j - lse_i).  query [B, Hq, L, D] with the LSE [B, Hq, L] of its attention over the same keys (for
    one query also [B, Hq], as decode_attention returns it); key [B, Hkv, S, D] of the query's dtype, or float8_e4m3fn
    codes with key_scale [B, Hkv, S / block].  Key j is visible to query i iff j < lengths[b] (S without lengths) and,
    when causal, j <= i + q_offset; with causal and lengths, queries at or past lengths[b] are padding and add nothing.
    Weights at or past lengths[b] are left as they are.  Returns ``weights``.
    """
    param = _h.AttentionWeightsParam(None if scale is None else float(scale), bool(is_causal), int(q_offset))
    return _h.AttentionWeightsOp(param).compute([weights, query, key, lse, lengths, key_scale])[0]


def kv_cache_evict(k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor, weights: torch.Tensor,
                   keep: int, recent: int, block: Optional[int] = None, k_scale: Optional[torch.Tensor] = None,
                   v_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Shrink each sequence of a padded cache to ``keep`` tokens by accumulated attention weight, in place.

    Every kv head keeps its last ``recent`` tokens and, of the others, those with the largest ``weights`` (fp32
    [B, Hkv, S_max], as attention_weight_accumulate sums them; of equal ones the first), in units of ``block`` tokens:
    1 by default, the tokens of a scale for an 8-bit cache with k_scale and v_scale.  What stays moves to the front in
    its order, its weights and scales with it; weights behind are zeroed and ``lengths`` shrinks.  A sequence of no
    more than keep / block blocks is left alone.  ``keep`` and ``recent`` are multiples of ``block``.  Returns the
    indices of the blocks that stayed, int32 [B, Hkv, keep / block], -1 past them.
    """
    param = _h.KvCacheEvictParam(int(keep), int(recent), 0 if block is None else int(block))
    return _h.KvCacheEvictOp(param).compute([k_cache, v_cache, lengths, weights, k_scale, v_scale])[0]


def kv_pages_fork(block_table: torch.Tensor, lengths: torch.Tensor, page_refs: torch.Tensor, parents: torch.Tensor) -> None:
    """Sequences of a paged cache continue their parents, in place and without copying a page.

    block_table int32 [B, max_pages] (slots outside the pool, such as -1, are empty), lengths int32 [B], page_refs int32
    [num_pages] (how many slots name each page), parents int32 [B], all on the device.  Row b and lengths[b] become what row
    parents[b] and its length were; a parent outside [0, B) frees the sequence.  B up to 8192.
    """
    _h.KvPagesForkOp().compute([block_table, lengths, page_refs, parents])


def kv_pages_reserve(pools: Sequence[torch.Tensor], block_table: torch.Tensor, lengths: torch.Tensor, page_refs: torch.Tensor,
                     n_new: int) -> torch.Tensor:
    """Pages of their own for the next ``n_new`` tokens of every sequence (copy on write), in place.

    pools: keys [num_pages, Hkv, page_size, D] first, then values, scales [num_pages, Hkv, page_size / block] or key bounds
    [num_pages, Hkv, page_size / block, D]; up to 8.  Empty slots take free pages (page_refs 0), the lowest first, sequence by
    sequence; a sequence whose next token falls into a page that others share takes a copy of its rows (of sequences that
    all write a page the last one keeps it).  Returns int32 [1] on the device: the pages that were lacking (0: none); slots
    that got none hold -1, and what was cached in them is lost to the sequence: they count as lacking in later calls too, until
    the sequence has gone on to its next page or has been freed.  lengths stay as they are.
    """
    return _h.KvPagesReserveOp(_h.TokenCountParam(int(n_new))).compute([block_table, lengths, page_refs, *pools])[0]


def kv_pages_compact(pools: Sequence[torch.Tensor], block_table: torch.Tensor, page_refs: torch.Tensor) -> torch.Tensor:
    """Move the pages in use to the front of the pool, in place.

    With U pages in use (page_refs > 0), those at or above index U move to the free ones below it, lowest to lowest, in
    every pool, with their counts; the table follows.  pools as for kv_pages_reserve.  Returns U, int32 [1] on the device.
    """
    return _h.KvPagesCompactOp().compute([block_table, page_refs, *pools])[0]


def decode_attention_shared(query: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor, prefix_lengths: torch.Tensor,
                            k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor,
                            scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """decode_attention of sequences behind a prefix that they share, which is read once for all of them.

    query [B, Hq, 1, D]; k_prefix / v_prefix [G, Hkv, S, D] with int32 prefix_lengths [G]: prefix g belongs to the B / G
    sequences from g * B / G on; k_cache / v_cache [B, Hkv, S_max, D] with int32 lengths [B]: each sequence's tokens behind it.
    bf16, fp16 or fp32, D up to 128.  Returns (O [B, Hq, 1, D], LSE [B, Hq] fp32).
    """
    op = _h.SdpaDecodeSharedOp(_h.SdpaDecodeSharedParam(None if scale is None else float(scale)))
    return tuple(op.compute([query, k_prefix, v_prefix, prefix_lengths, k_cache, v_cache, lengths]))


def decode_attention_shared_paged(query: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                                  lengths: torch.Tensor, prefix_lengths: torch.Tensor,
                                  scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """decode_attention_paged of sequences whose first pages are the same, which are read once for all of them.

    Arguments as for decode_attention_paged, and int32 prefix_lengths [G]: the first prefix_lengths[g] tokens (rounded down to whole
    pages) of the B / G sequences from g * B / G on lie in the same pages.  lengths count all tokens; sequences of length 0
    take no part.  Where a sequence is shorter than its group's prefix, the group shares no more than that sequence's whole pages.
    """
    op = _h.SdpaDecodeSharedPagedOp(_h.SdpaDecodeSharedParam(None if scale is None else float(scale)))
    return tuple(op.compute([query, k_pages, v_pages, block_table, lengths, prefix_lengths]))


def kv_key_bounds(k_cache: torch.Tensor, k_min: torch.Tensor, k_max: torch.Tensor, lengths: torch.Tensor, n_new: int) -> None:
    """Refresh the key bounds of the blocks that hold the last ``n_new`` tokens of each sequence, in place.

    k_cache [B, Hkv, S_max, D]; k_min / k_max [B, Hkv, S_max / block, D] of its dtype (the block, a power of two from 16 to 256,
    follows from the shapes): the smallest and the largest value of each dimension over a block's tokens, NaN passed over.
    Call it after the append of n_new tokens.
    """
    _h.KeyBoundsOp(_h.TokenCountParam(int(n_new))).compute([k_cache, k_min, k_max, lengths, None])


def kv_key_bounds_paged(k_pages: torch.Tensor, k_min: torch.Tensor, k_max: torch.Tensor, block_table: torch.Tensor,
                        lengths: torch.Tensor, n_new: int) -> None:
    """kv_key_bounds of a paged cache: bounds [num_pages, Hkv, page_size / block, D]."""
    _h.KeyBoundsOp(_h.TokenCountParam(int(n_new))).compute([k_pages, k_min, k_max, lengths, block_table])


def select_key_blocks(query: torch.Tensor, k_min: torch.Tensor, k_max: torch.Tensor, lengths: torch.Tensor, keep: int, recent: int,
                      block: int, scale: Optional[float] = None) -> torch.Tensor:
    """The blocks of a cache whose keys can score highest for a single-token query, by their key bounds (kv_key_bounds).

    For every kv head the last ``recent`` tokens' blocks and the best of the others, ``keep`` tokens in all (both multiples
    of ``block``): int32 [B, Hkv, keep / block], ascending, -1 behind the blocks of a shorter sequence.  A block's score is the
    largest over the kv head's query heads of the bound sum_d max(q_d k_min_d, q_d k_max_d), of equal ones the first
    counts.  Only the sign of ``scale`` matters.
    """
    param = _h.SelectKeyBlocksParam(int(keep), int(recent), int(block), None if scale is None else float(scale))
    return _h.SelectKeyBlocksOp(param).compute([query, k_min, k_max, lengths, None])[0]


def select_key_blocks_paged(query: torch.Tensor, k_min: torch.Tensor, k_max: torch.Tensor, block_table: torch.Tensor,
                            lengths: torch.Tensor, keep: int, recent: int, block: int,
                            scale: Optional[float] = None) -> torch.Tensor:
    """select_key_blocks of a paged cache (kv_key_bounds_paged)."""
    param = _h.SelectKeyBlocksParam(int(keep), int(recent), int(block), None if scale is None else float(scale))
    return _h.SelectKeyBlocksOp(param).compute([query, k_min, k_max, lengths, block_table])[0]


def decode_attention_blocks(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor,
                            blocks: torch.Tensor, block: int, scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """decode_attention over listed blocks of tokens only.

    blocks int32 [B, Hkv, n]: kv head hk of sequence b attends to tokens blocks[b, hk, i] * block + (0 .. block - 1) before
    lengths[b]; an index outside the sequence's blocks (-1) stands for none.  ``block`` is a power of two from 16 to 256.
    bf16, fp16 or fp32, D up to 128.  Returns (O [B, Hq, 1, D], LSE [B, Hq] fp32) over those tokens.
    """
    op = _h.SdpaDecodeBlocksOp(_h.SdpaDecodeBlocksParam(int(block), None if scale is None else float(scale)))
    return tuple(op.compute([query, k_cache, v_cache, lengths, blocks, None]))


def decode_attention_blocks_paged(query: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                                  lengths: torch.Tensor, blocks: torch.Tensor, block: int,
                                  scale: Optional[float] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """decode_attention_blocks over a paged cache whose pages hold whole blocks."""
    op = _h.SdpaDecodeBlocksOp(_h.SdpaDecodeBlocksParam(int(block), None if scale is None else float(scale)))
    return tuple(op.compute([query, k_pages, v_pages, lengths, blocks, block_table]))


def lse_merge(outs: Sequence[torch.Tensor], lses: Sequence[torch.Tensor],
              out_dtype: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Merge partial attention blocks over the same queries by their LSE."""
    if len(outs) != len(lses) or not outs:
        raise ValueError("lse_merge needs matching, non-empty lists of outputs and LSEs")
    ins: List[Optional[torch.Tensor]] = []
    for o, l in zip(outs, lses):
        ins += [o, l]
    return tuple(_h.LseMergeOp(out_dtype).compute(ins))


def ring_attention_step(query: torch.Tensor, k_chunks: Sequence[torch.Tensor], v_chunks: Sequence[torch.Tensor],
                        q_chunk_index: int, scale: Optional[float] = None, enable_gqa: bool = True,
                        return_blocks: bool = False):
    """One device's share of causal ring attention over equal-length sequence chunks.

    The Q chunk has global chunk index ``q_chunk_index``; KV chunk c is visible in full when
    c < q_chunk_index, causally (diagonal, offsets equal) when c == q_chunk_index, and not at all
    after.  Each visible block yields (O_c, LSE_c) with global offsets; the blocks are then merged by
    LSE.  This is the per-step arithmetic a true ring needs (the reference all-gathers K/V instead:
    python/dtorch/nn/scaled_dot_product_attention_with_cp.py:87-101).
    """
    L = query.shape[-2]
    blocks = []
    for c in range(min(q_chunk_index + 1, len(k_chunks))):
        diag = c == q_chunk_index
        o, lse = scaled_dot_product_attention_with_lse(
            query, k_chunks[c], v_chunks[c], is_causal=diag, scale=scale, enable_gqa=enable_gqa,
            q_offset=q_chunk_index * L, k_offset=c * k_chunks[c].shape[-2])
        blocks.append((o, lse))
    o, lse = lse_merge([b[0] for b in blocks], [b[1] for b in blocks])
    if return_blocks:
        return o, lse, blocks
    return o, lse


def quantize_fp8_per_head(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-head absmax e4m3fn quantization: (codes float8_e4m3fn [..., H, S, D], descale fp32 [..., H])."""
    codes, desc = _h.Fp8QuantizeOp().compute([x])
    return codes, desc


def device_peaks(device: int = 0):
    """MI355X peak table (CU count x clock x CDNA4 per-CU MFMA rate; HBM 8 TB/s)."""
    return _h.get_device_peaks(device)
