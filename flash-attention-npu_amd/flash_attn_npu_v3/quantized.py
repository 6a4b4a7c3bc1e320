"""Serving over a paged cache of 8-bit or 4-bit keys and values.

A serving step calls these three in turn: update_page_table gives the pages of
requests that ended to requests that grow and every new token its slot,
append_quantized_kvcache quantises the new k / v rows into their slots, and
flash_attn_with_quantized_kvcache attends to the cache. The reference has no
counterpart (its caches hold the type of q).

The cache: k_cache and v_cache are (num_pages, page_size, nheads_k, headdim),
torch.int8 or torch.float8_e4m3fn; k_scale and v_scale are fp32 (num_pages,
page_size // block, nheads_k). A scale holds for `block` tokens of a page and
one head: a stored code c stands for c * scale. block is a multiple of 16,
headdim one of 16 up to 256. A contiguous cache is (batch_size, seqlen_cache,
nheads_k, headdim) with scales (batch_size, seqlen_cache // block, nheads_k), and
no page table: slot b * seqlen_cache + j is row j of sequence b.

A 4-bit cache holds half the bytes (OCP Microscaling, MXFP4): k_cache and v_cache are (num_pages, page_size,
nheads_k, headdim // 2) of torch.float4_e2m1fn_x2 or of its bytes, torch.uint8 (the even channel in the
lower half); k_scale and v_scale are (num_pages, page_size, nheads_k, headdim // 32)
of torch.float8_e8m0fnu or its bytes, uint8: 32 channels of a token and head share one. A code (0, 0.5, 1, 1.5, 2, 3, 4
or 6, and their negatives) under the scale s stands for code * s. headdim is a multiple of 32 up to 256, page_size
one of 16. All the calls below take it in place of an 8-bit one.

read_quantized_kvcache gives rows of either cache back in 16 or 32 bits.
"""
from typing import Optional

import torch

from fa_mi355x import ops

from .interface import maybe_contiguous

_update_page_table, _append, _fwd, _read = (op.default for op in (ops.update_page_table, ops.quant_append, ops.quant_fwd,
                                                                  ops.quant_read))


def update_page_table(page_table, cache_seqlens, new_seqlens, free_pages, num_free, page_size, total_new,
                      cache_batch_idx: Optional[torch.Tensor] = None):
    """Bring the page table from one step's request lengths to the next, on the GPU.

    page_table (rows, max_pages) int32, written in place: the page of token j
    of request b is page_table[b, j // page_size], or with cache_batch_idx
    page_table[cache_batch_idx[b], j // page_size] (the rows of a step differ; a row outside the
    table has no pages). cache_seqlens and new_seqlens (batch_size,) int32: the
    tokens of each request before and after the step; a request grows by its new tokens,
    shrinks by those taken back, and ends with 0. free_pages (capacity,) int32,
    written in place, is a stack of the ids of free pages, num_free (1,) int32
    how many it holds; capacity for every page there is always suffices.

    Pages that are no longer needed go onto the stack first, then needed ones
    come off it, both in the order of the requests. Where the stack runs empty
    the table gets -1, and keeps it until the request shrinks below that page or ends: later steps
    count the page as held, and its tokens have no slots. Returns (slot_mapping, cu_seqlens_new, num_free_out):

      slot_mapping (total_new,) int64: the slots, page * page_size + row, of the
        new tokens of all requests in turn; -1 for a token without a page
        (stack empty, past max_pages * page_size) and behind the last one;
      cu_seqlens_new (batch_size + 1,) int32: their starts, at most 2 ** 31 - 1;
      num_free_out (1,) int32: the stack's new count, to be given to the next
        step, or less than 0 by as many pages as were missing.

    No new token is dropped if total_new is at least the sum of
    max(new_seqlens - cache_seqlens, 0). batch_size * max_pages is at most 2 ** 30. Nothing is read
    back to the host."""
    return _update_page_table(page_table, maybe_contiguous(cache_seqlens), maybe_contiguous(new_seqlens), free_pages,
                              num_free, int(page_size), int(total_new), maybe_contiguous(cache_batch_idx))


def append_quantized_kvcache(k, v, k_cache, v_cache, k_scale, v_scale, slot_mapping):
    """Quantise new k / v rows into the cache, in place.

    k, v: (total_new, nheads_k, headdim) fp16 or bf16. slot_mapping
    (total_new,) int64: the slot of each row; rows whose slot is not in the
    cache (-1) are skipped. No slot is given twice, and the rows of one block stand together,
    as update_page_table lays them out.

    The scale of a block and head becomes the smallest power of two s (at least
    2 ** -100) with max |x| <= 127 s (int8) or 448 s (e4m3) over the block's new
    rows. A block that earlier calls began (the first of its new rows here is not
    its row 0) keeps its scale if that is the larger; otherwise the codes before that row
    are rounded to the new scale. Codes are x / s rounded to the nearest, ties
    to even. +-inf counts as the type's largest finite value; NaN becomes 0 in
    int8 and NaN in e4m3. The new rows of one block and head are one workgroup's work, and so are the
    codes before them that move: blocks of thousands of tokens (a contiguous cache with one scale a
    sequence) are slow.

    4-bit cache: each 32 channels of a row get the smallest power of two s with max |x| <= 6 s (at least 2 ** -100, at most
    2 ** 13 for fp16 and 2 ** 125 for bf16, past which codes end at 6), and codes x / s rounded to the nearest, ties to
    the even code. +-inf counts as the type's largest finite value; a NaN makes its 32 channels NaN. Slots may
    come in any order, since no row touches another."""
    _append(k, v, k_cache, v_cache, k_scale, v_scale, maybe_contiguous(slot_mapping))


def flash_attn_with_quantized_kvcache(q, k_cache, v_cache, k_scale, v_scale, cache_seqlens,
                                      page_table: Optional[torch.Tensor] = None,
                                      cache_batch_idx: Optional[torch.Tensor] = None,
                                      cu_seqlens_q: Optional[torch.Tensor] = None,
                                      max_seqlen_q: Optional[int] = None, softmax_scale=None, causal=False,
                                      window_size=(-1, -1), softcap=0.0, return_softmax_lse=False):
    """Attention against a quantised cache (append_quantized_kvcache fills it).

    q: (batch_size, seqlen, nheads, headdim) fp16 or bf16 or, with cu_seqlens_q
    (batch_size + 1,) int32 and max_seqlen_q, at least the rows of each sequence,
    (total_q, nheads, headdim). Where cu_seqlens_q goes past total_q (update_page_table
    with too small a total_new), the tokens past it are not there, rows and keys.
    cache_seqlens (batch_size,) int32: the keys of each sequence, the tokens
    that this step appended among them (the last query row is aligned with the
    last key). page_table (rows, max_pages) int32 as from update_page_table, or
    None for a contiguous cache. cache_batch_idx (batch_size,) int32: the row
    of the page table (of the contiguous cache) of each sequence; one whose row is not there has
    no keys. Keys on a page whose id is not in the cache are not visible. A sequence holds at most 2 ** 30
    tokens, a call 2 ** 30 query rows x query heads of a kv head. The scales may have any value (scale * code in the range of fp32), and
    reach only the rows that see their keys. A NaN code of v_cache (e4m3) at a key that
    some row of the sequence sees may reach rows that do not see it, as a NaN of v does in
    flash_attn_with_kvcache.

    The scores are softmax_scale (default headdim ** -0.5) * k_scale * (q . c)
    of each key's codes, the weights of the values carry v_scale, and both
    products run on the codes without rounding them (fp32 sums). causal,
    window_size and softcap as in flash_attn_with_kvcache. A row that sees no
    key gets 0 and a softmax_lse of +inf. Of a 4-bit cache, the products run on the values that it holds, rounded to the type of q:
    bf16 holds them as they are, fp16 those from 2 ** -14 to 65504 (larger ones become inf, smaller ones lose bits). A value of
    v_cache that is NaN or inf so, at a key that some row of the sequence sees, may reach rows that do not see it. Rows behind the last sequence of cu_seqlens_q are not
    written: what out and softmax_lse hold there means nothing. Returns out, or (out, softmax_lse)
    with softmax_lse (batch_size, nheads, seqlen) or (nheads, total_q) fp32."""
    if softmax_scale is None:
        softmax_scale = q.shape[-1] ** (-0.5)
    if cu_seqlens_q is not None and max_seqlen_q is None:
        raise RuntimeError("max_seqlen_q is required with cu_seqlens_q")
    out, softmax_lse = _fwd(q, k_cache, v_cache, k_scale, v_scale, maybe_contiguous(cache_seqlens),
                            maybe_contiguous(page_table), maybe_contiguous(cache_batch_idx),
                            maybe_contiguous(cu_seqlens_q), int(max_seqlen_q or 0), float(softmax_scale), bool(causal),
                            int(window_size[0]), int(window_size[1]), float(softcap))
    return (out, softmax_lse) if return_softmax_lse else out


def read_quantized_kvcache(k_cache, v_cache, k_scale, v_scale, slot_mapping: Optional[torch.Tensor] = None,
                           cu_seqlens_k: Optional[torch.Tensor] = None, total_k: Optional[int] = None,
                           page_table: Optional[torch.Tensor] = None, cache_batch_idx: Optional[torch.Tensor] = None,
                           dtype=torch.bfloat16):
    """Rows of a quantised cache as values: (k, v), each (total, nheads_k, headdim) of dtype (bf16, fp16 or fp32).

    Which rows: those of slot_mapping (total,) int64, or the keys of sequences one behind the other, as
    flash_attn_varlen_func takes them: row cu_seqlens_k[b] + j, cu_seqlens_k (batch_size + 1,) int32, is key j
    of sequence b, which page_table and cache_batch_idx lead to as in flash_attn_with_quantized_kvcache; total_k is the number of
    rows of k and v, of which those behind the last sequence are 0. So is a row whose slot or page is not in the cache.

    A value is code * scale, rounded to fp32 and to dtype; of a 4-bit cache it is rounded to dtype alone."""
    if cu_seqlens_k is not None and total_k is None:
        raise RuntimeError("total_k is required with cu_seqlens_k")
    return _read(k_cache, v_cache, k_scale, v_scale, maybe_contiguous(slot_mapping), maybe_contiguous(cu_seqlens_k),
                 int(total_k or 0), maybe_contiguous(page_table), maybe_contiguous(cache_batch_idx), dtype)
