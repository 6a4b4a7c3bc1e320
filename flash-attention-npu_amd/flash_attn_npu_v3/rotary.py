"""Rotary positions: the tables of cosines and sines, for positions past the length
that a model was trained on too, and the rotation of q and k by them, with its
gradient.

flash_attn_with_kvcache turns q and the new keys itself and takes the same tables
(rotary_cos, rotary_sin: fp16 or bf16 as q there). The calls without a turn of their own take q
and k from apply_rotary_emb: flash_attn_func and flash_attn_varlen_func in training,
append_quantized_kvcache and flash_attn_with_quantized_kvcache in serving. The
reference has no counterpart.
"""
from typing import Optional

import torch

from fa_mi355x import capi, ops

from .interface import maybe_contiguous

_table, _rotary, _rotary_in_place = (op.default for op in (ops.rotary_table, ops.rotary, ops.rotary_))
_SCALING = {None: capi.FA_ROTARY_PLAIN, "linear": capi.FA_ROTARY_LINEAR, "ntk": capi.FA_ROTARY_NTK,
            "by_parts": capi.FA_ROTARY_BY_PARTS}


def rotary_cos_sin(positions, rotary_dim, base=10000.0, scaling=None, factor=1.0, original_length=0, low=1.0, high=32.0,
                   attention_factor=1.0, dtype=torch.float32):
    """Cosines and sines of positions (n,) int32 or int64: (cos, sin), each (n, rotary_dim // 2) of dtype (fp32, fp16
    or bf16). rotary_dim is a multiple of 16, at most 256.

    cos[j, i] = attention_factor * cos(positions[j] * f_i) with f_i = base ** (-2 i / rotary_dim), scaled for contexts
    that are `factor` times as long as the trained one:

      None        f_i
      "linear"    f_i / factor (positions interpolated)
      "ntk"       base * factor ** (rotary_dim / (rotary_dim - 2)) in place of base
      "by_parts"  f_i (g + (1 - g) / factor), where g goes from 0 to 1 while the turns that f_i makes over
                  original_length tokens, original_length * f_i / 2 pi, go from low to high

    Angles are formed in 64 bits, so that of position p is off by less than p * f_i * 2 ** -50; its cosine and sine are good to
    2 ** -22 of their value."""
    if scaling not in _SCALING:
        raise RuntimeError(f"scaling must be None, 'linear', 'ntk' or 'by_parts', got {scaling!r}")
    return _table(maybe_contiguous(positions), int(rotary_dim), float(base), _SCALING[scaling], float(factor),
                  float(original_length), float(low), float(high), float(attention_factor), dtype)


def apply_rotary_emb(q, k, rotary_cos, rotary_sin, positions: Optional[torch.Tensor] = None, seqlen_offsets=0,
                     cu_seqlens: Optional[torch.Tensor] = None, rotary_interleaved=True, inplace=False):
    """Turn the first rotary_dim channels of q and k (or of q alone, k None) by their positions; returns (q, k), or q.

    q: (batch_size, seqlen, nheads, headdim) or (total, nheads, headdim) fp16 or bf16, k the same with its own number of
    heads; headdim a multiple of 8. rotary_cos, rotary_sin: (seqlen_ro, rotary_dim // 2) fp32 or of the type of q,
    rotary_dim a multiple of 16. Pairs are channels (2 i, 2 i + 1) with rotary_interleaved (the default, as in
    flash_attn_with_kvcache), else (i, i + rotary_dim / 2); a pair (x1, x2) becomes (x1 cos - x2 sin, x2 cos + x1 sin).

    The position of a row is positions of it, (batch_size, seqlen) or (total,) int32 or int64, or its place in its
    sequence plus seqlen_offsets (a number, or (batch_size,) int32). Sequences of (total, nheads, headdim) are those
    of cu_seqlens (batch_size + 1,) int32, or one. Rows that belong to no sequence stay as they are. Positions outside
    the tables take their first or last row.

    inplace turns q and k themselves, without new memory; neither may hold a row twice, nor share memory with the other. What
    autograd does not let be changed (a leaf that requires a gradient, the pieces of a split) is refused and stays as it was.
    Gradients of q and k are turned back, which takes no saved rows; the tables get none. Forward-mode derivatives are refused."""
    offsets = maybe_contiguous(seqlen_offsets) if isinstance(seqlen_offsets, torch.Tensor) else None
    where = (positions, offsets, 0 if offsets is not None else int(seqlen_offsets), maybe_contiguous(cu_seqlens), bool(rotary_interleaved))
    if inplace:
        _rotary_in_place(q, k, rotary_cos, rotary_sin, *where, False)
        return (q, k) if k is not None else q
    turned_q, turned_k = _rotary(q, k, rotary_cos, rotary_sin, *where, False)
    return (turned_q, turned_k) if k is not None else turned_q
