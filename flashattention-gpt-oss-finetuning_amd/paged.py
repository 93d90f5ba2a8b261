"""Answering with a model: a paged key-value cache, attention of one new token a sequence over it, and eviction.

The reference takes whole sequences only (flash_attention_gpt_oss.py:348).  A layer's cache is a pool of pages,
``k_pages`` and ``v_pages`` [pages, Hkv, page_size, D]; row b of ``block_table`` (int32 [B, width], on the GPU) lists the
pages of sequence b in order, so its token t is entry t % page_size of page block_table[b, t // page_size].  A pool with
the slots before the heads in memory is passed as its transposed view; any strides that are multiples of 16
bytes are used in place.  ``lens`` (int32 [B], on the GPU) are the tokens of each sequence, the new ones included, so a
decoding step of all layers is::

    lens += 1                                                          # once for all layers
    paged_append(k, v, k_pages, v_pages, block_table, lens)            # k, v [B, Hkv, D]
    o = paged_attention(q, k_pages, v_pages, block_table, lens, window_size, sinks=module.sinks)   # q [B, Hq, D]

and a prompt goes through flash_swda_with_sink_varlen and, with its cu_seqlens, through paged_append.  Nothing waits for the
GPU, so a step can be captured into a HIP graph.  Entries of block_table that are no page (outside [0, pages)) are
masked when read and left out when written; a sequence with lens 0 is idle.

Pages are bfloat16, float16 or float32, as the call's other tensors, or float8_e4m3fn under bfloat16 or float16
tensors (D 64 or 128): a code stands for descale[0] (keys) or descale[1] (values) times its value.  Forward only: what
paged_attention returns for inputs that require a gradient raises in the backward pass, and what is in the pages has none.
Compute is in csrc/fa_paged_attn.hip and csrc/fa_paged_cache.hip; there is no CPU implementation.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _ops


class _NoBackward(torch.autograd.Function):
    """o as it is, but with an error in place of a silently missing gradient."""

    @staticmethod
    def forward(ctx, o, *inputs):
        ctx.mark_dirty(o)  # (returned as it is and not as a view, so that it can be written in place)
        return o

    @staticmethod
    def backward(ctx, do):
        raise NotImplementedError("paged_attention has no backward pass; train with flash_swda_with_sink and its kin, and "
                                  "answer under torch.no_grad()")


def paged_append(k, v, k_pages, v_pages, block_table, lens, cu_seqlens: Optional[torch.Tensor] = None,
                 descale=(1.0, 1.0)) -> None:
    """Writes new tokens' rows into the pages, in place: k, v [B, Hkv, D], one row a sequence, or packed
    [total, Hkv, D] with cu_seqlens [B + 1] (int32 or int64; on the host it is validated).  The n new rows of sequence b
    go to positions lens[b] - n .. lens[b] - 1; rows of no sequence and of positions outside the table are left
    out.  float8_e4m3fn pages get round-to-nearest-even codes of clamp(x / descale, -448, 448), as quantize_fp8 makes them."""
    cu = None
    if cu_seqlens is not None:
        cu = _ops.cu_seqlens_ready(cu_seqlens, k.shape[0], k_pages.device, None if cu_seqlens.device.type == "cpu" else 1)[0]
    _ops.paged_append(k, v, k_pages, v_pages, block_table, lens, cu, float(descale[0]), float(descale[1]))


def paged_attention(q, k_pages, v_pages, block_table, lens, window_size: Optional[int] = None, sink_size: int = 0,
                    sinks: Optional[torch.Tensor] = None, scale: Optional[float] = None, descale=(1.0, 1.0),
                    max_seqlen: Optional[int] = None, weight_sums: Optional[torch.Tensor] = None):
    """Attention of the last token of every sequence over its cache: q [B, Hq, D] -> o [B, Hq, D].  Of a sequence of n
    tokens it sees key k where n - 1 - k < window_size (None: every key) or k < sink_size; `sinks` [Hq] are GPT-OSS's
    learned sink logits.  A sequence without visible keys gets zeros.

    max_seqlen: a bound on lens (default: the table's tokens); a tighter one makes the launch and its workspace
    smaller.  weight_sums (float32 [B, Hkv, tokens], at least max_seqlen tokens) accumulates the softmax weights in place:
    weight_sums[b, h, k] += the sum of key k's weights over the query heads of KV head h, for paged_evict.  Its workspace is Hq / Hkv
    times as large as weight_sums of max_seqlen tokens: a tight max_seqlen keeps it small.  Sinks in float32 save a
    conversion on every call."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    most = 2 ** 31 - 1
    o = _ops.paged_attention(q, k_pages, v_pages, block_table, lens, most if window_size is None else int(window_size),
                             int(sink_size), sinks, float(scale), float(descale[0]), float(descale[1]),
                             most if max_seqlen is None else int(max_seqlen), weight_sums)
    if (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad or (sinks is not None and sinks.requires_grad)) \
            and torch.is_grad_enabled():
        return _NoBackward.apply(o, q, k_pages, v_pages, sinks)
    return o


def paged_evict(k_pages, v_pages, block_table, lens, weight_sums, keep: int, new_table, sink_size: int = 0, recent: int = 0,
                max_seqlen: Optional[int] = None):
    """Thins out every sequence of more than `keep` tokens to `keep` entries, each KV head by itself: the first sink_size and
    the last `recent` entries stay, and of the others those with the largest weight_sums [B, Hkv, tokens] (the lower
    position first among equals; a NaN counts as the largest).  The entries go, in order, to the pages of
    new_table (int32 [B, width]): pages that the call does not read, so that a prefix shared with other
    sequences stays whole; sequences of at most `keep` tokens are copied.  Entries on no page of block_table are none of
    the sequence's: they neither count nor stay.  Returns (new lens [B], new weight sums, shaped
    as weight_sums, zero behind the kept entries), to be used with new_table from then on.  An entry's place says
    nothing about its token's position any more: call paged_attention with window_size None and sink_size 0.

    max_seqlen: a bound on lens, as paged_attention's; weight_sums are that wide at least."""
    if max_seqlen is not None and max_seqlen < 1:
        raise ValueError(f"max_seqlen must be at least 1, got {max_seqlen}")
    return _ops.paged_evict(k_pages, v_pages, block_table, lens, weight_sums, int(keep), new_table, int(sink_size), int(recent),
                            0 if max_seqlen is None else min(int(max_seqlen), 2 ** 31 - 1))
