"""Paged 8-bit KV cache: requests of different lengths in blocks of tokens, tables kept on the GPU.

Beside ``NVFP4KVCache`` (one dense batch in 4 bits, rows of one length) this is the cache of a server whose
requests come and go: keys and values are e4m3 codes in blocks of 16 to 128 tokens with one scale for each block and
head, and which block holds which tokens is decided on the GPU, without a copy to the host, so that a whole step can
be captured in a CUDA graph.  (No counterpart in the reference.)

Layout, shared by every function here:

  k_cache, v_cache   [blocks, Hk, block_size, D] float8_e4m3fn: codes; heads dense, any stride between blocks
  k_scale, v_scale   [blocks, Hk] float32: value = code * scale (a power of two; attention also reads others, which calls of
                     many query rows a request round to eleven bits)
  block_table        [requests, width] int32: block of tokens j * block_size .. of a request, -1 where it has none.
                     Attention may read a block for several requests; reserve, write and trim take it to be one's own
  lengths            [requests] int32: tokens that a request holds
  free_blocks        [blocks] int32, free_count [1] int32: a stack of block ids, its top at free_count - 1

A step is ``paged_kv_reserve`` (blocks and slots for the new tokens), then in every layer ``fp8_kv_write`` and
``fp8_paged_decode`` or ``fp8_paged_attention``; ``paged_kv_trim`` takes tokens away again (rejected drafts, requests
that ended).  With trees of drafted tokens: ``draft_tree`` once, ``fp8_paged_tree_attention`` in every layer, ``verify_drafts``,
then ``paged_kv_keep_path`` for all layers in front of the trim.  ``FP8PagedKVCache`` holds the buffers of a model's layers and calls these.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib


class PagedStep(NamedTuple):
    """New tokens of one step, request by request: where each goes, its position, and where each request's begin."""

    slot_map: torch.Tensor      # [num_slots] int64: block * block_size + offset, -1 behind the last token
    positions: torch.Tensor     # [num_slots] int32: position in the request (for the caller's rotary embedding), 0 behind
    cu_seqlens: torch.Tensor    # [requests + 1] int32
    shortage: torch.Tensor      # [1] int32: 1 where nothing was reserved


class DraftTree(NamedTuple):
    """What the tokens of a step's trees see of each other, and where they stand."""

    tree_mask: torch.Tensor     # [T, ceil(max_tokens / 64)] int64: bit j of a token's row: token j of its request is it or above it
    positions: torch.Tensor     # [T] int32: position in the request along the token's own path


class VerifiedDrafts(NamedTuple):
    """The path that a verification keeps of every request's tree, and the token that follows it."""

    accepted: torch.Tensor      # [T] int32: from cu_seqlens[r] on the path's tokens as numbers within the request, 0 first, then -1
    num_accepted: torch.Tensor  # [requests] int32
    next_tokens: torch.Tensor   # [requests] int64, -1 for a request without tokens


def paged_kv_reserve(new_lens, lengths, block_table, free_blocks, free_count, num_slots: int, block_size: int) -> PagedStep:
    """Blocks and slots for ``new_lens[r]`` more tokens of every request r (int32 on the GPU; below 0 counts as 0).

    Pops the blocks that are needed off the stack in request order, enters them in ``block_table``, adds to
    ``lengths`` (all in place) and lists the slots and positions of the new tokens, padded to ``num_slots``.  All or
    nothing: where the stack, the table's width or ``num_slots`` does not suffice, ``shortage`` is 1, every slot -1,
    ``cu_seqlens`` 0 and the state as it was.
    """
    return PagedStep(*_lib.native().paged_reserve(new_lens, lengths, block_table, free_blocks, free_count, num_slots, block_size))


def paged_kv_trim(keep_lens, lengths, block_table, free_blocks, free_count, block_size: int) -> None:
    """Every request r keeps its first ``keep_lens[r]`` tokens (0: it ends); blocks that hold none of them go back on
    the stack.  In place.  Trimmed to the lengths in front of a reservation, stack and table are what they were; codes and scales are not
    touched, so a block that stays keeps the scale that a token taken away may have raised (see ``fp8_kv_write``)."""
    _lib.native().paged_trim(keep_lens, lengths, block_table, free_blocks, free_count, block_size)


def fp8_kv_write(key, value, slot_map, k_cache, v_cache, k_scale, v_scale) -> None:
    """Quantise the keys and values of new tokens ([T, Hk, D], or [Z, Hk, 1, D]) into their slots.

    Per block and head the scale is the smallest power of two 2^e with max|x| <= 448 * 2^e, so codes are the one
    rounding of exact quotients.  Tokens that a block holds in front of the call's first one stay; where the new
    ones need a larger scale, their codes are rounded again to it.  Infinities saturate and do not count for the scale,
    nor do NaN, which stay.  Slots below 0 are skipped.  A block's tokens stand next to each other in ``slot_map``,
    ascending by one, as ``paged_kv_reserve`` lists them; a block named in two places of one call is left with
    unspecified codes.  Two calls that write the same block are ordered by the caller (one stream, or events).
    """
    _lib.native().kv8_write(key, value, slot_map, k_cache, v_cache, k_scale, v_scale)


def fp8_paged_decode(query, k_cache, v_cache, k_scale, v_scale, block_table, lengths, scaling, num_key_value_groups=1,
                     return_lse=False):
    """Attention of one query token a request over its ``lengths[r]`` keys; lengths may differ and are read on the GPU.

    ``query`` ``[Z, H, 1, D]`` (bf16 / fp16 / fp32), row r for row r of ``block_table``.  Returns ``[Z, H, 1, D]``,
    with ``return_lse`` also the natural-log sums ``[Z, H]`` (fp32).  A request without keys gets zeros and -inf; entries of
    the table that are no block hide their keys.
    """
    out, lse = _lib.native().kv8_attention(query, None, k_cache, v_cache, k_scale, v_scale, block_table, lengths, scaling,
                                           num_key_value_groups, return_lse)
    return (out, lse) if return_lse else out


def fp8_paged_attention(query, cu_seqlens, k_cache, v_cache, k_scale, v_scale, block_table, lengths, scaling,
                        num_key_value_groups=1, return_lse=False):
    """Causal attention of several query tokens a request: drafts to verify, chunks of a prompt, or both in one batch.

    ``query`` ``[T, H, D]``; request r owns tokens ``cu_seqlens[r] .. cu_seqlens[r + 1]``, the last ones of its
    ``lengths[r]`` keys (written before the call): token i of n sees keys ``0 .. lengths[r] - n + i``.  The kernel is chosen by the query
    tokens a row of the table, idle rows among them: a long chunk is called with the rows of the table that it needs
    (``block_table[r:r + 1]``, ``lengths[r:r + 1]``) rather than with hundreds of idle ones.  A value that is NaN
    reaches the call's tokens in front of it too (their weight 0 times NaN), as in a masked softmax; keys, and what is
    behind ``lengths[r]`` in a block, reach nothing that does not see them.  Returns ``[T, H, D]``, with ``return_lse`` also ``[T, H]``; tokens without a key, or behind the last request's, get zeros and -inf.
    """
    if cu_seqlens is None:
        raise ValueError("fp8_paged_attention needs cu_seqlens (one token a request: fp8_paged_decode)")
    out, lse = _lib.native().kv8_attention(query, cu_seqlens, k_cache, v_cache, k_scale, v_scale, block_table, lengths, scaling,
                                           num_key_value_groups, return_lse)
    return (out, lse) if return_lse else out


def draft_tree(parents, cu_seqlens, lengths, max_tokens: int) -> DraftTree:
    """Tables of trees of drafted tokens, once a step for all layers.

    Request r's tokens are ``cu_seqlens[r] .. cu_seqlens[r + 1]``, the last ones of its ``lengths[r]`` (reserved before the call); token i
    hangs on the request's earlier token ``parents[t]`` (int32, counted within the request), and on the context alone where that names
    none (-1).  ``max_tokens`` (1 to 1024): tokens of the largest tree; what lies behind them sees the context alone, and
    ``verify_drafts`` with the same ``max_tokens`` never keeps it.  Tokens of no request have no bits and position 0.
    """
    return DraftTree(*_lib.native().draft_tree(parents, cu_seqlens, lengths, max_tokens))


def fp8_paged_tree_attention(query, cu_seqlens, tree_mask, k_cache, v_cache, k_scale, v_scale, block_table, lengths, scaling,
                             num_key_value_groups=1, return_lse=False):
    """``fp8_paged_attention`` of trees of drafted tokens: token i of a request's n sees the keys in front of them,
    ``0 .. lengths[r] - n - 1``, and of the n those whose bit its row of ``tree_mask`` has.

    ``tree_mask`` ``[T, words]`` int64, as ``draft_tree`` makes it or any other bits: bit j % 64 of word j / 64 is key
    ``lengths[r] - n + j``; bits from n on do not count, tokens from 64 * words on are seen by none.  A token that sees no key gets
    zeros and -inf.  A value that is NaN reaches all tokens of its request's tree (weight 0 times NaN); keys reach those that see them.
    """
    out, lse = _lib.native().kv8_tree_attention(query, cu_seqlens, tree_mask, k_cache, v_cache, k_scale, v_scale, block_table, lengths,
                                                scaling, num_key_value_groups, return_lse)
    return (out, lse) if return_lse else out


def verify_drafts(target_probs, tokens, parents, cu_seqlens, uniforms, draft_probs=None, max_tokens: int = 1024) -> VerifiedDrafts:
    """Which drafted tokens to keep, so that what is kept and the token behind it are distributed as the target's own draws.

    ``target_probs`` ``[T, vocabulary]`` (bf16 / fp16 / fp32): row t is the target's distribution behind token t.  A request's first
    token is given (the one that the step before ended with), the others are drafts: ``tokens`` ``[T]`` ids (int64 or int32),
    ``parents`` as for ``draft_tree`` (a draft that hangs on the context alone is never kept).  ``max_tokens`` (1 to 1024): what lies
    behind them in a tree is never kept; where trees may be larger than what ``draft_tree`` was told (a captured step, whose
    ``max_tokens`` stays as it was), the same number, as drafts behind it were attended without their ancestors.  ``uniforms`` ``[T]`` float32 in [0, 1): of a draft the number that tests it, of a request's first token
    the one that draws the next.

    At a token with row p, its children in order, R = p and M = 1.  With ``draft_probs`` (``[T, vocabulary]``, row t: what the children of
    t were drawn from independently, q) a child c is kept where ``u q(c) M < R(c)``; else R becomes max(R / M - q, 0) and M its sum.
    Without (drafts that were chosen, such as the likeliest tokens) it is kept where ``u M < R(c)``; else M loses R(c), and R(c) becomes 0.
    The walk goes on at the first child kept; where none is, the next token is the first v whose running sum of R exceeds w sum(R)
    (of p, where R is empty).  Sums are in 64 bits.  Entries that are no finite number above zero count as 0, as do ids outside the vocabulary.
    """
    return VerifiedDrafts(*_lib.native().verify_drafts(target_probs, tokens, parents, cu_seqlens, uniforms, draft_probs, max_tokens))


def paged_kv_keep_path(accepted, num_accepted, cu_seqlens, lengths, block_table, k_cache, v_cache, k_scale, v_scale) -> torch.Tensor:
    """Move the keys and values of the path that ``verify_drafts`` kept to the front of their request's newest tokens, in place.

    Of the n = ``cu_seqlens[r + 1] - cu_seqlens[r]`` last tokens of request r, token ``accepted[cu_seqlens[r] + j]`` goes to position
    ``lengths[r] - n + j``, for j below ``num_accepted[r]`` (a path ends in front of an entry that does not ascend).  Caches of one
    layer, ``[blocks, Hk, block_size, D]``, or of all, ``[layers, blocks, Hk, block_size, D]``, scales likewise.  Where a block receives
    codes of a larger scale that its own cannot hold, its scale becomes the smallest power of two that can, and its older codes are
    rounded again to it.  Returns ``keep_lens`` [requests] int32 for ``paged_kv_trim``.  The codes behind those tokens are left as they were,
    but the scale of the path's last block may have grown over them: what lies there is no token any more, with or without the trim.
    """
    return _lib.native().paged_keep_path(accepted, num_accepted, cu_seqlens, lengths, block_table, k_cache, v_cache, k_scale, v_scale)


class FP8PagedKVCache:
    """The paged 8-bit cache of a model's layers: one table for all of them, codes and scales for each.

    Args: ``num_layers``; ``num_blocks`` of ``block_size`` tokens shared by all requests; ``hk`` KV heads of head
    dim ``d`` (128 or 256); ``max_requests`` rows of the table; ``max_seq_len`` tokens that a request may hold.
    """

    def __init__(self, num_layers, num_blocks, hk, d, max_requests, max_seq_len, device, block_size=64):
        assert d in (128, 256), "D must be 128 or 256"
        assert block_size in (16, 32, 64, 128), "block_size must be 16, 32, 64 or 128"
        assert num_layers >= 1 and num_blocks >= 1 and hk >= 1 and max_requests >= 1 and max_seq_len >= 1
        self.num_layers, self.num_blocks, self.hk, self.d, self.block_size = num_layers, num_blocks, hk, d, block_size
        self.device = torch.device(device)
        dev = self.device
        shape = (num_layers, num_blocks, hk, block_size, d)
        self.k = torch.zeros(shape, dtype=torch.float8_e4m3fn, device=dev)
        self.v = torch.zeros(shape, dtype=torch.float8_e4m3fn, device=dev)
        self.k_scale = torch.zeros(num_layers, num_blocks, hk, device=dev)
        self.v_scale = torch.zeros(num_layers, num_blocks, hk, device=dev)
        width = -(-max_seq_len // block_size)
        self.block_table = torch.full((max_requests, width), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(max_requests, dtype=torch.int32, device=dev)
        self.free_blocks = torch.arange(num_blocks - 1, -1, -1, dtype=torch.int32, device=dev)
        self.free_count = torch.full((1,), num_blocks, dtype=torch.int32, device=dev)

    def reserve(self, new_lens: torch.Tensor, num_slots: int) -> PagedStep:
        """``paged_kv_reserve`` on this cache's table; ``num_slots`` is at least the sum of ``new_lens``."""
        return paged_kv_reserve(new_lens, self.lengths, self.block_table, self.free_blocks, self.free_count, num_slots,
                                self.block_size)

    def trim(self, keep_lens: torch.Tensor) -> None:
        """``paged_kv_trim`` on this cache's table."""
        paged_kv_trim(keep_lens, self.lengths, self.block_table, self.free_blocks, self.free_count, self.block_size)

    def write(self, layer: int, key: torch.Tensor, value: torch.Tensor, slot_map: torch.Tensor) -> None:
        """New tokens of one layer into the slots of a step."""
        fp8_kv_write(key, value, slot_map, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer])

    def decode(self, layer: int, query: torch.Tensor, scaling: float, g: int, return_lse: bool = False):
        """``fp8_paged_decode`` of ``[max_requests, H, 1, D]`` over one layer."""
        return fp8_paged_decode(query, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], self.block_table,
                                self.lengths, scaling, g, return_lse)

    def attend(self, layer: int, query: torch.Tensor, cu_seqlens: torch.Tensor, scaling: float, g: int, return_lse: bool = False):
        """``fp8_paged_attention`` of ``[T, H, D]`` over one layer."""
        return fp8_paged_attention(query, cu_seqlens, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer],
                                   self.block_table, self.lengths, scaling, g, return_lse)

    def attend_tree(self, layer: int, query: torch.Tensor, cu_seqlens: torch.Tensor, tree_mask: torch.Tensor, scaling: float, g: int,
                    return_lse: bool = False):
        """``fp8_paged_tree_attention`` of ``[T, H, D]`` over one layer."""
        return fp8_paged_tree_attention(query, cu_seqlens, tree_mask, self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer],
                                        self.block_table, self.lengths, scaling, g, return_lse)

    def tree(self, parents: torch.Tensor, cu_seqlens: torch.Tensor, max_tokens: int) -> DraftTree:
        """``draft_tree`` of the tokens that a step has reserved."""
        return draft_tree(parents, cu_seqlens, self.lengths, max_tokens)

    def keep_path(self, accepted: torch.Tensor, num_accepted: torch.Tensor, cu_seqlens: torch.Tensor) -> None:
        """``paged_kv_keep_path`` in all layers, then ``trim`` to what it keeps: the step's other tokens are gone."""
        self.trim(paged_kv_keep_path(accepted, num_accepted, cu_seqlens, self.lengths, self.block_table, self.k, self.v, self.k_scale,
                                     self.v_scale))

    def cache_bytes(self) -> int:
        """Bytes of codes and scales, all layers and blocks."""
        return 2 * self.num_layers * self.num_blocks * self.hk * (self.block_size * self.d + 4)

    def held_bytes(self) -> int:
        """Bytes of the blocks that requests hold, all layers (reads the stack's size: synchronises)."""
        return self.cache_bytes() // self.num_blocks * (self.num_blocks - int(self.free_count))
